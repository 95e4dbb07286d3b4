"""Paged, bounded key cache on the sm_100a kernels: the server's form of the decode cache of
src/sisa/generation.py:58-95.

A sequence's keys lie in pages of ``page_size`` slots named by its row of a block table, so sequences of
different lengths share one pool (:class:`KeyPages`, one per layer). The keys kept per sequence can be
bounded: the prompt's keys are weighed by the attention they received (:func:`attention_key_weights`), the
newest and the heaviest go into the pages (:func:`paged_fill`), and every further token takes the slot of
the lightest old key (:func:`paged_evict`, :func:`paged_append`) while the attention of the new token
(:func:`paged_attention`) adds to the weights. SISA keeps a key's position in its g, F and rotated b~, so
the slots may hold the keys in any order.

All functions run on torch's current stream and follow the check mode of :mod:`sisa_b200.backends`;
``block_table`` is (B, max_pages) int32, ``lengths`` and ``position`` are (B,) int32 on the device, so
that a captured CUDA graph serves every step. They are for serving and have no backward: an input that
requires a gradient, in grad mode, raises ValueError.

Rows of a block table may share pages (a common prefix) only in calls that read them: :func:`paged_attention`
without ``accumulate``. A page that a call writes, or whose weights it adds to, has to belong to one row.
"""
from __future__ import annotations

import torch
from torch import Tensor

from .. import _lib, backends

__all__ = ["KeyPages", "paged_attention", "paged_evict", "paged_append", "attention_key_weights", "paged_fill",
           "CARRY"]

PAGE_SIZES = (16, 32, 64, 128, 256)
#: fp32 values of the recurrent state per (sequence, head): the phases Phi 0..15, g and F of the last token.
CARRY = 18


class KeyPages:
    """One layer's pages: ``k``, ``v`` (P, H, page_size, 64) and ``b`` (P, H, page_size, 32) bf16 or fp16, the
    planes ``g``, ``f``, ``weight`` (P, H, page_size) fp32 and ``token`` int32. ``f`` may be None without a
    forget gate, ``weight`` and ``token`` where nothing is evicted. Page and head strides are free, the
    slots of one head in one page are dense; the planes share one set of strides."""

    def __init__(self, k: Tensor, v: Tensor, b: Tensor, g: Tensor, f: Tensor | None = None,
                 weight: Tensor | None = None, token: Tensor | None = None):
        if k.dim() != 4 or k.shape[-1] != 64 or k.shape[2] not in PAGE_SIZES:
            raise ValueError(f"k pages must be (P, H, page_size, 64) with page_size in {PAGE_SIZES}, got {tuple(k.shape)}")
        P, H, S, _ = k.shape
        if tuple(v.shape) != (P, H, S, 64) or tuple(b.shape) != (P, H, S, 32):
            raise ValueError(f"v and b pages must be {(P, H, S, 64)} and {(P, H, S, 32)}, got {tuple(v.shape)} and "
                             f"{tuple(b.shape)}")
        self.dtype_code = _lib.dtype_code(k.dtype)
        if v.dtype != k.dtype or b.dtype != k.dtype:
            raise TypeError(f"k, v and b pages differ in dtype: {k.dtype}, {v.dtype}, {b.dtype}")
        for name, t in (("k", k), ("v", v), ("b", b)):
            if t.stride(3) != 1 or t.stride(2) != t.shape[3]:
                raise ValueError(f"the rows of {name} pages must be dense within a page, got strides {t.stride()}")
        planes = [("g", g, torch.float32), ("f", f, torch.float32), ("weight", weight, torch.float32),
                  ("token", token, torch.int32)]
        for name, t, dt in planes:
            if t is None:
                continue
            if tuple(t.shape) != (P, H, S) or t.stride(2) != 1 or t.stride() != g.stride():
                raise ValueError(f"plane {name} must be {(P, H, S)} with unit slot stride and the strides of g, got "
                                 f"{tuple(t.shape)} {t.stride()}")
            if t.dtype != dt:
                raise TypeError(f"plane {name} must be {dt}, got {t.dtype}")
        if any(t is not None and t.device != k.device for t in (v, b, g, f, weight, token)):
            raise ValueError("all pages must lie on one device")
        if torch.is_grad_enabled():
            _refuse_grad("KeyPages", k, v, b, g, f, weight)
        self.k, self.v, self.b, self.g, self.f, self.weight, self.token = k, v, b, g, f, weight, token
        self.n_pages, self.n_head, self.page_size = P, H, S
        self.dtype, self.device = k.dtype, k.device
        c = _lib.Pages(k.data_ptr(), v.data_ptr(), b.data_ptr(), g.data_ptr(), _lib.ptr(f), _lib.ptr(weight),
                             _lib.ptr(token), k.stride(0), k.stride(1), v.stride(0), v.stride(1), b.stride(0), b.stride(1),
                             g.stride(0), g.stride(1), P, S)
        self.cbytes = bytes(c)                  # the struct every call passes, and its device's status word
        self.status = backends.status_word(self.device).data_ptr() if k.is_cuda else None
        self.ws_bytes: dict[tuple, int] = {}    # workspace sizes of the tables seen

    @classmethod
    def empty(cls, n_pages: int, n_head: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda",
              forget: bool = True, evict: bool = True) -> "KeyPages":
        """Uninitialised pages: 336 bytes per slot and head (328 without ``evict``)."""
        shape = (n_pages, n_head, page_size)
        k, v = (torch.empty(shape + (64,), dtype=dtype, device=device) for _ in range(2))
        b = torch.empty(shape + (32,), dtype=dtype, device=device)
        g = torch.empty(shape, dtype=torch.float32, device=device)
        f = torch.empty_like(g) if forget else None
        weight = torch.empty_like(g) if evict else None
        token = torch.empty(shape, dtype=torch.int32, device=device) if evict else None
        return cls(k, v, b, g, f, weight, token)


def _refuse_grad(what: str, *tensors: Tensor | None) -> None:
    """These operators serve; none has a backward. In grad mode (the caller looks) an input that requires a gradient
    raises, rather than a result that has lost it being returned."""
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError(f"{what} has no backward: call it under torch.no_grad() or with detached inputs")


def _table(pages: KeyPages, table: Tensor, B: int) -> tuple[int, int, int]:
    """(pointer, row stride, max_pages) of a block table."""
    shape = table.shape
    if len(shape) != 2 or shape[0] != B or shape[1] < 1 or table.dtype != torch.int32:
        raise ValueError(f"block_table must be ({B}, max_pages) int32, got {tuple(shape)} {table.dtype}")
    if table.device != pages.device:
        raise ValueError(f"block_table is on {table.device}, the pages on {pages.device}")
    row, one = table.stride()
    if one != 1 and shape[1] > 1:
        raise ValueError("block_table rows must be contiguous")
    return table.data_ptr(), (row if B > 1 else max(row, shape[1])), shape[1]


def _rows(t: Tensor, shape: tuple, name: str, pages: KeyPages) -> int:
    """The pointer of an int32 row tensor (positions, lengths, slots), checked."""
    if t.shape != shape or t.dtype != torch.int32 or not t.is_contiguous() or t.device != pages.device:
        raise ValueError(f"{name} must be a contiguous {shape} int32 tensor on {pages.device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    return t.data_ptr()


def _operand(t: Tensor) -> Tensor:
    """``t`` as the kernels read it: unit last stride, 16-byte aligned rows."""
    a, b, c, d = t.stride()
    if d == 1 and (a | b | c) % 8 == 0 and c > 0 and a >= 0 and b >= 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)      # (contiguous() keeps a dense tensor where it is, aligned or not)


def _f32(t: Tensor) -> Tensor:
    """``t`` in fp32, contiguous."""
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _check_query(q: Tensor, c: Tensor, pages: KeyPages) -> tuple[int, int]:
    shape, H = q.shape, pages.n_head
    if len(shape) != 4 or shape[2] != 1 or shape[3] != 64 or c.shape != (shape[0], shape[1], 1, 32):
        raise ValueError(f"paged_attention takes one query row with d_head 64 and d_state 32, got {tuple(shape)} and "
                         f"{tuple(c.shape)}")
    if shape[1] != H:
        raise ValueError(f"q has {shape[1]} heads, the pages {H}")
    if q.dtype != pages.dtype:
        raise TypeError(f"q dtype {q.dtype} differs from the pages' {pages.dtype}")
    if q.device != pages.device or c.device != pages.device:
        raise ValueError(f"q and c are on {q.device} and {c.device}, the pages on {pages.device}")
    return shape[0], H


def paged_attention(q: Tensor, c: Tensor, g: Tensor, fgate: Tensor | None, pages: KeyPages, block_table: Tensor,
                    lengths: Tensor, lam: Tensor, *, accumulate: bool = False, weight_out: Tensor | None = None,
                    return_lse: bool = False):
    """One new token per sequence over its paged keys. q (B, H, 1, 64), c (B, H, 1, 32) in the pages' dtype; g,
    fgate (B, H, 1) fp32 (fgate None: no forget gate); lengths (B,) int32, the keys of each sequence with the
    new token's own among them (0: idle row, y = 0); lam (H,) fp32. Returns y (B, H, 1, 64) in q.dtype and, with
    ``return_lse``, (y, lse) with lse (B, H) fp32 in log2 units (-inf for an idle row).

    With ``accumulate`` each key's softmax share is added to its weight: ``pages.weight`` in place, or
    ``weight_out`` = ``pages.weight`` + share where that plane is given (used slots only). No two rows may then
    share a page: both would add to the same weights, and one of the shares could be lost."""
    B, H = _check_query(q, c, pages)
    if torch.is_grad_enabled():
        _refuse_grad("paged_attention", q, c, g, fgate, lam, weight_out)
    lib = _lib.load()
    dev = pages.device
    tp, tsb, mp = _table(pages, block_table, B)
    lp = _rows(lengths, (B,), "lengths", pages)
    wo = None
    if accumulate:
        if pages.weight is None:
            raise ValueError("accumulate needs pages with a weight plane")
        wo = pages.weight if weight_out is None else weight_out
    if weight_out is not None:
        if not accumulate:
            raise ValueError("weight_out needs accumulate=True")
        if weight_out.shape != pages.weight.shape or weight_out.stride() != pages.weight.stride() \
                or weight_out.dtype != torch.float32 or weight_out.device != dev:
            raise ValueError("weight_out must be an fp32 plane with the shape and strides of pages.weight")
    if fgate is not None and pages.f is None:
        raise ValueError("fgate is given but the pages hold no f plane")
    for name, t in (("g", g), ("fgate", fgate)):
        if t is not None and (t.numel() != B * H or t.shape[0] != B or t.device != dev):
            raise ValueError(f"{name} must be ({B}, {H}, 1) on {dev}, got {tuple(t.shape)} on {t.device}")
    if lam.shape != (H,) or lam.device != dev:
        raise ValueError(f"lam must have shape {(H,)} on {dev}, got {tuple(lam.shape)} on {lam.device}")
    if c.dtype != q.dtype:
        c = c.to(q.dtype)
    q, c, gq, lam = _operand(q), _operand(c), _f32(g), _f32(lam)
    fq = None if fgate is None else _f32(fgate)
    y = torch.empty_like(q)                     # (less host time than torch.empty with a device)
    lse = lam.new_empty((B, H)) if return_lse else None
    key = (B, mp, accumulate)
    nbytes = pages.ws_bytes.get(key)
    if nbytes is None:
        if len(pages.ws_bytes) >= 1024:         # a long-running process with ever-changing tables
            pages.ws_bytes.clear()
        nbytes = pages.ws_bytes[key] = lib.sisa_paged_attn_workspace(B, H, mp * pages.page_size, accumulate)
    ws = lam.new_empty(nbytes // 4) if nbytes else None
    rc = lib.sisa_paged_attn(_lib.view4_bytes(q), _lib.view4_bytes(c), gq.data_ptr(), None if fq is None else fq.data_ptr(),
                             pages.cbytes, tp, tsb, mp, lp, lam.data_ptr(), B, H, pages.dtype_code, _lib.view4_bytes(y),
                             None if lse is None else lse.data_ptr(), None if wo is None else wo.data_ptr(),
                             None if ws is None else ws.data_ptr(),
                             pages.status, _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_attn")
    backends.after_call(dev)
    return (y, lse) if return_lse else y


def paged_evict(pages: KeyPages, block_table: Tensor, position: Tensor, budget: int, recent: int) -> Tensor:
    """The slot that the token ``position`` (B,) int32 takes per (sequence, head): the one whose key has the
    least accumulated weight among the keys older than the ``recent`` newest, the lowest slot where several
    weigh the same; -1 while the sequence holds fewer than ``budget`` keys. Returns (B, H) int32."""
    B, H = block_table.shape[0], pages.n_head
    tp, tsb, mp = _table(pages, block_table, B)
    pp = _rows(position, (B,), "position", pages)
    dev = pages.device
    slots = position.new_empty((B, H))
    rc = _lib.load().sisa_paged_evict(pages.cbytes, tp, tsb, mp, pp, B, H, int(budget), int(recent), slots.data_ptr(),
                                      pages.status, _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_evict")
    backends.after_call(dev)
    return slots


def paged_append(proj: Tensor, z: Tensor | None, pages: KeyPages, block_table: Tensor, position: Tensor, carry: Tensor,
                 *, carry_out: Tensor | None = None, slots: Tensor | None = None, budget: int | None = None,
                 lengths: Tensor | None = None):
    """The new token of every sequence from its fused projection row ``proj`` (B, 1, NPAD) and forget logits ``z``
    (B, 1, H) fp32 (None: no forget gate): continues g, F and Phi from ``carry`` (B, H, 18) fp32 (updated in place,
    or written to ``carry_out``), rotates c and b, and writes the key to slot ``position`` of its pages, or
    to ``slots`` (B, H) from :func:`paged_evict` where that is >= 0. ``position`` (B,) int32 is the token's index
    in its sequence, < 0 for an idle row (nothing is written). With ``lengths`` (B,) int32 the number of keys
    after the write, min(position + 1, budget), is stored for :func:`paged_attention`.

    Returns q (a view of proj's Q columns), c~ (B, H, 1, 32), g and F (B, H, 1) fp32 (F None without z)."""
    H, dev = pages.n_head, pages.device
    shape = proj.shape
    if len(shape) != 3 or shape[1] != 1 or shape[2] < 273 * H:
        raise ValueError(f"proj must be (B, 1, >= {273 * H}), got {tuple(shape)}")
    B, _, width = shape
    if proj.dtype != pages.dtype:
        raise TypeError(f"projection dtype {proj.dtype} differs from the pages' {pages.dtype}")
    if proj.device != dev:
        raise ValueError(f"proj is on {proj.device}, the pages on {dev}")
    if torch.is_grad_enabled():
        _refuse_grad("paged_append", proj, z, carry, carry_out)
    tp, tsb, mp = _table(pages, block_table, B)
    pp = _rows(position, (B,), "position", pages)
    sp = None if slots is None else _rows(slots, (B, H), "slots", pages)
    lp = None if lengths is None else _rows(lengths, (B,), "lengths", pages)
    co = carry if carry_out is None else carry_out
    for t in (carry, co):
        if t.shape != (B, H, CARRY) or t.dtype != torch.float32 or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"carry must be a contiguous {(B, H, CARRY)} fp32 tensor on {dev}, got {tuple(t.shape)} "
                             f"{t.dtype} on {t.device}")
    sb, _, sl = proj.stride()
    if sl != 1 or proj.data_ptr() % 16 or (B > 1 and (sb % 8 or sb < width)):    # (sb < width: rows shared or overlapping)
        proj = proj.clone(memory_format=torch.contiguous_format)
        sb = width
        if B > 1 and sb % 8:                    # rows of odd width: q's rows are read in 16-byte units
            wide = proj.new_empty((B, 1, -(-width // 8) * 8))
            wide[..., :width] = proj
            proj, sb = wide, wide.shape[2]
    c = proj.new_empty((B, H, 1, 32))
    g = carry.new_empty((B, H, 1))
    z2 = f = zp = fp = None
    if z is not None:
        if pages.f is None:
            raise ValueError("z is given but the pages hold no f plane")
        if z.numel() != B * H or z.shape[0] != B or z.device != dev:
            raise ValueError(f"z must be ({B}, 1, {H}) on {dev}, got {tuple(z.shape)} on {z.device}")
        z2 = _f32(z)
        f = torch.empty_like(g)
        zp, fp = z2.data_ptr(), f.data_ptr()
    rc = _lib.load().sisa_paged_append(proj.data_ptr(), sb if B > 1 else width, zp, H, pages.cbytes, tp, tsb, mp, pp, sp,
                                       int(budget or 0), B, H, pages.dtype_code, carry.data_ptr(), co.data_ptr(),
                                       c.data_ptr(), g.data_ptr(), fp, lp, pages.status,
                                       _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_append")
    backends.after_call(dev)
    return proj.as_strided((B, H, 1, 64), (sb, 64, 64, 1)), c, g, f


def attention_key_weights(q: Tensor, k: Tensor, c: Tensor, b: Tensor, pos: Tensor, lam: Tensor, lse: Tensor, *,
                          first_query: int = 0) -> Tensor:
    """The attention each prompt key received: w[b, h, j] = the sum over the queries i >= max(j, first_query) of
    softmax(s_i)_j. q, k (B, H, L, 64) and c, b (B, H, L, 32) views in bf16 or fp16 (rotated, as
    :func:`sisa_b200.ops.attn_fwd` takes them), ``pos`` its position planes, ``lse`` (B, H, L) fp32 the
    log-sum-exp it returned. Returns (B, H, L) fp32."""
    if q.dim() != 4 or q.shape[-1] != 64:
        raise ValueError(f"q must be (B, H, L, 64), got {tuple(q.shape)}")
    B, H, L, _ = q.shape
    if k.shape != (B, H, L, 64) or c.shape != (B, H, L, 32) or b.shape != (B, H, L, 32):
        raise ValueError(f"k, c and b must be {(B, H, L, 64)}, {(B, H, L, 32)} and {(B, H, L, 32)}, got "
                         f"{tuple(k.shape)}, {tuple(c.shape)} and {tuple(b.shape)}")
    if any(t.dtype != q.dtype for t in (k, c, b)):
        raise TypeError(f"q, k, c and b differ in dtype: {q.dtype}, {k.dtype}, {c.dtype}, {b.dtype}")
    if torch.is_grad_enabled():
        _refuse_grad("attention_key_weights", q, k, c, b, pos, lam, lse)
    lib = _lib.load()
    code = _lib.dtype_code(q.dtype)
    if pos.shape != (B, H, 4, lib.sisa_pos_len(L)) or not pos.is_contiguous() or pos.dtype != torch.float32:
        raise ValueError(f"pos must be the contiguous position planes {(B, H, 4, lib.sisa_pos_len(L))}, got "
                         f"{tuple(pos.shape)} {pos.dtype}")
    if lse.shape != (B, H, L) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be {(B, H, L)} fp32, got {tuple(lse.shape)} {lse.dtype}")
    lam = lam.float().contiguous()
    if lam.shape != (H,):
        raise ValueError(f"lam must have shape {(H,)}, got {tuple(lam.shape)}")
    dev = q.device
    if any(t.device != dev for t in (k, c, b, pos, lam, lse)) or not q.is_cuda:
        raise ValueError("attention_key_weights takes CUDA tensors on one device")
    # (a tensor map has no stride of 0: operands shared by sequences or heads are copied)
    q, k, c, b = (_operand(t if t.stride(0) and t.stride(1) else t.contiguous()) for t in (q, k, c, b))
    lse = lse.contiguous()
    w = lse.new_empty((B, H, L))
    rc = lib.sisa_attn_key_weights(*map(_lib.view4_bytes, (q, k, c, b)), pos.data_ptr(), lam.data_ptr(), lse.data_ptr(), B,
                                   H, L, int(first_query), code, w.data_ptr(), backends.status_word(dev).data_ptr(),
                                   _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_attn_key_weights")
    backends.after_call(dev)
    return w


def paged_fill(pages: KeyPages, block_table: Tensor, k: Tensor, v: Tensor, b: Tensor, g: Tensor, fgate: Tensor | None, *,
               weight: Tensor | None = None, keep: int | None = None, recent: int = 0) -> int:
    """A prompt's keys into pages: k, v (B, H, L, 64), b~ (B, H, L, 32), g and fgate (B, H, L) fp32. With ``keep``
    < L only the ``recent`` newest and the ``keep - recent`` heaviest of the others by ``weight`` (B, H, L) fp32 stay
    (the earlier position where two weigh the same), in ascending order from slot 0 on; their weights and
    token indices go along. Returns the number of keys per sequence."""
    if k.dim() != 4 or k.shape[-1] != 64:
        raise ValueError(f"k must be (B, H, L, 64), got {tuple(k.shape)}")
    B, H, L, _ = k.shape
    if H != pages.n_head or v.shape != (B, H, L, 64) or b.shape != (B, H, L, 32):
        raise ValueError(f"k, v and b must be (B, {pages.n_head}, L, 64), (.., 64) and (.., 32), got {tuple(k.shape)}, "
                         f"{tuple(v.shape)} and {tuple(b.shape)}")
    if k.dtype != pages.dtype or v.dtype != pages.dtype or b.dtype != pages.dtype:
        raise TypeError(f"k, v and b must be {pages.dtype} like the pages, got {k.dtype}, {v.dtype}, {b.dtype}")
    if torch.is_grad_enabled():
        _refuse_grad("paged_fill", k, v, b, g, fgate, weight)
    dev = pages.device
    for t in (k, v, b, g, fgate, weight):
        if t is not None and t.device != dev:
            raise ValueError(f"the prompt's keys must lie on {dev} like the pages")
    keep = L if keep is None else int(keep)
    if weight is not None:
        if weight.shape != (B, H, L) or weight.dtype != torch.float32:
            raise ValueError(f"weight must be {(B, H, L)} fp32, got {tuple(weight.shape)} {weight.dtype}")
        weight = weight.contiguous()
    for name, t in (("g", g), ("fgate", fgate)):
        if t is not None and (t.shape != (B, H, L) or t.dtype != torch.float32):
            raise ValueError(f"{name} must be {(B, H, L)} fp32, got {tuple(t.shape)} {t.dtype}")
    if fgate is not None and pages.f is None:
        raise ValueError("fgate is given but the pages hold no f plane")
    g, fgate = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (g, fgate))
    tp, tsb, mp = _table(pages, block_table, B)
    lib = _lib.load()
    ws = block_table.new_empty(max(B * H * min(keep, L), 4))             # the kept positions
    k, v, b = _operand(k), _operand(v), _operand(b)
    fs = (0, 0) if fgate is None else fgate.stride()[:2]
    rc = lib.sisa_paged_fill(pages.cbytes, tp, tsb, mp, *map(_lib.view4_bytes, (k, v, b)), g.data_ptr(), g.stride(0),
                             g.stride(1), _lib.ptr(fgate), *fs, _lib.ptr(weight), B, H, L, keep, int(recent), ws.data_ptr(),
                             pages.status, _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_fill")
    backends.after_call(dev)
    return keep
