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
that a captured CUDA graph serves every step.
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
        self.k, self.v, self.b, self.g, self.f, self.weight, self.token = k, v, b, g, f, weight, token
        self.n_pages, self.n_head, self.page_size = P, H, S
        self.dtype, self.device = k.dtype, k.device
        self._c = _lib.Pages(k.data_ptr(), v.data_ptr(), b.data_ptr(), g.data_ptr(), _lib.ptr(f), _lib.ptr(weight),
                             _lib.ptr(token), k.stride(0), k.stride(1), v.stride(0), v.stride(1), b.stride(0), b.stride(1),
                             g.stride(0), g.stride(1), P, S)

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

    def cref(self):
        return _lib.ctypes.byref(self._c)


def _table(pages: KeyPages, table: Tensor, B: int) -> tuple[int, int, int]:
    """(pointer, row stride, max_pages) of a block table."""
    if table.dim() != 2 or table.shape[0] != B or table.shape[1] < 1 or table.dtype != torch.int32:
        raise ValueError(f"block_table must be ({B}, max_pages) int32, got {tuple(table.shape)} {table.dtype}")
    if table.device != pages.device:
        raise ValueError(f"block_table is on {table.device}, the pages on {pages.device}")
    if table.stride(1) != 1 and table.shape[1] > 1:
        raise ValueError("block_table rows must be contiguous")
    return table.data_ptr(), max(table.stride(0), table.shape[1]) if B == 1 else table.stride(0), table.shape[1]


def _rows(t: Tensor, shape: tuple, name: str, pages: KeyPages) -> Tensor:
    """An int32 row tensor (positions, lengths, slots), checked."""
    if tuple(t.shape) != shape or t.dtype != torch.int32 or not t.is_contiguous() or t.device != pages.device:
        raise ValueError(f"{name} must be a contiguous {shape} int32 tensor on {pages.device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    return t


def _operand(t: Tensor) -> Tensor:
    """``t`` as the kernels read it: unit last stride, 16-byte aligned rows."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 and s >= 0 for s in t.stride()[:-1]) \
        and t.stride(-2) > 0
    return t if ok else t.contiguous()


def _check_query(q: Tensor, c: Tensor, pages: KeyPages) -> tuple[int, int]:
    if q.dim() != 4 or q.shape[2] != 1 or q.shape[3] != 64 or tuple(c.shape) != (q.shape[0], q.shape[1], 1, 32):
        raise ValueError(f"paged_attention takes one query row with d_head 64 and d_state 32, got {tuple(q.shape)} and "
                         f"{tuple(c.shape)}")
    if q.shape[1] != pages.n_head:
        raise ValueError(f"q has {q.shape[1]} heads, the pages {pages.n_head}")
    if q.dtype != pages.dtype:
        raise TypeError(f"q dtype {q.dtype} differs from the pages' {pages.dtype}")
    if q.device != pages.device:
        raise ValueError(f"q is on {q.device}, the pages on {pages.device}")
    return q.shape[0], q.shape[1]


def paged_attention(q: Tensor, c: Tensor, g: Tensor, fgate: Tensor | None, pages: KeyPages, block_table: Tensor,
                    lengths: Tensor, lam: Tensor, *, accumulate: bool = False, weight_out: Tensor | None = None,
                    return_lse: bool = False):
    """One new token per sequence over its paged keys. q (B, H, 1, 64), c (B, H, 1, 32) in the pages' dtype; g,
    fgate (B, H, 1) fp32 (fgate None: no forget gate); lengths (B,) int32, the keys of each sequence with the
    new token's own among them (0: idle row, y = 0); lam (H,) fp32. Returns y (B, H, 1, 64) in q.dtype and, with
    ``return_lse``, (y, lse) with lse (B, H) fp32 in log2 units (-inf for an idle row).

    With ``accumulate`` each key's softmax share is added to its weight: ``pages.weight`` in place, or
    ``weight_out`` = ``pages.weight`` + share where that plane is given (used slots only)."""
    B, H = _check_query(q, c, pages)
    lib = _lib.load()
    dev = q.device
    tp, tsb, mp = _table(pages, block_table, B)
    _rows(lengths, (B,), "lengths", pages)
    if accumulate and pages.weight is None:
        raise ValueError("accumulate needs pages with a weight plane")
    if weight_out is not None:
        if not accumulate:
            raise ValueError("weight_out needs accumulate=True")
        if tuple(weight_out.shape) != tuple(pages.weight.shape) or weight_out.stride() != pages.weight.stride() \
                or weight_out.dtype != torch.float32 or weight_out.device != dev:
            raise ValueError("weight_out must be an fp32 plane with the shape and strides of pages.weight")
    if fgate is not None and pages.f is None:
        raise ValueError("fgate is given but the pages hold no f plane")
    wo = None if not accumulate else (pages.weight if weight_out is None else weight_out)
    if c.dtype != q.dtype:
        c = c.to(q.dtype)
    q, c = _operand(q), _operand(c)
    gq = g.reshape(B, H).float().contiguous()
    fq = None if fgate is None else fgate.reshape(B, H).float().contiguous()
    lam = lam.float().contiguous()
    if lam.shape != (H,):
        raise ValueError(f"lam must have shape {(H,)}, got {tuple(lam.shape)}")
    y = torch.empty((B, H, 1, 64), device=dev, dtype=q.dtype)
    lse = torch.empty((B, H), device=dev, dtype=torch.float32) if return_lse else None
    nbytes = lib.sisa_paged_attn_workspace(B, H, mp * pages.page_size, int(accumulate))
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
    st = backends.status_word(dev)
    vq, vc, vy = _lib.view4(q), _lib.view4(c), _lib.view4(y)
    rc = lib.sisa_paged_attn(_lib.vref(vq), _lib.vref(vc), gq.data_ptr(), _lib.ptr(fq), pages.cref(), tp, tsb, mp,
                             lengths.data_ptr(), lam.data_ptr(), B, H, pages.dtype_code, _lib.vref(vy), _lib.ptr(lse),
                             _lib.ptr(wo), ws.data_ptr(), st.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_attn")
    backends.after_call(dev)
    return (y, lse) if return_lse else y


def paged_evict(pages: KeyPages, block_table: Tensor, position: Tensor, budget: int, recent: int) -> Tensor:
    """The slot that the token ``position`` (B,) int32 takes per (sequence, head): the one whose key has the
    least accumulated weight among the keys older than the ``recent`` newest, the lowest slot where several
    weigh the same; -1 while the sequence holds fewer than ``budget`` keys. Returns (B, H) int32."""
    B, H = block_table.shape[0], pages.n_head
    tp, tsb, mp = _table(pages, block_table, B)
    _rows(position, (B,), "position", pages)
    slots = torch.empty((B, H), dtype=torch.int32, device=pages.device)
    st = backends.status_word(pages.device)
    rc = _lib.load().sisa_paged_evict(pages.cref(), tp, tsb, mp, position.data_ptr(), B, H, int(budget), int(recent),
                                      slots.data_ptr(), st.data_ptr(), _lib.stream_ptr(pages.device))
    _lib.check(rc, "sisa_paged_evict")
    backends.after_call(pages.device)
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
    lib = _lib.load()
    H = pages.n_head
    if proj.dim() != 3 or proj.shape[1] != 1 or proj.shape[2] < 273 * H:
        raise ValueError(f"proj must be (B, 1, >= {273 * H}), got {tuple(proj.shape)}")
    B, dev = proj.shape[0], pages.device
    if proj.dtype != pages.dtype:
        raise TypeError(f"projection dtype {proj.dtype} differs from the pages' {pages.dtype}")
    if proj.device != dev:
        raise ValueError(f"proj is on {proj.device}, the pages on {dev}")
    tp, tsb, mp = _table(pages, block_table, B)
    _rows(position, (B,), "position", pages)
    if slots is not None:
        _rows(slots, (B, H), "slots", pages)
    if lengths is not None:
        _rows(lengths, (B,), "lengths", pages)
    for name, t in (("carry", carry), ("carry_out", carry_out)):
        if t is not None and (tuple(t.shape) != (B, H, CARRY) or t.dtype != torch.float32 or not t.is_contiguous()
                              or t.device != dev):
            raise ValueError(f"{name} must be a contiguous {(B, H, CARRY)} fp32 tensor on {dev}, got {tuple(t.shape)} "
                             f"{t.dtype} on {t.device}")
    if z is not None and pages.f is None:
        raise ValueError("z is given but the pages hold no f plane")
    co = carry if carry_out is None else carry_out
    proj2 = proj.reshape(B, proj.shape[-1])
    if proj2.stride(-1) != 1 or proj2.stride(0) % 8 or proj2.data_ptr() % 16:
        proj2 = proj2.contiguous()
    c = torch.empty((B, H, 1, 32), dtype=proj.dtype, device=dev)
    g = torch.empty((B, H, 1), dtype=torch.float32, device=dev)
    z2 = f = None
    if z is not None:
        z2 = z.reshape(B, H).float().contiguous()
        f = torch.empty((B, H, 1), dtype=torch.float32, device=dev)
    st = backends.status_word(dev)
    rc = lib.sisa_paged_append(proj2.data_ptr(), proj2.stride(0) if B > 1 else proj2.shape[1], _lib.ptr(z2), H,
                               pages.cref(), tp, tsb, mp, position.data_ptr(), _lib.ptr(slots), int(budget or 0), B, H,
                               pages.dtype_code, carry.data_ptr(), co.data_ptr(), c.data_ptr(), g.data_ptr(),
                               _lib.ptr(f), _lib.ptr(lengths), st.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_append")
    backends.after_call(dev)
    return proj2[:, :H * 64].view(B, H, 64).unsqueeze(2), c, g, f


def attention_key_weights(q: Tensor, k: Tensor, c: Tensor, b: Tensor, pos: Tensor, lam: Tensor, lse: Tensor, *,
                          first_query: int = 0) -> Tensor:
    """The attention each prompt key received: w[b, h, j] = the sum over the queries i >= max(j, first_query) of
    softmax(s_i)_j. q, k (B, H, L, 64) and c, b (B, H, L, 32) views in bf16 or fp16 (rotated, as
    :func:`sisa_b200.ops.attn_fwd` takes them), ``pos`` its position planes, ``lse`` (B, H, L) fp32 the
    log-sum-exp it returned. Returns (B, H, L) fp32."""
    if q.dim() != 4 or q.shape[-1] != 64:
        raise ValueError(f"q must be (B, H, L, 64), got {tuple(q.shape)}")
    B, H, L, _ = q.shape
    if tuple(k.shape) != (B, H, L, 64) or tuple(c.shape) != (B, H, L, 32) or tuple(b.shape) != (B, H, L, 32):
        raise ValueError(f"k, c and b must be {(B, H, L, 64)}, {(B, H, L, 32)} and {(B, H, L, 32)}, got "
                         f"{tuple(k.shape)}, {tuple(c.shape)} and {tuple(b.shape)}")
    if any(t.dtype != q.dtype for t in (k, c, b)):
        raise TypeError(f"q, k, c and b differ in dtype: {q.dtype}, {k.dtype}, {c.dtype}, {b.dtype}")
    lib = _lib.load()
    code = _lib.dtype_code(q.dtype)
    if tuple(pos.shape) != (B, H, 4, lib.sisa_pos_len(L)) or not pos.is_contiguous() or pos.dtype != torch.float32:
        raise ValueError(f"pos must be the contiguous position planes {(B, H, 4, lib.sisa_pos_len(L))}, got "
                         f"{tuple(pos.shape)} {pos.dtype}")
    if tuple(lse.shape) != (B, H, L) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be {(B, H, L)} fp32, got {tuple(lse.shape)} {lse.dtype}")
    lam = lam.float().contiguous()
    if lam.shape != (H,):
        raise ValueError(f"lam must have shape {(H,)}, got {tuple(lam.shape)}")
    dev = q.device
    if any(t.device != dev for t in (k, c, b, pos, lam, lse)) or not q.is_cuda:
        raise ValueError("attention_key_weights takes CUDA tensors on one device")
    q, k, c, b, lse = _operand(q), _operand(k), _operand(c), _operand(b), lse.contiguous()
    w = torch.empty((B, H, L), dtype=torch.float32, device=dev)
    st = backends.status_word(dev)
    vs = [_lib.view4(t) for t in (q, k, c, b)]
    rc = lib.sisa_attn_key_weights(*(_lib.vref(v) for v in vs), pos.data_ptr(), lam.data_ptr(), lse.data_ptr(), B, H, L,
                                   int(first_query), code, w.data_ptr(), st.data_ptr(), _lib.stream_ptr(dev))
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
    if H != pages.n_head or tuple(v.shape) != (B, H, L, 64) or tuple(b.shape) != (B, H, L, 32):
        raise ValueError(f"k, v and b must be (B, {pages.n_head}, L, 64), (.., 64) and (.., 32), got {tuple(k.shape)}, "
                         f"{tuple(v.shape)} and {tuple(b.shape)}")
    if any(t.dtype != pages.dtype for t in (k, v, b)):
        raise TypeError(f"k, v and b must be {pages.dtype} like the pages, got {k.dtype}, {v.dtype}, {b.dtype}")
    dev = pages.device
    if any(t is not None and t.device != dev for t in (k, v, b, g, fgate, weight)):
        raise ValueError(f"the prompt's keys must lie on {dev} like the pages")
    keep = L if keep is None else int(keep)
    if weight is not None:
        if tuple(weight.shape) != (B, H, L) or weight.dtype != torch.float32:
            raise ValueError(f"weight must be {(B, H, L)} fp32, got {tuple(weight.shape)} {weight.dtype}")
        weight = weight.contiguous()
    for name, t in (("g", g), ("fgate", fgate)):
        if t is not None and (tuple(t.shape) != (B, H, L) or t.dtype != torch.float32):
            raise ValueError(f"{name} must be {(B, H, L)} fp32, got {tuple(t.shape)} {t.dtype}")
    if fgate is not None and pages.f is None:
        raise ValueError("fgate is given but the pages hold no f plane")
    g, fgate = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (g, fgate))
    tp, tsb, mp = _table(pages, block_table, B)
    lib = _lib.load()
    ws = torch.empty(max(lib.sisa_paged_fill_workspace(B, H, keep), 16), dtype=torch.uint8, device=dev)
    k, v, b = _operand(k), _operand(v), _operand(b)
    vk, vv, vb = _lib.view4(k), _lib.view4(v), _lib.view4(b)
    fs = (0, 0) if fgate is None else fgate.stride()[:2]
    st = backends.status_word(dev)
    rc = lib.sisa_paged_fill(pages.cref(), tp, tsb, mp, _lib.vref(vk), _lib.vref(vv), _lib.vref(vb), g.data_ptr(),
                             g.stride(0), g.stride(1), _lib.ptr(fgate), *fs, _lib.ptr(weight), B, H, L, keep, int(recent),
                             ws.data_ptr(), st.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "sisa_paged_fill")
    backends.after_call(dev)
    return keep
