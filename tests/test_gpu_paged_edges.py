"""Rows and arguments at the edges of the paged operators: table entries that name no page, rows left without
any key, slots past a sequence's end. Tolerances are those of test_gpu_paged.py."""
from __future__ import annotations

import math

import pytest
import torch

from tests.helpers import max_abs
from tests.test_gpu_paged import HALF_ULP, SHARE_REL, attn_case, attn_truth, get, put, widen

pytestmark = pytest.mark.gpu


def call(pages, table, lengths, x, dev, **kw):
    """paged_attention without reading the status word (the caller does)."""
    from sisa_b200.kernels.paged import paged_attention

    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    return paged_attention(x["q"].to(dev), x["c"].to(dev), x["gq"].to(dev), x["fq"].to(dev), pages, table, ln,
                           x["lam"].to(dev), return_lse=True, **kw)


def check_row(y, lse, w, row, want):
    """One sequence's outputs against its fp64 truth (y (H, 64), lse (H,), w (H, n) on the host)."""
    yr, lr, p = want
    assert bool(((y.double() - yr).abs() <= HALF_ULP[y.dtype] * yr.abs() * (1 + 1e-3) + SHARE_REL * row["v"].abs().max()).all())
    assert max_abs(lse, lr) <= 5e-5 * max(1.0, float(lr.abs().max()) / 32)
    want_w = row["w"].double() + p
    assert bool(((w.double() - want_w).abs() <= SHARE_REL * p + 2.0 ** -23 * want_w + 1e-30).all())


# 5 keys: one page; 300: several warps of one CTA, or of several; 6000: many CTAs (joined by the second kernel)
@pytest.mark.parametrize("n,S,wide", [(5, 16, False), (5, 64, True), (300, 32, False), (300, 32, True), (6000, 64, False)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_row_whose_keys_are_all_left_out(cuda_dev, n, S, wide, accumulate):
    """Every table entry of row 0 names no page: y = 0 and lse = -inf as for a row with no keys, the status names the
    bad page and not a non-finite input, and the other row is not touched by it."""
    from sisa_b200 import backends

    lengths = [n, 70]
    pages, table, rows, x = attn_case(lengths, 2, S, torch.bfloat16, cuda_dev, seed=n)
    bad = widen(table) if wide else table.clone()
    bad[0, ::2], bad[0, 1::2] = -1, pages.n_pages
    before = pages.weight.clone()
    y, lse = call(pages, bad, lengths, x, cuda_dev, accumulate=accumulate)
    with pytest.raises(ValueError):
        backends.check_status(cuda_dev)
    assert bool((y[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    truth = attn_truth(rows, lengths, x)[1]
    w = get(pages.weight, table, 1, 70)
    if accumulate:
        check_row(y[1, :, 0].cpu(), lse[1].cpu(), w, rows[1], truth)
        put(pages.weight, table, 1, rows[1]["w"])
    assert torch.equal(pages.weight.nan_to_num(-1.0), before.nan_to_num(-1.0))


@pytest.mark.parametrize("n,S,wide", [(130, 16, False), (130, 32, True), (500, 64, False), (3001, 16, True)])
def test_keys_of_a_bad_page_are_left_out(cuda_dev, n, S, wide):
    """One of a row's pages is bad: the result is that of the other keys, whose weights alone grow."""
    from sisa_b200 import backends

    lengths = [n]
    pages, table, rows, x = attn_case(lengths, 3, S, torch.bfloat16, cuda_dev, seed=n + 1)
    bad = widen(table) if wide else table.clone()
    bad[0, 1] = pages.n_pages
    keep = torch.tensor([j for j in range(n) if j // S != 1])
    kept = {name: t[:, keep] if t.dim() > 1 and t.shape[1] == n else t for name, t in rows[0].items()}
    y, lse = call(pages, bad, lengths, x, cuda_dev, accumulate=True)
    with pytest.raises(ValueError):
        backends.check_status(cuda_dev)
    w = get(pages.weight, table, 0, n)
    check_row(y[0, :, 0].cpu(), lse[0].cpu(), w[:, keep], kept, attn_truth([kept], [len(keep)], x)[0])
    out = torch.tensor([j for j in range(n) if j // S == 1])
    assert torch.equal(w[:, out], rows[0]["w"][:, out])


@pytest.mark.parametrize("n,wide", [(3, False), (400, False), (400, True), (6000, False)])
def test_a_row_whose_scores_are_all_minus_infinity(cuda_dev, n, wide):
    """No key has a share: y = 0, lse = -inf, the weights keep their values, and the status says that an input was
    not finite."""
    from sisa_b200 import backends

    pages, table, rows, x = attn_case([n], 2, 32, torch.bfloat16, cuda_dev, seed=n + 2)
    put(pages.f, table, 0, torch.full((2, n), math.inf))
    y, lse = call(pages, widen(table) if wide else table, [n], x, cuda_dev, accumulate=True)
    with pytest.raises(FloatingPointError):
        backends.check_status(cuda_dev)
    assert bool((y == 0).all()) and bool((lse == -math.inf).all())
    assert torch.equal(get(pages.weight, table, 0, n), rows[0]["w"])


@pytest.mark.parametrize("wide", [False, True])
def test_rows_may_share_the_pages_they_read(cuda_dev, wide):
    """Four queries over a common prefix of three pages, each with an own page after it."""
    from sisa_b200 import backends

    S, H, lengths = 32, 3, [100, 128, 97, 121]
    pages, table, rows, x = attn_case([128] * 4, H, S, torch.bfloat16, cuda_dev, seed=8)
    shared = table.clone()
    shared[1:, :3] = table[0, :3]
    for i, n in enumerate(lengths):
        for name in ("k", "v", "b", "g", "f", "w"):
            rows[i][name] = torch.cat([rows[0][name][:, :96], rows[i][name][:, 96:n]], dim=1)
    before = pages.weight.clone()
    y, lse = call(pages, widen(shared) if wide else shared, lengths, x, cuda_dev)
    backends.check_status(cuda_dev)
    for i, (yr, lr, _) in enumerate(attn_truth(rows, lengths, x)):
        bound = HALF_ULP[y.dtype] * yr.abs() * (1 + 1e-3) + SHARE_REL * rows[i]["v"].abs().max()
        assert bool(((y[i, :, 0].double().cpu() - yr).abs() <= bound).all())
        assert max_abs(lse[i], lr) <= 5e-5 * max(1.0, float(lr.abs().max()) / 32)
    assert torch.equal(pages.weight.nan_to_num(-1.0), before.nan_to_num(-1.0))


def test_inputs_that_require_a_gradient_are_refused(cuda_dev):
    """None of the operators has a backward: in grad mode they raise, under no_grad they run as ever."""
    from sisa_b200.kernels import paged as K
    from tests.test_gpu_paged import prompt

    dev, bf = cuda_dev, torch.bfloat16
    pages, table, rows, x = attn_case([40], 2, 16, bf, dev, seed=1)
    d = {n: t.to(dev) for n, t in x.items()}
    ln, pos = (torch.tensor([n], dtype=torch.int32, device=dev) for n in (40, 3))
    proj, z, carry = torch.zeros(1, 1, 560, dtype=bf, device=dev), torch.zeros(1, 1, 2, device=dev), torch.zeros(1, 2, 18, device=dev)
    q, k, v, c, b, pl, lam, lse = prompt(1, 2, 40, bf, dev, seed=2)
    g, f, w = pl[:, :, 0, :40].contiguous(), pl[:, :, 1, :40].contiguous(), torch.rand(1, 2, 40, device=dev)
    calls = [(lambda *a: K.paged_attention(*a[:4], pages, table, ln, a[4]), [d["q"], d["c"], d["gq"], d["fq"], d["lam"]]),
             (lambda *a: K.paged_append(a[0], a[1], pages, table, pos, a[2]), [proj, z, carry]),
             (K.attention_key_weights, [q, k, c, b, pl, lam, lse]),
             (lambda *a: K.paged_fill(pages, table, *a[:5], weight=a[5]), [k, v, b, g, f, w]),
             (K.KeyPages, [pages.k, pages.v, pages.b, pages.g, pages.f, pages.weight])]
    for fn, args in calls:
        fn(*args)
        for i in range(len(args)):
            a = list(args)
            a[i] = a[i].detach().clone().requires_grad_(True)
            with pytest.raises(ValueError, match="no backward"):
                fn(*a)
            with torch.no_grad():
                fn(*a)


def test_per_row_values_of_another_order_are_refused(cuda_dev):
    """g, F and the forget logits as (H, B): as many values as are wanted, in the wrong order."""
    from sisa_b200.kernels import paged as K

    dev, B, H = cuda_dev, 3, 2
    pages, table, rows, x = attn_case([40, 7, 12], H, 16, torch.bfloat16, dev, seed=1)
    d = {n: t.to(dev) for n, t in x.items()}
    ln = torch.tensor([40, 7, 12], dtype=torch.int32, device=dev)
    proj, carry = torch.zeros(B, 1, 560, dtype=torch.bfloat16, device=dev), torch.zeros(B, H, 18, device=dev)
    z, idle = torch.zeros(B, 1, H, device=dev), torch.full((B,), -1, dtype=torch.int32, device=dev)
    args = (pages, table, ln, d["lam"])
    want = K.paged_attention(d["q"], d["c"], d["gq"], d["fq"], *args)
    assert torch.equal(want, K.paged_attention(d["q"], d["c"], d["gq"].view(B, H), d["fq"].view(B, 1, H), *args))
    K.paged_append(proj, z.view(B, H), pages, table, idle, carry)
    for g, f in ((d["gq"].transpose(0, 1), d["fq"]), (d["gq"], d["fq"].transpose(0, 1)), (d["gq"][:2], d["fq"])):
        with pytest.raises(ValueError, match="must be"):
            K.paged_attention(d["q"], d["c"], g, f, *args)
    with pytest.raises(ValueError, match="must be"):
        K.paged_append(proj, z.transpose(0, 2), pages, table, idle, carry)


# 13, 30 and 301 leave a ragged last group of four keys; the wide tables take the kernels that split the keys
@pytest.mark.parametrize("S,wide", [(16, False), (16, True), (64, False), (64, True), (256, True)])
def test_weights_are_written_in_used_slots_only(cuda_dev, S, wide):
    """Unused slots hold a sentinel in both planes: in place and into a plane of its own, every used slot becomes
    weight + share and no other value changes."""
    from sisa_b200 import backends

    lengths = [13, 0, 30, 301, 64, 1, 2 * S + 3]
    pages, table, rows, x = attn_case(lengths, 3, S, torch.bfloat16, cuda_dev, seed=S)
    t = widen(table) if wide else table
    used = torch.zeros_like(pages.weight, dtype=torch.bool)
    for i, n in enumerate(lengths):
        if n:
            put(used, table, i, torch.ones(pages.n_head, n, dtype=torch.bool))
    pages.weight[~used] = 17.25
    before = pages.weight.clone()
    out = torch.full_like(before, -3.5)
    y0, lse0 = call(pages, t, lengths, x, cuda_dev, accumulate=True, weight_out=out)
    backends.check_status(cuda_dev)
    assert torch.equal(pages.weight, before) and bool((out[~used] == -3.5).all())
    y1, lse1 = call(pages, t, lengths, x, cuda_dev, accumulate=True)
    backends.check_status(cuda_dev)
    assert bool((pages.weight[~used] == 17.25).all()) and torch.equal(pages.weight[used], out[used])
    assert torch.equal(y0, y1) and torch.equal(lse0, lse1)
    for i, want in enumerate(attn_truth(rows, lengths, x)):
        if want is not None:
            check_row(y0[i, :, 0].cpu(), lse0[i].cpu(), get(out, table, i, lengths[i]), rows[i], want)


@pytest.mark.parametrize("units,budget,S", [((1, 1), 4097, 16), ((2, 2), 8192, 64), ((1, 3), 5003, 128), ((3, 1), 40961, 256)])
def test_evict_by_clusters_of_eight(cuda_dev, units, budget, S):
    """Few units with a large budget: eight blocks share one, their minima meet in the first. The least weight lies in
    each block's part once, and ties across blocks go to the lowest slot."""
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_evict
    from tests.test_gpu_paged import make_pages, make_table

    B, H = units
    gen = torch.Generator().manual_seed(budget)
    table, P = make_table([budget] * B, S, 3, cuda_dev)
    pages = make_pages(P, H, S, torch.bfloat16, cuda_dev)
    tok = torch.stack([torch.stack([torch.randperm(budget, generator=gen) for _ in range(H)]) for _ in range(B)])
    w = torch.rand(B, H, budget, generator=gen) + 1.0
    for b in range(B):
        put(pages.token, table, b, tok[b].to(torch.int32))
    recent = 50
    pos = torch.full((B,), budget, dtype=torch.int32, device=cuda_dev)
    old = tok < budget - recent
    spots = [0, 3, 1023, 1024, 2047, 2048, 3500, 4095, budget - 1] + [k * 1024 + 5 for k in range(budget // 1024)]
    for j in spots:
        v = w.clone()
        v[..., j] = 0.5
        v[..., j + 700:j + 702] = 0.5                     # ties further on
        for b in range(B):
            put(pages.weight, table, b, v[b])
        got = paged_evict(pages, table, pos, budget, recent).cpu().long()
        backends.check_status(cuda_dev)
        masked = v.masked_fill(~old, math.inf)
        least = masked.min(-1, keepdim=True).values
        first = (masked == least).to(torch.int8).argmax(-1)          # the lowest slot of the least weight
        assert torch.equal(got, first), j


@pytest.mark.parametrize("L,keep,recent,S", [(5, 3, 0, 16), (700, 100, 37, 64), (1500, 1499, 1, 32)])
def test_fill_with_a_choice_in_fp16(cuda_dev, L, keep, recent, S):
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_fill
    from tests.test_gpu_paged import fill_truth, make_pages, make_table, prompt

    B, H = 2, 3
    q, k, v, c, b, pos, lam, lse = prompt(B, H, L, torch.float16, cuda_dev, seed=L)
    w = torch.rand(B, H, L, generator=torch.Generator().manual_seed(L))
    w[1, 1] = (w[1, 1] * 4).round()
    table, P = make_table([keep] * B, S, L, cuda_dev)
    pages = make_pages(P, H, S, torch.float16, cuda_dev, fill=0.25)
    pages.weight.fill_(7.5)
    pages.token.fill_(-9)
    g, f = pos[:, :, 0, :L], pos[:, :, 1, :L]
    assert paged_fill(pages, table, k, v, b, g, f, weight=w.to(cuda_dev), keep=keep, recent=recent) == keep
    backends.check_status(cuda_dev)
    idx = fill_truth(w, keep, recent)
    used = torch.zeros_like(pages.weight, dtype=torch.bool)
    for i in range(B):
        put(used, table, i, torch.ones(H, keep, dtype=torch.bool))
        at = idx[i]
        assert torch.equal(get(pages.token, table, i, keep).long(), at)
        for plane, src in ((pages.k, k), (pages.v, v), (pages.b, b)):
            assert torch.equal(get(plane, table, i, keep), src[i].cpu().gather(1, at.unsqueeze(-1).expand(-1, -1, src.shape[-1])))
        for plane, src in ((pages.g, g), (pages.f, f), (pages.weight, w)):
            assert torch.equal(get(plane, table, i, keep), src[i].cpu().gather(1, at))
    for plane, value in ((pages.k, 0.25), (pages.v, 0.25), (pages.b, 0.25), (pages.g, 0.25), (pages.f, 0.25), (pages.weight, 7.5),
                         (pages.token, -9)):
        assert bool((plane[~used] == value).all())


def test_queries_shared_by_broadcasting(cuda_dev):
    """A query row that several sequences share through a stride of 0 gives what copies of it give."""
    from sisa_b200.kernels import paged as K

    dev, lengths = cuda_dev, [40, 300, 77]
    pages, table, rows, x = attn_case(lengths, 2, 16, torch.bfloat16, dev, seed=5)
    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    q, c = x["q"][:1].to(dev).expand(3, 2, 1, 64), x["c"][:1, :1].to(dev).expand(3, 2, 1, 32)
    g, f = x["gq"][:1].to(dev).expand(3, 2, 1), x["fq"][:1].to(dev).expand(3, 2, 1)
    a = K.paged_attention(q, c, g, f, pages, table, ln, x["lam"].to(dev))
    b = K.paged_attention(q.contiguous(), c.contiguous(), g.contiguous(), f.contiguous(), pages, table, ln, x["lam"].to(dev))
    assert torch.equal(a, b)


def test_a_prompt_shared_by_broadcasting(cuda_dev):
    from sisa_b200 import backends
    from sisa_b200.kernels import paged as K
    from tests.test_gpu_paged import make_pages, make_table, prompt

    L = 130
    q, k, v, c, b, pl, lam, lse = prompt(1, 2, L, torch.bfloat16, cuda_dev, seed=2)
    w = K.attention_key_weights(q, k, c, b, pl, lam, lse)
    q3, k3, c3, b3, l3 = (t.expand(3, *t.shape[1:]) for t in (q, k, c, b, lse))
    assert torch.equal(K.attention_key_weights(q3, k3, c3, b3, pl.repeat(3, 1, 1, 1), lam, l3), w.expand(3, 2, L))
    heads = K.attention_key_weights(q, k[:, :1].expand(1, 2, L, 64), c, b, pl, lam, lse)       # keys shared by the heads
    assert torch.equal(heads, K.attention_key_weights(q, k[:, :1].repeat(1, 2, 1, 1), c, b, pl, lam, lse))
    table, P = make_table([50] * 3, 32, 4, cuda_dev)
    src = [t.expand(3, *t.shape[1:]) for t in (k, v, b, pl[:, :, 0, :L], pl[:, :, 1, :L], w)]
    filled = [make_pages(P, 2, 32, torch.bfloat16, cuda_dev, fill=0.5) for _ in range(2)]
    K.paged_fill(filled[0], table, *src[:5], weight=src[5], keep=50, recent=9)
    src = [t.contiguous() for t in src]
    K.paged_fill(filled[1], table, *src[:5], weight=src[5], keep=50, recent=9)
    backends.check_status(cuda_dev)
    for name in ("k", "v", "b", "g", "f", "weight", "token"):
        assert torch.equal(getattr(filled[0], name), getattr(filled[1], name)), name


@pytest.mark.parametrize("H", [2, 3])
def test_a_projection_row_shared_by_broadcasting(cuda_dev, H):
    """The same new token for three sequences, and rows that overlap."""
    from sisa_b200 import backends
    from sisa_b200.kernels import paged as K
    from tests.test_gpu_paged import make_pages, make_table

    dev, bf, n = cuda_dev, torch.bfloat16, 273 * H + 8
    gen = torch.Generator().manual_seed(H)
    flat = torch.randn(n + 32, generator=gen).to(bf).to(dev)
    z, carry = torch.randn(1, 1, H, generator=gen).to(dev), torch.zeros(3, H, 18, device=dev)
    pos = torch.tensor([5, 0, 49], dtype=torch.int32, device=dev)
    table, P = make_table([50] * 3, 32, 4, dev)
    for proj in (flat[:n].view(1, 1, n).expand(3, 1, n), flat.as_strided((3, 1, n), (16, n, 1))):
        got = []
        for p, zz in ((proj, z.expand(3, 1, H)), (proj.contiguous(), z.repeat(3, 1, 1))):
            pages, co = make_pages(P, H, 32, bf, dev, fill=0.5), carry.clone()
            out = K.paged_append(p, zz, pages, table, pos, co)
            got.append([*out, co, pages.k, pages.v, pages.b, pages.g, pages.f, pages.weight, pages.token])
        backends.check_status(dev)
        assert all(torch.equal(s, t) for s, t in zip(*got))


def shifted(t, elements=4):
    """A dense copy of t that starts off a 16-byte boundary."""
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    out = flat[elements:elements + t.numel()].view(t.shape)
    assert out.data_ptr() % 16
    return out.copy_(t)


def test_dense_operands_off_a_16_byte_boundary(cuda_dev):
    from sisa_b200 import backends
    from sisa_b200.kernels import paged as K
    from tests.test_gpu_paged import make_pages, make_table, prompt

    dev, bf, L = cuda_dev, torch.bfloat16, 70
    pages, table, rows, x = attn_case([40], 2, 16, bf, dev, seed=5)
    ln, d = torch.tensor([40], dtype=torch.int32, device=dev), {n: t.to(dev) for n, t in x.items()}
    want = K.paged_attention(d["q"], d["c"], d["gq"], d["fq"], pages, table, ln, d["lam"])
    got = K.paged_attention(shifted(d["q"]), shifted(d["c"]), shifted(d["gq"], 1), shifted(d["fq"], 1), pages, table, ln,
                            shifted(d["lam"], 1))
    assert torch.equal(got, want)
    q, k, v, c, b, pl, lam, lse = prompt(2, 2, L, bf, dev, seed=2)
    w = K.attention_key_weights(q, k, c, b, pl, lam, lse)
    moved = [shifted(t) for t in (q, k, c, b)]
    assert torch.equal(K.attention_key_weights(*moved, pl, shifted(lam, 1), shifted(lse, 1)), w)
    table, P = make_table([50, 50], 32, 4, dev)
    src, filled = [k, v, b, pl[:, :, 0, :L].contiguous(), pl[:, :, 1, :L].contiguous(), w], []
    for move in (False, True):
        pages = make_pages(P, 2, 32, bf, dev, fill=0.5)
        s = [shifted(t, 1 if t.dtype == torch.float32 else 4) for t in src] if move else src
        K.paged_fill(pages, table, *s[:5], weight=s[5], keep=50, recent=9)
        filled.append(pages)
    gen = torch.Generator().manual_seed(1)
    proj, z = torch.randn(2, 1, 560, generator=gen).to(bf).to(dev), torch.randn(2, 1, 2, generator=gen).to(dev)
    carry, pos = torch.zeros(2, 2, 18, device=dev), torch.tensor([7, 49], dtype=torch.int32, device=dev)
    one = K.paged_append(proj, z, filled[0], table, pos, carry.clone())
    for n in (1, 2):                                       # one row by itself too
        two = K.paged_append(shifted(proj)[:n], shifted(z, 1)[:n], filled[1], table[:n], pos[:n], carry[:n].clone())
        assert all(torch.equal(s[:n], t) for s, t in zip(one, two)) and two[0].data_ptr() % 16 == 0
    backends.check_status(dev)
    for name in ("k", "v", "b", "g", "f", "weight", "token"):
        assert torch.equal(getattr(filled[0], name), getattr(filled[1], name)), name


def test_calls_from_a_thread_without_a_context(cuda_dev):
    """A host thread that has not touched CUDA gets the context of its current device, here the owner's, as from any
    runtime call; a thread that has it current keeps it."""
    import ctypes
    import threading

    from sisa_b200 import _lib, backends
    from sisa_b200.kernels import paged as K

    pages, table, rows, x = attn_case([128], 2, 16, torch.bfloat16, cuda_dev, seed=3)
    put(pages.token, table, 0, torch.arange(128).expand(2, 128).to(torch.int32).contiguous())
    pos = torch.tensor([128], dtype=torch.int32, device=cuda_dev)
    want = K.paged_evict(pages, table, pos, 128, 16)
    slots, lib, driver = torch.zeros_like(want), _lib.load(), ctypes.CDLL("libcuda.so.1")
    args = (pages.cbytes, table.data_ptr(), table.shape[1], table.shape[1], pos.data_ptr(), 1, 2, 128, 16, slots.data_ptr(),
            pages.status, None)
    torch.cuda.synchronize(cuda_dev)

    def current():
        ctx = ctypes.c_void_p()
        assert driver.cuCtxGetCurrent(ctypes.byref(ctx)) == 0
        return ctx.value

    seen = []
    thread = threading.Thread(target=lambda: seen.extend([current(), lib.sisa_paged_evict(*args), current(),
                                                          lib.sisa_paged_evict(*args), current()]))
    thread.start()
    thread.join()
    here = current()
    assert here is not None and seen == [None, 0, here, 0, here]
    torch.cuda.synchronize(cuda_dev)
    assert torch.equal(slots, want)
    assert lib.sisa_paged_evict(*args) == 0 and current() == here
    backends.check_status(cuda_dev)
