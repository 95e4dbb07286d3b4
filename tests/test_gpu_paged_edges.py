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
