"""The paged-cache operators (sisa_b200/kernels/paged.py) against plain fp64 implementations on the host.

Tolerances, derived from the arithmetic: outputs stored in 16 bits carry one rounding (half an ulp: at most
2^-8 of the value in bf16 with its 8 significant bits, 2^-11 in fp16 with 11) on an fp32 result, whose own
error comes from the exponents. A score in log2 units of magnitude up to 2^5 that is summed from about a
hundred fp32 products is off by at most about 100 x 2^-24 x 2^5 = 2e-4 in the worst case and by 1e-5 in
practice, so shares and log-sum-exps are held to 5e-5 (relative to a share, absolute for a log-sum-exp of that
magnitude); choices and copies are exact.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests.helpers import max_abs

pytestmark = pytest.mark.gpu

SHARE_REL = 5e-5
LOG2E = 1.0 / math.log(2.0)
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_pages(P, H, S, dtype, dev, layout="split", fill=float("nan")):
    """KeyPages whose slots all hold ``fill``; ``layout`` "joint" takes k, v and b out of one buffer per page."""
    from sisa_b200.kernels.paged import KeyPages

    if layout == "joint":
        buf = torch.full((P, H, 3 * S * 64), fill, dtype=dtype, device=dev)
        k, v = buf[..., :S * 64].view(P, H, S, 64), buf[..., S * 64:2 * S * 64].view(P, H, S, 64)
        b = buf[..., 2 * S * 64:2 * S * 64 + S * 32].view(P, H, S, 32)
        pl = torch.full((P, H, 3 * S), fill, dtype=torch.float32, device=dev)
        g, f, w = (pl[..., i * S:(i + 1) * S] for i in range(3))
        tk = torch.zeros((P, H, 3 * S), dtype=torch.int32, device=dev)[..., :S]
        return KeyPages(k, v, b, g, f, w, tk)
    pg = KeyPages.empty(P, H, S, dtype, dev)
    for t in (pg.k, pg.v, pg.b, pg.g, pg.f, pg.weight):
        t.fill_(fill)
    pg.token.zero_()
    return pg


def make_table(lengths, S, seed, dev):
    need = [max(1, -(-n // S)) for n in lengths]
    total = sum(need) + 2
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lengths), max(need)), total - 1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = perm[at:at + m]
        at += m
    return table.to(dev), total


def widen(table, columns=300):
    """The table with further entries that name no page (they may not be read)."""
    return torch.cat([table, torch.full((table.shape[0], columns), -7, dtype=torch.int32, device=table.device)], dim=1)


def put(plane, table, b, values):
    """values (H, n, ...) into the first n slots of sequence b."""
    S, n = plane.shape[2], values.shape[1]
    j = torch.arange(n)
    pg, sl = table[b].long().cpu()[j // S], j % S
    plane[pg.to(plane.device), :, sl.to(plane.device)] = values.transpose(0, 1).to(plane.device)


def get(plane, table, b, n):
    S = plane.shape[2]
    j = torch.arange(n)
    pg, sl = table[b].long().cpu()[j // S], j % S
    return plane.cpu()[pg, :, sl].transpose(0, 1)


def attn_case(lengths, H, S, dtype, dev, seed, layout="split", qscale=1.0, frate=0.02, forget=True):
    gen = torch.Generator().manual_seed(seed)
    table, P = make_table(lengths, S, seed, dev)
    pages = make_pages(P, H, S, dtype, dev, layout)
    rows = []
    for i, n in enumerate(lengths):
        m = max(n, 1)
        r = dict(k=torch.randn(H, m, 64, generator=gen).to(dtype), v=torch.randn(H, m, 64, generator=gen).to(dtype),
                 b=torch.randn(H, m, 32, generator=gen).to(dtype),
                 g=-torch.cumsum(torch.rand(H, m, generator=gen) * 0.05, 1),
                 f=-torch.cumsum(torch.rand(H, m, generator=gen) * frate, 1), w=torch.rand(H, m, generator=gen))
        perm = torch.randperm(m, generator=gen)                     # keys lie in any slot order
        r["gq"], r["fq"] = r["g"][:, -1].clone(), r["f"][:, -1].clone()
        for name in ("k", "v", "b", "g", "f", "w"):
            r[name] = r[name][:, perm]
        rows.append(r)
        if n:
            for plane, name in ((pages.k, "k"), (pages.v, "v"), (pages.b, "b"), (pages.g, "g"), (pages.f, "f"),
                                (pages.weight, "w")):
                put(plane, table, i, r[name])
    B = len(lengths)
    q = (torch.randn(B, H, 1, 64, generator=gen) * qscale).to(dtype)
    c = torch.randn(B, H, 1, 32, generator=gen).to(dtype)
    lam = torch.linspace(0.2, 1.5, H)
    x = dict(q=q, c=c, lam=lam, gq=torch.stack([r["gq"] for r in rows])[..., None],
             fq=torch.stack([r["fq"] for r in rows])[..., None] if forget else None)
    return pages, table, rows, x


def attn_truth(rows, lengths, x):
    out = []
    for i, n in enumerate(lengths):
        if n == 0:
            out.append(None)
            continue
        r = {k: t.double() for k, t in rows[i].items()}
        s = torch.einsum("hd,hnd->hn", x["q"][i, :, 0].double(), r["k"]) / 8
        dec = torch.exp(torch.clamp(x["gq"][i].double() - r["g"], max=0.0))
        s = s + x["lam"].double()[:, None] * dec * torch.einsum("hd,hnd->hn", x["c"][i, :, 0].double(), r["b"])
        if x["fq"] is not None:
            s = s + x["fq"][i].double() - r["f"]
        p = torch.softmax(s, dim=1)
        out.append((torch.einsum("hn,hnd->hd", p, r["v"]), torch.logsumexp(s, 1) * LOG2E, p))
    return out


def run_attn(pages, table, lengths, x, dev, **kw):
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_attention

    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out = paged_attention(x["q"].to(dev), x["c"].to(dev), x["gq"].to(dev), None if x["fq"] is None else x["fq"].to(dev),
                          pages, table, ln, x["lam"].to(dev), return_lse=True, **kw)
    torch.cuda.synchronize(dev)
    backends.check_status(dev)
    return out


def check_attn(pages, table, rows, lengths, x, dev, accumulate=True):
    before = pages.weight.clone()
    y, lse = run_attn(pages, table, lengths, x, dev, accumulate=accumulate)
    half = HALF_ULP[y.dtype]
    for i, want in enumerate(attn_truth(rows, lengths, x)):
        if want is None:
            assert bool((y[i] == 0).all()) and bool((lse[i] == -math.inf).all())
            continue
        yr, lr, p = want
        got = y[i, :, 0].double().cpu()
        assert bool(((got - yr).abs() <= half * yr.abs() * (1 + 1e-3) + SHARE_REL * rows[i]["v"].abs().max()).all())
        assert max_abs(lse[i], lr) <= 5e-5 * max(1.0, float(lr.abs().max()) / 32)
        n = lengths[i]
        w = get(pages.weight, table, i, n).double()
        if accumulate:
            want_w = rows[i]["w"].double()[:, :n] + p
            assert bool(((w - want_w).abs() <= SHARE_REL * p + 2.0 ** -23 * want_w + 1e-30).all())
        else:
            assert torch.equal(w, rows[i]["w"].double()[:, :n])
    # nothing else was written
    used = torch.zeros_like(before, dtype=torch.bool)
    for i, n in enumerate(lengths):
        if n:
            put(used, table, i, torch.ones(pages.n_head, n, dtype=torch.bool))
    assert torch.equal(before[~used].isnan(), pages.weight[~used].isnan())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_lengths_around_pages_and_tiles(cuda_dev, S, dtype, wide):
    """``wide``: the same sequences under a table for many more keys (its further entries, which no length
    reaches, name no page): the kernels that split the keys serve them instead of the one-CTA-per-row kernel."""
    lengths = [1, 0, 2, S - 1, S, S + 1, 31, 32, 33, 63, 64, 65, 2 * S + 7, 300]
    pages, table, rows, x = attn_case(lengths, 3, S, dtype, cuda_dev, seed=S)
    check_attn(pages, widen(table) if wide else table, rows, lengths, x, cuda_dev)


@pytest.mark.parametrize("B,H,n,S", [(1, 1, 1, 64), (1, 8, 5003, 64), (1, 1, 20011, 16), (7, 5, 777, 32), (40, 2, 129, 128),
                                     (3, 4, 512, 64), (3, 4, 513, 64), (33, 3, 1500, 256)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention_shapes(cuda_dev, B, H, n, S, accumulate):
    gen = torch.Generator().manual_seed(n)
    lengths = [n] + torch.randint(0, n + 1, (B - 1,), generator=gen).tolist()
    pages, table, rows, x = attn_case(lengths, H, S, torch.bfloat16, cuda_dev, seed=n + B, layout="joint")
    check_attn(pages, table, rows, lengths, x, cuda_dev, accumulate)


def test_attention_large_scores_strong_forgetting_and_no_forget_gate(cuda_dev):
    """Scores of a few hundred (the maximum moves often, most shares underflow) and without F."""
    lengths = [513, 40, 1, 900]
    for kw in (dict(qscale=30.0, frate=3.0), dict(forget=False)):
        pages, table, rows, x = attn_case(lengths, 4, 64, torch.bfloat16, cuda_dev, seed=9, **kw)
        truth = attn_truth(rows, lengths, x)
        for i, (yr, lr, p), t in ((i, r, t) for t in (table, widen(table)) for i, r in enumerate(truth)):
            y, lse = run_attn(pages, t, lengths, x, cuda_dev)
            # scores of magnitude 2^10 are off by up to 2^-24 x 2^10 x a few in their fp32 sums
            assert max_abs(lse[i], lr) <= 2e-3
            assert bool(((y[i, :, 0].double().cpu() - yr).abs() <= HALF_ULP[y.dtype] * yr.abs() + 8e-3).all())


def test_attention_all_idle_and_minus_infinity_keys(cuda_dev):
    pages, table, rows, x = attn_case([0, 0], 2, 32, torch.bfloat16, cuda_dev, seed=1)
    for t in (table, widen(table)):
        y, lse = run_attn(pages, t, [0, 0], x, cuda_dev, accumulate=True)
        assert bool((y == 0).all()) and bool((lse == -math.inf).all())
    # a key whose score is -inf has no share, wherever it lies; whole tiles of them too
    lengths = [200]
    pages, table, rows, x = attn_case(lengths, 2, 32, torch.bfloat16, cuda_dev, seed=2)
    rows[0]["f"][:, :70] = math.inf
    rows[0]["f"][:, 133] = math.inf
    put(pages.f, table, 0, rows[0]["f"])
    before = pages.weight.clone()
    check_attn(pages, table, rows, lengths, x, cuda_dev)
    pages.weight.copy_(before)
    check_attn(pages, widen(table), rows, lengths, x, cuda_dev)


def test_attention_nan_key_reaches_output_and_status(cuda_dev):
    lengths = [150, 90]
    pages, table, rows, x = attn_case(lengths, 2, 64, torch.bfloat16, cuda_dev, seed=3)
    rows[0]["g"][1, 77] = math.nan
    put(pages.g, table, 0, rows[0]["g"])
    for t in (table, widen(table)):
        with pytest.raises(FloatingPointError):
            run_attn(pages, t, lengths, x, cuda_dev)
    from sisa_b200 import backends

    mode = backends.get_check_mode()
    backends.set_check_mode("off")
    try:
        from sisa_b200.kernels.paged import paged_attention

        ln = torch.tensor(lengths, dtype=torch.int32, device=cuda_dev)
        y = paged_attention(*(x[n].to(cuda_dev) for n in ("q", "c", "gq", "fq")), pages, table, ln, x["lam"].to(cuda_dev))
    finally:
        backends.set_check_mode(mode)
    assert bool(y[0, 1].isnan().all()) and bool(y[0, 0].isfinite().all()) and bool(y[1].isfinite().all())
    backends.status_word(cuda_dev).zero_()


def test_attention_is_deterministic_on_any_stream_and_layout(cuda_dev):
    lengths = [1500, 3, 0, 640]
    pages, table, rows, x = attn_case(lengths, 4, 64, torch.bfloat16, cuda_dev, seed=4)
    w_out = torch.zeros_like(pages.weight)
    y0, l0 = run_attn(pages, table, lengths, x, cuda_dev, accumulate=True, weight_out=w_out)
    stream = torch.cuda.Stream(cuda_dev)
    xs = dict(x)
    # q and c as strided views of wider rows
    wide = torch.randn(4, 4, 1, 160).to(torch.bfloat16)
    wide[..., 8:72], wide[..., 96:128] = x["q"], x["c"]
    wide = wide.to(cuda_dev)
    xs["q"], xs["c"] = wide[..., 8:72], wide[..., 96:128]
    w2 = torch.zeros_like(w_out)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        y1, l1 = run_attn(pages, table, lengths, xs, cuda_dev, accumulate=True, weight_out=w2)
    assert torch.equal(y0, y1) and torch.equal(l0, l1) and torch.equal(w_out, w2)


def test_attention_pages_past_32_bit_offsets(cuda_dev):
    """Two pages more than 2^31 elements apart (k and v share the rows)."""
    from sisa_b200.kernels.paged import KeyPages

    H, S, far = 2, 64, (1 << 31) + 4096
    buf = torch.empty(far + H * S * 64, dtype=torch.bfloat16, device=cuda_dev)
    k = buf.as_strided((2, H, S, 64), (far, S * 64, 64, 1))
    gen = torch.Generator().manual_seed(5)
    rows = dict(k=torch.randn(H, 128, 64, generator=gen).to(torch.bfloat16), b=torch.randn(H, 128, 32, generator=gen).to(torch.bfloat16),
                g=-torch.rand(H, 128, generator=gen), f=-torch.rand(H, 128, generator=gen))
    rows["v"], rows["w"] = rows["k"], torch.zeros(H, 128)
    pages = KeyPages(k, k, torch.empty((2, H, S, 32), dtype=torch.bfloat16, device=cuda_dev),
                     *(torch.empty((2, H, S), device=cuda_dev) for _ in range(2)),
                     weight=torch.zeros((2, H, S), device=cuda_dev))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=cuda_dev)
    for plane, name in ((pages.k, "k"), (pages.b, "b"), (pages.g, "g"), (pages.f, "f")):
        put(plane, table, 0, rows[name])
    x = dict(q=torch.randn(1, H, 1, 64, generator=gen).to(torch.bfloat16), c=torch.randn(1, H, 1, 32, generator=gen).to(torch.bfloat16),
             lam=torch.ones(H), gq=-torch.ones(1, H, 1), fq=-torch.ones(1, H, 1))
    check_attn(pages, table, [rows], [128], x, cuda_dev)


def test_attention_bad_table_and_length_set_the_status(cuda_dev):
    lengths = [128, 50]
    pages, table, rows, x = attn_case(lengths, 2, 32, torch.bfloat16, cuda_dev, seed=6)
    for page, wide in ((pages.n_pages, False), (-1, False), (pages.n_pages, True), (-1, True)):
        bad = widen(table) if wide else table.clone()
        bad[0, 1] = page
        for acc in (True, False):
            with pytest.raises(ValueError):
                run_attn(pages, bad, lengths, x, cuda_dev, accumulate=acc)
    with pytest.raises(ValueError):
        run_attn(pages, table, [129, 50], x, cuda_dev)


# ------------------------------------------------------------------------------------------------ evict
def evict_truth(w, tok, pos, budget, recent):
    out = []
    for b, p in enumerate(pos):
        if p < budget:
            out.append([-1] * w.shape[1])
            continue
        row = []
        for h in range(w.shape[1]):
            cand = [j for j in range(budget) if int(tok[b, h, j]) < p - recent]
            key = lambda j: (0, 0.0, j) if math.isnan(float(w[b, h, j])) else (1, float(w[b, h, j]), j)  # noqa: E731
            row.append(min(cand, key=key))
        out.append(row)
    return torch.tensor(out, dtype=torch.int32)


@pytest.mark.parametrize("budget,recent,S", [(1, 0, 16), (2, 1, 16), (33, 32, 16), (100, 0, 64), (500, 64, 32), (3000, 100, 128)])
def test_evict_matches_the_definition(cuda_dev, budget, recent, S):
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_evict

    B, H = 6, 3
    gen = torch.Generator().manual_seed(budget)
    table, P = make_table([budget] * B, S, budget, cuda_dev)
    pages = make_pages(P, H, S, torch.bfloat16, cuda_dev)
    pos = [budget, budget + 17, -1, budget - 1, 4 * budget, budget + 1]
    w = torch.rand(B, H, budget, generator=gen)
    w[1] = w[1].round()                                        # ties
    w[4, 0] = 0.0
    w[4, 1, ::2], w[4, 1, 1::2] = 0.0, -0.0                    # both zeros weigh the same
    w[5, 0, budget // 2] = math.nan
    w[5, 1] = -w[5, 1]
    w[5, 2] = math.inf
    tok = torch.stack([torch.stack([torch.randperm(budget, generator=gen) for _ in range(H)]) for _ in range(B)])
    for b, p in enumerate(pos):                                # the newest tokens are always held
        t = tok[b]
        tok[b] = torch.where(t < recent, p - 1 - t, t - recent)
        put(pages.weight, table, b, w[b])
        put(pages.token, table, b, tok[b].to(torch.int32))
    got = paged_evict(pages, table, torch.tensor(pos, dtype=torch.int32, device=cuda_dev), budget, recent)
    backends.check_status(cuda_dev)
    assert torch.equal(got.cpu(), evict_truth(w, tok, pos, budget, recent))


# ------------------------------------------------------------------------------------------------ append
def append_truth(proj, z, H, carry):
    """The recurrences in fp64 (oracle.prep over one token, from the carried state)."""
    from oracle import sisa_oracle as O

    pr = O.prep(proj.double(), None if z is None else z.double(), H)
    off = O.fused_layout(H)
    phi = carry[..., :16].double() + proj[:, 0, off["TH"]:off["TH"] + 16 * H].double().view(-1, H, 16)
    g = carry[..., 16].double() + pr["g"][:, :, 0]
    f = carry[..., 17].double() + (pr["F"][:, :, 0] if z is not None else 0.0)
    cols = lambda n: proj[:, 0, off[n]:off[n] + 32 * H].double().view(-1, H, 1, 32)  # noqa: E731
    rot = lambda t: O.rotate_pairs(t, phi.unsqueeze(2))  # noqa: E731
    return dict(q=pr["q"], k=pr["k"], v=pr["v"], c=rot(cols("C")), b=rot(cols("B")), g=g, f=f, phi=phi)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,S,gate", [(1, 8, 16, True), (5, 3, 64, True), (3, 2, 128, False), (9, 16, 32, True)])
def test_append_matches_fp64(cuda_dev, B, H, S, gate, dtype):
    from oracle import sisa_oracle as O
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_append

    proj, z, _ = O.make_proj_inputs(B, 1, H, seed=B * H)
    proj, z = proj.to(dtype), z if gate else None
    gen = torch.Generator().manual_seed(B)
    carry = torch.randn(B, H, 18, generator=gen) * 10
    cap = 2 * S
    table, P = make_table([cap] * B, S, B, cuda_dev)
    pages = make_pages(P, H, S, dtype, cuda_dev, fill=0.5)
    pos = [(7 * i + 3) % cap for i in range(B)]
    if B > 2:
        pos[1], pos[2] = -1, cap + 40                           # an idle row; one past the pages, into a reused slot
    slots = torch.full((B, H), -1, dtype=torch.int32)
    if B > 2:
        slots[2] = torch.randint(0, cap, (H,), generator=gen).to(torch.int32)
    want = append_truth(proj, z, H, carry)
    carry_d, lengths = carry.to(cuda_dev), torch.zeros(B, dtype=torch.int32, device=cuda_dev)
    before = {n: getattr(pages, n).clone() for n in ("k", "v", "b", "g", "f", "weight", "token")}
    q, c, g, f = paged_append(proj.to(cuda_dev), None if z is None else z.to(cuda_dev), pages, table,
                              torch.tensor(pos, dtype=torch.int32, device=cuda_dev), carry_d, slots=slots.to(cuda_dev),
                              budget=cap, lengths=lengths)
    backends.check_status(cuda_dev)
    half = HALF_ULP[dtype]
    assert lengths.tolist() == [min(p + 1, cap) for p in pos]
    assert torch.equal(q.cpu(), want["q"].to(dtype)) and (f is None) == (z is None)
    for i in range(B):
        if pos[i] < 0:
            assert bool((c[i] == 0).all()) and bool((g[i] == 0).all()) and torch.equal(carry_d[i].cpu(), carry[i])
            continue
        cr, br = want["c"][i], want["b"][i]
        # cos and sin of a phase of magnitude up to 2^6 held in fp32: its rounding moves the rotation by 2^-19
        assert bool(((c[i].double().cpu() - cr).abs() <= half * cr.abs() + 2e-5 * 8).all())
        assert max_abs(carry_d[i, :, :16], want["phi"][i]) <= 1e-5
        assert max_abs(carry_d[i, :, 16], want["g"][i]) <= 1e-5 and max_abs(carry_d[i, :, 17], want["f"][i]) <= 1e-5
        assert torch.equal(g[i, :, 0], carry_d[i, :, 16]) and (f is None or torch.equal(f[i, :, 0], carry_d[i, :, 17]))
        for h in range(H):
            s = int(slots[i, h]) if int(slots[i, h]) >= 0 else pos[i]
            page, at = int(table[i, s // S]), s % S
            assert torch.equal(pages.k[page, h, at].cpu(), want["k"][i, h, 0].to(dtype))
            assert torch.equal(pages.v[page, h, at].cpu(), want["v"][i, h, 0].to(dtype))
            assert bool(((pages.b[page, h, at].double().cpu() - br[h, 0]).abs() <= half * br[h, 0].abs() + 2e-5 * 8).all())
            assert float(pages.g[page, h, at]) == float(g[i, h, 0]) and float(pages.weight[page, h, at]) == 0.0
            assert float(pages.f[page, h, at]) == (float(f[i, h, 0]) if gate else 0.0)
            assert int(pages.token[page, h, at]) == pos[i]
            for n, t in before.items():                         # for the check that nothing else changed
                t[page, h, at] = getattr(pages, n)[page, h, at]
    for n, t in before.items():
        assert torch.equal(t, getattr(pages, n)), n


def test_append_outside_the_pages_sets_the_status_and_writes_nothing(cuda_dev):
    from oracle import sisa_oracle as O
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_append

    proj, z, _ = O.make_proj_inputs(1, 1, 2, seed=1)
    table, P = make_table([32], 16, 1, cuda_dev)
    pages = make_pages(P, 2, 16, torch.bfloat16, cuda_dev, fill=0.5)
    before = pages.k.clone()
    carry = torch.ones(1, 2, 18, device=cuda_dev)
    args = (proj.to(torch.bfloat16).to(cuda_dev), z.to(cuda_dev), pages, table)
    for pos, slot, budget in ((32, -1, None), (20, -1, 20), (0, 32, None), (100, 25, 25)):
        paged_append(*args, torch.tensor([pos], dtype=torch.int32, device=cuda_dev), carry, budget=budget,
                     slots=torch.full((1, 2), slot, dtype=torch.int32, device=cuda_dev))
        with pytest.raises(ValueError):
            backends.check_status(cuda_dev)
        assert torch.equal(pages.k, before) and bool((carry == 1).all())


# ------------------------------------------------------------------------------------------------ key weights
def prompt(B, H, L, dtype, dev, seed, a_mean=-3.0, z_mean=2.0):
    """A prompt's operands as the layer hands them over (k, v views of the projection), with the oracle's."""
    from oracle import sisa_oracle as O
    from sisa_b200 import ops

    proj, z, lam = O.make_proj_inputs(B, L, H, seed=seed, a_mean=a_mean, z_mean=z_mean)
    proj = proj.to(dtype).to(dev)
    lam = (lam * torch.linspace(0.5, 2.0, H)).to(dev)
    c, b, pos, _ = ops.prep_fwd(proj, z.to(dev), H)
    q, k, v = (ops.heads(proj, 64 * H * i, H, 64) for i in range(3))
    _, lse, _ = ops.attn_fwd(q, k, v, c, b, pos, lam, False)
    return q, k, v, c, b, pos, lam, lse


def weights_truth(q, k, c, b, pos, lam, lse, first):
    q, k, c, b, lse = (t.double().cpu() for t in (q, k, c, b, lse))
    L = q.shape[2]
    g, f = pos[:, :, 0, :L].double().cpu(), pos[:, :, 1, :L].double().cpu()
    s = q @ k.transpose(2, 3) / 8
    s = s + lam.double().cpu().view(1, -1, 1, 1) * torch.exp((g[..., :, None] - g[..., None, :]).clamp_max(0)) * (c @ b.transpose(2, 3))
    s = s + f[..., :, None] - f[..., None, :]
    i = torch.arange(L)
    p = torch.exp(s - lse[..., None] / LOG2E)
    return p.masked_fill(~((i[None] <= i[:, None]) & (i[:, None] >= first)), 0.0).sum(2)


@pytest.mark.parametrize("L", [1, 2, 17, 63, 64, 65, 127, 128, 129, 200, 257, 513, 1000])
def test_key_weights_match_fp64(cuda_dev, L):
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import attention_key_weights

    B, H = 2, 3
    q, k, v, c, b, pos, lam, lse = prompt(B, H, L, torch.bfloat16, cuda_dev, seed=L)
    for first in sorted({0, L // 3, max(0, L - 64), L - 1}):
        w = attention_key_weights(q, k, c, b, pos, lam, lse, first_query=first)
        backends.check_status(cuda_dev)
        want = weights_truth(q, k, c, b, pos, lam, lse, first)
        assert bool(((w.double().cpu() - want).abs() <= SHARE_REL * want + 1e-30).all()), (L, first)
        assert abs(float(w.double().sum()) / (B * H * (L - first)) - 1) <= 1e-4    # every query hands out one


@pytest.mark.parametrize("a_mean,z_mean", [(-5.0, 4.0), (2.0, -2.0), (-8.0, 9.0)])
def test_key_weights_decay_rates_and_fp16(cuda_dev, a_mean, z_mean):
    """Slow to fast decay and forgetting (most shares underflow in the middle case)."""
    from sisa_b200.kernels.paged import attention_key_weights

    q, k, v, c, b, pos, lam, lse = prompt(1, 2, 700, torch.float16, cuda_dev, seed=3, a_mean=a_mean, z_mean=z_mean)
    w = attention_key_weights(q, k, c, b, pos, lam, lse)
    want = weights_truth(q, k, c, b, pos, lam, lse, 0)
    # F falls by up to 2 per token: differences of F are exact to 2^-24 x 2^11 = 1e-4 of a score
    tol = SHARE_REL if z_mean > 0 else 3e-4
    assert bool(((w.double().cpu() - want).abs() <= tol * want + 1e-30).all())
    again = attention_key_weights(q.contiguous(), k.contiguous(), c, b, pos, lam, lse)
    assert torch.equal(w, again)


# ------------------------------------------------------------------------------------------------ fill
def fill_truth(w, keep, recent):
    L = w.shape[-1]
    out = torch.empty(w.shape[:2] + (keep,), dtype=torch.long)
    for b in range(w.shape[0]):
        for h in range(w.shape[1]):
            val = lambda j: (1, 0.0, j) if math.isnan(float(w[b, h, j])) else (0, -float(w[b, h, j]), j)  # noqa: E731
            top = sorted(range(L - recent), key=val)[:keep - recent]
            out[b, h] = torch.tensor(sorted(top) + list(range(L - recent, L)))
    return out


@pytest.mark.parametrize("L,keep,recent,S", [(1, 1, 0, 16), (1, 1, 1, 64), (5, 2, 2, 16), (5, 3, 0, 16), (200, 200, 10, 32),
                                             (513, 100, 37, 64), (700, 699, 1, 128), (3000, 1024, 100, 64)])
def test_fill_keeps_the_newest_and_the_heaviest(cuda_dev, L, keep, recent, S):
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_fill

    B, H = 2, 3
    q, k, v, c, b, pos, lam, lse = prompt(B, H, L, torch.bfloat16, cuda_dev, seed=L)
    w = torch.rand(B, H, L, generator=torch.Generator().manual_seed(L))
    w[0, 1] = (w[0, 1] * 4).round()                            # ties
    w[0, 2, ::2], w[0, 2, 1::2] = 0.0, -0.0
    w[1, 0, L // 2] = math.nan
    w[1, 1] = -w[1, 1]
    table, P = make_table([keep] * B, S, L, cuda_dev)
    pages = make_pages(P, H, S, torch.bfloat16, cuda_dev, fill=0.25)
    g, f = pos[:, :, 0, :L], pos[:, :, 1, :L]
    n = paged_fill(pages, table, k, v, b, g, f, weight=w.to(cuda_dev), keep=keep, recent=recent)
    backends.check_status(cuda_dev)
    assert n == keep
    idx = fill_truth(w, keep, recent)
    for i in range(B):
        at = idx[i]
        assert torch.equal(get(pages.token, table, i, keep).long(), at)
        for plane, src in ((pages.k, k), (pages.v, v), (pages.b, b)):
            assert torch.equal(get(plane, table, i, keep), src[i].cpu().gather(1, at.unsqueeze(-1).expand(-1, -1, src.shape[-1])))
        for plane, src in ((pages.g, g), (pages.f, f), (pages.weight, w)):
            assert torch.equal(get(plane, table, i, keep).nan_to_num(), src[i].cpu().gather(1, at).nan_to_num())
    used = torch.zeros_like(pages.weight, dtype=torch.bool)
    for i in range(B):
        put(used, table, i, torch.ones(H, keep, dtype=torch.bool))
    assert bool((pages.k[~used] == 0.25).all()) and bool((pages.g[~used] == 0.25).all())


def test_fill_whole_prompt_without_weights_or_planes(cuda_dev):
    from sisa_b200.kernels.paged import KeyPages, paged_fill

    q, k, v, c, b, pos, lam, lse = prompt(1, 2, 90, torch.float16, cuda_dev, seed=5)
    table, P = make_table([90], 32, 3, cuda_dev)
    pages = KeyPages.empty(P, 2, 32, torch.float16, cuda_dev, evict=False)
    assert paged_fill(pages, table, k, v, b, pos[:, :, 0, :90], pos[:, :, 1, :90]) == 90
    assert torch.equal(get(pages.v, table, 0, 90), v[0].cpu()) and torch.equal(get(pages.f, table, 0, 90), pos[0, :, 1, :90].cpu())


@pytest.mark.parametrize("levels", [None, 3])
@pytest.mark.parametrize("L,keep,recent", [(33000, 5000, 100), (70000, 9000, 0), (41000, 40999, 7)])
def test_fill_long_prompts(cuda_dev, L, keep, recent, levels):
    """Prompts past one chunk of the compaction and past the shared memory of the select; with ``levels`` the
    weights take three values only, so that no digit tells the candidates apart."""
    import numpy as np
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import paged_fill

    gen = torch.Generator().manual_seed(L + (levels or 0))
    w = torch.rand(1, 2, L, generator=gen)
    if levels:
        w = (w * levels).floor() / levels
    src = [torch.randn(1, 2, L, d, generator=gen).to(torch.bfloat16).to(cuda_dev) for d in (64, 64, 32)]
    g, f = (torch.randn(1, 2, L, generator=gen).to(cuda_dev) for _ in range(2))
    table, P = make_table([keep], 64, 1, cuda_dev)
    pages = make_pages(P, 2, 64, torch.bfloat16, cuda_dev, fill=0.25)
    paged_fill(pages, table, *src, g, f, weight=w.to(cuda_dev), keep=keep, recent=recent)
    backends.check_status(cuda_dev)
    old = L - recent
    idx = []
    for h in range(2):
        top = np.lexsort((np.arange(old), -w[0, h, :old].numpy()))[:keep - recent]
        idx.append(np.concatenate([np.sort(top), np.arange(old, L)]))
    idx = torch.from_numpy(np.stack(idx))
    assert torch.equal(get(pages.token, table, 0, keep).long(), idx)
    for plane, x in ((pages.k, src[0]), (pages.v, src[1]), (pages.b, src[2])):
        assert torch.equal(get(plane, table, 0, keep), x[0].cpu().gather(1, idx.unsqueeze(-1).expand(-1, -1, x.shape[-1])))
    for plane, x in ((pages.g, g), (pages.f, f), (pages.weight, w)):
        assert torch.equal(get(plane, table, 0, keep), x[0].cpu().gather(1, idx))


def test_attention_of_many_tiles(cuda_dev):
    """More tiles than one wave of warps takes (units spread over many CTAs, runs that cross units), against fp64
    on the GPU, with and without weights."""
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import KeyPages, paged_attention

    dev, H, S, lengths = cuda_dev, 16, 128, [90001, 40, 0, 12345]
    gen = torch.Generator(device=dev).manual_seed(1)
    table, P = make_table(lengths, S, 2, dev)
    rnd = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
    pages = KeyPages(rnd(P, H, S, 64).half(), rnd(P, H, S, 64).half(), rnd(P, H, S, 32).half(), -rnd(P, H, S).abs(),
                     -rnd(P, H, S).abs(), rnd(P, H, S).abs())
    q, c = rnd(4, H, 1, 64).half(), rnd(4, H, 1, 32).half()
    gq, fq, lam = -2 * torch.ones(4, H, 1, device=dev), -3 * torch.ones(4, H, 1, device=dev), torch.linspace(0.2, 1.0, H, device=dev)
    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    before = pages.weight.clone()
    y0, l0 = paged_attention(q, c, gq, fq, pages, table, ln, lam, return_lse=True)
    y, lse = paged_attention(q, c, gq, fq, pages, table, ln, lam, accumulate=True, return_lse=True)
    backends.check_status(dev)
    assert torch.equal(y, y0) and torch.equal(lse, l0)
    for b, n in enumerate(lengths):
        if n == 0:
            assert bool((y[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        j = torch.arange(n, device=dev)
        pg, sl = table[b].long()[j // S], j % S
        for h in range(H):
            s = pages.k[pg, h, sl].double() @ q[b, h, 0].double() / 8
            dec = torch.exp((gq[b, h].double() - pages.g[pg, h, sl].double()).clamp_max(0))
            s = s + lam[h].double() * dec * (pages.b[pg, h, sl].double() @ c[b, h, 0].double()) + fq[b, h].double() - pages.f[pg, h, sl].double()
            p = torch.softmax(s, 0)
            want, v = p @ pages.v[pg, h, sl].double(), pages.v[pg, h, sl]
            assert bool(((y[b, h, 0].double() - want).abs() <= 2.0 ** -11 * want.abs() + SHARE_REL * v.abs().max() + 2.0 ** -25).all())
            assert abs(float(lse[b, h]) - float(torch.logsumexp(s, 0)) * LOG2E) <= 5e-5
            ww = before[pg, h, sl].double() + p
            assert bool(((pages.weight[pg, h, sl].double() - ww).abs() <= SHARE_REL * p + 2.0 ** -23 * ww + 1e-30).all())


@pytest.mark.parametrize("L,first", [(5000, 0), (9001, 8000)])
def test_key_weights_long_prompts(cuda_dev, L, first):
    """Sums over thousands of queries, against fp64 on the GPU."""
    from sisa_b200 import backends
    from sisa_b200.kernels.paged import attention_key_weights

    q, k, v, c, b, pos, lam, lse = prompt(1, 2, L, torch.bfloat16, cuda_dev, seed=L)
    w = attention_key_weights(q, k, c, b, pos, lam, lse, first_query=first)
    backends.check_status(cuda_dev)
    want = torch.zeros(2, L, dtype=torch.float64, device=cuda_dev)
    g, f = pos[0, :, 0, :L].double(), pos[0, :, 1, :L].double()
    j = torch.arange(L, device=cuda_dev)
    for h in range(2):
        for i0 in range(first, L, 1000):
            i = torch.arange(i0, min(L, i0 + 1000), device=cuda_dev)
            s = q[0, h, i].double() @ k[0, h].double().t() / 8
            s = s + lam[h].double() * torch.exp((g[h, i, None] - g[h, None]).clamp_max(0)) * (c[0, h, i].double() @ b[0, h].double().t())
            s = s + f[h, i, None] - f[h, None] - lse[0, h, i, None].double() / LOG2E
            want[h] += torch.exp(s).masked_fill(j[None] > i[:, None], 0.0).sum(0)
    assert bool(((w[0].double() - want).abs() <= SHARE_REL * want + 1e-30).all())


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(cuda_dev):
    from sisa_b200.kernels import paged as K

    dev, bf = cuda_dev, torch.bfloat16
    pages, table, rows, x = attn_case([40], 2, 16, bf, dev, seed=1)
    d = {n: t.to(dev) for n, t in x.items()}
    ln = torch.tensor([40], dtype=torch.int32, device=dev)

    def attn(**kw):
        a = dict(q=d["q"], c=d["c"], g=d["gq"], fgate=d["fq"], pages=pages, block_table=table, lengths=ln, lam=d["lam"])
        extra = {n: kw.pop(n) for n in ("accumulate", "weight_out") if n in kw}
        a.update(kw)
        return K.paged_attention(*a.values(), **extra)

    attn()
    bare = K.KeyPages(pages.k, pages.v, pages.b, pages.g)
    for kw, err in ((dict(q=d["q"].half()), TypeError), (dict(q=d["q"][:, :1]), ValueError), (dict(q=d["q"].expand(1, 2, 2, 64)), ValueError),
                    (dict(c=d["c"][..., :16]), ValueError), (dict(lengths=ln.long()), ValueError), (dict(lengths=ln.cpu()), ValueError),
                    (dict(block_table=table.long()), ValueError), (dict(block_table=table[:, :0]), ValueError),
                    (dict(lam=d["lam"][:1]), ValueError), (dict(pages=bare), ValueError), (dict(weight_out=pages.weight), ValueError),
                    (dict(pages=bare, fgate=None, accumulate=True), ValueError),
                    (dict(accumulate=True, weight_out=pages.weight[:1]), ValueError)):
        with pytest.raises(err):
            attn(**kw)
    pos = torch.tensor([50], dtype=torch.int32, device=dev)
    for budget, recent in ((0, 0), (49, 0), (40, 40), (40, -1)):
        with pytest.raises(ValueError):
            K.paged_evict(pages, table, pos, budget, recent)
    with pytest.raises(ValueError):
        K.paged_evict(bare, table, pos, 40, 4)
    proj = torch.zeros(1, 1, 560, dtype=bf, device=dev)
    z, carry = torch.zeros(1, 1, 2, device=dev), torch.zeros(1, 2, 18, device=dev)
    for a, err in (((proj.half(), z, pages, table, pos, carry), TypeError), ((proj[..., :500], z, pages, table, pos, carry), ValueError),
                   ((proj, z, bare, table, pos, carry), ValueError), ((proj, z, pages, table, pos, carry.double()), ValueError),
                   ((proj, z, pages, table, pos.long(), carry), ValueError), ((proj, z, pages, table, pos, carry[..., :17]), ValueError)):
        with pytest.raises(err):
            K.paged_append(*a)
    with pytest.raises(ValueError):
        K.paged_append(proj, z, pages, table, pos, carry, budget=1000)
    q, k, v, c, b, pl, lam, lse = prompt(1, 2, 40, bf, dev, seed=2)
    for first in (-1, 40):
        with pytest.raises(ValueError):
            K.attention_key_weights(q, k, c, b, pl, lam, lse, first_query=first)
    for a, err in (((q.float(), k, c, b, pl, lam, lse), TypeError), ((q, k[:, :, :30], c, b, pl, lam, lse), ValueError),
                   ((q, k, c, b, pl[..., :20], lam, lse), ValueError), ((q, k, c, b, pl, lam, lse.half()), ValueError),
                   ((q, k, c, b, pl, lam[:1], lse), ValueError), ((q.cpu(), k, c, b, pl, lam, lse), ValueError)):
        with pytest.raises(err):
            K.attention_key_weights(*a)
    g, f, w = pl[:, :, 0, :40], pl[:, :, 1, :40], torch.rand(1, 2, 40, device=dev)
    for kw in (dict(keep=10), dict(keep=0), dict(keep=41), dict(keep=10, recent=11, weight=w), dict(keep=10, recent=-1, weight=w),
               dict(weight=w[..., :20])):
        with pytest.raises(ValueError):
            K.paged_fill(pages, table, k, v, b, g, f, **kw)
    with pytest.raises(ValueError):
        K.paged_fill(pages, table[:, :2], k, v, b, g, f)                 # 32 slots for 40 keys
    with pytest.raises(TypeError):
        K.paged_fill(pages, table, k.half(), v, b, g, f)
    with pytest.raises(ValueError):
        K.KeyPages(pages.k[:, :, :10], pages.v, pages.b, pages.g)        # no page size of ten
    with pytest.raises(ValueError):
        K.KeyPages(pages.k.transpose(2, 3).contiguous().transpose(2, 3), pages.v, pages.b, pages.g)
    with pytest.raises(TypeError):
        K.KeyPages(pages.k, pages.v.half(), pages.b, pages.g)
    with pytest.raises(TypeError):
        K.KeyPages(pages.k, pages.v, pages.b, pages.g, token=pages.g)
