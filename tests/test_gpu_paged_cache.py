"""The paged, bounded cache on the model (sisa_b200/paged_cache.py): against the dense cache where nothing is
dropped, against an fp64 simulation of the eviction, and its rows, pages and graph."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import sisa_oracle as O
from tests.helpers import max_abs

pytestmark = pytest.mark.gpu

LOGIT_TOL = 2e-2         # the tolerance of the fused decode step against the unfused one (test_gpu_decode.py)


def tiny(dev, dtype=torch.bfloat16):
    import sisa_b200 as sisa

    torch.manual_seed(0)
    cfg = sisa.SISAConfig(vocab_size=97, d_model=128, n_layer=2, n_head=2, d_ff=96, attn_impl="cuda", zero_init_c=False)
    model = sisa.SISAForCausalLM(cfg)
    with torch.no_grad():
        for layer in model.layers:
            layer.attn.theta_proj.weight.mul_(20)
            layer.attn.alpha_proj.bias.fill_(-2.0)
            layer.attn.forget_proj.bias.fill_(1.0)
    return model.to(dev).to(dtype)


def ids_of(shape, seed, dev):
    return torch.randint(0, 97, shape, generator=torch.Generator().manual_seed(seed)).to(dev)


@torch.no_grad()
def dense_logits(model, ids, prompt):
    from sisa_b200.generation import SISACache

    cache = SISACache()
    out = [model(ids[:, :prompt], cache=cache, logits_to_keep=1).logits[:, -1].float()]
    for t in range(prompt, ids.shape[1]):
        out.append(model(ids[:, t:t + 1], cache=cache, logits_to_keep=1).logits[:, -1].float())
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prompt,page_size,kind", [(70, 16, "max"), (1, 32, "max"), (129, 64, "budget"), (2, 16, "budget")])
@torch.no_grad()
def test_paged_steps_match_the_dense_cache(cuda_dev, prompt, page_size, kind, dtype):
    """Nothing is dropped (no budget, or one that is not reached): the same logits at every step."""
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev, dtype)
    ids = ids_of((3, prompt + 20), 1, cuda_dev)
    kw = dict(max_tokens=prompt + 20) if kind == "max" else dict(budget=prompt + 20, recent=5)
    cache = PagedCache(model.config, 3, page_size=page_size, dtype=dtype, device=cuda_dev, **kw)
    got = [model(ids[:, :prompt], cache=cache, logits_to_keep=1).logits[:, -1].float()]
    for t in range(prompt, ids.shape[1]):
        got.append(model(ids[:, t:t + 1], cache=cache, logits_to_keep=1).logits[:, -1].float())
    for a, b in zip(got, dense_logits(model, ids, prompt)):
        assert max_abs(a, b) <= LOGIT_TOL
    assert cache.tokens == [prompt + 20] * 3 and cache.position.tolist() == [prompt + 20] * 3
    if kind == "max":
        with pytest.raises(ValueError):
            model(ids[:, :1], cache=cache)                       # full


@torch.no_grad()
def test_rows_of_different_lengths_come_and_go(cuda_dev):
    """Prompts of 5, 90 and 33 tokens in rows 0, 2 and 3 decode together with row 1 idle; row 2 is released and
    its pages serve a new prompt. Every row's logits are those of its sequence alone."""
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    cache = PagedCache(model.config, 4, max_tokens=128, page_size=16, n_pages=17, device=cuda_dev)
    seqs = {0: ids_of((1, 30), 2, cuda_dev), 2: ids_of((1, 115), 3, cuda_dev), 3: ids_of((1, 58), 4, cuda_dev)}
    prompts = {0: 5, 2: 90, 3: 33}
    want = {r: dense_logits(model, s, prompts[r]) for r, s in seqs.items()}
    for r, s in seqs.items():
        got = model(s[:, :prompts[r]], cache=cache.row(r), logits_to_keep=1).logits[:, -1]
        assert max_abs(got, want[r][0]) <= LOGIT_TOL
    with pytest.raises(ValueError):
        model(seqs[0][:, :5], cache=cache.row(0))                # the row holds a prompt
    with pytest.raises(ValueError):
        model(ids_of((1, 128), 9, cuda_dev), cache=cache.row(1))  # too few pages left
    cache.release(1)
    for step in range(25):
        nxt = torch.zeros((4, 1), dtype=torch.long, device=cuda_dev)
        for r, s in seqs.items():
            nxt[r] = s[0, prompts[r] + step]
        got = model(nxt, cache=cache, logits_to_keep=1).logits[:, -1]
        for r in seqs:
            assert max_abs(got[r], want[r][step + 1][0]) <= LOGIT_TOL
    assert cache.tokens == [30, -1, 115, 58] and cache.lengths.tolist() == [30, 0, 115, 58]
    cache.release(2)
    s = ids_of((1, 60), 5, cuda_dev)
    w = dense_logits(model, s, 50)
    got = model(s[:, :50], cache=cache.row(2), logits_to_keep=1).logits[:, -1]
    assert max_abs(got, w[0]) <= LOGIT_TOL
    got = model(s[:, 50:51], cache=cache.row(2), logits_to_keep=1).logits[:, -1]   # a row stepped by itself
    assert max_abs(got, w[1]) <= LOGIT_TOL
    held = [p for pages in cache.row_pages for p in pages]
    assert len(set(held)) == len(held) and sorted(held + cache.free) == list(range(17))


@torch.no_grad()
def test_eviction_follows_an_fp64_simulation(cuda_dev):
    """One layer of a bounded cache from its first token on, against plain fp64: the shares, the running
    weights, the slot taken at every step, and the attention over what is left."""
    from sisa_b200 import backends
    from sisa_b200.kernels import paged as K

    B, H, S, budget, recent, steps = 2, 3, 16, 40, 7, 150
    proj, z, lam = O.make_proj_inputs(B, steps, H, seed=3, a_mean=-3.0, z_mean=3.0)
    proj = proj.to(torch.bfloat16).to(cuda_dev)
    z, lam_d = z.to(cuda_dev), lam.to(cuda_dev)
    pages = K.KeyPages.empty(B * 3, H, S, torch.bfloat16, cuda_dev)
    table = torch.randperm(B * 3, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(B, 3).to(cuda_dev)
    carry = torch.zeros(B, H, 18, device=cuda_dev)
    pos, lengths = torch.zeros(B, dtype=torch.int32, device=cuda_dev), torch.zeros(B, dtype=torch.int32, device=cuda_dev)
    sim_w = torch.zeros(B, H, budget, dtype=torch.float64)
    sim_tok = torch.full((B, H, budget), -1)

    def plane(t, b, n):
        j = torch.arange(n)
        return t[table[b].long()[j // S].to(cuda_dev), :, (j % S).to(cuda_dev)].transpose(0, 1).double().cpu()

    for t in range(steps):
        slots = K.paged_evict(pages, table, pos, budget, recent)
        q, c, g, f = K.paged_append(proj[:, t:t + 1], z[:, t:t + 1], pages, table, pos, carry, slots=slots, budget=budget,
                                    lengths=lengths)
        y, lse = K.paged_attention(q, c, g, f, pages, table, lengths, lam_d, accumulate=True, return_lse=True)
        backends.check_status(cuda_dev)
        n = min(t + 1, budget)
        assert lengths.tolist() == [n, n]
        for b in range(B):
            kp, vp, bp, gp, fp, wp = (plane(x, b, n) for x in (pages.k, pages.v, pages.b, pages.g, pages.f, pages.weight))
            for h in range(H):
                s = int(slots[b, h]) if t >= budget else t
                if t >= budget:
                    old = sim_tok[b, h] < t - recent
                    best = sim_w[b, h].masked_fill(~old, math.inf)
                    # the least weight (the running fp32 sums of up to 150 shares are off by 1e-5 at most)
                    assert bool(old[s]) and float(best[s]) <= float(best.min()) + 1e-5
                else:
                    assert int(slots[b, h]) == -1
                sim_w[b, h, s], sim_tok[b, h, s] = 0.0, t
                sc = kp[h] @ q[b, h, 0].double().cpu() / 8
                dec = torch.exp(torch.clamp(g[b, h].double().cpu() - gp[h], max=0.0))
                sc = sc + lam[h].double() * dec * (bp[h] @ c[b, h, 0].double().cpu()) + f[b, h].double().cpu() - fp[h]
                p = torch.softmax(sc, 0)
                sim_w[b, h, :n] += p
                want = p @ vp[h]
                assert bool(((y[b, h, 0].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 5e-5 * 4).all())
                assert max_abs(wp[h], sim_w[b, h, :n]) <= 1e-5
            assert torch.equal(plane(pages.token, b, n).long(), sim_tok[b, :, :n])
        pos += 1


@torch.no_grad()
def test_bounded_prompt_keeps_the_heaviest_and_newest(cuda_dev):
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    ids = ids_of((2, 200), 6, cuda_dev)
    cache = PagedCache(model.config, 2, budget=48, recent=16, page_size=16, device=cuda_dev)
    full = PagedCache(model.config, 2, budget=200, recent=16, page_size=16, device=cuda_dev)
    model(ids, cache=cache)
    model(ids, cache=full)
    assert cache.lengths.tolist() == [48, 48] and cache.tokens == [200, 200]
    for i in range(2):
        small, big = cache.pages[i], full.pages[i]
        for r in range(2):
            tok = small.token[cache.table[r].long()].transpose(0, 1).reshape(2, -1)[:, :48].cpu()
            w = big.weight[full.table[r].long()].transpose(0, 1).reshape(2, -1)[:, :200].cpu()
            for h in range(2):
                top = torch.sort(w[h, :184], descending=True, stable=True).indices[:32].sort().values
                assert torch.equal(tok[h].long(), torch.cat([top, torch.arange(184, 200)]))


def test_generate_paged_and_bounded(cuda_dev):
    """generate() over pages equals the dense generate where nothing is dropped (the first steps of greedy
    decoding, whose logits differ by rounding only), the graph equals the eager loop, and a small budget runs."""
    model = tiny(cuda_dev)
    ids = ids_of((4, 65), 7, cuda_dev)
    dense = model.generate(ids, max_new_tokens=24)
    paged = model.generate(ids, max_new_tokens=24, page_size=32)
    assert paged.shape == dense.shape
    eager = model.generate(ids, max_new_tokens=24, page_size=32, cuda_graph=False)
    assert torch.equal(paged, eager)
    for kw in (dict(cache_budget=32), dict(cache_budget=32, cache_recent=4, cache_observe=16, page_size=16), dict(cache_budget=80)):
        a = model.generate(ids, max_new_tokens=40, **kw)
        b = model.generate(ids, max_new_tokens=40, cuda_graph=False, **kw)
        assert a.shape == (4, 105) and torch.equal(a, b), kw
    one = model.generate(ids[0, :1], max_new_tokens=20, cache_budget=8)
    assert one.shape == (21,)


def test_paged_cache_refusals_on_the_model(cuda_dev):
    from sisa_b200.generation import DecodeGraph
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    ids = ids_of((2, 10), 8, cuda_dev)
    cache = PagedCache(model.config, 2, max_tokens=32, device=cuda_dev)
    with pytest.raises(ValueError):
        model(ids, cache=cache)                                  # with autograd on
    with torch.no_grad():
        with pytest.raises(ValueError):
            model(ids[:1], cache=cache)                          # one prompt for two rows
        model(ids, cache=cache)
        with pytest.raises(ValueError):
            model(ids, cache=cache)                              # several tokens onto a prompt
        with pytest.raises(ValueError):
            DecodeGraph(model, cache, 3)
        half = PagedCache(model.config, 2, max_tokens=32, dtype=torch.float16, device=cuda_dev)
        with pytest.raises((TypeError, ValueError)):
            model(ids, cache=half)
    model.set_attn_impl("torch")
    with pytest.raises(ValueError):
        model.generate(ids, max_new_tokens=3, cache_budget=8)
