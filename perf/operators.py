"""Timing and comparison cases of the paged-cache serving operators (``sisa_b200.kernels.paged``).

A serving process keeps every sequence's keys in pages and bounds what it keeps: the prompt's keys are
weighed by the attention they received, the heaviest and the newest go into pages, every new token
replaces the lightest old key, and one query row per sequence attends over the pages. Five operators:

* ``attention``  one new token over its paged keys, optionally adding each key's share to its weight
* ``evict``      the slot whose key has the least accumulated weight, outside the newest keys
* ``append``     the new token's recurrences, rotation and write into its slot
* ``key_weights`` the attention each prompt key received from the prompt's queries
* ``fill``       the choice of the prompt's keys by weight and their copy into pages

Scores, for query i and key j (d_head 64, d_state 32):
    s_ij = q_i.k_j / 8 + lam_h exp(min(g_i - g_j, 0)) (c_i.b_j) + (F_i - F_j)

Head counts and dtypes are those of the package's presets and tests; batch, length and page sizes span
what a server meets, from one short sequence to 64 sequences of 8192 keys.
"""
import math
import random

import torch

own = False

D, S = 64, 32
LOG2E = 1.0 / math.log(2.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one interactive user early in a conversation: launch latency is everything
        dict(name="attention-one-short", op="attention", batch=1, heads=8, keys=77, ragged=False, page=16,
             dtype="bf16", accumulate=False),
        # a continuous batch of sequences of all ages, idle slots and one-token sequences among them
        dict(name="attention-ragged-24", op="attention", batch=24, heads=12, keys=4001, ragged=True, page=64,
             dtype="bf16", accumulate=False),
        # one very long document: few rows, so the length has to be split
        dict(name="attention-one-long", op="attention", batch=1, heads=16, keys=131071, ragged=False, page=128,
             dtype="fp16", accumulate=False),
        # the full decode batch with bounded caches: every key's weight is updated as well
        dict(name="attention-batch-64-weights", op="attention", batch=64, heads=16, keys=8192, ragged=False, page=64,
             dtype="bf16", accumulate=True),
        # choosing the slot to reuse: a small bounded cache
        dict(name="evict-4-small", op="evict", batch=4, heads=8, budget=500, recent=64, page=32),
        # the same for the full decode batch
        dict(name="evict-64", op="evict", batch=64, heads=16, budget=8192, recent=512, page=64),
        # the new token of a single user
        dict(name="append-one", op="append", batch=1, heads=8, budget=0, page=16, dtype="bf16"),
        # the new tokens of a large batch into reused slots
        dict(name="append-64-reuse", op="append", batch=64, heads=16, budget=256, page=64, dtype="fp16"),
        # weights of a prompt's keys over all its queries, at the training length
        dict(name="weights-prompt-4x4096", op="key_weights", batch=4, heads=16, length=4096, first=0, dtype="bf16"),
        # weights from the last 512 queries of one long prompt of odd length
        dict(name="weights-window-16411", op="key_weights", batch=1, heads=12, length=16411, first=15899, dtype="fp16"),
        # a short prompt cut to a quarter
        dict(name="fill-2x1000", op="fill", batch=2, heads=8, length=1000, keep=250, recent=32, page=16, dtype="bf16"),
        # long prompts cut to 2048 keys each
        dict(name="fill-16x8192", op="fill", batch=16, heads=16, length=8192, keep=2048, recent=256, page=64,
             dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "evict", "append", "key_weights", "fill"])
    heads = rng.choice([5, 8, 12, 16])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    batch = _logint(rng, 1, 64)
    if op == "attention":
        keys = _logint(rng, 1, min(131072, (1 << 23) // (batch * heads)))
        return dict(op=op, batch=batch, heads=heads, keys=keys, ragged=rng.random() < 0.5, page=page, dtype=dtype,
                    accumulate=rng.random() < 0.5)
    if op == "evict":
        budget = _logint(rng, 16, min(65536, (1 << 23) // (batch * heads)))
        return dict(op=op, batch=batch, heads=heads, budget=budget, recent=rng.randint(1, max(1, budget // 2)), page=page)
    if op == "append":
        return dict(op=op, batch=batch, heads=heads, budget=rng.choice([0, _logint(rng, 16, 512)]), page=page, dtype=dtype)
    if op == "key_weights":
        # at most 4 x 16 heads x 4096 x 4097 / 2 = 5.4e8 (query, key) pairs
        batch = _logint(rng, 1, 8)
        length = _logint(rng, 1, int(math.sqrt(1.07e9 / (batch * heads))))
        first = rng.choice([0, rng.randint(0, length - 1), max(0, length - 256)])
        return dict(op=op, batch=batch, heads=heads, length=length, first=first, dtype=dtype)
    batch = _logint(rng, 1, 16)
    length = _logint(rng, 2, min(65536, (1 << 21) // (batch * heads)))
    keep = rng.choice([length, _logint(rng, 1, length), max(1, length // 4)])
    keep = min(keep, max(1, (1 << 19) // (batch * heads)))
    return dict(op=op, batch=batch, heads=heads, length=length, keep=keep, recent=rng.randint(0, keep), page=page,
                dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """Keys held by each sequence: all the same, or of all ages with idle and one-token rows among them."""
    B, n = case["batch"], case["keys"]
    if not case["ragged"]:
        return [n] * B
    rng = random.Random(seed * 7919 + 11)
    out = [rng.randint(0, n) for _ in range(B)]
    out[0] = n
    if B > 2:
        out[1], out[2] = 0, 1
    return out


def _gates(gen, B, H, n, dev):
    """Cumulative decay g and forget value F (B, H, n): heads from nearly no decay to fast decay."""
    rate = torch.logspace(-4.0, -1.5, H, device=dev).view(1, H, 1)
    fr = torch.logspace(-5.0, -2.0, H, device=dev).flip(0).view(1, H, 1)
    g = -torch.cumsum(torch.rand((B, H, n), generator=gen, device=dev) * 2 * rate, dim=2)
    f = -torch.cumsum(torch.rand((B, H, n), generator=gen, device=dev) * 2 * fr, dim=2)
    return g, f


def _table(lengths, page, gen, dev):
    """A block table over a pool in random order, with one page that belongs to nobody."""
    need = [max(1, -(-n // page)) for n in lengths]
    width = max(need)
    total = sum(need) + 1
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros((len(lengths), width), dtype=torch.int32, device=dev)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = perm[at:at + m]
        at += m
    return table, total


def _randn(gen, shape, dtype, dev):
    return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)


def _lam(H, dev):
    return torch.linspace(0.2, 1.1, H, device=dev)


def _slots(B, n, page, table, dev):
    """(page index, slot) of positions 0..n-1 of every sequence, each (B, n)."""
    j = torch.arange(n, device=dev)
    return table.long()[:, j // page], (j % page).expand(B, n)


def _scatter(plane, values, table, page):
    """Write values (B, H, n, ...) into the page plane (P, H, page, ...)."""
    B, H, n = values.shape[:3]
    pg, sl = _slots(B, n, page, table, plane.device)
    plane[pg.unsqueeze(1), torch.arange(H, device=plane.device).view(1, H, 1), sl.unsqueeze(1)] = values


def _gather(plane, table, n, page):
    """The first n positions of every sequence from a page plane: (B, H, n, ...)."""
    m = -(-n // page)
    x = plane[table.long()[:, :m]].transpose(1, 2)                  # (B, H, m, page, ...)
    return x.reshape(x.shape[0], x.shape[1], m * page, *x.shape[4:])[:, :, :n]


def _key_pages(st):
    """The package's handle of the pages, made once per state as a cache keeps it."""
    if "pages" not in st:
        from sisa_b200.kernels.paged import KeyPages

        st["pages"] = KeyPages(k=st["k"], v=st["v"], b=st["b"], g=st["g"], f=st["f"], weight=st.get("weight"),
                               token=st.get("token"))
    return st["pages"]


def _planes(g, f):
    """The position planes (B, H, 4, Lp) that a prompt's preparation leaves: g, F, and each position's decay
    from the start and to the end of its block of 64."""
    B, H, L = g.shape
    out = torch.zeros((B, H, 4, (L + 3) // 4 * 4), device=g.device)
    j = torch.arange(L, device=g.device)
    start = j // 64 * 64
    out[:, :, 0, :L], out[:, :, 1, :L] = g, f
    out[:, :, 2, :L] = torch.exp((g - g[:, :, start]).clamp_max(0.0))
    out[:, :, 3, :L] = torch.exp((g[:, :, (start + 63).clamp_max(L - 1)] - g).clamp_max(0.0))
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    B, H = case["batch"], case["heads"]
    st = dict(case=dict(case))
    if op == "attention":
        dt, page = DTYPES[case["dtype"]], case["page"]
        lens = _lengths(case, seed)
        N = max(lens)
        table, P = _table(lens, page, gen, dev)
        st.update(table=table, lengths=torch.tensor(lens, dtype=torch.int32, device=dev), N=N, lam=_lam(H, dev))
        # whatever the pages' last owners left stays in the slots past a sequence's end
        st["k"] = _randn(gen, (P, H, page, D), dt, dev)
        st["v"] = _randn(gen, (P, H, page, D), dt, dev)
        st["b"] = _randn(gen, (P, H, page, S), dt, dev)
        g, f = _gates(gen, B, H, N, dev)
        st["g"] = torch.zeros((P, H, page), device=dev)
        st["f"] = torch.zeros((P, H, page), device=dev)
        live = [i for i, n in enumerate(lens) if n]
        for i in live:
            _scatter(st["g"], g[i:i + 1, :, :lens[i]], table[i:i + 1], page)
            _scatter(st["f"], f[i:i + 1, :, :lens[i]], table[i:i + 1], page)
        last = (st["lengths"].long() - 1).clamp_min(0).view(B, 1, 1).expand(B, H, 1)
        st["gq"], st["fq"] = g.gather(2, last).contiguous(), f.gather(2, last).contiguous()
        st["q"] = _randn(gen, (B, H, 1, D), dt, dev)
        st["c"] = _randn(gen, (B, H, 1, S), dt, dev)
        if case["accumulate"]:
            # what earlier steps gave: a few heavy keys, most of them light
            st["weight"] = torch.rand((P, H, page), generator=gen, device=dev).pow_(6).mul_(3.0)
            st["weight_out"] = st["weight"].clone()
    elif op == "evict":
        page, n = case["page"], case["budget"]
        table, P = _table([n] * B, page, gen, dev)
        rng = random.Random(seed * 31 + 5)
        # most sequences are past their budget, some still grow, some rows are idle
        pos = [n + rng.randint(0, 4 * n) for _ in range(B)]
        for i in range(1, B):
            if i % 7 == 3:
                pos[i] = rng.randint(0, n - 1)
            if i % 11 == 5:
                pos[i] = -1
        st.update(table=table, position=torch.tensor(pos, dtype=torch.int32, device=dev))
        w = torch.rand((B, H, n), generator=gen, device=dev).pow_(6).mul_(3.0)
        w = torch.where(w < 1e-6, torch.zeros_like(w), w)           # forgotten keys end at exactly zero
        # slots are reused, so the tokens a cache holds lie in any order; the newest are all held
        p = st["position"].clamp_min(n).view(B, 1, 1)
        tok = torch.rand((B, H, n), generator=gen, device=dev).argsort(dim=2)
        tok = torch.where(tok < case["recent"], p - 1 - tok, tok - case["recent"]).to(torch.int32)
        st["weight"] = torch.zeros((P, H, page), device=dev)
        st["token"] = torch.zeros((P, H, page), dtype=torch.int32, device=dev)
        _scatter(st["weight"], w, table, page)
        _scatter(st["token"], tok, table, page)
        # the pages' other planes are not read
        for name, x in (("k", D), ("v", D), ("b", S)):
            st[name] = torch.empty((P, H, page, x), dtype=torch.bfloat16, device=dev)
        st["g"], st["f"] = torch.empty_like(st["weight"]), torch.empty_like(st["weight"])
    elif op == "append":
        dt, page, budget = DTYPES[case["dtype"]], case["page"], case["budget"]
        n = budget if budget else 96
        table, P = _table([n] * B, page, gen, dev)
        rng = random.Random(seed * 17 + 3)
        pos = [n + rng.randint(0, 5000) if budget else rng.randint(0, n - 1) for _ in range(B)]
        if B > 4:
            pos[3], pos[4] = -1, 0                                   # an idle row and a first token
        st.update(table=table, position=torch.tensor(pos, dtype=torch.int32, device=dev))
        slots = [[rng.randint(0, n - 1) if p >= n else -1 for _ in range(H)] for p in pos]
        st["slots"] = torch.tensor(slots, dtype=torch.int32, device=dev) if budget else None
        npad = (273 * H + 15) // 16 * 16
        proj = torch.randn((B, 1, npad), generator=gen, device=dev)
        proj[..., 256 * H:272 * H] *= 0.2                            # rotation rates
        proj[..., 272 * H:273 * H] = proj[..., 272 * H:273 * H] * 0.45 - 5.0
        st["proj"] = proj.to(dt)
        st["z"] = torch.randn((B, 1, H), generator=gen, device=dev) * 0.45 + 4.0
        carry = torch.randn((B, H, 18), generator=gen, device=dev) * 20.0
        carry[..., 16:] = -carry[..., 16:].abs()
        st["carry"], st["carry_out"] = carry, torch.zeros_like(carry)
        for name, x in (("k", D), ("v", D), ("b", S)):
            st[name] = _randn(gen, (P, H, page, x), dt, dev)
        for name in ("g", "f", "weight"):
            st[name] = torch.rand((P, H, page), generator=gen, device=dev)
        st["token"] = torch.zeros((P, H, page), dtype=torch.int32, device=dev)
        st["lengths"] = torch.zeros(B, dtype=torch.int32, device=dev)
    else:
        dt, L = DTYPES[case["dtype"]], case["length"]
        # the prompt's keys and values are head views of the fused projection, as the layer hands them over
        npad = (273 * H + 15) // 16 * 16
        proj = torch.randn((B, L, npad), generator=gen, device=dev).to(dt)
        st["proj"] = proj
        for i, name in enumerate(("q", "k", "v")):
            st[name + "p"] = proj[..., i * H * D:(i + 1) * H * D].view(B, L, H, D).transpose(1, 2)
        st["bp"] = _randn(gen, (B, H, L, S), dt, dev)
        st["gp"], st["fp"] = _gates(gen, B, H, L, dev)
        if op == "key_weights":
            st["c"] = _randn(gen, (B, H, L, S), dt, dev)
            st["lam"] = _lam(H, dev)
            lse = torch.zeros((B, H, L), device=dev)                 # rows before `first` are not read
            for b, h, i0, i1 in _blocks(case):
                s = _scores(st, b, h, i0, i1, torch.float32)
                lse[b, h, i0:i1] = torch.logsumexp(s, dim=-1) * LOG2E
            st["lse"] = lse
            st["pos"] = _planes(st["gp"], st["fp"])
        else:
            page, K = case["page"], case["keep"]
            table, P = _table([K] * B, page, gen, dev)
            w = torch.rand((B, H, L), generator=gen, device=dev).pow_(8).mul_(5.0)
            st.update(table=table, w=torch.where(w < 1e-5, torch.zeros_like(w), w))
            for name, x in (("k", D), ("v", D), ("b", S)):
                st[name] = torch.zeros((P, H, page, x), dtype=dt, device=dev)
            for name in ("g", "f", "weight"):
                st[name] = torch.zeros((P, H, page), device=dev)
            st["token"] = torch.zeros((P, H, page), dtype=torch.int32, device=dev)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    return (_OWN if own else _PLAIN)[op](st)


def _own_attention(st):
    from sisa_b200.kernels.paged import paged_attention

    y, lse = paged_attention(st["q"], st["c"], st["gq"], st["fq"], _key_pages(st), st["table"], st["lengths"], st["lam"],
                             accumulate=st["case"]["accumulate"], weight_out=st.get("weight_out"), return_lse=True)
    return [y, lse] + ([st["weight_out"]] if st["case"]["accumulate"] else [])


def _own_evict(st):
    from sisa_b200.kernels.paged import paged_evict

    return paged_evict(_key_pages(st), st["table"], st["position"], st["case"]["budget"], st["case"]["recent"])


def _own_append(st):
    from sisa_b200.kernels.paged import paged_append

    q, c, g, f = paged_append(st["proj"], st["z"], _key_pages(st), st["table"], st["position"], st["carry"],
                              carry_out=st["carry_out"], slots=st["slots"], budget=st["case"]["budget"] or None,
                              lengths=st["lengths"])
    return [q, c, g, f, st["carry_out"], st["lengths"]] + [st[n] for n in ("k", "v", "b", "g", "f", "weight", "token")]


def _own_key_weights(st):
    from sisa_b200.kernels.paged import attention_key_weights

    return attention_key_weights(st["qp"], st["kp"], st["c"], st["bp"], st["pos"], st["lam"], st["lse"],
                                 first_query=st["case"]["first"])


def _own_fill(st):
    from sisa_b200.kernels.paged import paged_fill

    case = st["case"]
    paged_fill(_key_pages(st), st["table"], st["kp"], st["vp"], st["bp"], st["gp"], st["fp"], weight=st["w"],
               keep=case["keep"], recent=case["recent"])
    return [st[n] for n in ("k", "v", "b", "g", "f", "weight", "token")]


_OWN = dict(attention=_own_attention, evict=_own_evict, append=_own_append, key_weights=_own_key_weights,
            fill=_own_fill)


def _plain_attention(st):
    case = st["case"]
    page, N = case["page"], st["N"]
    B, H = case["batch"], case["heads"]
    dt = st["q"].dtype
    if N == 0:
        k = torch.zeros((B, H, 0, D), device=st["q"].device)
        return [torch.zeros_like(st["q"]), k.sum((2, 3)) - math.inf]
    mask = (torch.arange(N, device=st["q"].device) < st["lengths"].view(B, 1)).view(B, 1, N)
    k = _gather(st["k"], st["table"], N, page).float()
    x = (st["q"].float() * k).sum(-1) * 0.125 if B * H <= 16 else (k @ st["q"].float().transpose(2, 3))[..., 0] * 0.125
    del k
    b = _gather(st["b"], st["table"], N, page).float()
    cb = (b @ st["c"].float().transpose(2, 3))[..., 0]
    del b
    g, f = _gather(st["g"], st["table"], N, page), _gather(st["f"], st["table"], N, page)
    x = x + st["lam"].view(1, H, 1) * torch.exp((st["gq"] - g).clamp_max(0.0)) * cb + (st["fq"] - f)
    x = torch.where(mask, x, torch.full_like(x, -math.inf))
    m = x.max(dim=-1, keepdim=True).values
    m0 = torch.where(m > -math.inf, m, torch.zeros_like(m))          # idle rows attend to nothing
    p = torch.exp(x - m0)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    v = _gather(st["v"], st["table"], N, page).float()
    y = (p.unsqueeze(2) @ torch.where(mask.unsqueeze(-1), v, torch.zeros_like(v))).to(dt)
    out = [y, ((m0 + torch.log(l)) * LOG2E)[..., 0]]
    if case["accumulate"]:
        w = _gather(st["weight"], st["table"], N, page) + p
        wo = st["weight_out"]
        if case["ragged"]:
            # the positions past a sequence's end go to a page behind the pool
            pool = torch.cat([wo, torch.zeros_like(wo[:1])])
            past = torch.arange(-(-N // page), device=w.device) * page >= st["lengths"].view(B, 1)
            keep = torch.where(mask, w, _gather(wo, st["table"], N, page))
            _scatter(pool, keep, torch.where(past, wo.shape[0], st["table"]), page)
            wo.copy_(pool[:-1])
        else:
            _scatter(wo, w, st["table"], page)
        out.append(wo)
    return out


def _plain_evict(st):
    case = st["case"]
    page, n = case["page"], case["budget"]
    pos = st["position"].view(-1, 1, 1)
    w = _gather(st["weight"], st["table"], n, page)
    tok = _gather(st["token"], st["table"], n, page)
    w = torch.where(tok >= pos - case["recent"], torch.full_like(w, math.inf), w)
    low = w.min(dim=-1, keepdim=True).values
    idx = torch.arange(n, device=w.device, dtype=torch.int32).expand_as(w)
    first = torch.where(w == low, idx, torch.full_like(idx, n)).min(dim=-1).values
    return torch.where(pos[..., 0] >= n, first, torch.full_like(first, -1))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp_max(20))))


def _append_math(st, dt):
    """The new token's values in dtype ``dt``: q, k, v, rotated c and b, g, F, phase."""
    B, H = st["case"]["batch"], st["case"]["heads"]
    x = st["proj"].to(dt).view(B, -1)
    parts, at = [], 0
    for w in (D, D, D, S, S, S // 2, 1):
        parts.append(x[:, at:at + H * w].view(B, H, w))
        at += H * w
    q, k, v, b, c, th, a = parts
    carry = st["carry"].to(dt)
    z = st["z"].to(dt).view(B, H)
    phi = carry[..., :16] + th
    g = carry[..., 16] - _softplus(a[..., 0])
    f = carry[..., 17] + torch.minimum(z, torch.zeros_like(z)) - torch.log1p(torch.exp(-z.abs()))
    cs, sn = torch.cos(phi), torch.sin(phi)

    def rot(t):
        e, o = t[..., 0::2], t[..., 1::2]
        return torch.stack([e * cs - o * sn, e * sn + o * cs], dim=-1).reshape(B, H, S)

    return q, k, v, rot(c), rot(b), g, f, phi


def _append(st, dt, low, planes, carry_out, lengths):
    """Write the new token into ``planes`` (a dict of page planes) and return the query side."""
    case = st["case"]
    B, H, page = case["batch"], case["heads"], case["page"]
    dev = st["proj"].device
    q, k, v, c, b, g, f, phi = _append_math(st, dt)
    pos = st["position"].long()
    live = pos >= 0
    slot = pos.view(B, 1).expand(B, H)
    if st["slots"] is not None:
        slot = torch.where(st["slots"] >= 0, st["slots"].long(), slot)
    slot = torch.where(live.view(B, 1), slot, torch.zeros_like(slot))
    pg = st["table"].long().gather(1, slot // page)
    hh = torch.arange(H, device=dev).expand(B, H)
    sel = torch.nonzero(live.view(B, 1).expand(B, H), as_tuple=True)           # an idle row writes nothing
    at = (pg[sel], hh[sel], (slot % page)[sel])
    for name, val in (("k", k), ("v", v), ("b", b), ("g", g), ("f", f), ("weight", torch.zeros_like(g)),
                      ("token", pos.view(B, 1).expand(B, H))):
        planes[name][at] = val[sel].to(planes[name].dtype)
    new = torch.cat([phi, g.unsqueeze(-1), f.unsqueeze(-1)], dim=-1)
    on = live.view(B, 1, 1)
    carry_out.copy_(torch.where(on, new, st["carry"].to(dt)))
    n = pos + 1
    lengths.copy_(n.clamp(max=case["budget"]) if case["budget"] else n)
    zero = torch.zeros_like
    return [q.unsqueeze(2).to(low), torch.where(on, c, zero(c)).unsqueeze(2).to(low),
            torch.where(on[..., 0], g, zero(g)).unsqueeze(-1), torch.where(on[..., 0], f, zero(f)).unsqueeze(-1)]


def _plain_append(st):
    names = ("k", "v", "b", "g", "f", "weight", "token")
    out = _append(st, torch.float32, st["proj"].dtype, {n: st[n] for n in names}, st["carry_out"], st["lengths"])
    return out + [st["carry_out"], st["lengths"]] + [st[n] for n in names]


def _blocks(case):
    """(b, h, i0, i1): the query rows from ``first`` on, in blocks of at most 2^26 scores."""
    L, first = case["length"], case["first"]
    step = max(1, min(L, (1 << 26) // L))
    for b in range(case["batch"]):
        for h in range(case["heads"]):
            for i0 in range(first, L, step):
                yield b, h, i0, min(L, i0 + step)


def _scores(st, b, h, i0, i1, dt):
    """Masked scores of queries i0..i1-1 of one head in dtype ``dt``."""
    q, k = st["qp"][b, h, i0:i1].to(dt), st["kp"][b, h, :i1].to(dt)
    c, bm = st["c"][b, h, i0:i1].to(dt), st["bp"][b, h, :i1].to(dt)
    g, f = st["gp"][b, h].to(dt), st["fp"][b, h].to(dt)
    s = (q @ k.t()) * 0.125
    s = s + st["lam"][h].to(dt) * torch.exp((g[i0:i1, None] - g[None, :i1]).clamp_max(0.0)) * (c @ bm.t())
    s = s + (f[i0:i1, None] - f[None, :i1])
    i, j = torch.arange(i0, i1, device=s.device)[:, None], torch.arange(i1, device=s.device)[None]
    return torch.where(j <= i, s, torch.full_like(s, -math.inf))


def _weigh(st, dt):
    case = st["case"]
    w = torch.zeros((case["batch"], case["heads"], case["length"]), dtype=dt, device=st["qp"].device)
    for b, h, i0, i1 in _blocks(case):
        s = _scores(st, b, h, i0, i1, dt)
        w[b, h, :i1] += torch.exp(s - st["lse"][b, h, i0:i1, None].to(dt) / LOG2E).sum(0)
    return w


def _plain_key_weights(st):
    return _weigh(st, torch.float32)


def _plain_fill(st):
    case = st["case"]
    B, H, L, K, R, page = (case[n] for n in ("batch", "heads", "length", "keep", "recent", "page"))
    dev = st["w"].device
    # the newest `recent` keys stay; of the rest the heaviest, the earlier one where two weigh the same
    key = torch.where(torch.arange(L, device=dev) >= L - R, torch.full_like(st["w"], math.inf), st["w"])
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :K]
    idx = torch.sort(order, dim=-1).values
    for name, src in (("k", st["kp"]), ("v", st["vp"]), ("b", st["bp"])):
        _scatter(st[name], src.gather(2, idx.unsqueeze(-1).expand(B, H, K, src.shape[-1])), st["table"], page)
    for name, src in (("g", st["gp"]), ("f", st["fp"]), ("weight", st["w"])):
        _scatter(st[name], src.gather(2, idx), st["table"], page)
    _scatter(st["token"], idx.to(torch.int32), st["table"], page)
    return [st[n] for n in ("k", "v", "b", "g", "f", "weight", "token")]


_PLAIN = dict(attention=_plain_attention, evict=_plain_evict, append=_plain_append, key_weights=_plain_key_weights,
              fill=_plain_fill)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    op = case["op"]
    st = prepare(case, seed)
    f64 = torch.float64
    if op == "attention":
        page, H = case["page"], case["heads"]
        lens = st["lengths"].tolist()
        y = torch.zeros(st["q"].shape, dtype=f64, device=st["q"].device)
        lse = torch.full(st["q"].shape[:2], -math.inf, dtype=f64, device=y.device)
        wo = st["weight"].double() if case["accumulate"] else None
        for i, n in enumerate(lens):
            if n == 0:
                continue
            rows = st["table"][i].long()
            j = torch.arange(n, device=y.device)
            pg, sl = rows[j // page], j % page
            for h in range(H):
                s = st["k"][pg, h, sl].to(f64) @ st["q"][i, h, 0].to(f64) / 8.0
                dec = torch.exp(torch.clamp(st["gq"][i, h].to(f64) - st["g"][pg, h, sl].to(f64), max=0.0))
                s = s + st["lam"][h].to(f64) * dec * (st["b"][pg, h, sl].to(f64) @ st["c"][i, h, 0].to(f64))
                s = s + st["fq"][i, h].to(f64) - st["f"][pg, h, sl].to(f64)
                p = torch.softmax(s, dim=0)
                y[i, h, 0] = p @ st["v"][pg, h, sl].to(f64)
                lse[i, h] = torch.logsumexp(s, dim=0) / math.log(2.0)
                if wo is not None:
                    wo[pg, h, sl] = wo[pg, h, sl] + p
        return [y, lse] + ([wo] if wo is not None else [])
    if op == "append":
        names = ("k", "v", "b", "g", "f", "weight")
        planes = {n: st[n].to(f64) for n in names}
        planes["token"] = st["token"].clone()
        carry, lengths = torch.zeros_like(st["carry"], dtype=f64), torch.zeros_like(st["lengths"])
        out = _append(st, f64, f64, planes, carry, lengths)
        return out + [carry, lengths] + [planes[n] for n in names] + [planes["token"]]
    if op == "key_weights":
        return _weigh(st, f64)
    if op == "evict":
        return None                                                   # a choice: no computed number
    # fill: every head's choice on the host, then copies
    import numpy as np

    L, K, R, page = case["length"], case["keep"], case["recent"], case["page"]
    w = st["w"].cpu().numpy()
    idx = np.empty((case["batch"], case["heads"], K), dtype=np.int64)
    for b, h in np.ndindex(*idx.shape[:2]):
        old = np.lexsort((np.arange(L - R), -w[b, h, :L - R]))[:K - R]          # by weight, then by position
        idx[b, h] = np.concatenate([np.sort(old), np.arange(L - R, L)])
    idx = torch.from_numpy(idx).to(st["w"].device)
    out = []
    for name, src in (("k", st["kp"]), ("v", st["vp"]), ("b", st["bp"]), ("g", st["gp"]), ("f", st["fp"]),
                      ("weight", st["w"])):
        plane = torch.zeros(st[name].shape, dtype=f64, device=idx.device)
        at = idx if src.dim() == 3 else idx.unsqueeze(-1).expand(*idx.shape, src.shape[-1])
        _scatter(plane, src.gather(2, at).to(f64), st["table"], page)
        out.append(plane)
    token = torch.zeros_like(st["token"])
    _scatter(token, idx.to(torch.int32), st["table"], page)
    return out + [token]


def work(case):
    """Each input read once, each output written once; multiply-adds of the products as two operations."""
    op, B, H = case["op"], case["batch"], case["heads"]
    key = 2 * (D + D + S) + 8                                         # k, v, b~ in 16 bits, g and F in 32
    if op == "attention":
        # ragged rows are spread evenly over 0 .. keys
        n = B * H * case["keys"] * (0.5 if case["ragged"] and B > 1 else 1.0)
        return {"bytes": n * (key + (8 if case["accumulate"] else 0)) + B * H * (2 * (2 * D + S) + 12),
                "flops": n * 2 * (D + S + D)}
    if op == "evict":
        n = B * H * case["budget"]
        return {"bytes": 8 * n + 4 * B * H, "flops": 2 * n}
    if op == "append":
        # the projection row, the state in and out, the written key and the query side
        return {"bytes": B * H * (2 * 273 + 4 + 2 * 72 + key + 8 + 2 * S + 8), "flops": B * H * 200}
    L = case["length"]
    if op == "key_weights":
        M = L - case["first"]
        pairs = B * H * (M * case["first"] + M * (M + 1) / 2)
        return {"bytes": B * H * (M * (2 * (D + S) + 12) + L * (2 * (D + S) + 8 + 4)), "flops": pairs * 2 * (D + S)}
    K = case["keep"]
    return {"bytes": B * H * (4 * L + K * (2 * key + 8)), "flops": B * H * L}
