"""A paged, bounded decode cache for many sequences (the server's form of src/sisa/generation.py:58-136).

The reference's cache holds one rectangular batch and grows with the text. :class:`PagedCache` holds ``rows``
independent sequences whose keys lie in pages of one pool per layer, so sequences of different lengths decode
in one batch, and rows come and go. With a ``budget`` a row keeps at most that many keys per head: the
prompt's heaviest by attention received (plus the ``recent`` newest), and from then on every new token takes
the slot of the lightest old key (:mod:`sisa_b200.kernels.paged`).

    cache = PagedCache(model.config, rows=8, page_size=64, budget=4096, recent=512)
    model(prompt_a, cache=cache.row(0), logits_to_keep=1)      # prompts of any lengths, row by row
    model(prompt_b, cache=cache.row(3), logits_to_keep=1)
    logits = model(next_ids, cache=cache).logits               # (8, 1) ids; idle rows' logits mean nothing
    cache.release(3)

It runs on the ``cuda`` attention path only and raises elsewhere.
"""
from __future__ import annotations

from typing import TYPE_CHECKING

import torch
from torch import Tensor

from .kernels import paged as K

if TYPE_CHECKING:  # pragma: no cover
    from .config import SISAConfig

__all__ = ["PagedCache", "PagedRows", "PagedLayer"]


def resolve_recent(budget: int, recent: int | None, observe: int | None) -> int:
    """The number of newest keys that are never evicted, by default a quarter of the budget, with the eviction's
    arguments checked."""
    if budget < 1:
        raise ValueError(f"budget must be >= 1, got {budget}")
    recent = budget // 4 if recent is None else recent
    if not 0 <= recent < budget:
        raise ValueError(f"recent must lie in [0, budget), got {recent} with a budget of {budget}")
    if observe is not None and observe < 1:
        raise ValueError(f"observe must be >= 1, got {observe}")
    return recent


class PagedLayer:
    """One layer of some rows of a :class:`PagedCache`, as the attention's decode step uses it."""

    paged = True

    def __init__(self, rows: "PagedRows", layer_idx: int):
        self.rows, self.layer_idx = rows, layer_idx
        self.pages = rows.cache.pages[layer_idx]

    @property
    def k_buf(self) -> Tensor:
        return self.pages.k

    def step(self, proj: Tensor, z: Tensor, lam: Tensor) -> Tensor:
        """The attention of one new token per row from its fused projection ``proj`` (rows, 1, NPAD) and forget
        logits ``z`` (rows, 1, H): slot choice, append, attention. Returns y (rows, H, 1, 64)."""
        rows, cache, pages = self.rows, self.rows.cache, self.pages
        if proj.shape[0] != rows.count:
            raise ValueError(f"the cache has {rows.count} rows, the step {proj.shape[0]}")
        if self.layer_idx == 0:
            rows.before_step()
        slots = None
        if cache.budget is not None and rows.may_evict():
            slots = K.paged_evict(pages, rows.table, rows.position, cache.budget, cache.recent)
        q, c, g, f = K.paged_append(proj, z, pages, rows.table, rows.position, rows.carry(self.layer_idx), slots=slots,
                                    budget=cache.budget, lengths=rows.lengths)
        y = K.paged_attention(q, c, g, f, pages, rows.table, rows.lengths, lam, accumulate=cache.budget is not None)
        if self.layer_idx == cache.n_layer - 1:
            rows.after_step()
        return y


class PagedRows:
    """Rows [first, first + count) of a :class:`PagedCache`; what the model takes as ``cache``."""

    paged = True

    def __init__(self, cache: "PagedCache", first: int, count: int):
        # the whole cache does not refer to itself: a cycle would keep its pages allocated until the garbage collector runs
        self._cache = None if cache is self else cache
        self.first, self.count = first, count
        span = slice(first, first + count)
        self.table, self.position, self.lengths = cache.table[span], cache.position[span], cache.lengths[span]
        self._live = cache.live[span]
        self._range = range(first, first + count)

    @property
    def cache(self) -> "PagedCache":
        return self if self._cache is None else self._cache

    def carry(self, layer_idx: int) -> Tensor:
        return self.cache.carries[layer_idx, self.first:self.first + self.count]

    def get(self, layer_idx: int) -> PagedLayer | None:
        """The layer's state, or None while no row of these holds keys of it (a prompt then fills them)."""
        if all(self.cache.filled[r] <= layer_idx for r in self._range):
            return None
        return PagedLayer(self, layer_idx)

    def __len__(self) -> int:
        return max(self.cache.filled[r] for r in self._range)

    @property
    def seq_len(self) -> int:
        """Tokens seen by the longest row."""
        return max(self.cache.tokens[r] for r in self._range)

    # ------------------------------------------------------------------------------------ prompt
    def weigh_from(self, length: int) -> int | None:
        """The first prompt query whose attention weighs the keys, or None where no weights are needed."""
        c = self.cache
        if c.budget is None:
            return None
        return 0 if c.observe is None else max(0, length - c.observe)

    def fill(self, layer_idx: int, k: Tensor, v: Tensor, b: Tensor, g: Tensor, fgate: Tensor, phi: Tensor,
             weight: Tensor | None) -> None:
        """One layer's prompt into these rows: k, v (rows, H, L, 64), b~ (rows, H, L, 32), g and F (rows, H, L) fp32, the
        phase at the last position (rows, H, 16), and with a budget the keys' weights (rows, H, L)."""
        cache = self.cache
        n, _, L, _ = k.shape
        if n != self.count:
            raise ValueError(f"the cache has {self.count} rows, the prompt {n}")
        if any(cache.filled[r] != layer_idx for r in self._range):
            raise ValueError("a prompt goes into empty rows of a paged cache (release them first)")
        keep = min(L, cache.capacity)
        if layer_idx == 0:
            if cache.budget is None and L > cache.capacity:
                raise ValueError(f"the prompt has {L} tokens, a row of the cache holds {cache.capacity}")
            self._take_pages([-(-keep // cache.page_size)] * n)
        K.paged_fill(cache.pages[layer_idx], self.table, k, v, b, g, fgate, weight=weight, keep=keep,
                     recent=min(cache.recent, keep) if cache.budget is not None else 0)
        carry = self.carry(layer_idx)
        carry[..., :16].copy_(phi)
        carry[..., 16].copy_(g[..., -1])
        carry[..., 17].copy_(fgate[..., -1])
        for r in self._range:
            cache.filled[r] = layer_idx + 1
        if layer_idx == cache.n_layer - 1:
            self.position.fill_(L)
            self.lengths.fill_(keep)
            self._live.fill_(1)
            for r in self._range:
                cache.tokens[r] = L

    def _take_pages(self, need: list[int]) -> None:
        """Give row first + i its first need[i] pages, all or none."""
        cache = self.cache
        missing = [max(0, m - len(cache.row_pages[r])) for r, m in zip(self._range, need)]
        if sum(missing) > len(cache.free):
            raise ValueError(f"the page pool is exhausted: {sum(missing)} pages needed, {len(cache.free)} free")
        for r, m in zip(self._range, missing):
            if m:
                at = len(cache.row_pages[r])
                new = [cache.free.pop() for _ in range(m)]
                cache.row_pages[r] += new
                cache.table[r, at:at + m] = torch.tensor(new, dtype=torch.int32).to(cache.table.device)

    # ------------------------------------------------------------------------------------ steps
    def may_evict(self) -> bool:
        """Whether a row may be at its budget (a captured step serves every later position, so it always may)."""
        cache = self.cache
        return torch.cuda.is_current_stream_capturing() or any(cache.tokens[r] >= cache.budget for r in self._range)

    def before_step(self) -> None:
        """Pages for the next token of every live row. A captured step finds them there already."""
        if torch.cuda.is_current_stream_capturing():
            return
        cache = self.cache
        need = []
        for r in self._range:
            t = cache.tokens[r]
            if 0 <= t and cache.budget is None and t >= cache.capacity:
                raise ValueError(f"row {r} of the paged cache is full ({cache.capacity} tokens)")
            need.append(0 if t < 0 else min(t, cache.capacity - 1) // cache.page_size + 1)
        self._take_pages(need)

    def after_step(self) -> None:
        """Advance the live rows by one token (the device counters with the captured step, the host's outside)."""
        self.position.add_(self._live)
        if not torch.cuda.is_current_stream_capturing():
            self.advance_host()

    def advance_host(self) -> None:
        tokens = self.cache.tokens
        for r in self._range:
            if tokens[r] >= 0:
                tokens[r] += 1

    def room(self) -> int:
        """Steps left before a live row is full (rows with a budget never are)."""
        cache = self.cache
        if cache.budget is not None:
            return (1 << 31) - 1 - max(self.seq_len, 0)
        left = [cache.capacity - cache.tokens[r] for r in self._range if cache.tokens[r] >= 0]
        return min(left) if left else 0


class PagedCache(PagedRows):
    """``rows`` sequences over one page pool per layer. A row holds up to ``max_tokens`` keys per head, or
    ``budget`` with eviction (the ``recent`` newest, by default a quarter, are never evicted; the prompt's keys are
    weighed by its last ``observe`` queries, by default all). ``n_pages`` defaults to what every row at its largest
    needs; with fewer, rows share what there is and a step that finds none raises ValueError."""

    def __init__(self, config: "SISAConfig", rows: int, *, max_tokens: int | None = None, budget: int | None = None,
                 recent: int | None = None, observe: int | None = None, page_size: int = 64, n_pages: int | None = None,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        if rows < 1:
            raise ValueError(f"rows must be >= 1, got {rows}")
        if (max_tokens is None) == (budget is None):
            raise ValueError("give either max_tokens or, for eviction, budget")
        if page_size not in K.PAGE_SIZES:
            raise ValueError(f"page_size must be one of {K.PAGE_SIZES}, got {page_size}")
        capacity = max_tokens if budget is None else budget
        if budget is None and max_tokens < 1:
            raise ValueError(f"max_tokens must be >= 1, got {max_tokens}")
        if budget is None and (recent is not None or observe is not None):
            raise ValueError("recent and observe need a budget")
        recent = 0 if budget is None else resolve_recent(budget, recent, observe)
        if config.d_head != 64 or config.d_state != 32:
            raise ValueError("the paged cache needs d_head 64 and d_state 32")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"the paged cache holds bf16 or fp16 keys, got {dtype}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"the paged cache runs on the cuda path only, got device {device}")
        self.budget, self.recent, self.observe = budget, recent, observe
        self.capacity, self.page_size, self.n_layer = capacity, page_size, config.n_layer
        per_row = -(-capacity // page_size)
        n_pages = rows * per_row if n_pages is None else n_pages
        if n_pages < 1:
            raise ValueError(f"n_pages must be >= 1, got {n_pages}")
        self.pages = [K.KeyPages.empty(n_pages, config.n_head, page_size, dtype, device, evict=budget is not None)
                      for _ in range(config.n_layer)]
        dev = self.pages[0].device
        self.carries = torch.zeros((config.n_layer, rows, config.n_head, K.CARRY), dtype=torch.float32, device=dev)
        self.table = torch.zeros((rows, per_row), dtype=torch.int32, device=dev)
        self.position = torch.full((rows,), -1, dtype=torch.int32, device=dev)    # index of a row's next token
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=dev)           # keys a row holds
        self.live = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.free = list(range(n_pages - 1, -1, -1))
        self.row_pages: list[list[int]] = [[] for _ in range(rows)]
        self.filled = [0] * rows                                                   # layers that hold the row's prompt
        self.tokens = [-1] * rows                                                  # tokens seen; -1: idle
        super().__init__(self, 0, rows)

    def row(self, r: int) -> PagedRows:
        """Row ``r`` alone (for its prompt, or to step it by itself)."""
        if not 0 <= r < self.count:
            raise ValueError(f"row {r} outside [0, {self.count})")
        return PagedRows(self, r, 1)

    def release(self, r: int) -> None:
        """Make row ``r`` idle and give its pages back."""
        rows = self.row(r)
        rows.position.fill_(-1)
        rows.lengths.zero_()
        rows._live.zero_()
        self.free += reversed(self.row_pages[r])
        self.row_pages[r], self.filled[r], self.tokens[r] = [], 0, -1

    def reset(self) -> None:
        for r in range(self.count):
            self.release(r)
