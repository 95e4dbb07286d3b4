"""The host side of the paged cache: argument checks that need no GPU."""
from __future__ import annotations

import pytest
import torch

import sisa_b200 as sisa
from sisa_b200.paged_cache import PagedCache


def test_arguments():
    cfg = sisa.SISAConfig(vocab_size=97, d_model=128, n_layer=2, n_head=2, d_ff=96)
    for kw in (dict(rows=0, budget=8), dict(rows=2), dict(rows=2, budget=8, max_tokens=8), dict(rows=2, budget=0),
               dict(rows=2, budget=8, recent=8), dict(rows=2, budget=8, recent=-1), dict(rows=2, max_tokens=8, recent=2),
               dict(rows=2, max_tokens=8, observe=2), dict(rows=2, budget=8, observe=0), dict(rows=2, budget=8, page_size=24),
               dict(rows=2, budget=8, device="cpu")):
        with pytest.raises(ValueError):
            PagedCache(cfg, **kw)
    with pytest.raises(TypeError):
        PagedCache(cfg, rows=2, budget=8, dtype=torch.float32)
    with pytest.raises(ValueError):
        PagedCache(sisa.SISAConfig(vocab_size=97, d_model=128, n_layer=1, n_head=4, d_ff=96), rows=1, budget=8)


def test_generate_needs_the_cuda_path():
    cfg = sisa.SISAConfig(vocab_size=97, d_model=128, n_layer=1, n_head=2, d_ff=96)
    model = sisa.SISAForCausalLM(cfg)
    ids = torch.zeros((1, 4), dtype=torch.long)
    for kw in (dict(page_size=16), dict(cache_budget=8), dict(cache_recent=2), dict(cache_observe=2)):
        with pytest.raises(ValueError):
            model.generate(ids, max_new_tokens=2, **kw)
