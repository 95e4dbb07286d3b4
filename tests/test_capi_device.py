"""Every launching entry point makes the device that owns its data current before its first launch (no GPU).

A call whose data lies on a GPU other than the current one must not launch on the current one. Two GPUs are not
needed to see that the owner is looked up: with arguments that pass every check and addresses that belong to no
device, the call has to end at that look-up (``cudaPointerGetAttributes``), not at a kernel launch. The test is
for machines without a GPU only, where no launch is possible whatever the library does."""
from __future__ import annotations

import ctypes

import pytest
import torch

from sisa_b200 import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of no device: only where nothing can launch")

A = 0x10000          # 16-byte aligned, in no allocation
BF16 = _lib.BF16


def view(width, rows=200, B=3, H=2):
    return _lib.vref(_lib.View4(A, rows * width * H, width, width * H))


def paged_calls(lib):
    H, S = 2, 64
    pg = _lib.Pages(A, A, A, A, A, A, A, 64 * S * H, 64 * S, 64 * S * H, 64 * S, 32 * S * H, 32 * S, S * H, S, 8, S)
    p, one = ctypes.byref(pg), lambda w: _lib.vref(_lib.View4(A, 2 * w, w, w))
    return {
        "sisa_paged_attn": lambda: lib.sisa_paged_attn(one(64), one(32), A, A, p, A, 4, 4, A, A, 3, 2, BF16, one(64), None,
                                                       None, A, None, None),
        "sisa_paged_evict": lambda: lib.sisa_paged_evict(p, A, 4, 4, A, 3, 2, 100, 8, A, None, None),
        "sisa_paged_append": lambda: lib.sisa_paged_append(A, 560, A, 2, p, A, 4, 4, A, None, 0, 3, 2, BF16, A, A, A, A, A,
                                                           None, None, None),
        "sisa_paged_fill": lambda: lib.sisa_paged_fill(p, A, 4, 4, view(64), view(64), view(32), A, 400, 200, A, 400, 200, A,
                                                       3, 2, 200, 100, 10, A, None, None),
        "sisa_attn_key_weights": lambda: lib.sisa_attn_key_weights(view(64), view(64), view(32), view(32), A, A, A, 3, 2, 200,
                                                                   0, BF16, A, None, None),
    }


def ends_at_the_look_up(call):
    rc = call()
    message = _lib.last_error()
    return rc != 0 and ("cudaPointerGetAttributes" in message or "not device memory" in message), (rc, message)


@pytest.mark.parametrize("name", ["sisa_paged_attn", "sisa_paged_evict", "sisa_paged_append", "sisa_paged_fill",
                                  "sisa_attn_key_weights"])
def test_paged_calls_bind_the_device_of_their_pages(name):
    ok, got = ends_at_the_look_up(paged_calls(_lib.load())[name])
    assert ok, got
