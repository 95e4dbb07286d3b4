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


def other_calls(lib):
    k, b = view(64), view(32)
    nf, nb = _lib.NormFwdArgs(), _lib.NormBwdArgs()
    for a in (nf, nb):
        for name, value in (("weight", A), ("rstd", A), ("rows", 4), ("d", 64)):
            setattr(a, name, value)
    nf.x, nf.x_ld, nf.x_dtype, nf.n_out, nf.eps = A, 64, BF16, 1, 1e-6
    nf.y[0], nf.y_ld[0], nf.y_dtype[0] = A, 64, BF16
    nb.v, nb.v_ld, nb.v_dtype, nb.dx, nb.dx_ld, nb.dx_dtype = A, 64, BF16, A, 64, BF16
    nb.dy[0], nb.dy_ld[0], nb.dy_dtype[0] = A, 64, BF16
    attn = (k, b, A, A, k, k, b, A, A, 200, A, 3, 2)
    prep = (A, 560, A, 2, 3, 2, BF16, k, k, b, A, A, 200)
    return {
        "sisa_prep_fwd": lambda: lib.sisa_prep_fwd(A, 3, 200, 2, 560 * 200, 560, BF16, A, 400, 2, A, A, A, A, None, None),
        "sisa_pack_positions": lambda: lib.sisa_pack_positions(A, 400, 200, 1, A, 400, 200, 1, 3, 2, 200, A, None, None),
        "sisa_prep_bwd": lambda: lib.sisa_prep_bwd(A, 3, 200, 2, 560 * 200, 560, BF16, A, 400, 2, A, A, A, A, A, A, 560 * 200, 560,
                                                   A, A, None, None),
        "sisa_decode_attn": lambda: lib.sisa_decode_attn(*attn, 200, BF16, k, A, None, None),
        "sisa_decode_attn_dpos": lambda: lib.sisa_decode_attn_dpos(*attn, A, 200, BF16, k, A, None, None),
        "sisa_decode_prep": lambda: lib.sisa_decode_prep(*prep, 7, A, A, A, A, None, None),
        "sisa_decode_prep_dpos": lambda: lib.sisa_decode_prep_dpos(*prep, A, 100, A, A, A, A, None, None),
        "sisa_lce_grad": lambda: lib.sisa_lce_grad(A, 128, 4, 100, 128, BF16, A, -100, A, 1.0, 1, A, A, None, None),
        "sisa_norm_fwd": lambda: lib.sisa_norm_fwd(_lib.vref(nf), None, None),
        "sisa_norm_bwd": lambda: lib.sisa_norm_bwd(_lib.vref(nb), None, None),
        "sisa_swiglu_fwd": lambda: lib.sisa_swiglu_fwd(A, 64, A, 64, 4, 64, BF16, A, 64, None, None),
        "sisa_swiglu_bwd": lambda: lib.sisa_swiglu_bwd(A, 64, A, 64, A, 64, 4, 64, BF16, A, 64, A, 64, None, None),
        "sisa_selftest_wait": lambda: lib.sisa_selftest_wait(1, 1000000, None, A, None),
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


@pytest.mark.parametrize("name", ["sisa_prep_fwd", "sisa_pack_positions", "sisa_prep_bwd", "sisa_decode_attn",
                                  "sisa_decode_attn_dpos", "sisa_decode_prep", "sisa_decode_prep_dpos", "sisa_lce_grad",
                                  "sisa_norm_fwd", "sisa_norm_bwd", "sisa_swiglu_fwd", "sisa_swiglu_bwd", "sisa_selftest_wait"])
def test_the_other_calls_bind_the_device_of_their_data(name):
    ok, got = ends_at_the_look_up(other_calls(_lib.load())[name])
    assert ok, got
