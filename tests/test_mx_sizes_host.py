"""Products of microscaled rows without a GPU: sizes of more threads than a launch takes."""
import ctypes
import os

import pytest

import iris_testlib as tl
import mx_reference as mx

P = 1 << 20   # a 16-byte aligned address that nothing reads


@pytest.mark.parametrize("M,N,K", [(1, 1 << 27, 4096), (16, 1 << 30, 1024), (1, 1 << 30, 10240), (1 << 30, 128, 64),
                                   (1 << 30, 1 << 30, 64)])
def test_past_a_launch(M, N, K):
    """Refused before anything is launched."""
    lib = mx.bind(ctypes.CDLL(os.path.join(tl.ROOT, "iris.c_amd", "libiris_hip.so")))
    a, w = (mx.Mx(P, P, mx.ld_codes(f, K), mx.ld_scales(K), f) for f in (mx.FP8, mx.FP4))
    g = mx.MxGemm(a, w, P, None, M, N, K, N, 0, mx.Mx())
    assert lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0) < 0
    assert b"threads" in lib.iris_hip_last_error()
