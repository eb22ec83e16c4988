"""Microscaled matrices without a GPU: row strides, calls of no rows, and what
is refused before anything is launched."""
import ctypes
import os

import numpy as np
import pytest

import iris_testlib as tl
import mx_reference as mx

P = 1 << 20   # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return mx.bind(ctypes.CDLL(os.path.join(tl.ROOT, "iris.c_amd", "libiris_hip.so")))


def mat(fmt, cols, /, **kw):
    m = mx.Mx(P, P, mx.ld_codes(fmt, cols), mx.ld_scales(cols), fmt)
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def test_strides(lib):
    for cols in (1, 31, 32, 127, 128, 129, 512, 513, 2560, 3840, 9728):
        for fmt in (mx.FP8, mx.FP4):
            assert lib.iris_hip_mx_ld_codes(fmt, cols) == mx.ld_codes(fmt, cols)
        assert lib.iris_hip_mx_ld_scales(cols) == mx.ld_scales(cols)


def test_reference_formats():
    """The test's own tables: every e2m1 and e4m3 code is its own nearest code."""
    for fmt in (mx.FP8, mx.FP4):
        g = mx.GRID[fmt]
        x = np.zeros((len(g), 32))
        x[:, 0], x[:, 1] = mx.TOP[fmt], g
        code, s = mx.quantize(x, fmt)
        assert (code[:, 1] == np.arange(len(g))).all() and (s[:, 0] == 127).all()


BAD_MATS = [dict(q=None), dict(s=None), dict(q=P + 8), dict(s=P + 4), dict(ld_q=24), dict(ld_s=8), dict(ld_q=64),
            dict(ld_s=16), dict(fmt=2), dict(fmt=-1)]


@pytest.mark.parametrize("bad", BAD_MATS)
def test_bad_matrices(lib, bad):
    m = mat(mx.FP4, 1000, **bad)
    ok = mat(mx.FP8, 1000)
    assert lib.iris_hip_mx_quantize(ctypes.byref(m), P, 0, 1000, 4, 1000) < 0
    assert lib.iris_hip_mx_dequantize(P, 0, 1000, ctypes.byref(m), 4, 1000) < 0
    n = mx.MxNorm(P, 1000, None, 0, 0, None, None, 0, P, None, m, 4, 1000, 1e-6)
    assert lib.iris_hip_mx_rmsnorm(ctypes.byref(n)) < 0
    for a, w in ((m, mat(mx.FP4, 1000)), (ok, m)):
        g = mx.MxGemm(a, w, P, None, 4, 64, 1000, 64, 0, mx.Mx())
        assert lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0) < 0
    if "q" not in bad or bad["q"] is not None:
        g = mx.MxGemm(ok, mat(mx.FP4, 1000), None, None, 4, 2048, 1000, 0, 3, mat(mx.FP4, 1024, **bad))
        if bad.get("ld_s") != 16:      # wide enough for 1024 columns is 32
            assert lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0) < 0


def test_refusals(lib):
    m = mat(mx.FP8, 100)
    r = ctypes.byref(m)
    assert lib.iris_hip_mx_quantize(None, P, 0, 100, 4, 100) < 0
    assert lib.iris_hip_mx_quantize(r, None, 0, 100, 4, 100) < 0
    assert lib.iris_hip_mx_quantize(r, P, 0, 99, 4, 100) < 0
    assert b"stride" in lib.iris_hip_last_error()
    assert lib.iris_hip_mx_dequantize(None, 0, 100, r, 4, 100) < 0
    assert lib.iris_hip_mx_dequantize(P, 0, 100, None, 4, 100) < 0
    assert lib.iris_hip_mx_dequantize(P, 1, 99, r, 4, 100) < 0
    assert lib.iris_hip_mx_rmsnorm(None) < 0

    def norm(**kw):
        n = mx.MxNorm(P, 100, P, 100, 0, None, P, 100, P, None, m, 4, 100, 1e-6)
        for k, v in kw.items():
            setattr(n, k, v)
        return lib.iris_hip_mx_rmsnorm(ctypes.byref(n))
    for kw in (dict(x=None), dict(w=None), dict(x_out=None), dict(ldx=99), dict(ldd=99), dict(ldxo=99),
               dict(d=None, gate=P), dict(x_out=P, ldxo=104)):
        assert norm(**kw) < 0, kw

    def gemm(**kw):
        g = mx.MxGemm(m, mat(mx.FP4, 100), P, None, 4, 64, 100, 64, 0, mx.Mx())
        for k, v in kw.items():
            setattr(g, k, v)
        return lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0)
    for kw in (dict(W=m), dict(out=None), dict(K=0), dict(K=-1), dict(K=129), dict(ldo=63), dict(epi=4), dict(epi=6),
               dict(epi=-1), dict(epi=3, N=96), dict(epi=3, vec=P), dict(epi=3, ldo=31), dict(mx_out=mat(mx.FP8, 64)),
               dict(epi=3, N=32)):
        assert gemm(**kw) < 0, kw
    # sizes that would pass 32 bits within a kernel
    for kw in (dict(M=(1 << 30) + 1), dict(M=2 ** 31 - 1), dict(N=2 ** 31 - 1, ldo=2 ** 31 - 1)):
        assert gemm(**kw) < 0 and b"output" in lib.iris_hip_last_error(), kw
    assert lib.iris_hip_mx_gemm(None, None, 0) < 0


def test_nothing_to_do(lib):
    """No rows or columns: done, whatever the pointers."""
    m, g = mx.Mx(), mx.MxGemm()
    assert lib.iris_hip_mx_quantize(ctypes.byref(m), None, 0, 0, 0, 64) == 0
    assert lib.iris_hip_mx_quantize(ctypes.byref(m), None, 0, 0, 64, 0) == 0
    assert lib.iris_hip_mx_dequantize(None, 0, 0, ctypes.byref(m), 0, 64) == 0
    assert lib.iris_hip_mx_rmsnorm(ctypes.byref(mx.MxNorm())) == 0
    assert lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0) == 0
