"""Microscaled operators where a call is cut: products with SwiGLU split over K,
more rows than one launch takes, quotients past the range of f32."""
import ctypes

import numpy as np
import pytest

import iris_testlib as tl
import mx_reference as mx
from mx_reference import FP4, FP8, Mat
from test_gpu_mx import EPI_SWIGLU, WS, Product, done, kernels

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return mx.bind(tl.hip())


@pytest.fixture(scope="module")
def ws():
    return tl.Dev(WS)


@pytest.mark.parametrize("M,N,K", [(5, 128, 20000), (37, 320, 9728), (300, 192, 9000)])
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("mx_fmt", [None, FP8, FP4])
def test_swiglu_of_split_products(lib, ws, M, N, K, afmt, mx_fmt):
    """The ranges' sums through SwiGLU into bf16 and microscaled rows, whose
    padding (64 of 128, 160 of 256, 96 of 128 columns) is written by lanes of its
    own; strides as narrow and wider than they have to be, and without a
    workspace, unsplit."""
    p = Product(M, N, K, afmt, EPI_SWIGLU, mx_fmt=mx_fmt)
    names = kernels(lib, lambda: p.check(p.run(lib, ws.ptr)))
    assert "mx_reduce_kernel" in " ".join(k for k, _ in names), names
    names = kernels(lib, lambda: p.check(p.run(lib, None, 0)))
    assert "mx_reduce_kernel" not in " ".join(k for k, _ in names), names
    if mx_fmt is not None:
        m = Mat(mx_fmt, M, p.nout, pad=2, more=1)
        done(lib, lib.iris_hip_mx_gemm(ctypes.byref(p.args(None, m)), ws.ptr, WS))
        p.check(m)
        q, s = m.get()
        assert (q[:, mx.ld_codes(mx_fmt, p.nout):] == 0xA5).all() and (s[:, mx.ld_scales(p.nout):] == 0xA5).all()
        m.close()
    p.close()


def test_quantize_of_many_rows(lib):
    """More rows than one launch counts lanes for (2^26 of one column)."""
    rows, period = (1 << 26) + 5, 1 << 20
    x = np.random.default_rng(2).standard_normal(period).astype(np.float32)
    dx, q, s = tl.Dev(rows * 4), tl.Dev(rows * 64), tl.Dev(rows * 16)
    for i in range(0, rows, period):
        n = min(period, rows - i)
        assert lib.iris_hip_memcpy_h2d(dx.ptr + i * 4, x.ctypes.data, n * 4) == 0
    m = mx.Mx(q.ptr, s.ptr, 64, 16, FP4)
    done(lib, lib.iris_hip_mx_quantize(ctypes.byref(m), dx.ptr, 0, 1, rows, 1))
    code, sc = mx.quantize(x[:, None], FP4)
    code = mx.pack(code, FP4)
    for at, n in ((0, 1000), (1 << 25, 1000), ((1 << 26) - 500, 505)):
        gq, gs = np.empty((n, 64), np.uint8), np.empty((n, 16), np.uint8)
        assert lib.iris_hip_memcpy_d2h(gq.ctypes.data, q.ptr + at * 64, gq.nbytes) == 0
        assert lib.iris_hip_memcpy_d2h(gs.ctypes.data, s.ptr + at * 16, gs.nbytes) == 0
        r = (at + np.arange(n)) % period
        assert np.array_equal(gq, code[r]) and np.array_equal(gs[:, :4], sc[r])
    for d in (dx, q, s):
        d.close()


@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_quotients_past_f32(lib, fmt):
    """A quotient past the range of f32 counts as its largest number."""
    cols = 320
    x = np.ones((2, cols), np.float32)
    x[0, 3], x[0, 40] = 1e6, -1e6
    w = np.full(cols, 3e38, np.float32)
    dx, dw = tl.Dev.of(x), tl.Dev.of(w)
    m = Mat(fmt, 2, cols)
    a = mx.MxNorm(dx.ptr, cols, None, 0, 0, None, None, 0, dw.ptr, None, m.c, 2, cols, 1e-6)
    done(lib, lib.iris_hip_mx_rmsnorm(ctypes.byref(a)))
    t = x.astype(np.float64)
    y = t / np.sqrt((t * t).mean(1, keepdims=True) + np.float64(np.float32(1e-6))) * w
    top = np.float64(np.finfo(np.float32).max)
    assert (np.abs(y) > top).any()
    code, s = mx.quantize(np.clip(y, -top, top), fmt)
    got, gs, _ = m.read()
    assert np.array_equal(got, code) and np.array_equal(gs, s)
    for d in (dx, dw, m):
        d.close()
