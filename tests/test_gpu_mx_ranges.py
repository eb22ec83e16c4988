"""Microscaled operators where a call is cut: products split over K, SwiGLU behind
them, captured ones, more rows than one launch takes, quotients past the range of
f32."""
import ctypes

import numpy as np
import pytest

import iris_testlib as tl
import mx_reference as mx
from mx_reference import FP4, FP8, Mat
from test_gpu_mx import EPI_BF16, EPI_F32, EPI_GATED_ADD, EPI_SWIGLU, WS, Product, done, kernels

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


@pytest.mark.parametrize("M,N,K,want", [(3, 70, 100000, "direct_kernel"), (40, 64, 100000, "rows_kernel"),
                                        (300, 192, 30000, "tile_kernel")])
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_GATED_ADD])
def test_long_sums(lib, ws, M, N, K, want, afmt, epi):
    """Ten times the longest row of a model, in ranges and in one; a range that ends inside a step."""
    p = Product(M, N, K, afmt, epi)
    names = " ".join(k for k, _ in kernels(lib, lambda: p.check(p.run(lib, ws.ptr))))
    assert want in names and "mx_reduce_kernel" in names, names
    p.check(p.run(lib, None, 0))
    p.close()


@pytest.mark.parametrize("M,N,K,epi,mx_fmt,launches", [(37, 320, 9728, EPI_SWIGLU, FP8, 2), (64, 320, 9000, EPI_GATED_ADD, None, 2),
                                                       (4400, 4160, 2000, EPI_BF16, None, 2)])
def test_captured(lib, ws, M, N, K, epi, mx_fmt, launches):
    """A product of several launches in a graph, replayed with eager products
    that use the same workspace between: the eager bits each time."""
    p = Product(M, N, K, FP8, epi, mx_fmt=mx_fmt)
    x0 = tl.to_bf16(p.x0) if p.bf16 else p.x0
    m = Mat(mx_fmt, M, p.nout) if mx_fmt is not None else None
    o = None if m else tl.Dev.of(x0)
    g = p.args(o.ptr if o else None, m)

    def put():
        if m:
            m.q.put(np.full(m.shape_q, 0xA5, np.uint8))
            m.s.put(np.full(m.shape_s, 0xA5, np.uint8))
        else:
            o.put(x0)

    def get():
        assert lib.iris_hip_sync() == 0
        return m.get() if m else (o.get(x0.dtype, x0.shape),)
    names = kernels(lib, lambda: done(lib, lib.iris_hip_mx_gemm(ctypes.byref(g), ws.ptr, WS)))
    assert sum(("mx_" in k) for k, _ in names) >= launches, names
    want = get()
    lib.iris_hip_graph_end.restype = ctypes.c_void_p
    lib.iris_hip_graph_launch.argtypes = lib.iris_hip_graph_destroy.argtypes = [ctypes.c_void_p]
    assert lib.iris_hip_graph_begin() == 0
    rc = lib.iris_hip_mx_gemm(ctypes.byref(g), ws.ptr, WS)
    graph = lib.iris_hip_graph_end()
    assert rc == 0 and graph
    e = Product(64, 320, 9000, FP8, EPI_F32)
    for _ in range(4):
        put()
        e.check(e.run(lib, ws.ptr))
        assert lib.iris_hip_graph_launch(graph) == 0
        for a, b in zip(get(), want):
            assert np.array_equal(a, b)
    lib.iris_hip_graph_destroy(graph)
    for v in (p, e, m or o):
        v.close()


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
