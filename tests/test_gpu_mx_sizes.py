"""Products of microscaled rows at the ends of what a launch and 32-bit offsets reach."""
import ctypes

import numpy as np
import pytest

import iris_testlib as tl
import mx_reference as mx
from mx_reference import FP4, FP8, Mat
from test_gpu_mx import EPI_BF16, EPI_F32, EPI_SWIGLU, WS, Product, done, kernels

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return mx.bind(tl.hip())


@pytest.fixture(scope="module")
def ws():
    return tl.Dev(WS)


def put(lib, dev, at, x):
    assert lib.iris_hip_memcpy_h2d(dev.ptr + at, x.ctypes.data, x.nbytes) == 0


def test_many_columns(lib):
    """One row by 2^27 columns of W: 2^23 blocks. W is 2^20 rows over and over."""
    N, K, period = 1 << 27, 100, 1 << 20
    rng = np.random.default_rng(1)
    a = Mat.of(rng.standard_normal((1, K)), FP8)
    code, s = mx.quantize(rng.standard_normal((period, K)).astype(np.float32), FP4)
    q = np.ascontiguousarray(mx.pack(code, FP4))
    sc = np.zeros((period, 16), np.uint8)
    sc[:, :s.shape[1]] = s
    dq, ds, out = tl.Dev(N * 64), tl.Dev(N * 16), tl.Dev(N * 4)
    for i in range(0, N, period):
        put(lib, dq, i * 64, q)
        put(lib, ds, i * 16, sc)
    assert lib.iris_hip_sync() == 0
    g = mx.MxGemm(a.c, mx.Mx(dq.ptr, ds.ptr, 64, 16, FP4), out.ptr, None, 1, N, K, N, EPI_F32, mx.Mx())
    done(lib, lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0))
    got = out.get(np.float32, (N // period, period))
    want = mx.values(code, s, FP4, K) @ a.values[0]
    tol = K * 2.0 ** -24 * (np.abs(mx.values(code, s, FP4, K)) @ np.abs(a.values[0]))
    assert (np.abs(got[0] - want) <= tol).all()
    assert (got == got[0]).all()
    for d in (a, dq, ds, out):
        d.close()


class Far:
    """A matrix with its rows `ld` bytes of codes apart, in memory that ends with the last row's codes."""

    def __init__(self, lib, m, ld):
        rows, width = m.rows, mx.ld_codes(m.fmt, m.cols)
        q, _ = m.get()
        self.q = tl.Dev((rows - 1) * ld + width)
        for r in range(rows):
            put(lib, self.q, r * ld, np.ascontiguousarray(q[r, :width]))
        assert lib.iris_hip_sync() == 0
        self.c = mx.Mx(self.q.ptr, m.s.ptr, ld, m.ld_s, m.fmt)

    def close(self):
        self.q.close()


@pytest.mark.parametrize("ld,want", [((1 << 23) - 16, None), (1 << 23, "direct_kernel<AF, 1, 4>"),
                                     ((1 << 23) + 128, "direct_kernel<AF, 1, 4>")])
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("epi,mx_fmt", [(EPI_F32, None), (EPI_BF16, None), (EPI_SWIGLU, None), (EPI_SWIGLU, FP8),
                                        (EPI_SWIGLU, FP4)])
def test_rows_far_apart(lib, ws, ld, want, afmt, epi, mx_fmt):
    """The last stride of the 32-bit kernels and the first ones behind it, for A
    and for W, a few rows (M 5), some (40) and tiles (150): every output."""
    for M, which in ((5, "W"), (40, "A"), (40, "W"), (150, "A"), (150, "W")):
        p = Product(M, 192, 200, afmt, epi, mx_fmt=mx_fmt)
        far = Far(lib, getattr(p, which), ld)
        keep = getattr(p, which).c
        getattr(p, which).c = far.c
        got = []
        names = kernels(lib, lambda: got.append(p.run(lib, ws.ptr)))
        flat = " ".join(k for k, _ in names)
        assert ("direct_kernel<AF, 1, 4>" in flat) == (want is not None), flat
        p.check(got[0])
        getattr(p, which).c = keep
        far.close()
        p.close()
