"""Microscaled quantisation, RMSNorm of an updated stream and products with
4-bit weights against their definitions in 64 bits.

Codes and scales are compared for equality. Tolerances of products: the
factors are exact in f32 and so are their products, a sum of K of them in f32
in any order is off by at most K 2^-24 sum |a w|, an epilogue adds a few
roundings of 2^-24 and an output type half a step (bf16 2^-8)."""
import ctypes

import numpy as np
import pytest

import iris_testlib as tl
import mx_reference as mx
from mx_reference import FP4, FP8, Mat

pytestmark = pytest.mark.gpu
EPI_F32, EPI_BF16, EPI_GATED_ADD, EPI_SWIGLU, _, EPI_ADD = range(6)
U = 2.0 ** -24
WS = 64 << 20


@pytest.fixture(scope="module")
def lib():
    return mx.bind(tl.hip())


@pytest.fixture(scope="module")
def ws():
    return tl.Dev(WS)


def done(lib, rc):
    assert rc == 0, lib.iris_hip_last_error()
    assert lib.iris_hip_sync() == 0


def rows_for(rows, cols, seed):
    """Blocks of very different sizes, zeros, ties of both formats, the ends of the range."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    b = -(-cols // 32)
    x *= np.repeat(np.exp2(rng.integers(-30, 30, (rows, b))), 32, 1)[:, :cols].astype(np.float32)
    ties = rng.random((rows, cols)) < 0.3
    x[ties] = (rng.integers(-64, 65, ties.sum()) / 8.0 * np.exp2(rng.integers(-4, 5, ties.sum()))).astype(np.float32)
    for r in range(rows):
        k = rng.integers(0, b) * 32
        x[r, k:k + 32] = [0.0, -0.0, 1e-40, 3.4e38, 1e-38, 2.0 ** -127, -1e-45][(r + seed) % 7]
        if (r + seed) % 11 == 0:
            x[r, min(cols - 1, k + 5)] = [np.inf, -np.inf, np.nan][r % 3]
    return x


# ---------------------------------------------------------------- quantisation

SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 127), (2, 128), (17, 129), (3, 512), (2, 1000), (300, 257), (7, 2560),
          (1, 9728)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("bf16", [0, 1])
def test_quantize(lib, rows, cols, fmt, bf16):
    """Every byte: codes, scales, their padding; the bytes behind them and the
    rows behind the last stay. Aligned rows, and rows that start anywhere."""
    x = rows_for(rows, cols, rows + cols)
    if bf16:
        x = tl.bf16_to_f32(tl.to_bf16(x))
    code, s = mx.quantize(x, fmt)
    p = mx.pack(code, fmt)
    for more, off, pad in ((0, 0, 0), (3, 1, 1)):
        flat = np.zeros(off + rows * (cols + more), np.float32)
        flat[off:].reshape(rows, -1)[:, :cols] = x
        flat[off:].reshape(rows, -1)[:, cols:] = 77.0
        d = tl.Dev.of(tl.to_bf16(flat) if bf16 else flat)
        m = Mat(fmt, rows, cols, pad, more=2)
        done(lib, lib.iris_hip_mx_quantize(ctypes.byref(m.c), d.ptr + off * (2 if bf16 else 4), bf16, cols + more, rows,
                                           cols))
        q, sc = m.get()
        assert np.array_equal(q[:rows, :p.shape[1]], p)
        assert np.array_equal(sc[:rows, :s.shape[1]], s)
        assert (q[rows:] == 0xA5).all() and (sc[rows:] == 0xA5).all()
        assert (q[:, p.shape[1]:] == 0xA5).all() and (sc[:, s.shape[1]:] == 0xA5).all()
        d.close()
        m.close()


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("bf16", [0, 1])
def test_dequantize(lib, fmt, bf16):
    """Every code under scales from the smallest to NaN, odd widths and strides."""
    n = 256 if fmt == FP8 else 16
    for cols in (n, n - 3, 1):
        code = np.zeros((8, 256), np.uint8)
        code[:, :cols] = np.arange(cols) % n
        s = np.broadcast_to(np.array([0, 1, 2, 100, 127, 200, 254, 255], np.uint8)[:, None], (8, 8))
        m = Mat(fmt, 8, 256)
        m.q.put(mx.pack(code, fmt))
        sc = np.zeros(m.shape_s, np.uint8)
        sc[:, :8] = s
        m.s.put(sc)
        with np.errstate(over="ignore"):
            want = mx.values(code, s, fmt, cols).astype(np.float32)
        for ldy in (cols, cols + 5):
            y = tl.Dev.of(np.full((8, ldy), 0x4141, np.uint16) if bf16 else np.full((8, ldy), 7.0, np.float32))
            done(lib, lib.iris_hip_mx_dequantize(y.ptr, bf16, ldy, ctypes.byref(m.c), 8, cols))
            got = y.get(np.uint16 if bf16 else np.float32, (8, ldy))
            assert (got[:, cols:] == (0x4141 if bf16 else 7.0)).all()
            got = tl.bf16_to_f32(got[:, :cols]) if bf16 else got[:, :cols]
            ref = np.where(np.isnan(want), want, tl.bf16_to_f32(tl.to_bf16(want))) if bf16 else want
            assert np.array_equal(got, ref, equal_nan=True)
            y.close()
        m.close()


def test_offsets_past_32_bits(lib):
    """Rows 2.4 GB apart: the third row's offset passes 2^32 bytes and 2^31 elements."""
    ld, cols = 1 << 30, 200
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, cols)).astype(np.float32)
    big = tl.Dev(2 * ld * 4 + cols * 4)
    for r in range(3):
        assert lib.iris_hip_memcpy_h2d(big.ptr + r * ld * 4, x[r].ctypes.data, cols * 4) == 0
    m = Mat(FP4, 3, cols)
    done(lib, lib.iris_hip_mx_quantize(ctypes.byref(m.c), big.ptr, 0, ld, 3, cols))
    code, s = mx.quantize(x, FP4)
    got, sc, v = m.read()
    assert np.array_equal(got, code) and np.array_equal(sc, s)
    # the same rows as a product's operand, 2 GiB - 128 bytes apart
    lq = (1 << 31) - 128
    q, _ = m.get()
    for r in range(3):
        assert lib.iris_hip_memcpy_h2d(big.ptr + r * lq, q[r].ctypes.data, q.shape[1]) == 0
    w = rng.standard_normal((70, cols)).astype(np.float32)
    wm = Mat.of(w, FP4)
    out = tl.Dev(3 * 70 * 4)
    for a, b, M, N in ((mx.Mx(big.ptr, m.s.ptr, lq, m.ld_s, FP4), wm.c, 3, 70),
                       (wm.c, mx.Mx(big.ptr, m.s.ptr, lq, m.ld_s, FP4), 70, 3)):
        g = mx.MxGemm(a, b, out.ptr, None, M, N, cols, N, EPI_F32, mx.Mx())
        done(lib, lib.iris_hip_mx_gemm(ctypes.byref(g), None, 0))
        y = out.get(np.float32, (M, N))
        want = v @ wm.values.T if M == 3 else wm.values @ v.T
        assert tl.rel_l2(y, want) < 1e-6
    for d in (big, m, wm, out):
        d.close()


# ---------------------------------------------------------------- RMSNorm

def norm_reference(x, d, gate, w, scale, eps):
    t = x if d is None else (x.astype(np.float64) + (1.0 if gate is None else gate.astype(np.float64)) * d).astype(np.float32)
    y = t.astype(np.float64)
    y = y / np.sqrt((y * y).mean(1, keepdims=True) + np.float64(np.float32(eps))) * w
    return t, y if scale is None else y * scale


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (2, 128), (5, 2047), (37, 2048), (4, 2049), (2, 2560), (9, 3840),
                                       (2, 4104), (3, 8192), (2, 8193), (1, 20000), (4, 500), (4, 1000), (1100, 2100)])
@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("add", ["none", "f32", "bf16"])
def test_rmsnorm(lib, rows, cols, fmt, add):
    """Codes, scales and the updated stream bit for bit; aligned and unaligned
    rows, with and without gate and scale, into other rows and in place."""
    rng = np.random.default_rng(rows + cols + len(add))
    for more, with_gate, with_scale, in_place in ((0, False, False, False), (3, True, True, True)):
        ld = cols + more
        x = (rng.standard_normal((rows, ld)) * np.exp2(rng.integers(-3, 4, (rows, ld)))).astype(np.float32)
        x[-1] *= 1e-3 if rows > 1 else 1.0
        if rows > 2:
            x[1] = 0.0
        d = rng.standard_normal((rows, ld)).astype(np.float32)
        if add == "bf16":
            d = tl.bf16_to_f32(tl.to_bf16(d))
        if rows > 2:
            d[1] = 0.0      # a row of zeros stays one
        w, gate, scale = (rng.standard_normal(cols).astype(np.float32) + 1 for _ in range(3))
        use_gate = with_gate and add != "none"
        t, y = norm_reference(x[:, :cols], None if add == "none" else d[:, :cols], gate if use_gate else None, w,
                              scale if with_scale else None, 1e-6)
        code, s = mx.quantize(y, fmt)
        dx, dd = tl.Dev.of(x), tl.Dev.of(tl.to_bf16(d) if add == "bf16" else d)
        dw, dg, ds = (tl.Dev.of(v) for v in (w, gate, scale))
        o = dx if in_place else tl.Dev.of(np.full((rows, ld), 5.0, np.float32))
        m = Mat(fmt, rows, cols, more=1)
        a = mx.MxNorm(dx.ptr, ld, None if add == "none" else dd.ptr, ld, int(add == "bf16"), dg.ptr if use_gate else None,
                      o.ptr, ld, dw.ptr, ds.ptr if with_scale else None, m.c, rows, cols, 1e-6)
        done(lib, lib.iris_hip_mx_rmsnorm(ctypes.byref(a)))
        got = o.get(np.float32, (rows, ld))
        if add == "none":
            assert np.array_equal(got, x if in_place else np.full_like(x, 5.0))
        else:
            assert np.array_equal(got[:, :cols], t)
            assert np.array_equal(got[:, cols:], x[:, cols:] if in_place else np.full((rows, more), 5.0))
        gc, gs, _ = m.read()
        assert np.array_equal(gs, s)
        # a zero's sign is the sign of t w
        assert np.array_equal(gc, code)
        q, sc = m.get()
        assert (q[rows:] == 0xA5).all() and (sc[rows:] == 0xA5).all()
        for v in (dx, dd, dw, dg, ds, o, m):
            v.close()


def test_rmsnorm_of_millions_of_rows(lib):
    """More rows than one launch holds threads for."""
    rows, cols = (1 << 22) + 5, 3
    rng = np.random.default_rng(11)
    x, d = rng.standard_normal((rows, cols), np.float32), rng.standard_normal((rows, cols), np.float32)
    w = np.array([1.0, 2.0, -0.5], np.float32)
    dx, dd, dw, do = tl.Dev.of(x), tl.Dev.of(d), tl.Dev.of(w), tl.Dev(x.nbytes)
    m = Mat(FP4, rows, cols)
    a = mx.MxNorm(dx.ptr, cols, dd.ptr, cols, 0, None, do.ptr, cols, dw.ptr, None, m.c, rows, cols, 1e-6)
    done(lib, lib.iris_hip_mx_rmsnorm(ctypes.byref(a)))
    assert np.array_equal(do.get(np.float32, (rows, cols)), x + d)
    pick = np.r_[0:7, rows // 2:rows // 2 + 7, rows - 12:rows]
    _, y = norm_reference(x[pick], d[pick], None, w, None, 1e-6)
    code, s = mx.quantize(y, FP4)
    q, sc = m.get()
    assert np.array_equal(q[pick, 0] & 15, code[:, 0]) and np.array_equal(q[pick, 0] >> 4, code[:, 1])
    assert np.array_equal(q[pick, 1], code[:, 2]) and not q[pick, 2:64].any()
    assert np.array_equal(sc[pick, 0], s[:, 0])
    for v in (dx, dd, dw, do, m):
        v.close()


def test_rmsnorm_of_nan(lib):
    """A NaN in a row makes that row NaN and no other."""
    x = np.ones((3, 300), np.float32)
    x[1, 299] = np.nan
    dx, dw = tl.Dev.of(x), tl.Dev.of(np.ones(300, np.float32))
    m = Mat(FP8, 3, 300)
    a = mx.MxNorm(dx.ptr, 300, None, 0, 0, None, None, 0, dw.ptr, None, m.c, 3, 300, 1e-6)
    done(lib, lib.iris_hip_mx_rmsnorm(ctypes.byref(a)))
    _, s, v = m.read()
    assert np.isnan(v[1]).all() and np.isfinite(v[[0, 2]]).all()
    assert (s[1, :10] == 255).all() and (s[1, 10:] == 0).all()   # 10 blocks hold columns


# ---------------------------------------------------------------- products

class Product:
    """out = A W^T with seeded operands; run() on fresh output memory, check() against 64 bits."""

    def __init__(self, M, N, K, afmt, epi, pad=0, seed=0, mx_fmt=None):
        rng = np.random.default_rng(M * 7 + N + 3 * K + epi + seed)
        a = rng.standard_normal((M, K)) * np.exp2(rng.integers(-3, 4, (M, 1)))
        w = rng.standard_normal((N, K)) * 0.05 * np.exp2(rng.integers(-2, 3, (N, 1)))
        self.A, self.W = Mat.of(a, afmt, pad), Mat.of(w, FP4, pad)
        self.M, self.N, self.K, self.epi, self.mx_fmt = M, N, K, epi, mx_fmt
        self.nout = N // 2 if epi == EPI_SWIGLU else N
        self.ldo = self.nout + 3 * pad
        self.vec = rng.standard_normal(N).astype(np.float32)
        self.dvec = tl.Dev.of(self.vec)
        self.x0 = rng.standard_normal((M, self.ldo)).astype(np.float32)
        self.bf16 = epi in (EPI_BF16, EPI_SWIGLU)
        self.use_vec = epi != EPI_SWIGLU
        self.ab = np.abs(self.A.values) @ np.abs(self.W.values).T
        self.y = self.A.values @ self.W.values.T
        if afmt == FP8 and self.bf16:
            # e4m3 A with 16- or 8-bit outputs may be summed by the single instruction, which drops, in each
            # group of 8 columns, bits of a product below 2^-13 of the largest one's power of two
            g = lambda t: np.abs(np.pad(t, ((0, 0), (0, -t.shape[1] % 8)))).reshape(len(t), -1, 8).max(2)  # noqa: E731
            self.ab = self.ab + 8 * 2.0 ** -13 / (K * U) * (g(self.A.values) @ g(self.W.values).T)

    def args(self, out, m=None):
        return mx.MxGemm(self.A.c, self.W.c, out, self.dvec.ptr if self.use_vec else None, self.M, self.N, self.K,
                         self.ldo, self.epi, m.c if m else mx.Mx())

    def run(self, lib, ws, nbytes=WS):
        if self.mx_fmt is not None:
            m = Mat(self.mx_fmt, self.M, self.nout, more=1)
            done(lib, lib.iris_hip_mx_gemm(ctypes.byref(self.args(None, m)), ws, nbytes))
            return m
        o = tl.Dev.of(tl.to_bf16(self.x0) if self.bf16 else self.x0)
        done(lib, lib.iris_hip_mx_gemm(ctypes.byref(self.args(o.ptr)), ws, nbytes))
        r = o.get(np.uint16 if self.bf16 else np.float32, (self.M, self.ldo))
        o.close()
        return r

    def exact(self):
        """(values, how far f32 arithmetic may be off)"""
        y, e = self.y, self.K * U * self.ab
        if self.epi == EPI_SWIGLU:
            grp = lambda t: t.reshape(self.M, -1, 2, 32)  # noqa: E731
            g, u = grp(y)[:, :, 0], grp(y)[:, :, 1]
            eg, eu = grp(e)[:, :, 0], grp(e)[:, :, 1]
            s = g / (1 + np.exp(-g))
            # |silu'| <= 1.1; exp, the sum, the quotient and the product a few roundings each
            return (s * u).reshape(self.M, -1), (1.1 * eg * (np.abs(u) + eu) + np.abs(s) * eu + 8 * U * np.abs(s * u)).reshape(self.M, -1)
        v = self.vec.astype(np.float64) if self.use_vec else (1.0 if self.epi == EPI_GATED_ADD else 0.0)
        x0 = self.x0[:, :self.nout].astype(np.float64)
        if self.epi == EPI_GATED_ADD:
            r = x0 + v * y
            return r, np.abs(v) * e + 2 * U * (np.abs(v * y) + np.abs(r))
        if self.epi == EPI_ADD:
            r = x0 + v + y
            return r, e + 2 * U * (np.abs(y + v) + np.abs(r))
        return y + v, e + U * np.abs(y + v)

    def check(self, got):
        want, err = self.exact()
        if self.mx_fmt is not None:
            code, s, v = got.read()
            q, sc = got.get()
            assert (q[self.M:] == 0xA5).all() and (sc[self.M:] == 0xA5).all()
            nb = -(-self.nout // 32)
            assert (code[:, self.nout:] == 0).all() and (s[:, nb:] == 0).all()
            # the scale is that of a maximum within its error
            b, eb = np.abs(want).reshape(self.M, nb, 32), err.reshape(self.M, nb, 32)
            lo, hi = (b - eb).max(2), (b + eb).max(2)
            two = np.exp2(s[:, :nb].astype(np.float64) - 127 + mx.EMAX[self.mx_fmt])
            assert ((two <= hi) & (2 * two > lo)).all()
            two = np.repeat(np.exp2(s[:, :nb].astype(np.float64) - 127), 32, 1)
            half = {FP8: np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * two),
                    FP4: np.maximum(2.0 ** -2 * np.abs(want), 0.25 * two)}[self.mx_fmt]
            over = np.abs(want) - mx.TOP[self.mx_fmt] * two
            assert (np.abs(v - want) <= np.maximum(half, over) + 2 * err).all()
            return
        g = tl.bf16_to_f32(got) if self.bf16 else got
        fill = tl.bf16_to_f32(tl.to_bf16(self.x0)) if self.bf16 else self.x0
        assert np.array_equal(g[:, self.nout:], fill[:, self.nout:])
        tol = err + (2.0 ** -8 * np.abs(want) if self.bf16 else 0.0)
        assert (np.abs(g[:, :self.nout] - want) <= tol * (1 + 1e-6) + 1e-37).all()

    def close(self):
        for v in (self.A, self.W, self.dvec):
            v.close()


GEMMS = [(1, 1, 1), (1, 64, 32), (2, 65, 100), (1, 2560, 2560), (16, 128, 128), (17, 192, 129), (37, 320, 1000),
         (64, 16, 4096), (77, 448, 640), (128, 256, 512), (129, 257, 1056), (200, 130, 9728), (255, 512, 384),
         (300, 1344, 256), (513, 576, 2560)]


@pytest.mark.parametrize("M,N,K", GEMMS)
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_BF16, EPI_GATED_ADD, EPI_ADD])
def test_gemm(lib, ws, M, N, K, afmt, epi):
    """One row to several tiles, edges in every direction, K that ends inside a
    step, padded strides; with a workspace, with a small one and without."""
    for pad in (0, 1):
        p = Product(M, N, K, afmt, epi, pad)
        p.check(p.run(lib, ws.ptr))
        if pad == 0:
            p.check(p.run(lib, None, 0))
            p.check(p.run(lib, ws.ptr, 4 * M * N + 16))
        p.close()


@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (1, 19456, 256), (37, 320, 1000), (130, 448, 640), (300, 1344, 512)])
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("mx_fmt", [None, FP8, FP4])
def test_gemm_swiglu(lib, ws, M, N, K, afmt, mx_fmt):
    for pad in (0, 1):
        p = Product(M, N, K, afmt, EPI_SWIGLU, pad, mx_fmt=mx_fmt)
        p.check(p.run(lib, ws.ptr))
        p.check(p.run(lib, None, 0))
        p.close()


@pytest.mark.parametrize("epi", [EPI_F32, EPI_BF16, EPI_GATED_ADD, EPI_ADD])
def test_gemm_without_vec(lib, ws, epi):
    p = Product(37, 100, 300, FP8, epi)
    p.use_vec = False
    p.check(p.run(lib, ws.ptr))
    p.close()


@pytest.mark.parametrize("M,N,K", [(2113, 3905, 200), (2100, 4000, 1056), (2304, 3840, 512)])
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_BF16, EPI_GATED_ADD])
def test_gemm_large_tiles(lib, ws, M, N, K, afmt, epi):
    """More than half a round of 256 x 256 tiles, with part tiles and without."""
    p = Product(M, N, K, afmt, epi, pad=0 if M == 2304 else 1)
    p.check(p.run(lib, ws.ptr))
    p.close()


@pytest.mark.parametrize("M,N,K,epi", [(301, 1349, 640, EPI_BF16), (2113, 4005, 200, EPI_BF16), (301, 1344, 640, EPI_SWIGLU),
                                       (2113, 4032, 200, EPI_SWIGLU), (301, 1349, 640, EPI_F32), (40, 1349, 640, EPI_BF16)])
@pytest.mark.parametrize("afmt", [FP8, FP4])
def test_gemm_cut_tiles_with_aligned_rows(lib, ws, M, N, K, epi, afmt):
    """Rows and columns that end inside a tile, output rows on 16 bytes: the
    columns behind and the rows below stay as they were."""
    p = Product(M, N, K, afmt, epi, pad=N % 8 != 0)
    assert p.ldo % 8 == 0
    x0 = tl.to_bf16(p.x0) if p.bf16 else p.x0
    o = tl.Dev.of(np.concatenate([x0, np.full((300, p.ldo), 7, x0.dtype)]))
    done(lib, lib.iris_hip_mx_gemm(ctypes.byref(p.args(o.ptr)), ws.ptr, WS))
    got = o.get(x0.dtype, (M + 300, p.ldo))
    p.check(got[:M])
    assert (got[M:] == 7).all()
    o.close()
    p.close()


@pytest.mark.parametrize("M,N,K", [(2113, 4032, 200), (2304, 4096, 640)])
@pytest.mark.parametrize("afmt", [FP8, FP4])
@pytest.mark.parametrize("mx_fmt", [None, FP8, FP4])
def test_gemm_large_tiles_swiglu(lib, ws, M, N, K, afmt, mx_fmt):
    p = Product(M, N, K, afmt, EPI_SWIGLU, mx_fmt=mx_fmt)
    p.check(p.run(lib, ws.ptr))
    p.close()


@pytest.mark.parametrize("afmt,epi,mx_fmt", [(FP8, EPI_BF16, None), (FP4, EPI_F32, None), (FP8, EPI_SWIGLU, FP8),
                                             (FP4, EPI_SWIGLU, None)])
def test_gemm_rows_behind_whole_rounds(lib, ws, afmt, epi, mx_fmt):
    """More than 256 tiles of 256 x 256: whole rounds, and the rows behind them by themselves."""
    p = Product(4400, 4160, 2000, afmt, epi, pad=1, mx_fmt=mx_fmt)
    assert len(kernels(lib, lambda: p.check(p.run(lib, ws.ptr)))) >= 2
    p.close()


def kernels(lib, call):
    """The (kernel, blocks) pairs that a call launches."""
    lib.iris_hip_profile_read.argtypes = [ctypes.c_void_p, ctypes.c_int]
    assert lib.iris_hip_profile_enable(1) == 0
    call()
    rec = (tl.KernelTime * 64)()
    n = lib.iris_hip_profile_read(ctypes.byref(rec), 64)
    assert lib.iris_hip_profile_enable(0) == 0
    return [(r.kernel.decode(), r.grid) for r in rec[:n]]


@pytest.mark.parametrize("M,N,K,afmt,epi,want", [
    (1, 320, 1000, FP8, EPI_F32, "direct_kernel<AF, 1, 1>"), (16, 64, 5000, FP4, EPI_BF16, "direct_kernel<AF, 1, 1>"),
    (5, 128, 9000, FP8, EPI_SWIGLU, "rows_kernel<AF, FM, FN>"),
    (20, 320, 9000, FP4, EPI_F32, "rows_kernel<AF, FM, FN>"), (40, 320, 9000, FP8, EPI_BF16, "rows_kernel<AF, FM, FN>"),
    (64, 320, 9000, FP8, EPI_BF16, "rows_kernel<AF, FM, FN>"), (64, 320, 9000, FP8, EPI_BF16, "mx_reduce_kernel"),
    (500, 2000, 640, FP8, EPI_F32, "tile_kernel<0, 1, 128, 128>"), (500, 2000, 640, FP8, EPI_BF16, "tile_kernel<0, 0, 128, 128>"),
    (500, 2000, 640, FP4, EPI_F32, "tile_kernel<1, 0, 128, 128>"), (4096, 4096, 512, FP8, EPI_BF16, "tile_kernel<0, 0, 256, 256>"),
    (4096, 4096, 512, FP4, EPI_F32, "tile_kernel<1, 0, 256, 256>")])
def test_every_kernel_is_reached(lib, ws, M, N, K, afmt, epi, want):
    p = Product(M, N, K, afmt, epi)
    names = [k for k, _ in kernels(lib, lambda: p.check(p.run(lib, ws.ptr)))]
    flat = " ".join(names).replace("IRIS_MX_FP8", "0").replace("IRIS_MX_FP4", "1").replace("false", "0").replace("true", "1")
    assert want in flat, flat
    p.close()


@pytest.mark.parametrize("M,N,K", [(3, 70, 200), (300, 600, 640), (37, 512, 4096)])
@pytest.mark.parametrize("afmt", [FP8, FP4])
def test_gemm_nan_blocks(lib, ws, M, N, K, afmt):
    """A block of scale 255 makes its row of the output (A) or its column (W) NaN and nothing else."""
    p = Product(M, N, K, afmt, EPI_F32)
    for m, r in ((p.A, 2), (p.W, 65)):
        s = m.s.get(np.uint8, m.shape_s)
        s[r, K // 64] = 255
        m.s.put(s)
    got = p.run(lib, ws.ptr)
    nan = np.zeros((M, N), bool)
    nan[2], nan[:, 65] = True, True
    assert np.array_equal(np.isnan(got), nan)
    want, err = p.exact()
    assert (np.abs(got - want) <= err)[~nan].all()
    p.close()


def test_gemm_extreme_scales(lib, ws):
    """Scales at both ends: sums that overflow are infinite, tiny ones exact."""
    a, w = np.full((2, 64), 2.0 ** 126, np.float32), np.full((3, 64), 1.0, np.float32)
    a[1], w[1], w[2] = 2.0 ** -120, 2.0 ** 100, 2.0 ** -20
    A, W, o = Mat.of(a, FP8), Mat.of(w, FP4), tl.Dev(2 * 3 * 4)
    g = mx.MxGemm(A.c, W.c, o.ptr, None, 2, 3, 64, 3, EPI_F32, mx.Mx())
    done(lib, lib.iris_hip_mx_gemm(ctypes.byref(g), ws.ptr, WS))
    with np.errstate(over="ignore"):
        want = (A.values @ W.values.T).astype(np.float32)
    assert np.array_equal(o.get(np.float32, (2, 3)), want)


# ---------------------------------------------------------------- together

def test_chain_and_graph(lib, ws):
    """A feed-forward block as a model runs it: the norm of an updated stream,
    gate and up into microscaled rows, the down product added to the stream,
    the attention's rows quantised for another product. Eager against 64 bits
    from each stage's own codes; captured and replayed with eager work between
    the replays, the same bits each time."""
    M, h, inter = 45, 320, 704
    rng = np.random.default_rng(5)
    x = rng.standard_normal((M, h)).astype(np.float32)
    d = tl.bf16_to_f32(tl.to_bf16(rng.standard_normal((M, h)).astype(np.float32)))
    w = (1 + 0.1 * rng.standard_normal(h)).astype(np.float32)
    gu, dn = Mat.of(0.1 * rng.standard_normal((2 * inter, h)), FP4), Mat.of(0.1 * rng.standard_normal((h, inter)), FP4)
    dx, dd, dw = tl.Dev.of(x), tl.Dev.of(tl.to_bf16(d)), tl.Dev.of(w)
    xo, att = tl.Dev(M * h * 4), tl.Dev.of(tl.to_bf16(x))
    a1, a2, a3 = Mat(FP8, M, h), Mat(FP8, M, inter), Mat(FP4, M, h)
    out = tl.Dev(M * h * 4)
    n = mx.MxNorm(dx.ptr, h, dd.ptr, h, 1, None, xo.ptr, h, dw.ptr, None, a1.c, M, h, 1e-6)
    g1 = mx.MxGemm(a1.c, gu.c, None, None, M, 2 * inter, h, 0, EPI_SWIGLU, a2.c)
    g2 = mx.MxGemm(a2.c, dn.c, xo.ptr, None, M, h, inter, h, EPI_GATED_ADD, mx.Mx())
    g3 = mx.MxGemm(a3.c, gu.c, out.ptr, None, M, h, h, h, EPI_F32, mx.Mx())

    def block():
        assert lib.iris_hip_mx_rmsnorm(ctypes.byref(n)) == 0
        assert lib.iris_hip_mx_gemm(ctypes.byref(g1), ws.ptr, WS) == 0
        assert lib.iris_hip_mx_gemm(ctypes.byref(g2), ws.ptr, WS) == 0
        assert lib.iris_hip_mx_quantize(ctypes.byref(a3.c), att.ptr, 1, h, M, h) == 0
        assert lib.iris_hip_mx_gemm(ctypes.byref(g3), ws.ptr, WS) == 0

    def result():
        assert lib.iris_hip_sync() == 0
        return [xo.get(np.float32, (M, h)), out.get(np.float32, (M, h)), *a1.get(), *a2.get(), *a3.get()]

    block()
    first = result()
    t, y = norm_reference(x, d, None, w, None, 1e-6)
    code, _ = mx.quantize(y, FP8)
    assert np.array_equal(a1.read()[0], code)
    yy = (a1.read()[2] @ gu.values.T).reshape(M, -1, 2, 32)
    act = (yy[:, :, 0] / (1 + np.exp(-yy[:, :, 0])) * yy[:, :, 1]).reshape(M, -1)
    assert tl.rel_l2(a2.read()[2], act) < 2.0 ** -4
    want = t + a2.read()[2] @ dn.values.T
    assert np.abs(first[0] - want).max() <= inter * U * (np.abs(a2.read()[2]) @ np.abs(dn.values).T).max() + 4 * U * np.abs(want).max()
    assert tl.rel_l2(first[1], a3.read()[2] @ gu.values[:h].T) < 1e-6

    lib.iris_hip_graph_end.restype = ctypes.c_void_p
    lib.iris_hip_graph_launch.argtypes = lib.iris_hip_graph_destroy.argtypes = [ctypes.c_void_p]
    assert lib.iris_hip_graph_begin() == 0
    block()
    graph = lib.iris_hip_graph_end()
    assert graph
    for _ in range(3):
        for buf in (xo, out, a1.q, a2.q, a2.s, a3.q):
            buf.put(np.full(buf.n, 0xA5, np.uint8))
        p = Product(5, 64, 200, FP8, EPI_F32)     # eager work that uses the same workspace
        p.check(p.run(lib, ws.ptr))
        p.close()
        assert lib.iris_hip_graph_launch(graph) == 0
        for u, v in zip(result(), first):
            assert np.array_equal(u, v)
    lib.iris_hip_graph_destroy(graph)


def test_side_stream(lib, ws):
    """Two products beside each other, one on the side stream with a workspace of its own: the bits of one after the other."""
    p, q = Product(40, 640, 2560, FP8, EPI_F32), Product(33, 320, 2560, FP4, EPI_BF16)
    a, b = p.run(lib, ws.ptr), q.run(lib, ws.ptr)
    ws2 = tl.Dev(WS)
    oa, ob = tl.Dev.of(p.x0), tl.Dev.of(tl.to_bf16(q.x0))
    ga, gb = p.args(oa.ptr), q.args(ob.ptr)
    for _ in range(4):
        assert lib.iris_hip_fork() == 0
        lib.iris_hip_side(1)
        rc = lib.iris_hip_mx_gemm(ctypes.byref(ga), ws2.ptr, WS)
        lib.iris_hip_side(0)
        assert rc == 0 and lib.iris_hip_mx_gemm(ctypes.byref(gb), ws.ptr, WS) == 0 and lib.iris_hip_join() == 0
    assert lib.iris_hip_sync() == 0
    assert np.array_equal(oa.get(np.float32, a.shape), a) and np.array_equal(ob.get(np.uint16, b.shape), b)
