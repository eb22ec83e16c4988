"""Microscaled formats in 64 bits, from their definition (include/iris_hip.h),
and ctypes mirrors of the argument structures."""
import ctypes

import numpy as np

import iris_testlib as tl

FP8, FP4 = 0, 1
EMAX, TOP = {FP8: 8, FP4: 2}, {FP8: 448.0, FP4: 6.0}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
E4M3 = np.array([m / 512 for m in range(8)] + [2.0 ** e * (1 + m / 8) for e in range(-6, 9) for m in range(8)][:-1])
GRID = {FP8: E4M3, FP4: E2M1}

VP, I, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float


class Mx(ctypes.Structure):
    _fields_ = [("q", VP), ("s", VP), ("ld_q", I), ("ld_s", I), ("fmt", I)]


class MxNorm(ctypes.Structure):
    _fields_ = [("x", VP), ("ldx", I), ("d", VP), ("ldd", I), ("d_bf16", I), ("gate", VP), ("x_out", VP),
                ("ldxo", I), ("w", VP), ("scale", VP), ("out", Mx), ("rows", I), ("cols", I), ("eps", F)]


class MxGemm(ctypes.Structure):
    _fields_ = [("A", Mx), ("W", Mx), ("out", VP), ("vec", VP), ("M", I), ("N", I), ("K", I), ("ldo", I),
                ("epi", I), ("mx_out", Mx)]


def bind(lib):
    lib.iris_hip_mx_quantize.argtypes = [VP, VP, I, I, I, I]
    lib.iris_hip_mx_dequantize.argtypes = [VP, I, I, VP, I, I]
    lib.iris_hip_mx_rmsnorm.argtypes = [VP]
    lib.iris_hip_mx_gemm.argtypes = [VP, VP, ctypes.c_size_t]
    lib.iris_hip_last_error.restype = ctypes.c_char_p
    return lib


def ld_codes(fmt, cols):
    return -(-cols // 128) * 128 // (2 if fmt == FP4 else 1)


def ld_scales(cols):
    return -(-cols // 512) * 16


def blocks(x):
    """[rows][blocks][32], zero padded to whole 128 columns."""
    rows, cols = x.shape
    p = np.zeros((rows, -(-cols // 128) * 128), x.dtype)
    p[:, :cols] = x
    return p.reshape(rows, -1, 32)


def quantize(x, fmt):
    """(code of each element, scale bytes) over the padded columns."""
    b = blocks(np.asarray(x, np.float64))
    with np.errstate(invalid="ignore"):
        top = np.abs(b).max(2)
    bad = ~np.isfinite(b).all(2)
    top[bad] = 1.0
    _, e = np.frexp(top)
    s = np.where(top > 0, np.clip(e - 1 - EMAX[fmt], -127, None) + 127, 0)
    v = np.where(bad[:, :, None], 0.0, b) * np.exp2(127.0 - s)[:, :, None]
    a = np.minimum(np.abs(v), TOP[fmt])
    g = GRID[fmt]
    hi = np.minimum(np.searchsorted(g, a), len(g) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - g[lo], g[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = code | np.where(np.signbit(v), 8 if fmt == FP4 else 128, 0)
    return code.reshape(len(b), -1).astype(np.uint8), np.where(bad, 255, s).astype(np.uint8)


def pack(code, fmt):
    return code if fmt == FP8 else code[:, 0::2] | code[:, 1::2] << 4


def values(code, s, fmt, cols):
    """What codes (one per element) and scale bytes stand for."""
    mag, sign = (code & 7, code >> 3) if fmt == FP4 else (code & 127, code >> 7)
    g = GRID[fmt] if fmt == FP4 else np.append(E4M3, np.nan)
    v = g[mag] * (1.0 - 2.0 * sign)
    two = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127.0))
    return (v.reshape(len(v), -1, 32) * two[:, :v.shape[1] // 32, None]).reshape(len(v), -1)[:, :cols]


def unpack(q, fmt):
    return q if fmt == FP8 else np.stack([q & 15, q >> 4], 2).reshape(len(q), -1)


class Mat:
    """A microscaled matrix on the device, its strides wider than needed by
    pad 16-byte units, every byte at first `fill`, `more` rows behind the last."""

    def __init__(self, fmt, rows, cols, pad=0, fill=0xA5, more=0):
        self.fmt, self.rows, self.cols = fmt, rows, cols
        self.ld_q, self.ld_s = ld_codes(fmt, cols) + 16 * pad, ld_scales(cols) + 16 * pad
        self.shape_q, self.shape_s = (rows + more, self.ld_q), (rows + more, self.ld_s)
        self.q = tl.Dev.of(np.full(self.shape_q, fill, np.uint8))
        self.s = tl.Dev.of(np.full(self.shape_s, fill, np.uint8))
        self.c = Mx(self.q.ptr, self.s.ptr, self.ld_q, self.ld_s, fmt)

    @classmethod
    def of(cls, x, fmt, pad=0):
        """x quantised by the reference."""
        code, s = quantize(x, fmt)
        m = cls(fmt, x.shape[0], x.shape[1], pad)
        q0, s0 = np.full(m.shape_q, 0xA5, np.uint8), np.full(m.shape_s, 0xA5, np.uint8)
        p = pack(code, fmt)
        q0[:, :p.shape[1]], s0[:, :s.shape[1]] = p, s
        m.q.put(q0)
        m.s.put(s0)
        m.values = values(code, s, fmt, x.shape[1])
        return m

    def get(self):
        """All bytes of codes and scales."""
        return self.q.get(np.uint8, self.shape_q), self.s.get(np.uint8, self.shape_s)

    def read(self):
        """(code of each element, scale bytes) over the padded columns, and the values."""
        q, s = self.get()
        code = unpack(q[:self.rows, :ld_codes(self.fmt, self.cols)], self.fmt)
        s = s[:self.rows, :code.shape[1] // 32]
        return code, s, values(code, s, self.fmt, self.cols)

    def close(self):
        self.q.close()
        self.s.close()
