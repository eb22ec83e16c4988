"""Microscaled operators of this library, measured through its C entry points
(include/iris_hip.h): rows quantised to 4- and 8-bit codes with one power of
two per 32 columns, RMSNorm of an updated residual stream with such an output,
and the products of such activations with 4-bit weights, the text encoder's
and the denoisers' linears.

The format (OCP microscaling): a block of 32 columns of a row shares the scale
2^(s - 127) in one byte s, with s - 127 = max(floor(log2 max|x|) - emax, -127),
emax 2 for e2m1 (4 bits: 0 .5 1 1.5 2 3 4 6) and 8 for e4m3 (8 bits, up to
448); a code is x / scale rounded to the nearest value, ties to even, clamped.
Codes are row-major, e2m1 two to a byte with the even column in the low
nibble, rows zero padded to 128 columns; scales are row-major, rows padded to
16 bytes, a block of zeros has scale byte 0.

listed() names the cases, draw() draws more of the same ranges, prepare()
makes what a program has in hand, run() is one pass, exact() its results in 64
bits.
"""
import ctypes
import functools
import math
import os

import torch

own = False

HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FP8, FP4 = 0, 1                       # IRIS_MX_FP8, IRIS_MX_FP4
EPI = {"f32": 0, "bf16": 1, "swiglu": 3, "swiglu_mx": 3}
EMAX, TOP = {FP8: 8, FP4: 2}, {FP8: 448.0, FP4: 6.0}
FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
WS_BYTES = 64 << 20


# ------------------------------------------------------------------ the cases

def _quant(fmt, bf16, rows, cols):
    return {"kind": "quant", "fmt": fmt, "bf16": bf16, "rows": rows, "cols": cols}


def _norm(fmt, rows, cols, add, gate=False):
    return {"kind": "norm", "fmt": fmt, "rows": rows, "cols": cols, "add": add, "gate": gate}


def _gemm(afmt, epi, m, n, k):
    return {"kind": "gemm", "afmt": afmt, "epi": epi, "m": m, "n": n, "k": k}


def listed():
    return [
        # a text encoder's gate and up weights taken to 4 bits as the model is loaded, and read back
        dict(_quant(FP4, True, 19456, 2560), name="quant_weights_fp4"),
        # the attention output of a padded prompt before its output projection
        dict(_quant(FP8, True, 512, 4096), name="quant_rows_fp8"),
        # f32 caption features of an odd length
        dict(_quant(FP4, False, 203, 2560), name="quant_caption_fp4"),
        # one token's residual stream after a projection: latency
        dict(_norm(FP8, 1, 2560, "bf16"), name="norm_token"),
        # the text encoder's stream of a padded prompt
        dict(_norm(FP8, 512, 2560, "f32"), name="norm_prompt"),
        # a denoiser's stream of a 1024 x 1024 image and its caption, gated
        dict(_norm(FP8, 4608, 3840, "bf16", True), name="norm_image"),
        # one token through the Q, K and V projection: weights at memory rate
        dict(_gemm(FP8, "bf16", 1, 6144, 2560), name="gemm_token_qkv"),
        # a short prompt through gate and up, the product's rows microscaled for the next product
        dict(_gemm(FP8, "swiglu_mx", 37, 19456, 2560), name="gemm_prompt_gate_up"),
        # a padded prompt through the down projection: few tiles, a long sum
        dict(_gemm(FP8, "f32", 512, 2560, 9728), name="gemm_prompt_down"),
        # 4-bit activations of a 512 x 512 image's stream, an odd caption beside it
        dict(_gemm(FP4, "bf16", 1227, 11520, 3840), name="gemm_image_qkv_fp4"),
        # gate and up of a 1024 x 1024 image, 8-bit activations
        dict(_gemm(FP8, "swiglu", 4608, 20480, 3840), name="gemm_image_gate_up"),
        # and with 4-bit activations, its down projection
        dict(_gemm(FP4, "bf16", 4608, 3840, 10240), name="gemm_image_down_fp4"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "norm", "gemm", "gemm"])
    if kind == "quant":
        rows, cols = _between(rng, 1, 20000), _between(rng, 32, 10240)
        rows = min(rows, max(1, 19456 * 2560 // cols))
        return _quant(rng.choice([FP8, FP4]), rng.random() < 0.5, rows, cols)
    if kind == "norm":
        rows, cols = _between(rng, 1, 8192), _between(rng, 64, 10240)
        rows = min(rows, max(1, 4608 * 3840 // cols))
        return _norm(rng.choice([FP8, FP8, FP4]), rows, cols, rng.choice(["bf16", "f32", "none"]), rng.random() < 0.5)
    epi = rng.choice(["f32", "bf16", "swiglu", "swiglu_mx"])
    m, n, k = _between(rng, 1, 4608), _between(rng, 64, 20480), _between(rng, 64, 10240)
    if epi.startswith("swiglu"):
        n = (n + 63) // 64 * 64
    m = min(m, max(1, 4608 * 20480 * 3840 // (n * k)))
    return _gemm(rng.choice([FP8, FP4]), epi, m, n, k)


def _mx_bytes(fmt, rows, cols):
    """Codes and scales of a matrix, without padding."""
    return rows * ((cols if fmt == FP8 else (cols + 1) // 2) + (cols + 31) // 32)


def work(c):
    """Each input read once, each output written once; a product's 2 M N K, a few operations an element elsewhere."""
    if c["kind"] == "quant":
        n = c["rows"] * c["cols"]
        # read, codes written and read, values written
        return {"bytes": n * (2 if c["bf16"] else 4) + 2 * _mx_bytes(c["fmt"], c["rows"], c["cols"]) + 2 * n, "flops": 4 * n}
    if c["kind"] == "norm":
        n, add = c["rows"] * c["cols"], {"bf16": 2, "f32": 4, "none": 0}[c["add"]]
        b = n * (4 + add + (4 if add else 0)) + _mx_bytes(c["fmt"], c["rows"], c["cols"]) + 4 * c["cols"]
        if c["fmt"] == FP4:
            b += _mx_bytes(FP4, c["rows"], c["cols"]) + 2 * n
        return {"bytes": b, "flops": 8 * n}
    m, n, k = c["m"], c["n"], c["k"]
    out = {"f32": 4 * m * n, "bf16": 2 * m * n, "swiglu": m * n, "swiglu_mx": _mx_bytes(FP8, m, n // 2)}[c["epi"]]
    return {"bytes": _mx_bytes(c["afmt"], m, k) + _mx_bytes(FP4, n, k) + out, "flops": 2 * m * n * k}


# ------------------------------------------------------------ the plain forms

def _pad(x, to):
    """Columns zero padded to a multiple of `to`."""
    more = -x.shape[1] % to
    return x if not more else torch.cat([x, x.new_zeros(x.shape[0], more)], 1)


def _scale_bytes(x, fmt):
    """The scale byte of each block of 32 columns."""
    top = _pad(x, 32).view(x.shape[0], -1, 32).abs().amax(2).double()
    _, e = torch.frexp(top)                        # top = m 2^e, m in [1/2, 1)
    s = (e - 1 - EMAX[fmt] + 127).clamp(0, 254)
    return torch.where(top > 0, s, torch.zeros_like(s)).to(torch.uint8)


def _quantized(x, fmt):
    """(code values, scale bytes) of the rows of x, code values in x's type."""
    s = _scale_bytes(x, fmt)
    two = torch.exp2(127.0 - s.double()).to(torch.float64)
    v = _pad(x, 32).view(x.shape[0], -1, 32).double() * two[:, :, None]
    v = v.clamp(-TOP[fmt], TOP[fmt])
    # the step between neighbouring codes around v: its power of two, over 2 (e2m1) or 8 (e4m3)
    _, e = torch.frexp(v)
    bits, least = (1, 0) if fmt == FP4 else (3, -6)
    step = torch.exp2(((e - 1).clamp(min=least) - bits).double())
    v = torch.round(v / step) * step               # ties to even
    return v.view(x.shape[0], -1)[:, :x.shape[1]], s


def _dequantized(v, s):
    """Code values times their blocks' scales."""
    two = torch.exp2(s.double() - 127.0).repeat_interleave(32, 1)[:, :v.shape[1]]
    return v.double() * two


def _fp4_codes(v):
    """e2m1 codes, two to a byte, rows padded to 128 columns."""
    a = _pad(v, 128).abs()
    code = sum((a >= t).to(torch.uint8) for t in FP4_VALUES[1:])
    code = code + torch.where(torch.signbit(_pad(v, 128)), 8, 0).to(torch.uint8)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()


def _codes(x, fmt):
    """(codes, scales) as the library lays them out."""
    v, s = _quantized(x, fmt)
    q = _fp4_codes(v) if fmt == FP4 else _pad(v.float(), 128).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.contiguous(), _pad(s, 16).contiguous()


def _values(q, s, fmt, cols):
    """What codes and scales stand for, f32."""
    if fmt == FP8:
        v = q.view(torch.float8_e4m3fn).to(torch.float32)
    else:
        table = torch.tensor(FP4_VALUES + tuple(-v for v in FP4_VALUES), device=q.device)
        v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], 2).view(q.shape[0], -1)
    blocks = (cols + 31) // 32
    two = torch.exp2(s[:, :blocks].float() - 127.0)
    return (_pad(v[:, :cols], 32).view(q.shape[0], blocks, 32) * two[:, :, None]).view(q.shape[0], -1)[:, :cols]


def _swiglu(y):
    """silu(gate) * up of 32-column gate and up groups."""
    y = y.view(y.shape[0], -1, 2, 32)
    g, u = y[:, :, 0], y[:, :, 1]
    return (g / (1 + torch.exp(-g)) * u).reshape(y.shape[0], -1)


def _plain(s):
    c = s["case"]
    if c["kind"] == "quant":
        return _dequantized(*_quantized(s["x"].float(), c["fmt"])).to(torch.bfloat16)
    if c["kind"] == "norm":
        x = s["x"]
        if c["add"] != "none":
            d = s["d"].double()
            x = (x.double() + (d * s["gate"].double() if c["gate"] else d)).float()
        # a value next to the border of two codes: 64 bits
        t = x.double()
        y = t / torch.sqrt(t.square().mean(1, keepdim=True) + EPS) * s["w"].double()
        v, sc = _quantized(y, c["fmt"])
        if c["fmt"] == FP4:
            out = {"y": _dequantized(v, sc).to(torch.bfloat16)}
        else:
            out = {"q": v.float().to(torch.float8_e4m3fn), "s": sc.view(torch.float8_e8m0fnu)}
        return out if c["add"] == "none" else dict(out, x=x)
    y = torch.matmul(_values(s["aq"], s["as"], c["afmt"], c["k"]), _values(s["wq"], s["ws"], FP4, c["k"]).t())
    if c["epi"] == "f32":
        return y + s["bias"]
    if c["epi"] == "bf16":
        return (y + s["bias"]).to(torch.bfloat16)
    y = _swiglu(y)
    if c["epi"] == "swiglu":
        return y.to(torch.bfloat16)
    v, sc = _quantized(y, FP8)
    return {"q": v.float().to(torch.float8_e4m3fn), "s": sc.view(torch.float8_e8m0fnu)}


# ------------------------------------------------------------ library calls

VP, I, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float


class _Mx(ctypes.Structure):          # iris_mx_t
    _fields_ = [("q", VP), ("s", VP), ("ld_q", I), ("ld_s", I), ("fmt", I)]


class _MxNorm(ctypes.Structure):      # iris_mx_norm_t
    _fields_ = [("x", VP), ("ldx", I), ("d", VP), ("ldd", I), ("d_bf16", I), ("gate", VP), ("x_out", VP),
                ("ldxo", I), ("w", VP), ("scale", VP), ("out", _Mx), ("rows", I), ("cols", I), ("eps", F)]


class _MxGemm(ctypes.Structure):      # iris_mx_gemm_t
    _fields_ = [("A", _Mx), ("W", _Mx), ("out", VP), ("vec", VP), ("M", I), ("N", I), ("K", I), ("ldo", I),
                ("epi", I), ("mx_out", _Mx)]


@functools.lru_cache(maxsize=1)
def _lib():
    torch.cuda.init()                 # one HIP runtime in the process: torch's
    lib = ctypes.CDLL(os.path.join(HERE, "iris.c_amd", "libiris_hip.so"))
    lib.iris_hip_last_error.restype = ctypes.c_char_p
    lib.iris_hip_mx_quantize.argtypes = [VP, VP, I, I, I, I]
    lib.iris_hip_mx_dequantize.argtypes = [VP, I, I, VP, I, I]
    lib.iris_hip_mx_rmsnorm.argtypes = [VP]
    lib.iris_hip_mx_gemm.argtypes = [VP, VP, ctypes.c_size_t]
    if lib.iris_hip_init(0):
        raise RuntimeError("iris: %s" % lib.iris_hip_last_error().decode())
    return lib


def _ok(rc):
    if rc:
        raise RuntimeError("iris: %s" % _lib().iris_hip_last_error().decode())


def _mx(q, s, fmt):
    return _Mx(q.data_ptr(), s.data_ptr(), q.shape[1], s.shape[1], fmt)


def _calls(s):
    """The argument structures of this state's buffers, as a program keeps them."""
    c = s["case"]
    if c["kind"] == "quant":
        return _mx(s["q"], s["s"], c["fmt"])
    if c["kind"] == "norm":
        add, cols = c["add"] != "none", c["cols"]
        return _MxNorm(s["x"].data_ptr(), cols, s["d"].data_ptr() if add else None, cols, int(c["add"] == "bf16"),
                       s["gate"].data_ptr() if add and c["gate"] else None, s["x_out"].data_ptr() if add else None, cols,
                       s["w"].data_ptr(), None, _mx(s["q"], s["s"], c["fmt"]), c["rows"], cols, EPS)
    mx = c["epi"] == "swiglu_mx"
    return _MxGemm(_mx(s["aq"], s["as"], c["afmt"]), _mx(s["wq"], s["ws"], FP4), None if mx else s["out"].data_ptr(),
                   s["bias"].data_ptr() if c["epi"] in ("f32", "bf16") else None, c["m"], c["n"], c["k"],
                   0 if mx else s["out"].shape[1], EPI[c["epi"]], _mx(s["q"], s["s"], FP8) if mx else _Mx())


def _own(s):
    lib, c = _lib(), s["case"]
    if "call" not in s:
        s["call"] = _calls(s)
    call = ctypes.byref(s["call"])
    if c["kind"] == "quant":
        _ok(lib.iris_hip_mx_quantize(call, s["x"].data_ptr(), int(c["bf16"]), c["cols"], c["rows"], c["cols"]) or
            lib.iris_hip_mx_dequantize(s["y"].data_ptr(), 1, c["cols"], call, c["rows"], c["cols"]))
        return s["y"]
    if c["kind"] == "norm":
        _ok(lib.iris_hip_mx_rmsnorm(call))
        if c["fmt"] == FP4:
            _ok(lib.iris_hip_mx_dequantize(s["y"].data_ptr(), 1, c["cols"], ctypes.byref(s["call"].out), c["rows"],
                                           c["cols"]))
        return s["result"]
    _ok(lib.iris_hip_mx_gemm(call, s["work"].data_ptr(), WS_BYTES))
    return s["result"]


# ------------------------------------------------------------ inputs, one pass

def _stream(g, rows, cols):
    """Rows of a residual stream: a few columns far larger than the rest, as language models have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    big = torch.randint(0, cols, (max(1, cols // 512),), generator=g, device="cuda")
    x[:, big] *= 24.0
    return x * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))


def _inputs(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if c["kind"] == "quant":
        x = _stream(g, c["rows"], c["cols"])
        if c["rows"] > 64:                         # padding: rows of zeros
            x[-(c["rows"] // 16):] = 0.0
        return {"x": x.to(torch.bfloat16) if c["bf16"] else x}
    if c["kind"] == "norm":
        s = {"x": _stream(g, c["rows"], c["cols"]), "w": 1 + 0.1 * torch.randn(c["cols"], generator=g, device="cuda")}
        if c["add"] != "none":
            d = 0.3 * torch.randn(c["rows"], c["cols"], generator=g, device="cuda")
            s["d"] = d.to(torch.bfloat16) if c["add"] == "bf16" else d
            s["gate"] = torch.tanh(torch.randn(c["cols"], generator=g, device="cuda"))
        return s
    s = {"bias": 0.1 * torch.randn(c["n"], generator=g, device="cuda")}
    s["aq"], s["as"] = _codes(_stream(g, c["m"], c["k"]), c["afmt"])
    s["wq"], s["ws"] = _codes(0.02 * torch.randn(c["n"], c["k"], generator=g, device="cuda"), FP4)
    return s


def _room(fmt, rows, cols):
    """Empty codes and scales of a matrix."""
    ld = -(-cols // 128) * 128 // (2 if fmt == FP4 else 1)
    return (torch.empty(rows, ld, dtype=torch.uint8, device="cuda"),
            torch.empty(rows, -(-cols // 512) * 16, dtype=torch.uint8, device="cuda"))


def _seen(q, s, cols):
    """The values of 8-bit codes and of their scales, in place."""
    return {"q": q.view(torch.float8_e4m3fn)[:, :cols], "s": s.view(torch.float8_e8m0fnu)[:, :(cols + 31) // 32]}


def prepare(c, seed):
    s = dict(_inputs(c, seed), case=c)
    if c["kind"] == "gemm":
        m, n = c["m"], c["n"]
        s["work"] = torch.empty(WS_BYTES, dtype=torch.uint8, device="cuda")
        if c["epi"] == "swiglu_mx":
            s["q"], s["s"] = _room(FP8, m, n // 2)
            s["result"] = _seen(s["q"], s["s"], n // 2)
        else:
            s["out"] = torch.empty(m, n // 2 if c["epi"] == "swiglu" else n, device="cuda",
                                   dtype=torch.float32 if c["epi"] == "f32" else torch.bfloat16)
            s["result"] = s["out"]
    else:
        rows, cols = c["rows"], c["cols"]
        s["q"], s["s"] = _room(c["fmt"], rows, cols)
        s["y"] = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
        if c["kind"] == "norm":
            s["result"] = _seen(s["q"], s["s"], cols) if c["fmt"] == FP8 else {"y": s["y"]}
            if c["add"] != "none":
                s["x_out"] = torch.empty(rows, cols, device="cuda")
                s["result"]["x"] = s["x_out"]
    torch.cuda.synchronize()          # the library works on a stream of its own
    return s


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------- the same in 64 bits

def _nearest(y, fmt):
    """(code values, scales) of the definition: the neighbour of smaller distance, of two the one of even code."""
    if fmt == FP4:
        grid = list(FP4_VALUES)
    else:
        grid = [m / 512.0 for m in range(8)] + [math.ldexp(1 + m / 8.0, e) for e in range(-6, 9) for m in range(8)][:-1]
    grid = torch.tensor(grid, dtype=torch.float64, device=y.device)
    rows, cols = y.shape
    blocks = -(-cols // 32)
    full = y.new_zeros(rows, blocks * 32)
    full[:, :cols] = y
    full = full.reshape(-1, 32)
    top = full.abs().max(1).values
    power = torch.floor(torch.log2(top))
    power = power + (torch.exp2(power + 1) <= top).double() - (torch.exp2(power) > top).double()
    scale = torch.exp2((power - EMAX[fmt]).clamp(min=-127.0))
    scale = torch.where(top > 0, scale, torch.full_like(scale, 2.0 ** -127))
    out = torch.empty_like(full)
    for at in range(0, full.shape[0], 1 << 19):
        a = (full[at:at + (1 << 19)] / scale[at:at + (1 << 19), None])
        hi = torch.searchsorted(grid, a.abs()).clamp(max=grid.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        dh, dl = grid[hi] - a.abs(), a.abs() - grid[lo]
        pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        out[at:at + (1 << 19)] = grid[pick] * torch.sign(a)
    return out.view(rows, -1)[:, :cols], scale.view(rows, blocks)


def _decoded(q, s, fmt, cols):
    """Codes and scales in 64 bits, from their fields."""
    q = q.to(torch.int64)
    if fmt == FP4:
        q = torch.stack([q & 15, q >> 4], 2).reshape(q.shape[0], -1)
        sign, e, m, low, bits = q >> 3, (q >> 1) & 3, q & 1, 1, 1
    else:
        sign, e, m, low, bits = q >> 7, (q >> 3) & 15, q & 7, 7, 3
    f = m.double() / (1 << bits) + (e > 0).double()
    v = torch.ldexp(f, e.clamp(min=1) - low) * (1 - 2 * sign.double())
    two = torch.ldexp(torch.ones_like(s, dtype=torch.float64), s.to(torch.int64) - 127)
    return v[:, :cols] * two.repeat_interleave(32, 1)[:, :cols]


def exact(c, seed):
    s = _inputs(c, seed)
    if c["kind"] == "quant":
        v, scale = _nearest(s["x"].double(), c["fmt"])
        return v * scale.repeat_interleave(32, 1)[:, :c["cols"]]
    if c["kind"] == "norm":
        x = s["x"].double()
        if c["add"] != "none":
            x = torch.addcmul(x, s["d"].double(), s["gate"].double()) if c["gate"] else x + s["d"].double()
        # the norm is taken of the stream as it is kept, in f32
        t = x.float().double() if c["add"] != "none" else x
        y = t * torch.rsqrt((t * t).sum(1, keepdim=True) / c["cols"] + EPS) * s["w"].double()
        v, scale = _nearest(y, c["fmt"])
        if c["fmt"] == FP4:
            out = {"y": v * scale.repeat_interleave(32, 1)[:, :c["cols"]]}
        else:
            out = {"q": v, "s": scale}
        return out if c["add"] == "none" else dict(out, x=x)
    y = _decoded(s["aq"], s["as"], c["afmt"], c["k"]) @ _decoded(s["wq"], s["ws"], FP4, c["k"]).t().contiguous()
    if not c["epi"].startswith("swiglu"):
        return y + s["bias"].double()
    g = y.unflatten(1, (-1, 64))
    y = (g[..., :32] * torch.sigmoid(g[..., :32]) * g[..., 32:]).flatten(1)
    if c["epi"] == "swiglu":
        return y
    v, scale = _nearest(y, FP8)
    return {"q": v, "s": scale}
