/*
 * mx.hip - microscaled matrices (4-bit e2m1 and 8-bit e4m3 codes, one power of
 * two per 32 columns of a row): quantisation, RMSNorm of an updated residual
 * stream with such an output, and the product with 4-bit weights on the
 * scaled matrix instructions. No counterpart in the reference, whose linears
 * are f32 and bf16 (iris_kernels.c:146-336).
 *
 * Block scale: with E the biased exponent of the block's largest magnitude,
 * floor(log2 max) = E - 127, so the scale byte is max(E - emax, 0) for zero,
 * subnormal and normal values alike, emax the exponent of the largest code (2
 * or 8). x / scale is exact in f32 wherever the result is not far below the
 * smallest code.
 */
#include "iris_internal.h"

#include <math.h>
#include <mutex>

namespace {

constexpr int NT = 256;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

/* 8 f32 values, the 8 columns of a lane; the 4 lanes of a quad hold a block of 32 */
struct Row8 {
    float v[8];
};

__device__ __forceinline__ uint32_t quad_maxu(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
}

/* scale byte of a block whose largest magnitude has these f32 bits */
template <int FMT> __device__ __forceinline__ int mx_scale(uint32_t top) {
    constexpr int EMAX = FMT == IRIS_MX_FP4 ? 2 : 8;
    return top >= 0x7f800000u ? 255 : max((int)(top >> 23) - EMAX, 0);
}

/* 1 / scale; 0 for a block that holds a NaN or an infinity */
__device__ __forceinline__ float mx_inv(int s) { return s == 255 ? 0.0f : __int_as_float((254 - s) << 23); }

/* codes of 4 values, code of v[0] lowest. e2m1 conversion saturates by
 * itself; e4m3 has a NaN above 448, hence the clamp. */
__device__ __forceinline__ uint32_t mx_fp8x4(float a, float b, float c, float d, float inv) {
    auto y = [inv](float v) { return inv == 0.0f ? 0.0f : __builtin_amdgcn_fmed3f(v * inv, -448.0f, 448.0f); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(y(a), y(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y(c), y(d), r, true);
}
__device__ __forceinline__ uint32_t mx_fp4x4(float a, float b, float c, float d, float inv) {
    auto y = [inv](float v) { return inv == 0.0f ? 0.0f : v * inv; };
    uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y(a), y(b), 1.0f, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y(c), y(d), 1.0f, 1) & 0xffffu;
}

/* the lane's 8 columns from c (a multiple of 8) on, of one row */
template <int FMT> __device__ __forceinline__ void mx_put8(uint8_t *q, uint8_t *s, int c, const Row8 &x) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x.v[i]) & 0x7fffffffu);
    const int sb = mx_scale<FMT>(quad_maxu(top));
    const float inv = mx_inv(sb);
    if constexpr (FMT == IRIS_MX_FP8) {
        *(uint2 *)(q + c) = make_uint2(mx_fp8x4(x.v[0], x.v[1], x.v[2], x.v[3], inv),
                                       mx_fp8x4(x.v[4], x.v[5], x.v[6], x.v[7], inv));
    } else {
        *(uint32_t *)(q + c / 2) = mx_fp4x4(x.v[0], x.v[1], x.v[2], x.v[3], inv) |
                                   mx_fp4x4(x.v[4], x.v[5], x.v[6], x.v[7], inv) << 16;
    }
    if ((threadIdx.x & 3) == 0) s[c / 32] = (uint8_t)sb;
}

/* 8 columns from c on of a row of f32 or bf16, zeros past cols; vec: 16-byte accesses are allowed */
template <bool BF16> __device__ __forceinline__ Row8 load8(const void *row, int c, int cols, bool vec) {
    Row8 x;
    if (vec && c + 8 <= cols) {
        if constexpr (BF16) {
            const u32x4 t = *(const u32x4 *)((const uint16_t *)row + c);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x.v[2 * i] = __uint_as_float(t[i] << 16);
                x.v[2 * i + 1] = __uint_as_float(t[i] & 0xffff0000u);
            }
        } else {
            const float4 a = *(const float4 *)((const float *)row + c), b = *(const float4 *)((const float *)row + c + 4);
            x.v[0] = a.x; x.v[1] = a.y; x.v[2] = a.z; x.v[3] = a.w;
            x.v[4] = b.x; x.v[5] = b.y; x.v[6] = b.z; x.v[7] = b.w;
        }
        return x;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (BF16) x.v[i] = c + i < cols ? bf2f(((const uint16_t *)row)[c + i]) : 0.0f;
        else x.v[i] = c + i < cols ? ((const float *)row)[c + i] : 0.0f;
    }
    return x;
}

/* One lane per 8 columns, rows one after the other (cpr = padded columns / 8
 * lanes each, a multiple of 16, so a quad stays in its block). Bound by the
 * bytes: 19456 x 2560 bf16 to e2m1 27.5 us, 4.6 TB/s; 512 x 4096 bf16 to e4m3
 * 3.4 us, a launch. */
template <int FMT, bool BF16>
__global__ __launch_bounds__(NT) void mx_quantize_kernel(uint8_t *q, uint8_t *s, int ld_q, int ld_s, const void *x,
                                                         int ldx, int cols, uint32_t cpr, uint32_t n, bool vec) {
    const uint32_t i = blockIdx.x * NT + threadIdx.x;
    if (i >= n) return;
    const uint32_t row = i / cpr;
    const int c = (int)(i - row * cpr) * 8;
    const void *xr = (const char *)x + (size_t)row * ldx * (BF16 ? 2 : 4);
    mx_put8<FMT>(q + (size_t)row * ld_q, s + (size_t)row * ld_s, c, load8<BF16>(xr, c, cols, vec));
}

/* 2^(s - 127); NaN for 255 */
__device__ __forceinline__ float mx_two(int s) {
    return s == 255 ? __int_as_float(0x7fc00000) : s ? __int_as_float(s << 23) : __int_as_float(0x00400000);
}

/* 19456 x 2560 e2m1 to bf16: 21.0 us, 6.0 TB/s (the codes from the caches). */
template <int FMT, bool BF16>
__global__ __launch_bounds__(NT) void mx_dequantize_kernel(void *y, int ldy, const uint8_t *q, const uint8_t *s,
                                                           int ld_q, int ld_s, int cols, uint32_t cpr, uint32_t n,
                                                           bool vec) {
    const uint32_t i = blockIdx.x * NT + threadIdx.x;
    if (i >= n) return;
    const uint32_t row = i / cpr;
    const int c = (int)(i - row * cpr) * 8;
    const uint8_t *qr = q + (size_t)row * ld_q;
    const float two = mx_two(s[(size_t)row * ld_s + c / 32]);
    float v[8];
    if constexpr (FMT == IRIS_MX_FP8) {
        const uint2 t = *(const uint2 *)(qr + c);
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)t.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)t.x, true);
        const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)t.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)t.y, true);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = d.x; v[5] = d.y; v[6] = e.x; v[7] = e.y;
    } else {
        const uint32_t t = *(const uint32_t *)(qr + c / 2);
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(t, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(t, 1.0f, 1);
        const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(t, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(t, 1.0f, 3);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = d.x; v[5] = d.y; v[6] = e.x; v[7] = e.y;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= two;
    if constexpr (BF16) {
        uint16_t *yr = (uint16_t *)y + (size_t)row * ldy;
        u32x4 t;
#pragma unroll
        for (int j = 0; j < 4; j++) t[j] = (uint32_t)f2bf_hw(v[2 * j]) | (uint32_t)f2bf_hw(v[2 * j + 1]) << 16;
        if (vec && c + 8 <= cols) *(u32x4 *)(yr + c) = t;
        else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < cols) yr[c + j] = (uint16_t)(t[j >> 1] >> (16 * (j & 1)));
    } else {
        float *yr = (float *)y + (size_t)row * ldy;
        if (vec && c + 8 <= cols) {
            *(float4 *)(yr + c) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4 *)(yr + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < cols) yr[c + j] = v[j];
    }
}

/* ---- RMSNorm of an updated stream ----
 * t = f32(x + gate d) into x_out; y = t / sqrt(mean t^2 + eps) w (scale),
 * quantised. Codes are those of the formula in exact arithmetic: the sum of
 * squares and y are held in 64 bits, and y goes to f32 rounded to odd (toward
 * zero, last bit set where anything was cut off), which keeps its exponent
 * and every later rounding to fewer bits as of y itself. So a code depends
 * neither on the order of the sum nor on an f32 rounding next to a border of
 * two codes (5e-6 of all elements otherwise). */
struct NormParams {
    const float *x, *gate, *w, *scale;
    const void *d;
    float *x_out;
    uint8_t *q, *s;
    int ldx, ldd, ldxo, ld_q, ld_s, cols, cols_pad;
    float eps;
    bool vx, vd, vo, vg, vw, vs;   /* 16-byte accesses to x, d, x_out, gate, w, scale */
};

__device__ __forceinline__ float to_odd(double y) {
    const float h = (float)y;
    uint32_t u = __float_as_uint(h);
    if (fabs((double)h) > fabs(y)) u--;         /* toward zero; an infinity becomes the largest number */
    if ((double)h != y) u |= 1;                 /* a NaN stays one */
    return __uint_as_float(u);
}

template <int DT> __device__ __forceinline__ Row8 norm_row8(const NormParams &P, size_t row, int c, bool store) {
    Row8 x = load8<false>(P.x + row * P.ldx, c, P.cols, P.vx);
    if constexpr (DT) {
        const Row8 d = load8<DT == 2>((const char *)P.d + row * P.ldd * (DT == 2 ? 2 : 4), c, P.cols, P.vd);
        if (P.gate) {
            const Row8 g = load8<false>(P.gate, c, P.cols, P.vg);
#pragma unroll
            for (int i = 0; i < 8; i++) x.v[i] = fmaf(g.v[i], d.v[i], x.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x.v[i] += d.v[i];
        }
        if (store) {
            float *o = P.x_out + row * P.ldxo + c;
            if (P.vo && c + 8 <= P.cols) {
                /* streaming: 4608 x 3840 that no cache holds 51 -> 46 us */
                st_stream((float4 *)o, make_float4(x.v[0], x.v[1], x.v[2], x.v[3]));
                st_stream((float4 *)(o + 4), make_float4(x.v[4], x.v[5], x.v[6], x.v[7]));
            } else
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (c + i < P.cols) o[i] = x.v[i];
        }
    }
    return x;
}

/* Bound by the bytes, one pass over them: 4608 x 3840, bf16 d and gate, 41.0 us
 * (4.8 TB/s); 512 x 2560, f32 d, 4.7 us; one row 3.5 us, a launch.
 * DT: 0 no d, 1 f32, 2 bf16. One block of TH threads per row, R chunks of 8
 * columns a thread held in registers; R 0: any length, the row read twice (the second
 * time from x_out where there is a d: the thread's own stores). */
template <int FMT, int DT, int TH, int R> __global__ __launch_bounds__(TH) void mx_rmsnorm_kernel(const NormParams P) {
    __shared__ double red[TH / IRIS_WAVE];
    const size_t row = blockIdx.x;
    Row8 t[R ? R : 1];
    double ss = 0.0;
    auto square = [&](const Row8 &x) {
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fma((double)x.v[i], (double)x.v[i], ss);
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int c = (r * TH + (int)threadIdx.x) * 8;
            if (c < P.cols_pad) {
                t[r] = norm_row8<DT>(P, row, c, true);
                square(t[r]);
            }
        }
    } else {
        for (int c = (int)threadIdx.x * 8; c < P.cols_pad; c += TH * 8) square(norm_row8<DT>(P, row, c, true));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < TH / IRIS_WAVE; i++) ss += red[i];
    const double inv = 1.0 / sqrt(ss / P.cols + (double)P.eps);
    auto put = [&](const Row8 &x, int c) {
        const Row8 w = load8<false>(P.w, c, P.cols, P.vw);   /* zeros past the row's end */
        double v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (double)x.v[i] * inv * (double)w.v[i];
        if (P.scale) {
            const Row8 g = load8<false>(P.scale, c, P.cols, P.vs);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] *= (double)g.v[i];
        }
        Row8 y;
#pragma unroll
        for (int i = 0; i < 8; i++) y.v[i] = c + i < P.cols ? to_odd(v[i]) : 0.0f;   /* 0 inv may be NaN */
        mx_put8<FMT>(P.q + row * P.ld_q, P.s + row * P.ld_s, c, y);
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int c = (r * TH + (int)threadIdx.x) * 8;
            if (c < P.cols_pad) put(t[r], c);
        }
    } else {
        NormParams P2 = P;
        if constexpr (DT != 0) {
            P2.x = P.x_out;
            P2.ldx = P.ldxo;
            P2.vx = P.vo;
        }
        for (int c = (int)threadIdx.x * 8; c < P.cols_pad; c += TH * 8) put(norm_row8<0>(P2, row, c, false), c);
    }
}

/* ---- product ----
 * out[m][n] = sum over K of A[m][k] W[n][k] on v_mfma_scale_f32_16x16x128:
 * W is the first operand, so a lane ends with 4 consecutive n of one m. Lane
 * l = 16 g + r of an operand holds row r: of e2m1 columns 32 g .. 32 g + 31
 * (16 bytes), of e4m3 columns 16 g .. 16 g + 15 and 64 + 16 g .. (two times
 * 16 bytes), and the scale of block g of the row in its byte. */
struct MxGemm {
    const uint8_t *aq, *as, *wq, *ws;
    int lda, ldas, ldw, ldws;
    void *out;
    const float *vec;
    int M, N, steps, ldo, epi;
    uint8_t *oq, *os;      /* SWIGLU: microscaled output, NULL: bf16 into out */
    int ldoq, ldos, ofmt;
    /* blocks: tiles_m x tiles_n of them for each of `chunks` ranges of per_chunk
     * K steps; with more than one, out is f32 [chunk][M][N] partial sums */
    int tiles_m, tiles_n, chunks, per_chunk;
};

/* The K range of chunk c: operands from its first step on, partial sums out.
 * per_chunk is a multiple of 4 steps, 16 scale bytes. */
template <int AF> __device__ __forceinline__ void mx_chunk(MxGemm &P, int c) {
    if (P.chunks == 1) return;
    const int k0 = c * P.per_chunk;
    P.aq += (size_t)k0 * (AF == IRIS_MX_FP8 ? 128 : 64);
    P.wq += (size_t)k0 * 64;
    P.as += (size_t)k0 * 4;
    P.ws += (size_t)k0 * 4;
    P.steps = min(P.per_chunk, P.steps - k0);
    P.out = (float *)P.out + (size_t)c * P.M * P.N;
}

/* The instruction adds its products in groups of 8 neighbouring columns and
 * keeps, of a group, bits down to 2^-13 of the largest product's power of two
 * (measured; between groups and with the accumulator it keeps f32). Products
 * of two e2m1 codes span 2^6 and lose nothing; those with e4m3 codes span more:
 * one pass leaves sums of ordinary rows 2e-5 off (512 x 2560 x 9728), and one
 * large product among small ones takes these away altogether. So A's e4m3 codes
 * go through it twice, in every kernel and for every output type, those of
 * magnitude 2 and more (exponents 1 .. 8) and those below (lowest bit 2^-9 to
 * 2^0): with W's lowest bit 2^-1 and highest 2^2 either span is within 13 powers
 * of two, and the sums are f32 sums. 4608 x 20480 x 3840 with SwiGLU takes 490 to
 * 505 us so, 254 with one pass. */
template <int AF>
__device__ __forceinline__ f32x4 mx_mfma(const u32x4 &w, const i32x8 &a, const f32x4 &c, int sw, int sa) {
    const i32x8 w8 = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a, c, 4, AF == IRIS_MX_FP8 ? 0 : 4, 0, sw, 0, sa);
}

/* of e2m1 codes, scales in byte OP */
template <int OP>
__device__ __forceinline__ f32x4 mx_mfma4(const u32x4 &w, const i32x8 &a, const f32x4 &c, int sw, int sa) {
    const i32x8 w8 = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a, c, 4, 4, OP, sw, OP, sa);
}

/* the e4m3 codes of magnitude 2 and more (bit 6 set), or the others */
template <bool BIG> __device__ __forceinline__ i32x8 mx_part(const i32x8 &a) {
    i32x8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t x = (uint32_t)a[i], big = ((x >> 6) & 0x01010101u) * 255u;
        r[i] = (int)(BIG ? x & big : x & ~big);
    }
    return r;
}

/* one lane's 4 columns n .. n + 3 of row m through the plain epilogues */
__device__ __forceinline__ void mx_store4(const MxGemm &P, int m, int n, const f32x4 &x, bool aligned) {
    const float vd = P.epi == IRIS_EPI_GATED_ADD ? 1.0f : 0.0f;
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = P.vec && n + r < P.N ? P.vec[n + r] : vd;
    const size_t o = (size_t)m * P.ldo + n;
    if (aligned && n + 4 <= P.N) {
        if (P.epi == IRIS_EPI_BF16) {
            *(uint2 *)((uint16_t *)P.out + o) =
                make_uint2((uint32_t)f2bf_hw(x[0] + v[0]) | (uint32_t)f2bf_hw(x[1] + v[1]) << 16,
                           (uint32_t)f2bf_hw(x[2] + v[2]) | (uint32_t)f2bf_hw(x[3] + v[3]) << 16);
            return;
        }
        float4 *dst = (float4 *)((float *)P.out + o);
        float4 y = make_float4(x[0] + v[0], x[1] + v[1], x[2] + v[2], x[3] + v[3]);
        if (P.epi == IRIS_EPI_GATED_ADD) {
            y = *dst;
            y.x += v[0] * x[0]; y.y += v[1] * x[1]; y.z += v[2] * x[2]; y.w += v[3] * x[3];
        } else if (P.epi == IRIS_EPI_ADD) {
            const float4 t = *dst;
            y.x += t.x; y.y += t.y; y.z += t.z; y.w += t.w;
        }
        *dst = y;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (n + r >= P.N) continue;
        float *f = (float *)P.out + o + r;
        if (P.epi == IRIS_EPI_BF16) ((uint16_t *)P.out)[o + r] = f2bf_hw(x[r] + v[r]);
        else if (P.epi == IRIS_EPI_GATED_ADD) *f += v[r] * x[r];
        else if (P.epi == IRIS_EPI_ADD) *f = x[r] + v[r] + *f;
        else *f = x[r] + v[r];
    }
}

/* The same in every kernel. The hardware's exponential and reciprocal would be
 * |x| units of 2^-24 off, and 0 below -87, where 1 + exp(-x) has no normal
 * reciprocal and the result still has 16 bits; they would save 20 to 25 of 490 us
 * of 4608 x 20480 x 3840. */
__device__ __forceinline__ float mx_silu(float x) { return x / (1.0f + expf(-x)); }

/* a 64-column gate / up group from n on (gate tiles 0, 1, up tiles 2, 3): 8
 * values of row m in each of 4 lanes 16 apart, one block of 32 columns of the
 * output. Whole waves call it: the block's maximum is taken over the lanes. */
__device__ __forceinline__ void mx_store_swiglu(const MxGemm &P, int m, int n, const f32x4 &g0, const f32x4 &g1,
                                                const f32x4 &u0, const f32x4 &u1, bool aligned) {
    const int lg = (threadIdx.x >> 4) & 3, col = n / 2 + 4 * lg;
    const bool in = m < P.M && n < P.N;   /* N % 64 == 0: the whole group or nothing */
    float y[8];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        y[r] = mx_silu(g0[r]) * u0[r];
        y[4 + r] = mx_silu(g1[r]) * u1[r];
    }
    if (!P.oq) {
        if (!in) return;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint16_t *dst = (uint16_t *)P.out + (size_t)m * P.ldo + col + 16 * h;
            uint16_t b[4];
#pragma unroll
            for (int r = 0; r < 4; r++) b[r] = f2bf_hw(y[4 * h + r]);
            if (aligned)
                *(uint2 *)dst = make_uint2((uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16);
            else
#pragma unroll
                for (int r = 0; r < 4; r++) dst[r] = b[r];
        }
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    if (!in) return;
    uint8_t *q = P.oq + (size_t)m * P.ldoq, *s = P.os + (size_t)m * P.ldos;
    int sb;
    if (P.ofmt == IRIS_MX_FP8) {
        sb = mx_scale<IRIS_MX_FP8>(top);
        const float inv = mx_inv(sb);
        *(uint32_t *)(q + col) = mx_fp8x4(y[0], y[1], y[2], y[3], inv);
        *(uint32_t *)(q + col + 16) = mx_fp8x4(y[4], y[5], y[6], y[7], inv);
    } else {
        sb = mx_scale<IRIS_MX_FP4>(top);
        const float inv = mx_inv(sb);
        *(uint16_t *)(q + col / 2) = (uint16_t)mx_fp4x4(y[0], y[1], y[2], y[3], inv);
        *(uint16_t *)(q + col / 2 + 8) = (uint16_t)mx_fp4x4(y[4], y[5], y[6], y[7], inv);
    }
    if (lg == 0) s[n / 64] = (uint8_t)sb;
    /* zero blocks up to the padded width, behind the last group */
    if (n + 64 == P.N)
        for (int b = P.N / 64; b & 3; b++) {
            if (P.ofmt == IRIS_MX_FP8) *(uint2 *)(q + 32 * b + 8 * lg) = make_uint2(0, 0);
            else *(uint32_t *)(q + 16 * b + 4 * lg) = 0;
            if (lg == 0) s[b] = 0;
        }
}

constexpr int waitcnt_imm(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }
typedef __attribute__((address_space(3))) void lds_void;
constexpr int GROUP_M = 8;


/* 64 lanes' 16 bytes from a buffer to LDS, one after the other from place at on
 * (rows past the buffer's end: zeros). Not the builtin: before reads of one
 * stage the compiler waits for the builtin's loads into the others too, which
 * takes the ring's depth away. The caller waits (vmcnt) before a barrier. */
__device__ __forceinline__ uint32_t lds_at(const void *p) { return (uint32_t)(uintptr_t)(const lds_void *)p; }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   /* m0 is reserved: the compiler keeps nothing in it, but may write it for its own use */
__device__ __forceinline__ void load_lds16(const u32x4 &rsrc, uint32_t at, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(at), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ u32x4 buffer_of(const void *p, int bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    return (u32x4){(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)),
                   (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

/* byte j of word i to byte i of word j */
__device__ __forceinline__ u32x4 bytes4x4(const u32x4 &x) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602);
    const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602);
    return (u32x4){__builtin_amdgcn_perm(c, a, 0x05040100), __builtin_amdgcn_perm(c, a, 0x07060302),
                   __builtin_amdgcn_perm(d, b, 0x05040100), __builtin_amdgcn_perm(d, b, 0x07060302)};
}

template <int V> struct Const {
    static constexpr int value = V;
};

/* explicit waits stay where they are written, and memory accesses on their side */
#define WAIT(vm, lgkm)                                              \
    do {                                                            \
        asm volatile("" ::: "memory");                              \
        __builtin_amdgcn_sched_barrier(0);                          \
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(vm, lgkm));          \
        __builtin_amdgcn_sched_barrier(0);                          \
        asm volatile("" ::: "memory");                              \
    } while (0)

/* part[0] + part[stride] + .. of n waves, in order; 4 reads in flight */
__device__ __forceinline__ f32x4 mx_sum_waves(const f32x4 *part, int stride, int n) {
    f32x4 s = part[0];
    for (int w = 1; w < n; w += 4) {
        f32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = part[min(w + k, n - 1) * stride];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (w + k < n) s += v[k];
    }
    return s;
}

/* ---- product of few rows ----
 * Bound by W's bytes and by the number of 128-byte lines that loads touch (1.5
 * ns each and CU), not by the matrix instructions. A block's waves share 16 FM
 * rows of A and 16 FN of W; a wave takes every waves-th unit of 256 columns,
 * through a part of LDS of its own: loads of 8 rows x 128 bytes, straight into
 * LDS (16-byte chunks XORed with the row number, as in the tiles below), while
 * the unit before is multiplied. Fragments straight from global memory touch
 * each line twice, and a wave's loads in registers leave room for half the
 * waves: gate and up of 37 rows 24.8 us. Scales of 4096 columns are loaded by
 * the whole block, a line a row. The waves' sums are added in wave order.
 * Measured, e4m3 A: 37 x 19456 x 2560 with SwiGLU 14.7 us (26.5 MB of W at 1.8
 * TB/s; of a block's 10 us a third is launch, first loads and scales, a third
 * instructions, a third sums and epilogue), 37 x 6144 x 2560 8.6; e2m1 A: 37 x
 * 11520 x 3840 7.3 (3.2 TB/s). <e2m1, 4, 4> spills 7 registers, addresses of the
 * next unit's loads, and waits for the loads in flight at each reload: 256 x 3840
 * x 10240 22.7 us. */
template <int AF, int FM, int FN> struct RowsShape {
    static constexpr int A_ROW = AF == IRIS_MX_FP8 ? 256 : 128;    /* bytes of 256 columns */
    static constexpr int A_BYTES = FM * 16 * A_ROW, UNIT = A_BYTES + FN * 2048;
    static constexpr int SCALES = 16 * (FM + FN) * 128;            /* bytes of 4096 columns */
    static constexpr int fit(int bytes) { return bytes / UNIT > 16 ? 16 : bytes / UNIT; }
    static constexpr int WAVES = fit(163840 - SCALES), WAVES2 = fit(81920 - SCALES);   /* one block per CU, two */
};

template <int AF, int FM, int FN>
__global__ __launch_bounds__((64 * RowsShape<AF, FM, FN>::WAVES)) void mx_gemm_rows_kernel(MxGemm P) {
    using Sh = RowsShape<AF, FM, FN>;
    constexpr bool F8 = AF == IRIS_MX_FP8;
    constexpr int SEG = 32;                    /* steps whose scales are in LDS */
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   /* scales, then a unit per wave; sums at the end */
    const int tiles = P.tiles_m * P.tiles_n;
    const int chunk = (int)blockIdx.x / tiles, t = (int)blockIdx.x - chunk * tiles;
    const int off = chunk * P.per_chunk;
    mx_chunk<AF>(P, chunk);
    const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
    const int m0 = t / P.tiles_n * 16 * FM, n0 = t % P.tiles_n * 16 * FN;
    const int a_rows = min(16 * FM, P.M - m0), w_rows = min(16 * FN, P.N - n0);
    /* rows past the end read as zeros */
    const u32x4 a_rsrc = buffer_of(P.aq + (size_t)m0 * P.lda, a_rows * P.lda - off * (F8 ? 128 : 64));
    const u32x4 w_rsrc = buffer_of(P.wq + (size_t)n0 * P.ldw, w_rows * P.ldw - off * 64);
    const u32x4 as_rsrc = buffer_of(P.as + (size_t)m0 * P.ldas, a_rows * P.ldas - off * 4);
    const u32x4 ws_rsrc = buffer_of(P.ws + (size_t)n0 * P.ldws, w_rows * P.ldws - off * 4);
    uint8_t *const mine = lds + Sh::SCALES + wave * Sh::UNIT;
    const uint32_t scl0 = lds_at(lds), at0 = lds_at(mine);
    const int units = (P.steps + 1) / 2;

    /* a load of 8 rows x 128 bytes: lane l row l / 8, place l % 8, chunk place
     * ^ (row % 8); chunks: how many of the 8 lie within the row's data, the
     * others read the first */
    const int row8 = lane >> 3, ch8 = (lane & 7) ^ row8;
    auto load8rows = [&](const u32x4 &rsrc, uint32_t at, int row0, int ld, int soff, int chunks) {
        load_lds16(rsrc, at, (row0 + row8) * ld + (ch8 < chunks ? ch8 << 4 : 0), soff);
    };
    auto load_unit = [&](int u) {
        const int n = min(2, P.steps - 2 * u);   /* steps of 128 columns */
#pragma unroll
        for (int i = 0; i < 2 * FN; i++)
            if (8 * i < w_rows) load8rows(w_rsrc, at0 + Sh::A_BYTES + i * 1024, 8 * i, P.ldw, u * 128, 4 * n);
#pragma unroll
        for (int i = 0; i < 2 * FM; i++)
            if (8 * i < a_rows) {
                load8rows(a_rsrc, at0 + i * 1024, 8 * i, P.lda, u * Sh::A_ROW, F8 ? 8 : 4 * n);
                if (F8 && n == 2) load8rows(a_rsrc, at0 + FM * 2048 + i * 1024, 8 * i, P.lda, u * 256 + 128, 8);
            }
    };
    auto load_scales = [&](int seg) {
        const int chunks = min(8, (P.steps - seg * SEG + 3) / 4);
        for (int i = wave; i < 2 * (FM + FN); i += waves) {
            if (i < 2 * FM) {
                if (8 * i < a_rows) load8rows(as_rsrc, scl0 + i * 1024, 8 * i, P.ldas, seg * 128, chunks);
            } else if (8 * i - 16 * FM < w_rows) load8rows(ws_rsrc, scl0 + i * 1024, 8 * i - 16 * FM, P.ldws, seg * 128, chunks);
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    /* places of a fragment row's chunk c, and of its scale byte of step k: rows 16 apart are stored alike */
    const int frow = lr * 128;
    auto piece = [&](int c) { return frow + ((c ^ (lr & 7)) << 4); };
    auto scale = [&](int tile, int k) { return (int)lds[tile * 2048 + piece((k & (SEG - 1)) >> 2) + (k & 3) * 4 + lg]; };
    auto unit = [&](int u, int n, int next) {
        u32x4 w[2][FN], a[2][FM][2];
        int sw[2][FN], sa[2][FM];
        WAIT(0, 15);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (h >= n) break;
#pragma unroll
            for (int j = 0; j < FN; j++) {
                w[h][j] = *(const u32x4 *)(mine + Sh::A_BYTES + j * 2048 + piece(4 * h + lg));
                sw[h][j] = scale(FM + j, 2 * u + h);
            }
#pragma unroll
            for (int i = 0; i < FM; i++) {
                const uint8_t *x = mine + (F8 ? h * FM * 2048 : 0) + i * 2048;
                a[h][i][0] = *(const u32x4 *)(x + piece(F8 ? lg : 4 * h + lg));
                a[h][i][1] = F8 ? *(const u32x4 *)(x + piece(4 + lg)) : (u32x4){0, 0, 0, 0};
                sa[h][i] = scale(i, 2 * u + h);
            }
        }
        WAIT(63, 0);
        if (next >= 0) load_unit(next);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (h >= n) break;
#pragma unroll
            for (int i = 0; i < FM; i++) {
                const u32x4 x = a[h][i][0], y = a[h][i][1];
                const i32x8 x8 = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
                const i32x8 hi = F8 ? mx_part<true>(x8) : x8, lo = mx_part<false>(x8);
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    acc[i][j] = mx_mfma<AF>(w[h][j], hi, acc[i][j], sw[h][j], sa[h][i]);
                    if constexpr (F8) acc[i][j] = mx_mfma<AF>(w[h][j], lo, acc[i][j], sw[h][j], sa[h][i]);
                }
            }
        }
    };
    int u = wave;
    if (u < units) load_unit(u);
    for (int seg = 0; seg * SEG < P.steps; seg++) {
        if (seg) __syncthreads();   /* everyone is done with the scales before */
        load_scales(seg);
        WAIT(0, 0);
        __syncthreads();
        const int end = min(units, (seg + 1) * (SEG / 2));
        for (; u < end; u += waves) {
            const int next = u + waves < units ? u + waves : -1;
            if (2 * u + 1 < P.steps) unit(u, 2, next);
            else unit(u, 1, next);
        }
    }
    __syncthreads();
    f32x4 *const part = (f32x4 *)lds;   /* [waves][FM * FN tiles][64 lanes] */
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) part[(wave * FM * FN + i * FN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    auto sum = [&](int i, int j) { return mx_sum_waves(part + (i * FN + j) * 64 + lane, FM * FN * 64, waves); };
    const bool aligned = (P.ldo & 3) == 0 && ((uintptr_t)P.out & 15) == 0;
    if constexpr (FN == 4) {
        if (P.epi == IRIS_EPI_SWIGLU) {
            for (int i = wave; i < FM; i += waves)
                mx_store_swiglu(P, m0 + 16 * i + lr, n0, sum(i, 0), sum(i, 1), sum(i, 2), sum(i, 3), aligned);
            return;
        }
    }
    for (int q = wave; q < FM * FN; q += waves) {
        const int m = m0 + 16 * (q / FN) + lr;
        const f32x4 s = sum(q / FN, q % FN);
        if (m < P.M) mx_store4(P, m, n0 + 16 * (q % FN) + 4 * lg, s, aligned);
    }
}

/* ---- product without LDS staging ----
 * Fragments straight from global memory by 64-bit pointers, a wave per group
 * of 512 columns in turn: for one to 16 rows of A (plain epilogues), and for
 * rows further apart than the other kernels' 32-bit offsets reach. Whole
 * 128-byte lines of the codes and one 16-byte load of scales a row for 4
 * steps (a 4-byte load per step touched as many lines as W). One row x 6144 x
 * 2560: 4.5 us, of which 3 are the launch; W's 8.4 MB at 1.9 TB/s. */
template <int AF, int FM, int FN> __global__ __launch_bounds__(512) void mx_gemm_direct_kernel(MxGemm P) {
    extern __shared__ f32x4 part[];   /* [waves][FM * FN tiles][64 lanes] */
    const int tiles = P.tiles_m * P.tiles_n;
    const int chunk = (int)blockIdx.x / tiles, t = (int)blockIdx.x - chunk * tiles;
    mx_chunk<AF>(P, chunk);
    const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
    const int m0 = t / P.tiles_n * 16 * FM, n0 = t % P.tiles_n * 16 * FN;
    const uint8_t *ap[FM], *sap[FM], *wp[FN], *swp[FN];
#pragma unroll
    for (int i = 0; i < FM; i++) {
        const size_t m = min(m0 + 16 * i + lr, P.M - 1);   /* rows past the end repeat the last; not stored */
        ap[i] = P.aq + m * P.lda + 16 * lg;
        sap[i] = P.as + m * P.ldas;
    }
#pragma unroll
    for (int j = 0; j < FN; j++) {
        const size_t n = min(n0 + 16 * j + lr, P.N - 1);
        wp[j] = P.wq + n * P.ldw + 16 * lg;
        swp[j] = P.ws + n * P.ldws;
    }
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    /* steps 4 g .. 4 g + n - 1 */
    auto group = [&](int g, int n) {
        u32x4 sw[FN], sa[FM], w[4][FN], a[4][FM][2];
#pragma unroll
        for (int j = 0; j < FN; j++) sw[j] = *(const u32x4 *)(swp[j] + (size_t)g * 16);
#pragma unroll
        for (int i = 0; i < FM; i++) sa[i] = *(const u32x4 *)(sap[i] + (size_t)g * 16);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (u >= n) break;
            const size_t k = (size_t)g * 4 + u;
#pragma unroll
            for (int j = 0; j < FN; j++) w[u][j] = *(const u32x4 *)(wp[j] + k * 64);
#pragma unroll
            for (int i = 0; i < FM; i++) {
                const uint8_t *x = ap[i] + k * (AF == IRIS_MX_FP8 ? 128 : 64);
                a[u][i][0] = *(const u32x4 *)x;
                a[u][i][1] = AF == IRIS_MX_FP8 ? *(const u32x4 *)(x + 64) : (u32x4){0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (u >= n) break;
#pragma unroll
            for (int i = 0; i < FM; i++) {
                const u32x4 x = a[u][i][0], y = a[u][i][1];
                const i32x8 x8 = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
                const i32x8 hi = AF == IRIS_MX_FP8 ? mx_part<true>(x8) : x8, lo = mx_part<false>(x8);
                const int s = (int)(sa[i][u] >> 8 * lg);
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    const int r = (int)(sw[j][u] >> 8 * lg);
                    acc[i][j] = mx_mfma<AF>(w[u][j], hi, acc[i][j], r, s);
                    if constexpr (AF == IRIS_MX_FP8) acc[i][j] = mx_mfma<AF>(w[u][j], lo, acc[i][j], r, s);
                }
            }
        }
    };
    const int whole = P.steps / 4;
    int g = wave;
    for (; g < whole; g += waves) group(g, 4);
    if (g == whole && (P.steps & 3)) group(g, P.steps & 3);
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) part[(wave * FM * FN + i * FN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    auto sum = [&](int i, int j) { return mx_sum_waves(part + (i * FN + j) * 64 + lane, FM * FN * 64, waves); };
    const bool aligned = (P.ldo & 3) == 0 && ((uintptr_t)P.out & 15) == 0;
    if constexpr (FN == 4) {
        if (P.epi == IRIS_EPI_SWIGLU) {
            for (int i = wave; i < FM; i += waves)
                mx_store_swiglu(P, m0 + 16 * i + lr, n0, sum(i, 0), sum(i, 1), sum(i, 2), sum(i, 3), aligned);
            return;
        }
    }
    for (int q = wave; q < FM * FN; q += waves) {
        const int m = m0 + 16 * (q / FN) + lr;
        const f32x4 s = sum(q / FN, q % FN);
        if (m < P.M) mx_store4(P, m, n0 + 16 * (q % FN) + 4 * lg, s, aligned);
    }
}

/* ---- sums of a split product ----
 * One lane per 8 output columns: the chunks' partial sums in order, then the
 * epilogue. 512 x 2560 of 3 chunks: 7.6 us, 5 where they are still in the
 * caches (4 TB/s). */
__global__ __launch_bounds__(NT) void mx_reduce_kernel(const MxGemm P, const float *part, uint32_t n, uint32_t cpr) {
    const uint32_t i = blockIdx.x * NT + threadIdx.x;
    if (i >= n) return;
    const uint32_t m = i / cpr;
    const int c = (int)(i - m * cpr) * 8;
    const bool swiglu = P.epi == IRIS_EPI_SWIGLU;
    const size_t stride = (size_t)P.M * P.N;
    const bool vec = (P.N & 3) == 0 && ((uintptr_t)part & 15) == 0;
    auto sum8 = [&](int col) {
        const float *row = part + (size_t)m * P.N;
        Row8 s = load8<false>(row, col, P.N, vec);
        for (int k = 1; k < P.chunks; k += 3) {   /* 3 chunks' loads in flight */
            Row8 x[3];
#pragma unroll
            for (int i = 0; i < 3; i++) x[i] = load8<false>(row + min(k + i, P.chunks - 1) * stride, col, P.N, vec);
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (k + i < P.chunks)
#pragma unroll
                    for (int j = 0; j < 8; j++) s.v[j] += x[i].v[j];
        }
        return s;
    };
    if (!swiglu) {
        const Row8 s = sum8(c);
        const bool aligned = (P.ldo & 3) == 0 && ((uintptr_t)P.out & 15) == 0;
        mx_store4(P, (int)m, c, (f32x4){s.v[0], s.v[1], s.v[2], s.v[3]}, aligned);
        if (c + 4 < P.N) mx_store4(P, (int)m, c + 4, (f32x4){s.v[4], s.v[5], s.v[6], s.v[7]}, aligned);
        return;
    }
    /* columns c .. c + 7 of the output: gate and up columns of one 64-column group */
    Row8 y;
    if (c < P.N / 2) {
        const Row8 g = sum8((c >> 5) * 64 + (c & 31)), u = sum8((c >> 5) * 64 + 32 + (c & 31));
#pragma unroll
        for (int j = 0; j < 8; j++) y.v[j] = mx_silu(g.v[j]) * u.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) y.v[j] = 0.0f;   /* a microscaled row's padding */
    }
    if (P.oq) {
        uint8_t *q = P.oq + (size_t)m * P.ldoq, *sc = P.os + (size_t)m * P.ldos;
        if (P.ofmt == IRIS_MX_FP8) mx_put8<IRIS_MX_FP8>(q, sc, c, y);
        else mx_put8<IRIS_MX_FP4>(q, sc, c, y);
        return;
    }
    uint16_t *o = (uint16_t *)P.out + (size_t)m * P.ldo + c;
    u32x4 b;
#pragma unroll
    for (int j = 0; j < 4; j++) b[j] = (uint32_t)f2bf_hw(y.v[2 * j]) | (uint32_t)f2bf_hw(y.v[2 * j + 1]) << 16;
    if ((P.ldo & 7) == 0 && ((uintptr_t)P.out & 15) == 0) *(u32x4 *)o = b;
    else
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = (uint16_t)(b[j >> 1] >> (16 * (j & 1)));
}

/* ---- product on LDS tiles ----
 * 8 waves, 4 along M x 2 along N, block tile BM x BN. LDS holds two stages of
 * A and two of W, rows of 128 bytes (e4m3: 128 columns, one K step; e2m1: 256):
 * a load costs the CU's address and cache path 1.5 ns per row it touches, 128
 * bytes or less, and with rows of 64 bytes that path, not the matrix
 * instructions, took the time. 16-byte chunks of a row are stored XORed with
 * its row number, so that the loads, which place 64 lanes' 16 bytes one after
 * the other, give fragment reads without bank conflicts. Waves w and w + 4
 * share a SIMD: group 0 (waves 0..3, the tile's upper half) and group 1 take
 * turns, one reading a K step's fragments while the other runs its matrix
 * instructions (phases as described at the loop).
 * Scales: 16 bytes of a row are 512 columns. They are loaded into LDS as they
 * are, then a lane transposes the 4 x 4 bytes of a row so that the bytes of
 * lane group g (block g of each 128 columns) make one word; a fragment's lane
 * reads its word once per 512 columns and shifts it by a byte per 128.
 * Measured on 256 x 256 tiles: e4m3 A, 4608 x 20480 x 3840 with SwiGLU 490 to
 * 505 us, 1.45 PFLOP/s: bound by the matrix instructions of A's two parts, 4220
 * cycles per K step, at the clock that such a kernel is given (with the
 * hardware's SwiGLU 482, on 128 x 128 tiles 534). It spills one sum in one of
 * four steps of group 1 (24 bytes a lane); the compiler's wait for the reload also
 * waits for the loads in flight. e2m1 A, 4352 x 3840 x 10240 86.6 us, 3.95
 * PFLOP/s: 3310 cycles per 256 columns, the instructions 2050; reading a step's
 * fragments beside the loads into LDS takes 1500 of a phase's 1650. 128 x 128
 * tiles, e4m3 A, f32: 512 x 2560 x 9728 in 3 ranges 33 us and their sum. 4 waves
 * of 128 x 128 each read a third less from LDS, but have to issue the loads
 * between their own matrix instructions and wait for the address path there: 126
 * to 130 us on 4096 x 4096 x 15360 e2m1 on either, and 60 for 44 us where tiles
 * are cut.
 * F32: f32 rows of an e4m3 A, without the code of the other outputs: 96 registers
 * for 101, 512 x 6144 x 2560 24.6 us for 24.9. */
__device__ __forceinline__ bool rows16_ok(const void *p, int ld) { return ((uintptr_t)p & 15) == 0 && (ld & 7) == 0; }

template <int AF, bool F32, int BM, int BN>
__global__ __launch_bounds__(512, BM == 128 ? 4 : 2) void mx_gemm_tile_kernel(MxGemm P) {
    constexpr bool F8 = AF == IRIS_MX_FP8;
    constexpr int KS = F8 ? 1 : 2, PER = 4 / KS;   /* 128 columns per step, steps per 512 columns */
    constexpr int TWM = BM / 4, TWN = BN / 2, FM = TWM / 16, FN = TWN / 16;
    constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128;
    constexpr int A_LD = BM / 64, W_LD = BN / 32 / (F8 ? 2 : 1);   /* loads of a wave: half of A's rows; W's per step */
    constexpr int SC_LD = (BM + BN + 255) / 256;                  /* and of scales */
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * (A_BYTES + W_BYTES)];
    __shared__ u32x4 raw[BM + BN];
    __shared__ u32x4 scl[BM + BN];
    const int tiles = P.tiles_m * P.tiles_n, per_xcd = (tiles * P.chunks + 7) / 8;
    const int L = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (L >= tiles * P.chunks) return;
    const int chunk = L / tiles, t = L - chunk * tiles;
    const int first_m = t / (GROUP_M * P.tiles_n) * GROUP_M, gsz = min(P.tiles_m - first_m, GROUP_M);
    const int tg = t - first_m * P.tiles_n, tn = tg / gsz;
    const int m0 = (first_m + tg - tn * gsz) * BM, n0 = tn * BN;
    const int off = chunk * P.per_chunk;   /* the buffers below end where the rows do */
    mx_chunk<AF>(P, chunk);

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = wave >> 2, gw = wave & 3;
    const int wm = wave >> 1, wn = wave & 1;

    /* rows past the end read as zeros */
    const u32x4 a_rsrc = buffer_of(P.aq + (size_t)m0 * P.lda, min(BM, P.M - m0) * P.lda - off * (F8 ? 128 : 64));
    const u32x4 w_rsrc = buffer_of(P.wq + (size_t)n0 * P.ldw, min(BN, P.N - n0) * P.ldw - off * 64);
    const u32x4 as_rsrc = buffer_of(P.as + (size_t)m0 * P.ldas, min(BM, P.M - m0) * P.ldas - off * 4);
    const u32x4 ws_rsrc = buffer_of(P.ws + (size_t)n0 * P.ldws, min(BN, P.N - n0) * P.ldws - off * 4);
    const int nk = (P.steps + KS - 1) / KS, nw = (P.steps + 1) / 2, ng = (P.steps + 3) / 4;
    const uint32_t at0 = lds_at(lds), raw0 = lds_at(raw);
    auto hidden_lane = [&]() {   /* places are computed anew in each step: registers are short */
        int zero = 0;
        asm volatile("" : "+s"(zero));
        return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (unsigned)zero));
    };
    /* A load covers 8 rows: lane l row l / 8, place l % 8, chunk place ^ (row /
     * 2 % 8), which depends on the load by its parity. Of 256 columns that the
     * row has only half of, that half is read twice, not what lies behind. */
    auto place = [](int l, int ld, int row0, int par, int chunks) {
        return (row0 + (l >> 3)) * ld + ((((l & 7) ^ ((4 * par + (l >> 4)) & 7)) & chunks) << 4);
    };
    /* half h of A's rows, step kt, into stage dst % 2 */
    auto load_a = [&](int h, int kt, int dst, int l, int i) {
        const int j0 = h * (BM / 16) + gw * A_LD, par = i & 1;
        const int ch = !F8 && 2 * kt + 1 >= P.steps ? 3 : 7;
        load_lds16(a_rsrc, at0 + (dst & 1) * A_BYTES + (j0 + i) * 1024,
                   place(l, P.lda, (j0 + par) * 8, par, ch) + (i - par) * 8 * P.lda, kt * 128);
    };
    /* W's rows, 256 columns kw, into stage dst % 2; e4m3: half s of the loads */
    auto load_w = [&](int kw, int dst, int s, int l, int i) {
        const int j0 = (s * 4 + gw) * W_LD, par = i & 1;
        const int ch = 2 * kw + 1 >= P.steps ? 3 : 7;
        load_lds16(w_rsrc, at0 + 2 * A_BYTES + (dst & 1) * W_BYTES + (j0 + i) * 1024,
                   place(l, P.ldw, (j0 + par) * 8, par, ch) + (i - par) * 8 * P.ldw, kw * 128);
    };
    /* scales of 512 columns g: wave w of group 1 rows 64 (w + 4 i) .. of A's and then W's */
    auto load_scales = [&](int g) {
        const int l = hidden_lane();
#pragma unroll
        for (int i = 0; i < SC_LD; i++) {
            const int r = (gw + 4 * i) * 64;
            if (r < BM) load_lds16(as_rsrc, raw0 + r * 16, (r + l) * P.ldas, g * 16);
            else if (r < BM + BN) load_lds16(ws_rsrc, raw0 + r * 16, (r - BM + l) * P.ldws, g * 16);
        }
    };
    auto put_scales = [&]() {
        const int l = hidden_lane();
#pragma unroll
        for (int i = 0; i < SC_LD; i++) {
            const int r = (gw + 4 * i) * 64;
            if (r < BM + BN) scl[r + l] = bytes4x4(raw[r + l]);
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 a[2][FM], w[KS][FN];   /* e4m3: A's two halves of a row; e2m1: 128 columns each */
    int sa[FM], sw[FN];
    /* fragments of step kt, loads of later steps spread over the reads (either
     * alone takes most of a phase). Rows 16 apart are stored alike, chunk 4 +
     * lg is chunk lg XOR 4. */
    auto frags = [&](int kt, auto &&load, auto loads) {
        const int l = hidden_lane(), r = l & 15, c = ((l >> 4) ^ (r >> 1)) << 4;
        const int pa = (kt & 1) * A_BYTES + wm * TWM * 128 + r * 128 + c;
        const int pw = 2 * A_BYTES + ((F8 ? kt >> 1 : kt) & 1) * W_BYTES + wn * TWN * 128 + r * 128 + (F8 && (kt & 1) ? c ^ 64 : c);
        constexpr int LOADS = decltype(loads)::value, AR = 2 * FM, READS = AR + KS * FN;
        int at = 0;
#pragma unroll
        for (int i = 0; i < READS; i++) {
            if (i * LOADS / READS == at && at < LOADS) {
                __builtin_amdgcn_sched_barrier(0);
                load(l, at++);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i < AR) a[i / FM][i % FM] = *(const u32x4 *)(lds + (i < FM ? pa : pa ^ 64) + (i % FM) * 2048);
            else w[(i - AR) / FN][(i - AR) % FN] = *(const u32x4 *)(lds + (i - AR < FN ? pw : pw ^ 64) + ((i - AR) % FN) * 2048);
        }
    };
    auto scales = [&](bool first) {
        if (first) {
            const int l = hidden_lane(), at = (l & 15) * 16 + (l >> 4) * 4, pa = wm * TWM * 16 + at, pw = (BM + wn * TWN) * 16 + at;
#pragma unroll
            for (int i = 0; i < FM; i++) sa[i] = *(const int *)((const uint8_t *)scl + pa + i * 256);
#pragma unroll
            for (int j = 0; j < FN; j++) sw[j] = *(const int *)((const uint8_t *)scl + pw + j * 256);
        } else {
#pragma unroll
            for (int i = 0; i < FM; i++) sa[i] = (int)((uint32_t)sa[i] >> 8 * KS);
#pragma unroll
            for (int j = 0; j < FN; j++) sw[j] = (int)((uint32_t)sw[j] >> 8 * KS);
        }
    };
    auto mfmas = [&](bool both) {
        if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < FM; i++) {
                const u32x4 x = a[0][i], y = a[1][i];
                const i32x8 x8 = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
                const i32x8 hi = mx_part<true>(x8);
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = mx_mfma<AF>(w[0][j], hi, acc[i][j], sw[j], sa[i]);
                __builtin_amdgcn_sched_barrier(0);   /* one part in registers at a time */
                const i32x8 lo = mx_part<false>(x8);
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = mx_mfma<AF>(w[0][j], lo, acc[i][j], sw[j], sa[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (h && !both) break;
#pragma unroll
                for (int i = 0; i < FM; i++) {
                    const u32x4 x = a[h][i];
                    const i32x8 x8 = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < FN; j++) acc[i][j] = h ? mx_mfma4<1>(w[KS - 1][j], x8, acc[i][j], sw[j], sa[i]) : mx_mfma4<0>(w[0][j], x8, acc[i][j], sw[j], sa[i]);
                }
            }
        }
    };
    /* the compiler takes the scaled instruction for one that it may move past
     * barriers and into branches, and then keeps a K step's operands for it */
    auto pin = [&]() {
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) asm volatile("" ::"v"(acc[i][j]));
    };
    auto barrier = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };
    /* Phases between barriers: group 0 runs L(t), C(t) in phases 2t, 2t + 1,
     * group 1 in phases 2t + 1, 2t + 2; L reads step t's fragments, C runs its
     * matrix instructions. Loads are issued in L only (one that waits for the
     * address path holds up the instructions behind it), each into memory that
     * was last read in an earlier phase:
     *  - A's upper half is read by group 0 alone, in phase 2t: group 1 issues
     *    that of step t + 2 in L(t), phase 2t + 1, and waits for it at the end
     *    of L(t + 1), one phase before it is read;
     *  - A's lower half is read by group 1 alone, in phase 2t + 1, W by both:
     *    group 0 issues in L(t) W's next (e4m3: of the next 256 columns, half
     *    in either of two steps), waited for at the end of C(t), and A's lower
     *    half of step t + 1, waited for at the end of L(t + 1).
     * Loads of a wave complete in order, so a wait names the number of younger
     * ones. Scales of the next 512 columns: group 1 loads them in the first
     * step of 512 columns, behind its part of A, and writes them to their place
     * in the last; both groups read them in the first. Past the end the loads
     * repeat the last step's, into a stage that nothing reads again. */
    auto step0 = [&](int kt, auto s_) {
        constexpr int S = decltype(s_)::value;
        const int kw = min((F8 ? kt >> 1 : kt) + 1, nw - 1), ka = min(kt + 1, nk - 1);
        const int wdst = (F8 ? kt >> 1 : kt) + 1;
        scales(S == 0);
        frags(kt, [&](int l, int i) {
            if (i < W_LD) load_w(kw, wdst, F8 ? kt & 1 : 0, l, i);
            else load_a(1, ka, kt + 1, l, i - W_LD);
        }, Const<W_LD + A_LD>{});
        WAIT(W_LD + A_LD, 0);
        barrier();
        mfmas(2 * kt + 1 < P.steps);
        pin();
        WAIT(A_LD, 0);
        barrier();
    };
    auto step1 = [&](int kt, auto s_) {
        constexpr int S = decltype(s_)::value;
        if constexpr (S == PER - 1) {
            if constexpr (PER == 2) WAIT(0, 15);
            put_scales();
        }
        scales(S == 0);
        const int ka = min(kt + 2, nk - 1);
        frags(kt, [&](int l, int i) { load_a(0, ka, kt, l, i); }, Const<A_LD>{});
        if constexpr (S == 0) load_scales(min(kt / PER + 1, ng - 1));
        WAIT(A_LD + (S == 0 ? SC_LD : 0), 0);
        barrier();
        mfmas(2 * kt + 1 < P.steps);
        pin();
        if (kt + 1 < nk) barrier();
    };
    {
        const int l = hidden_lane(), k1 = min(1, nk - 1);
        if (grp) {
#pragma unroll
            for (int i = 0; i < A_LD; i++) load_a(0, 0, 0, l, i);
#pragma unroll
            for (int i = 0; i < A_LD; i++) load_a(0, k1, 1, l, i);
            load_scales(0);
            WAIT(0, 0);
            put_scales();
            WAIT(63, 0);
        } else {
#pragma unroll
            for (int s = 0; s < (F8 ? 2 : 1); s++)
#pragma unroll
                for (int i = 0; i < W_LD; i++) load_w(0, 0, s, l, i);
#pragma unroll
            for (int i = 0; i < A_LD; i++) load_a(1, 0, 0, l, i);
            WAIT(0, 0);
        }
    }
    barrier();
    const int whole = nk / PER * PER;
    if (grp) {
        barrier();
        for (int kt = 0; kt < whole; kt += PER) {
            step1(kt, Const<0>{});
            step1(kt + 1, Const<1>{});
            if constexpr (PER == 4) {
                step1(kt + 2, Const<2>{});
                step1(kt + 3, Const<3>{});
            }
        }
        if (whole < nk) step1(whole, Const<0>{});
        if constexpr (PER == 4) {
            if (whole + 1 < nk) step1(whole + 1, Const<1>{});
            if (whole + 2 < nk) step1(whole + 2, Const<2>{});
        }
    } else {
        for (int kt = 0; kt < whole; kt += PER) {
            step0(kt, Const<0>{});
            step0(kt + 1, Const<1>{});
            if constexpr (PER == 4) {
                step0(kt + 2, Const<2>{});
                step0(kt + 3, Const<3>{});
            }
        }
        if (whole < nk) step0(whole, Const<0>{});
        if constexpr (PER == 4) {
            if (whole + 1 < nk) step0(whole + 1, Const<1>{});
            if (whole + 2 < nk) step0(whole + 2, Const<2>{});
        }
    }
    WAIT(0, 0);   /* no load outstanding at exit */
    const int lane = hidden_lane(), lr = lane & 15, lg = lane >> 4;
    /* 16-bit output leaves through LDS, two of a wave's 16-row tiles at a time,
     * so that a row's part of a wave (256, 128 or 64 bytes) is written by
     * neighbouring lanes: 8-byte stores of 16 rows each took 10 us more of 4096
     * x 4096 x 2560, and of 1227 x 11520 x 3840, of whose tiles a fifth are cut,
     * 42.7 us rather than 35.5. */
    uint8_t *const st = lds + wave * 8192;
    static_assert(sizeof(lds) >= 8 * 8192, "a wave's part");
    if (!F32 && P.epi == IRIS_EPI_BF16 && rows16_ok(P.out, P.ldo)) {
        __syncthreads();   /* every wave is done with the stages */
#pragma unroll
        for (int ip = 0; ip < FM; ip += 2) {
#pragma unroll
            for (int j = 0; j < FN; j++) {
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (P.vec)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int n = n0 + wn * TWN + j * 16 + 4 * lg + r;
                        v[r] = n < P.N ? P.vec[n] : 0.0f;
                    }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const f32x4 x = acc[ip + i][j];
                    const int row = i * 16 + lr;
                    *(uint2 *)(st + row * (TWN * 2) + (((2 * j + (lg >> 1)) ^ (row & (FN * 2 - 1))) << 4) + (lg & 1) * 8) =
                        make_uint2((uint32_t)f2bf_hw(x[0] + v[0]) | (uint32_t)f2bf_hw(x[1] + v[1]) << 16,
                                   (uint32_t)f2bf_hw(x[2] + v[2]) | (uint32_t)f2bf_hw(x[3] + v[3]) << 16);
                }
            }
            const int m = m0 + wm * TWM + ip * 16, n = n0 + wn * TWN;
            constexpr int CPR = FN * 2;
#pragma unroll
            for (int k = 0; k < 32 * CPR / 64; k++) {
                const int c = k * 64 + lane, row = c / CPR, ch = c % CPR, col = n + ch * 8;
                const u32x4 x = *(const u32x4 *)(st + row * (TWN * 2) + ((ch ^ (row & (CPR - 1))) << 4));
                uint16_t *const out = (uint16_t *)P.out + (size_t)(m + row) * P.ldo + col;
                if (m + row >= P.M) continue;
                if (col + 8 <= P.N) *(u32x4 *)out = x;
                else
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (col + j < P.N) out[j] = (uint16_t)(x[j >> 1] >> (16 * (j & 1)));
            }
        }
        return;
    }
    if (!F32 && P.epi == IRIS_EPI_SWIGLU && !P.oq && rows16_ok(P.out, P.ldo)) {
        __syncthreads();
#pragma unroll
        for (int ip = 0; ip < FM; ip += 2) {
#pragma unroll
            for (int j = 0; j < FN / 4; j++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const f32x4 g = acc[ip + i][4 * j + h], u = acc[ip + i][4 * j + 2 + h];
                        uint16_t y[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) y[r] = f2bf_hw(mx_silu(g[r]) * u[r]);
                        const int row = i * 16 + lr;
                        *(uint2 *)(st + row * TWN + (((4 * j + 2 * h + (lg >> 1)) ^ (row & (FN - 1))) << 4) + (lg & 1) * 8) =
                            make_uint2((uint32_t)y[0] | (uint32_t)y[1] << 16, (uint32_t)y[2] | (uint32_t)y[3] << 16);
                    }
            const int m = m0 + wm * TWM + ip * 16, n = (n0 + wn * TWN) / 2;
            constexpr int CPR = FN;
#pragma unroll
            for (int k = 0; k < 32 * CPR / 64; k++) {
                const int c = k * 64 + lane, row = c / CPR, ch = c % CPR, col = n + ch * 8;
                const u32x4 x = *(const u32x4 *)(st + row * TWN + ((ch ^ (row & (CPR - 1))) << 4));
                /* N / 2 is a multiple of 32: 8 columns are inside or none */
                if (m + row < P.M && col < P.N / 2) *(u32x4 *)((uint16_t *)P.out + (size_t)(m + row) * P.ldo + col) = x;
            }
        }
        return;
    }
    const bool aligned = (P.ldo & 3) == 0 && ((uintptr_t)P.out & 15) == 0;
    if (!F32 && P.epi == IRIS_EPI_SWIGLU) {
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j += 4)
                mx_store_swiglu(P, m0 + wm * TWM + i * 16 + lr, n0 + wn * TWN + j * 16, acc[i][j], acc[i][j + 1],
                                acc[i][j + 2], acc[i][j + 3], aligned);
        return;
    }
#pragma unroll
    for (int i = 0; i < FM; i++) {
        const int m = m0 + wm * TWM + i * 16 + lr;
        if (m < P.M)
#pragma unroll
            for (int j = 0; j < FN; j++) mx_store4(P, m, n0 + wn * TWN + j * 16 + 4 * lg, acc[i][j], aligned);
    }
}

/* ---- argument checks ---- */
int pad_to(long long v, int to) { return (int)((v + to - 1) / to * to); }

int check_mx(const char *what, const iris_mx_t &a, int cols) {
    if (a.fmt != IRIS_MX_FP8 && a.fmt != IRIS_MX_FP4) return iris_set_error("%s: format %d", what, a.fmt);
    if (!a.q || !a.s) return iris_set_error("%s: null codes or scales", what);
    if (cols > (1 << 30)) return iris_set_error("%s: %d columns", what, cols);
    if (((uintptr_t)a.q & 15) || ((uintptr_t)a.s & 15) || (a.ld_q & 15) || (a.ld_s & 15))
        return iris_set_error("%s: codes and scales need 16-byte aligned rows", what);
    if (a.ld_q < iris_hip_mx_ld_codes(a.fmt, cols) || a.ld_s < iris_hip_mx_ld_scales(cols))
        return iris_set_error("%s: row strides %d, %d hold less than %d columns", what, a.ld_q, a.ld_s, cols);
    return 0;
}

bool rows16(const void *p, long long ld, int elt) { return ((uintptr_t)p & 15) == 0 && (ld * elt & 15) == 0; }

}  // namespace

extern "C" {

int iris_hip_mx_ld_codes(int fmt, int cols) {
    return fmt == IRIS_MX_FP4 ? pad_to(cols, 128) / 2 : pad_to(cols, 128);
}
int iris_hip_mx_ld_scales(int cols) { return pad_to(cols, 512) / 32; }

/* rows per launch: lanes counted in 32 bits */
static int rows_per_launch(uint32_t cpr) { return (int)((1u << 30) / cpr); }

int iris_hip_mx_quantize(const iris_mx_t *out, const void *x, int is_bf16, int ldx, int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    if (!out || !x) return iris_set_error("mx_quantize: null argument");
    if (check_mx("mx_quantize", *out, cols)) return -1;
    if (ldx < cols) return iris_set_error("mx_quantize: row stride %d of %d columns", ldx, cols);
    if (!iris_hip_available()) return -1;
    const int es = is_bf16 ? 2 : 4;
    const uint32_t cpr = (uint32_t)pad_to(cols, 128) / 8;
    const bool vec = rows16(x, ldx, es);
    for (int r0 = 0, nr; r0 < rows; r0 += nr) {
        nr = rows - r0 < rows_per_launch(cpr) ? rows - r0 : rows_per_launch(cpr);
        const uint32_t n = (uint32_t)nr * cpr;
        const dim3 grid((n + NT - 1) / NT);
        uint8_t *q = out->q + (size_t)r0 * out->ld_q, *s = out->s + (size_t)r0 * out->ld_s;
        const void *xr = (const char *)x + (size_t)r0 * ldx * es;
#define MX_Q(F, B)                                                                                                   \
    IRIS_LAUNCH((mx_quantize_kernel<F, B>), grid, dim3(NT), 0, iris_stream(), q, s, out->ld_q, out->ld_s, xr, ldx,   \
                cols, cpr, n, vec)
        if (out->fmt == IRIS_MX_FP8) {
            if (is_bf16) MX_Q(IRIS_MX_FP8, true);
            else MX_Q(IRIS_MX_FP8, false);
        } else {
            if (is_bf16) MX_Q(IRIS_MX_FP4, true);
            else MX_Q(IRIS_MX_FP4, false);
        }
#undef MX_Q
        if (iris_launch_check("mx_quantize_kernel")) return -1;
    }
    return 0;
}

int iris_hip_mx_dequantize(void *y, int is_bf16, int ldy, const iris_mx_t *a, int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    if (!a || !y) return iris_set_error("mx_dequantize: null argument");
    if (check_mx("mx_dequantize", *a, cols)) return -1;
    if (ldy < cols) return iris_set_error("mx_dequantize: row stride %d of %d columns", ldy, cols);
    if (!iris_hip_available()) return -1;
    const int es = is_bf16 ? 2 : 4;
    const uint32_t cpr = (uint32_t)(cols + 7) / 8;
    const bool vec = rows16(y, ldy, es);
    for (int r0 = 0, nr; r0 < rows; r0 += nr) {
        nr = rows - r0 < rows_per_launch(cpr) ? rows - r0 : rows_per_launch(cpr);
        const uint32_t n = (uint32_t)nr * cpr;
        const dim3 grid((n + NT - 1) / NT);
        const uint8_t *q = a->q + (size_t)r0 * a->ld_q, *s = a->s + (size_t)r0 * a->ld_s;
        void *yr = (char *)y + (size_t)r0 * ldy * es;
#define MX_D(F, B)                                                                                                   \
    IRIS_LAUNCH((mx_dequantize_kernel<F, B>), grid, dim3(NT), 0, iris_stream(), yr, ldy, q, s, a->ld_q, a->ld_s,     \
                cols, cpr, n, vec)
        if (a->fmt == IRIS_MX_FP8) {
            if (is_bf16) MX_D(IRIS_MX_FP8, true);
            else MX_D(IRIS_MX_FP8, false);
        } else {
            if (is_bf16) MX_D(IRIS_MX_FP4, true);
            else MX_D(IRIS_MX_FP4, false);
        }
#undef MX_D
        if (iris_launch_check("mx_dequantize_kernel")) return -1;
    }
    return 0;
}

}  /* extern "C" */

namespace {
/* Threads per row, us (rows that no cache holds; 128 / 256 / 512): 20000 x 320
 * 19.9 / 25.9 / 42.4; 512 x 2560 6.8 / 6.0 / 5.5; 8192 x 2160 50.7 / 48.3 /
 * 49.7; 4608 x 3840 50.8 / 45.5 / 44.1 (4.4 TB/s); 1000 x 10240 36.5 / 34.3 /
 * 25.9 */
template <int FMT, int DT> void launch_norm(const NormParams &P, int rows) {
    const int lanes = P.cols_pad / 8;
#define MX_N(TH, R) IRIS_LAUNCH((mx_rmsnorm_kernel<FMT, DT, TH, R>), dim3(rows), dim3(TH), 0, iris_stream(), P)
    if (lanes <= 64) MX_N(64, 1);
    else if (lanes <= 128) MX_N(128, 1);
    else if (lanes <= 256) MX_N(256, 1);
    else if (lanes <= 384 && rows >= 1024) MX_N(256, 2);
    else if (lanes <= 512) MX_N(512, 1);
    else if (lanes <= 1024) MX_N(512, 2);
    else if (lanes <= 2048) MX_N(512, 4);
    else MX_N(512, 0);
#undef MX_N
}
}  // namespace

extern "C" int iris_hip_mx_rmsnorm(const iris_mx_norm_t *a) {
    if (!a) return iris_set_error("mx_rmsnorm: null argument");
    if (a->rows <= 0 || a->cols <= 0) return 0;
    if (!a->x || !a->w || (a->d && !a->x_out) || (a->gate && !a->d)) return iris_set_error("mx_rmsnorm: null argument");
    if (check_mx("mx_rmsnorm", a->out, a->cols)) return -1;
    if (a->d && a->x_out == a->x && a->ldxo != a->ldx)
        return iris_set_error("mx_rmsnorm: in place with row strides %d and %d", a->ldx, a->ldxo);
    if (a->ldx < a->cols || (a->d && (a->ldd < a->cols || a->ldxo < a->cols)))
        return iris_set_error("mx_rmsnorm: row strides %d, %d, %d of %d columns", a->ldx, a->ldd, a->ldxo, a->cols);
    if (!iris_hip_available()) return -1;
    NormParams P;
    P.x = a->x; P.gate = a->gate; P.w = a->w; P.scale = a->scale; P.d = a->d; P.x_out = a->x_out;
    P.q = a->out.q; P.s = a->out.s; P.ld_q = a->out.ld_q; P.ld_s = a->out.ld_s;
    P.ldx = a->ldx; P.ldd = a->ldd; P.ldxo = a->ldxo;
    P.cols = a->cols; P.cols_pad = pad_to(a->cols, 128); P.eps = a->eps;
    P.vx = rows16(a->x, a->ldx, 4);
    P.vd = rows16(a->d, a->ldd, a->d_bf16 ? 2 : 4);
    P.vo = rows16(a->x_out, a->ldxo, 4);
    P.vg = rows16(a->gate, 0, 4);
    P.vw = rows16(a->w, 0, 4);
    P.vs = rows16(a->scale, 0, 4);
    const int dt = !a->d ? 0 : a->d_bf16 ? 2 : 1;
    const int most = 1 << 22;   /* rows of 512 threads in one launch, which takes 2^32 threads */
    for (int r0 = 0, nr; r0 < a->rows; r0 += nr) {
        nr = a->rows - r0 < most ? a->rows - r0 : most;
        if (a->out.fmt == IRIS_MX_FP8) {
            if (dt == 0) launch_norm<IRIS_MX_FP8, 0>(P, nr);
            else if (dt == 1) launch_norm<IRIS_MX_FP8, 1>(P, nr);
            else launch_norm<IRIS_MX_FP8, 2>(P, nr);
        } else {
            if (dt == 0) launch_norm<IRIS_MX_FP4, 0>(P, nr);
            else if (dt == 1) launch_norm<IRIS_MX_FP4, 1>(P, nr);
            else launch_norm<IRIS_MX_FP4, 2>(P, nr);
        }
        if (iris_launch_check("mx_rmsnorm_kernel")) return -1;
        P.x += (size_t)nr * P.ldx;
        if (dt) {
            P.d = (const char *)P.d + (size_t)nr * P.ldd * (dt == 2 ? 2 : 4);
            P.x_out += (size_t)nr * P.ldxo;
        }
        P.q += (size_t)nr * P.ld_q;
        P.s += (size_t)nr * P.ld_s;
    }
    return 0;
}

/* ---- which kernel, and whether K is split ---- */
namespace {
enum { MX_ROWS, MX_DIRECT, MX_TILE128, MX_TILE256 };
struct MxPlan {
    int kind, fm, fn, tiles_m, tiles_n, chunks, per_chunk;
};

/* waves that LDS holds of mx_gemm_rows_kernel, one block per CU and two */
template <int AF> void rows_waves(int fm, int *one, int *two) {
    switch (fm) {
    case 1: *one = RowsShape<AF, 1, 4>::WAVES; *two = RowsShape<AF, 1, 4>::WAVES2; break;
    case 2: *one = RowsShape<AF, 2, 4>::WAVES; *two = RowsShape<AF, 2, 4>::WAVES2; break;
    case 3: *one = RowsShape<AF, 3, 4>::WAVES; *two = RowsShape<AF, 3, 4>::WAVES2; break;
    default: *one = RowsShape<AF, 4, 4>::WAVES; *two = RowsShape<AF, 4, 4>::WAVES2; break;
    }
}

/* waves of a block: units of 256 columns, as evenly as those that LDS holds take
 * them; two blocks on a CU where there are more than CUs (37 x 19456 x 2560, 304
 * blocks: 17.0 us, 21.8 with one block of all waves) */
template <int AF> int rows_block_waves(int fm, int per_chunk, long long blocks) {
    int one, two;
    rows_waves<AF>(fm, &one, &two);
    const int most = blocks <= iris_cu_count() ? one : two;
    const int units = (per_chunk + 1) / 2;
    /* rounds of a unit per wave: its loads, about two units' instructions, and
     * the instructions of the SIMD with the most waves */
    int waves = 1;
    for (int w = 2, least = 3 * units; w <= most && w <= units; w++) {
        const int full = units / w, rest = units % w;
        const int cost = 2 * (full + (rest > 0)) + full * ((w + 3) / 4) + (rest + 3) / 4;
        if (cost < least) least = cost, waves = w;
    }
    return waves;
}
/* and of mx_gemm_direct_kernel: a wave per 512 columns, as evenly as 8 waves take them */
int direct_block_waves(int per_chunk) {
    const int groups = (per_chunk + 3) / 4, rounds = (groups + 7) / 8;
    return (groups + rounds - 1) / rounds;
}

template <int AF, int FM, int FN> int launch_rows_of(const MxGemm &P, unsigned blocks, int waves) {
    using Sh = RowsShape<AF, FM, FN>;
    const int smem = Sh::SCALES + waves * Sh::UNIT;
    static_assert(Sh::UNIT >= FM * FN * 1024, "the sums fit where the units were");
    static std::once_flag once;
    static hipError_t attr = hipSuccess;
    std::call_once(once, [] {
        attr = hipFuncSetAttribute((const void *)mx_gemm_rows_kernel<AF, FM, FN>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   Sh::SCALES + Sh::WAVES * Sh::UNIT);
    });
    if (iris_check(attr, "mx_gemm_rows smem attribute")) return -1;
    IRIS_LAUNCH((mx_gemm_rows_kernel<AF, FM, FN>), dim3(blocks), dim3(64 * waves), smem, iris_stream(), P);
    return 0;
}
template <int AF> int launch_rows(const MxGemm &P, const MxPlan &plan, unsigned blocks, int waves) {
    if (plan.kind == MX_DIRECT) {
        if (plan.fn == 1) IRIS_LAUNCH((mx_gemm_direct_kernel<AF, 1, 1>), dim3(blocks), dim3(64 * waves), waves * 1024, iris_stream(), P);
        else IRIS_LAUNCH((mx_gemm_direct_kernel<AF, 1, 4>), dim3(blocks), dim3(64 * waves), waves * 4096, iris_stream(), P);
        return 0;
    }
    if (plan.fm == 1) return launch_rows_of<AF, 1, 4>(P, blocks, waves);
    if (plan.fm == 2) return launch_rows_of<AF, 2, 4>(P, blocks, waves);
    if (plan.fm == 3) return launch_rows_of<AF, 3, 4>(P, blocks, waves);
    return launch_rows_of<AF, 4, 4>(P, blocks, waves);
}

/* The kernel, the tile and the number of K ranges of least estimated time (us),
 * over 190 products of 20 to 4608 rows 2 % slower than the fastest measured
 * choice on average, 13 of them by more than 10 % (64 to 130 rows x 19456 x 2560
 * through mx_gemm_rows_kernel, up to 26 % with e4m3 A and 47 % with e2m1). A
 * launch with its first loads and last stores is 6; a round of 256 x 256 tiles 3
 * and per K step 0.85 (e2m1 A) or 2.5 (e4m3); one of 128 x 128 tiles 2 and 0.32
 * or 0.72. f32 rows of an e4m3 A take the small tiles, which were never slower
 * for them. A split's partial sums and their second launch are 3 and their bytes
 * at 4 TB/s. Measured, us, e4m3 A to bf16: 300 x 19456 x 2560 35.2 on 128 x 128
 * tiles, 56.9 on 256 x 256; 1500 rows 133 and 122; 512 x 2560 x 9728 63.1
 * unsplit, 36.2 in 3 ranges; 64 x 6144 x 2560 11.1 through mx_gemm_rows_kernel,
 * 16.1 on tiles in 3 ranges. */
/* f32 rows of an e4m3 A: on 128 x 128 tiles only */
bool mx_f32_rows(const iris_mx_gemm_t &p) {
    return p.A.fmt == IRIS_MX_FP8 && p.epi != IRIS_EPI_SWIGLU && p.epi != IRIS_EPI_BF16;
}

MxPlan mx_plan(const iris_mx_gemm_t &p, int steps, size_t ws_bytes, double *estimate) {
    const int cus = iris_cu_count() > 0 ? iris_cu_count() : 1;
    /* the staging kernels reach rows by 32-bit offsets */
    long long ld = p.A.ld_q;
    for (int v : {p.W.ld_q, p.A.ld_s, p.W.ld_s}) ld = v > ld ? v : ld;
    const bool far = ld * 256 > 0x7fffffffLL;
    const bool f8 = p.A.fmt == IRIS_MX_FP8;
    MxPlan best;
    double least = 0.0;
    best.chunks = 0;
    auto consider = [&](int kind, int fm, int fn, int bm, int bn) {
        MxPlan q;
        q.kind = kind;
        q.fm = fm;
        q.fn = fn;
        q.tiles_m = (p.M + bm - 1) / bm;
        q.tiles_n = (p.N + bn - 1) / bn;
        const double tiles = (double)q.tiles_m * q.tiles_n, mn = (double)p.M * p.N;
        for (int c : {1, 2, 3, 4, 6, 8, 12, 16}) {
            q.per_chunk = c == 1 ? steps : ((steps + c - 1) / c + 3) / 4 * 4;
            q.chunks = (steps + q.per_chunk - 1) / q.per_chunk;
            if (c > 1 && (q.chunks == 1 || q.chunks * mn * 4 > (double)ws_bytes || mn > 1e9)) break;
            const double blocks = tiles * q.chunks;
            double us;
            if (kind == MX_TILE128 || kind == MX_TILE256) {
                const bool big = kind == MX_TILE256;
                const double step = f8 ? (big ? 2.5 : 0.72) : big ? 0.85 : 0.32;
                us = 6 + ceil(blocks / cus) * ((big ? 3 : 2) + step * q.per_chunk);
            } else if (kind == MX_ROWS) {
                int one, two;
                if (f8) rows_waves<IRIS_MX_FP8>(fm, &one, &two);
                else rows_waves<IRIS_MX_FP4>(fm, &one, &two);
                const int units = (q.per_chunk + 1) / 2, waves = blocks > cus ? two : one;
                us = 8 + ceil(blocks / (2.0 * cus)) * ((units + waves - 1) / waves) * (1.2 + (f8 ? 0.35 : 0.25) * fm) * (blocks > cus ? 0.85 : 1.0);
            } else us = 6 + ceil(blocks / (4.0 * cus)) * (q.per_chunk + 31) / 32 * 2.0;   /* 8 waves of 4 steps each */
            if (q.chunks > 1) us += 3 + q.chunks * mn * 8 / 4e6;
            if (!best.chunks || us < least) {
                best = q;
                least = us;
            }
        }
    };
    if (far) consider(MX_DIRECT, 1, 4, 16, 64);
    else if (p.M <= 16 && p.epi != IRIS_EPI_SWIGLU) {
        /* 16 rows of W per block keep enough blocks in flight without LDS
         * (6144 x 2560, one row: 4.9 us, 5.4 through LDS); a gate / up group
         * needs 64 */
        consider(MX_DIRECT, 1, 1, 16, 16);
    } else {
        const int fm = p.M < 64 ? (p.M + 15) / 16 : 4;
        if (p.M <= 256) consider(MX_ROWS, fm, 4, 16 * fm, 64);
        if (p.M > 16) {
            consider(MX_TILE128, 0, 0, 128, 128);
            if (!mx_f32_rows(p)) consider(MX_TILE256, 0, 0, 256, 256);
        }
    }
    *estimate = least;
    return best;
}

/* Rows of A for a launch of their own: as many as fill whole rounds of 256 x
 * 256 tiles, where those behind them, planned by themselves, take less than
 * their part of a last round (4608 x 3840 x 10240 e2m1, 270 tiles for 256 CUs:
 * 132 -> 110 us). 0: one launch. */
int mx_main_rows(const iris_mx_gemm_t &p, int steps, size_t ws_bytes, double whole) {
    const int cus = iris_cu_count() > 0 ? iris_cu_count() : 1;
    const int tm = (p.M + 255) / 256, tn = (p.N + 255) / 256;
    const long long rounds = (long long)tm * tn / cus;
    if (mx_f32_rows(p) || rounds < 1 || rounds * cus < tn) return 0;
    const int rows = (int)(rounds * cus / tn) * 256;
    if (rows >= p.M) return 0;
    iris_mx_gemm_t part = p;
    double us[2];
    part.M = rows;
    (void)mx_plan(part, steps, ws_bytes, &us[0]);
    part.M = p.M - rows;
    (void)mx_plan(part, steps, ws_bytes, &us[1]);
    return us[0] + us[1] < 0.95 * whole ? rows : 0;
}
/* a checked problem; ws_bytes 0: no workspace */
int mx_run(const iris_mx_gemm_t *p, float *ws, size_t ws_bytes) {
    const bool swiglu = p->epi == IRIS_EPI_SWIGLU, mx = swiglu && p->mx_out.q;
    const int nout = swiglu ? p->N / 2 : p->N;
    MxGemm P;
    P.aq = p->A.q; P.as = p->A.s; P.lda = p->A.ld_q; P.ldas = p->A.ld_s;
    P.wq = p->W.q; P.ws = p->W.s; P.ldw = p->W.ld_q; P.ldws = p->W.ld_s;
    P.out = p->out; P.vec = p->vec; P.M = p->M; P.N = p->N; P.ldo = p->ldo; P.epi = p->epi;
    P.steps = pad_to(p->K, 128) / 128;
    P.oq = mx ? p->mx_out.q : nullptr; P.os = p->mx_out.s;
    P.ldoq = p->mx_out.ld_q; P.ldos = p->mx_out.ld_s; P.ofmt = p->mx_out.fmt;
    double whole;
    const MxPlan plan = mx_plan(*p, P.steps, ws_bytes, &whole);
    if (const int rows = mx_main_rows(*p, P.steps, ws_bytes, whole)) {
        iris_mx_gemm_t part = *p;
        part.M = rows;
        if (mx_run(&part, ws, ws_bytes)) return -1;
        part.M = p->M - rows;
        part.A.q += (size_t)rows * p->A.ld_q;
        part.A.s += (size_t)rows * p->A.ld_s;
        if (mx) {
            part.mx_out.q += (size_t)rows * p->mx_out.ld_q;
            part.mx_out.s += (size_t)rows * p->mx_out.ld_s;
        } else part.out = (char *)p->out + (size_t)rows * p->ldo * (swiglu || p->epi == IRIS_EPI_BF16 ? 2 : 4);
        return mx_run(&part, ws, ws_bytes);
    }
    P.tiles_m = plan.tiles_m; P.tiles_n = plan.tiles_n; P.chunks = plan.chunks; P.per_chunk = plan.per_chunk;
    const bool f8 = p->A.fmt == IRIS_MX_FP8;
    long long blocks = (long long)plan.tiles_m * plan.tiles_n * plan.chunks;
    if (plan.kind > MX_DIRECT) blocks = (blocks + 7) / 8 * 8;   /* as many for each XCD */
    const int waves = plan.kind > MX_DIRECT ? 8
                    : plan.kind == MX_DIRECT ? direct_block_waves(plan.per_chunk)
                    : f8 ? rows_block_waves<IRIS_MX_FP8>(plan.fm, plan.per_chunk, blocks)
                         : rows_block_waves<IRIS_MX_FP4>(plan.fm, plan.per_chunk, blocks);
    if (blocks * 64 * waves > 0xffffffffLL)
        return iris_set_error("mx_gemm: %d x %d output of K %d, more than 2^32 threads", p->M, p->N, p->K);
    if (!iris_hip_available()) return -1;
    MxGemm R = P;
    if (plan.chunks > 1) {
        P.out = ws; P.ldo = p->N; P.vec = nullptr; P.epi = IRIS_EPI_F32; P.oq = nullptr;
    }
    if (plan.kind <= MX_DIRECT) {
        if (f8 ? launch_rows<IRIS_MX_FP8>(P, plan, (unsigned)blocks, waves)
               : launch_rows<IRIS_MX_FP4>(P, plan, (unsigned)blocks, waves))
            return -1;
    } else {
        const dim3 grid((unsigned)blocks);
#define MX_T(F, X, T) IRIS_LAUNCH((mx_gemm_tile_kernel<F, X, T, T>), grid, dim3(512), 0, iris_stream(), P)
        if (plan.kind == MX_TILE256) {
            if (!f8) MX_T(IRIS_MX_FP4, false, 256);
            else MX_T(IRIS_MX_FP8, false, 256);
        } else {
            if (!f8) MX_T(IRIS_MX_FP4, false, 128);
            else if (P.epi != IRIS_EPI_BF16 && P.epi != IRIS_EPI_SWIGLU) MX_T(IRIS_MX_FP8, true, 128);
            else MX_T(IRIS_MX_FP8, false, 128);
        }
#undef MX_T
    }
    if (iris_launch_check("mx_gemm kernel")) return -1;
    if (plan.chunks > 1) {
        const int cols = mx ? pad_to(nout, 128) : nout;
        const uint32_t cpr = (uint32_t)(cols + 7) / 8, n = (uint32_t)p->M * cpr;
        IRIS_LAUNCH(mx_reduce_kernel, dim3((n + NT - 1) / NT), dim3(NT), 0, iris_stream(), R, (const float *)ws, n, cpr);
        return iris_launch_check("mx_reduce_kernel");
    }
    return 0;
}
}  // namespace

extern "C" int iris_hip_mx_gemm(const iris_mx_gemm_t *p, float *ws, size_t ws_bytes) {
    if (!p) return iris_set_error("mx_gemm: null problem");
    if (p->M <= 0 || p->N <= 0) return 0;
    if (p->K <= 0) return iris_set_error("mx_gemm: K %d", p->K);
    if (p->M > (1 << 30) || p->N > (1 << 30)) return iris_set_error("mx_gemm: %d x %d output", p->M, p->N);
    if (check_mx("mx_gemm A", p->A, p->K) || check_mx("mx_gemm W", p->W, p->K)) return -1;
    if (p->W.fmt != IRIS_MX_FP4) return iris_set_error("mx_gemm: weights of format %d, not IRIS_MX_FP4", p->W.fmt);
    const bool swiglu = p->epi == IRIS_EPI_SWIGLU, mx = swiglu && p->mx_out.q;
    if (!swiglu && p->epi != IRIS_EPI_F32 && p->epi != IRIS_EPI_BF16 && p->epi != IRIS_EPI_GATED_ADD &&
        p->epi != IRIS_EPI_ADD)
        return iris_set_error("mx_gemm: epilogue %d", p->epi);
    if (swiglu && (p->N % 64 || p->vec)) return iris_set_error("mx_gemm: SWIGLU needs N %% 64 == 0 (%d) and no vec", p->N);
    if (!swiglu && p->mx_out.q) return iris_set_error("mx_gemm: mx_out is for SWIGLU");
    const int nout = swiglu ? p->N / 2 : p->N;
    if (mx ? check_mx("mx_gemm output", p->mx_out, nout) : !p->out ? iris_set_error("mx_gemm: null output") : 0) return -1;
    if (!mx && p->ldo < nout) return iris_set_error("mx_gemm: output row stride %d of %d columns", p->ldo, nout);
    (void)iris_hip_available();   /* the plan counts the device's CUs; sizes are refused without one, too */
    return mx_run(p, ws, ((uintptr_t)ws & 15) || !ws ? 0 : ws_bytes);
}
