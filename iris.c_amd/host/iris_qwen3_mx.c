/*
 * iris_qwen3_mx.c - the Qwen3 text encoder with microscaled linears: weights of
 * 4 bits, their inputs 8-bit rows (iris_hip.h's iris_mx_t). No counterpart in
 * the reference, whose linears are f32 (iris_qwen3.c:496-538); the layer is the
 * one of iris_qwen3.c with other products and norms.
 */
#include "iris_qwen3_model.h"

#include <stdio.h>
#include <string.h>

static int fail(const char *what) {
    fprintf(stderr, "qwen3: %s: %s\n", what, iris_hip_last_error());
    return -1;
}

#define CK(x) do { if (x) return fail(#x); } while (0)

static void release(iris_mx_t *a) {
    iris_hip_free(a->q);
    iris_hip_free(a->s);
    memset(a, 0, sizeof(*a));
}

static int room(iris_mx_t *a, int fmt, size_t rows, int cols) {
    a->fmt = fmt;
    a->ld_q = iris_hip_mx_ld_codes(fmt, cols);
    a->ld_s = iris_hip_mx_ld_scales(cols);
    a->q = (uint8_t *)iris_hip_malloc(rows * a->ld_q);
    a->s = (uint8_t *)iris_hip_malloc(rows * a->ld_s);
    return a->q && a->s ? 0 : -1;
}

static void free_all(qwen3_model_t *m) {
    for (int i = 0; m->L && i < m->layers; i++) {
        qlayer_t *l = &m->L[i];
        release(&l->qkv_mx); release(&l->o_mx); release(&l->gate_up_mx); release(&l->down_mx);
    }
    release(&m->a_mx); release(&m->attn_mx); release(&m->mlp_mx);
    iris_hip_free(m->d_mx);
    m->d_mx = NULL;
}

/* residual stream += d (NULL: as it is), then the RMSNorm of it in 8 bits */
static int mx_rms(qwen3_model_t *m, const float *d, const float *w, int S) {
    iris_mx_norm_t a;
    memset(&a, 0, sizeof(a));
    a.x = a.x_out = m->x; a.ldx = a.ldxo = m->hidden;
    a.d = d; a.ldd = m->hidden;
    a.w = w; a.out = m->a_mx; a.rows = S; a.cols = m->hidden; a.eps = QWEN3_RMS_NORM_EPS;
    if (!d) a.x_out = NULL;
    return iris_hip_mx_rmsnorm(&a);
}

static int mx_gemm(qwen3_model_t *m, const iris_mx_t *A, const iris_mx_t *W, void *out, int ldo, int M, int N, int K, int epi,
                   const iris_mx_t *mx_out) {
    iris_mx_gemm_t p;
    memset(&p, 0, sizeof(p));
    p.A = *A; p.W = *W; p.out = out; p.ldo = ldo; p.M = M; p.N = N; p.K = K; p.epi = epi;
    if (mx_out) p.mx_out = *mx_out;
    return iris_hip_mx_gemm(&p, m->ws, m->ws_bytes);
}

static int first(qwen3_model_t *m, int S) { return mx_rms(m, NULL, m->L[0].ln1, S); }

/* a layer, from its normalised input rows to those of the next layer: the
 * residual's additions, of f32 sums as in the bf16 layer, run in the norms that
 * read the stream next; the last layer's, which no norm follows, in its product */
static int layer(qwen3_model_t *m, const qlayer_t *l, const float *next_ln1, int S, int n_real) {
    const int h = m->hidden, qd = m->heads * HD, kd = m->kv_heads * HD, I = m->inter;
    CK(mx_gemm(m, &m->a_mx, &l->qkv_mx, m->qkv, qd + 2 * kd, S, qd + 2 * kd, h, IRIS_EPI_BF16, NULL));
    if (iris_qwen3_attend(m, l, S, n_real)) return -1;
    CK(iris_hip_mx_quantize(&m->attn_mx, m->attn, 1, qd, S, qd));
    CK(mx_gemm(m, &m->attn_mx, &l->o_mx, m->d_mx, h, S, h, qd, IRIS_EPI_F32, NULL));
    CK(mx_rms(m, m->d_mx, l->ln2, S));
    CK(mx_gemm(m, &m->a_mx, &l->gate_up_mx, NULL, 0, S, 2 * I, h, IRIS_EPI_SWIGLU, &m->mlp_mx));
    if (!next_ln1) {
        CK(mx_gemm(m, &m->mlp_mx, &l->down_mx, m->x, h, S, h, I, IRIS_EPI_GATED_ADD, NULL));
        return 0;
    }
    CK(mx_gemm(m, &m->mlp_mx, &l->down_mx, m->d_mx, h, S, h, I, IRIS_EPI_F32, NULL));
    CK(mx_rms(m, m->d_mx, next_ln1, S));
    return 0;
}

int qwen3_model_quantize(qwen3_model_t *m) {
    if (!m) return -1;
    if (m->mx_layer) return 0;
    const int h = m->hidden, I = m->inter, qd = m->heads * HD, kd = m->kv_heads * HD, S = QWEN3_MAX_SEQ_LEN;
    int rc = room(&m->a_mx, IRIS_MX_FP8, S, h) || room(&m->attn_mx, IRIS_MX_FP8, S, qd) ||
             room(&m->mlp_mx, IRIS_MX_FP8, S, I) || !(m->d_mx = (float *)iris_hip_malloc((size_t)S * h * sizeof(float)));
    for (int i = 0; !rc && i < m->layers; i++) {
        qlayer_t *l = &m->L[i];
        rc = room(&l->qkv_mx, IRIS_MX_FP4, (size_t)qd + 2 * kd, h) || room(&l->o_mx, IRIS_MX_FP4, h, qd) ||
             room(&l->gate_up_mx, IRIS_MX_FP4, 2 * (size_t)I, h) || room(&l->down_mx, IRIS_MX_FP4, h, I) ||
             iris_hip_mx_quantize(&l->qkv_mx, l->qkv, 1, h, qd + 2 * kd, h) ||
             iris_hip_mx_quantize(&l->o_mx, l->o, 1, qd, h, qd) ||
             iris_hip_mx_quantize(&l->gate_up_mx, l->gate_up, 1, h, 2 * I, h) ||
             iris_hip_mx_quantize(&l->down_mx, l->down, 1, I, h, I);
    }
    if (iris_hip_sync() || rc) {
        fail("quantize");
        free_all(m);
        return -1;
    }
    for (int i = 0; i < m->layers; i++) {
        qlayer_t *l = &m->L[i];
        iris_hip_free(l->qkv); iris_hip_free(l->o); iris_hip_free(l->gate_up); iris_hip_free(l->down);
        l->qkv = l->o = l->gate_up = l->down = NULL;
    }
    m->mx_first = first;
    m->mx_layer = layer;
    m->mx_free = free_all;
    return 0;
}
