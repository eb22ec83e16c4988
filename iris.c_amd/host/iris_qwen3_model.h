/* iris_qwen3_model.h - the text encoder's model as its translation units see it:
 * iris_qwen3.c (bf16 linears, the forward) and iris_qwen3_mx.c (microscaled
 * linears). */
#ifndef IRIS_QWEN3_MODEL_H
#define IRIS_QWEN3_MODEL_H

#include "../../include/iris_hip.h"
#include "../../include/iris_qwen3.h"

#define HD 128

typedef struct {
    uint16_t *qkv;       /* [(Hq + 2 Hkv) * 128][h]: Q rows, K rows (head dims permuted), V rows */
    uint16_t *o;         /* [h][Hq * 128] */
    uint16_t *gate_up;   /* [2 I][h], gate and up rows interleaved in 32-row groups */
    uint16_t *down;      /* [h][I] */
    float *ln1, *ln2;    /* [h] */
    float *q_norm, *k_norm;   /* [128], permuted like the Q / K rows */
    iris_mx_t qkv_mx, o_mx, gate_up_mx, down_mx;   /* the same rows in 4 bits, instead (quantized models) */
} qlayer_t;

struct qwen3_model {
    int hidden, inter, heads, kv_heads, vocab, layers;
    float rope_theta;
    int mode;                 /* 0 Flux, 1 Z-Image */
    uint16_t *embed;          /* [vocab][h] */
    qlayer_t *L;
    /* work buffers for QWEN3_MAX_SEQ_LEN tokens */
    int *ids;
    float *x, *out;           /* x [S][h] residual stream; out: the extracted layers, [3][S][h] or [S][3h] */
    float *host_out;          /* pinned copy of out, one extracted layer after the other; or NULL */
    uint16_t *a, *qkv, *q, *k, *vt, *attn, *mlp;
    float *rope_cos, *rope_sin;   /* [S][128], value of pair p at 2p and 2p+1 */
    float *rp_cos, *rp_sin;       /* [S][64], value of pair p at p (the attention's Q prologue) */
    float *ws;                    /* split-K partial products */
    size_t ws_bytes;
    /* microscaled linears (qwen3_model_quantize; NULL: bf16): the first norm, a
     * layer, and what they hold, with the inputs of the products */
    int (*mx_first)(qwen3_model_t *m, int S);
    int (*mx_layer)(qwen3_model_t *m, const qlayer_t *l, const float *next_ln1, int S, int n_real);
    void (*mx_free)(qwen3_model_t *m);
    iris_mx_t a_mx, attn_mx, mlp_mx;
    float *d_mx;                  /* [S][h], what a product adds to the stream */
};

/* Q, K, V rows of a layer (m->qkv) to its attention output (m->attn) */
int iris_qwen3_attend(qwen3_model_t *m, const qlayer_t *l, int S, int n_real);

#endif
