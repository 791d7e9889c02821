/*
 * atlas_train.h — C-ABI of the MI355X (gfx950) kernels of a retriever TRAINING step (libatlas_train.so).
 *
 * The retriever's training forward and backward (src/atlas.py:452-465 over src/modeling_bert.py) are PyTorch operators in the
 * reference. These entry points compute its layers on packed tokens (only real tokens are rows):
 *   attention with its backward pass, dense layers with a fused epilogue and theirs, activations kept in 8 bits for the
 *   backward pass, and BERT's layer norm (uncentred second moment, modeling_bert.py:104-114) with its backward pass.
 *
 * Conventions (all entry points): those of atlas_hip.h
 *   - plain pointers and sizes; every buffer is caller-owned DEVICE memory; structs are host memory and read before the call returns
 *   - nothing allocates, frees or synchronises; work is enqueued on `stream` (a hipStream_t as void*; NULL = the null stream) of the
 *     CURRENT device, which has to be the buffers' device; capturable into a hipGraph (kernels only, no memset nodes)
 *   - no mutable state, no environment variables: everything a call needs is in its arguments. Two calls at once need two workspaces
 *   - results are the same bits from call to call: no atomics
 *   - return value: 0 = enqueued, > 0 = hipError_t of a launch, < 0 = ATLAS_TRAIN_E_*
 *   - element types ATLAS_TRAIN_F16 | _F32 | _BF16 of inputs, outputs and gradients; sums and statistics are fp32
 */
#ifndef ATLAS_TRAIN_H
#define ATLAS_TRAIN_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ATLAS_TRAIN_ABI_VERSION 3

#define ATLAS_TRAIN_E_BADARG      (-1)
#define ATLAS_TRAIN_E_WORKSPACE   (-2)
#define ATLAS_TRAIN_E_UNSUPPORTED (-3)

#define ATLAS_TRAIN_F16  0
#define ATLAS_TRAIN_F32  1
#define ATLAS_TRAIN_BF16 2

int atlas_train_abi_version(void);

/* ---- attention over packed sequences ---------------------------------------------------------------------------------
 *   S = scale * q k^T,  P = softmax over the sequence's visible keys,  out = (P * keep * keep_scale) v
 * Sequence b owns query rows q_offsets[b] .. q_offsets[b+1]-1 and key rows k_offsets[b] .. k_offsets[b+1]-1 (int32 [batch+1] on the
 * device, non-decreasing; values outside [0, total] are clamped into it). Query head h reads key head h / (heads / kv_heads).
 *   q, dout            [total_q][heads][dim] by strides in ELEMENTS (rows, heads); dim contiguous; every row 16-byte aligned, and
 *                      no row stride of 2^24 bytes or more
 *   k, v               [total_k][kv_heads][dim] likewise
 *   key_mask           NULL or uint8 [total_k]: 0 hides the key. A hidden key's k and v rows are never used (NaN there is harmless)
 *   keep               forward: NULL or uint8 [total_q][heads][keep_cols] by strides, each 0 or 1: 0 drops the probability (dropout);
 *                      key j of a sequence is column j; columns from keep_cols on count as dropped; no row stride of 2^26 or more
 *   keep_bits          uint32 [heads][total_q][(keep_cols + 31) / 32]: the same decisions as bits. Written by the forward pass (NULL: not
 *                      wanted) as far as sequences reach, read by the backward pass (NULL: no dropout), which does not look at keep
 *   max_q, max_k       launch sizes: the longest sequence (a longer one is still computed, more slowly)
 *   out, dq            [total_q][heads][dim] contiguous;  dk, dv: [total_k][kv_heads][dim] contiguous. Rows of no sequence: zeros
 *   lse                fp32 [heads][total_q]: log2 of the row's sum of 2^(S log2 e); +inf for a row without a visible key, whose
 *                      output and gradients are zeros
 *   out_rest           NULL or uint8 [total_q][heads][64 (dim <= 64) or 128], 16-byte aligned, 16-bit types only: what rounding left of out, in 1/128ths of half
 *                      a step and an order of its own. Written by the forward pass as far as sequences reach, read by the backward pass: rowsum(dout . out), whose
 *                      error every dS of the row has, is then that of the output before it was rounded
 *   delta              fp32 [heads][total_q], workspace of the backward pass
 *   ws                 fp32 sums of parts where a few long walks are split over workgroups (each then takes a second launch that joins
 *                      them in a fixed order): atlas_attention_workspace_bytes(), which looks at everything in the struct but ws;
 *                      16-byte aligned; 0 = none needed
 * dim: a multiple of 8, at most 128; total_q and total_k below 2^31 - 255. The backward pass recomputes P from lse: two launches (dq
 * and delta; dk and dv).
 */
typedef struct {
    const void *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    const int32_t *q_offsets, *k_offsets;
    int64_t total_q, total_k;
    int batch, heads, kv_heads, dim, max_q, max_k, dtype, keep_cols;
    const uint8_t *key_mask, *keep;
    int64_t keep_row, keep_head;
    uint32_t* keep_bits;
    float scale, keep_scale;
    void* out;
    float* lse;
    uint8_t* out_rest;
    /* backward pass only */
    const void* dout;
    int64_t dout_row, dout_head;
    void *dq, *dk, *dv;
    float* delta;
    void* ws;
    size_t ws_bytes;
} atlas_attention_args;
size_t atlas_attention_workspace_bytes(const atlas_attention_args* a, int backward);
int atlas_attention_forward(const atlas_attention_args* a, void* stream);
int atlas_attention_backward(const atlas_attention_args* a, void* stream);

/* ---- dense layer -----------------------------------------------------------------------------------------------------
 * atlas_gemm: C[m][n] = sum_k A(m,k) B(k,n) with an optional epilogue, products on the matrix cores, sums in fp32
 *   a_layout 0: A stored [m][k] (lda = row stride), 1: stored [k][m];  b_layout 0: B stored [n][k] (a Linear weight), 1: [k][n]
 *   b_codes: B ([k][n], b_layout 1) is given as 8-bit codes (see atlas_compress) instead of `b`: codes uint8 [k][ldb], scales uint8
 *            [k][ldb/32], ldb a multiple of 32
 *   epilogue, in this order, each optional: z = C + bias[n]; save z as `dtype` (save_z) or as 8-bit codes of the fp32 value
 *            (save_z_codes / save_z_scales, row strides n rounded up to 32 and that / 32); y = gelu(z) (act 1: the exact erf form);
 *            y *= keep ? keep_scale : 0; y += residual; y is rounded once into c
 *   ws:      fp32 partial products where k is split over workgroups (a second launch joins them in a fixed order and has the epilogue):
 *            atlas_gemm_workspace_bytes(), which looks at everything in the struct but ws; 16-byte aligned; 0 = none needed
 */
typedef struct {
    const void *a, *b;
    int64_t lda, ldb, ldc;
    int m, n, k, dtype, a_layout, b_layout;
    const uint8_t *b_codes, *b_scales;
    const void* bias;
    int act;
    void* save_z;
    uint8_t *save_z_codes, *save_z_scales;
    const uint8_t* keep;           /* [m][n] contiguous */
    float keep_scale;
    const void* residual;          /* [m][n], row stride ld_residual */
    int64_t ld_residual;
    void* c;
    void* ws;
    size_t ws_bytes;
} atlas_gemm_args;
size_t atlas_gemm_workspace_bytes(const atlas_gemm_args* a);
int atlas_gemm(const atlas_gemm_args* a, void* stream);

/* dz = dy * (keep ? keep_scale : 0) * gelu'(z), db = sum over rows of dz (fp32, before dz is rounded)
 *   z (contiguous [m][n]) or z_codes / z_scales (as atlas_gemm saved them), or neither (no activation); keep or NULL;
 *   dz NULL: only the sums;  db NULL: only dz.  dy by row stride; dz contiguous.  ws (only with db): floats, atlas_linear_dz_workspace_bytes(m, n) */
size_t atlas_linear_dz_workspace_bytes(int64_t m, int n);
int atlas_linear_dz(const void* dy, int64_t ld_dy, const void* z, const uint8_t* z_codes, const uint8_t* z_scales, const uint8_t* keep,
                    float keep_scale, int64_t m, int n, int dtype, void* dz, void* db, void* ws, size_t ws_bytes, void* stream);

/* ---- activations in 8 bits ---------------------------------------------------------------------------------------------
 * Every 32 consecutive values of a row (the last group of a row may be shorter) share a power of two s = 2^e, the smallest
 * with amax / s <= 448, e in [-126, 120]; a value is stored as the e4m3 code of x / s (round to nearest even), s as the byte e + 127.
 * Where the nearest code stands for more than the largest finite value of x's type, the code below it is taken (saved pre-activations: of fp32).
 * A value that is not finite becomes the code NaN and does not count for amax; a group without a finite value other than 0 has e = -126.
 *   x [m][n] row stride ldx;  codes [m][ld], scales [m][ld/32], ld = n rounded up to 32 (codes behind a row's end are 0)
 */
int atlas_compress(const void* x, int64_t ldx, int64_t m, int n, int dtype, uint8_t* codes, uint8_t* scales, void* stream);
int atlas_decompress(const uint8_t* codes, const uint8_t* scales, int64_t m, int n, int dtype, void* out, void* stream);

/* ---- layer norm with the uncentred second moment --------------------------------------------------------------------------
 *   mu = mean(x), r = (mean(x^2) + eps)^-1/2, y = w (x - mu) r + b         stats: fp32 [m][2] = (mu, r) for the backward pass
 *   backward: g = w dy; dx = r (g - mean(g)) - x r^3 mean(g (x - mu)); dw = sum_rows dy (x - mu) r; db = sum_rows dy
 * x, dy: [m][n] by row stride; y, dx contiguous; dx, (dw, db) may be NULL.  ws (only with dw): floats, atlas_layer_norm_workspace_bytes(m, n)
 */
int atlas_layer_norm_forward(const void* x, int64_t ldx, const void* w, const void* b, float eps, int64_t m, int n, int dtype, void* y, float* stats,
                             void* stream);
size_t atlas_layer_norm_workspace_bytes(int64_t m, int n);
int atlas_layer_norm_backward(const void* x, int64_t ldx, const void* w, const float* stats, const void* dy, int64_t ld_dy, int64_t m, int n, int dtype,
                              void* dx, void* dw, void* db, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ATLAS_TRAIN_H */
