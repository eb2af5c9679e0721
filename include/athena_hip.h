/* libathena_hip.so -- C ABI of the MI355X (gfx950) kernels behind Athena's hybrid
 * attention/CTC ASR training step.
 *
 * The reference has no native interface on this path: its arithmetic is delegated to
 * TensorFlow/Keras ops and Horovod from Python.  Each entry point below therefore cites the
 * reference call site (file:line under athena/ of the reference) whose TensorFlow op(s) it
 * replaces; the Python side of the drop-in binds them with ctypes (athena_amd/_lib.py).
 *
 * Conventions
 *   - every buffer is device memory owned by the caller; the library never allocates, frees or
 *     keeps a pointer after the call returns;
 *   - all work is enqueued on ``stream``; no call synchronises the device;
 *   - tensors are row-major and batch-major; ``dtype`` arguments take ATHENA_F32 or ATHENA_BF16
 *     and name the storage type of activations (arithmetic is fp32 everywhere; bf16 GEMMs
 *     accumulate in fp32 on the matrix cores); parameters, their gradients, statistics and
 *     losses are always fp32;
 *   - return value 0 on success, a negative ATHENA_E_* code otherwise, with a message kept
 *     per thread for athena_last_error(); nothing throws or aborts.
 */
#ifndef ATHENA_HIP_H
#define ATHENA_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* athena_stream_t; /* a hipStream_t */

enum { ATHENA_OK = 0, ATHENA_E_SHAPE = -1, ATHENA_E_ALIGN = -2, ATHENA_E_LAUNCH = -3, ATHENA_E_UNSUPPORTED = -4 };
enum { ATHENA_F32 = 0, ATHENA_BF16 = 1 };
enum {
    ATHENA_ACT_NONE = 0,
    ATHENA_ACT_RELU6 = 1,      /* tf.nn.relu6 */
    ATHENA_ACT_GELU = 2,       /* tanh-form gelu, athena/layers/functional.py:101-112 */
    ATHENA_ACT_MUL_DGELU = 3,  /* backward: multiply by gelu'(aux), aux = saved pre-activation */
    ATHENA_ACT_MUL_DRELU6 = 4, /* backward: multiply by [0 < aux < 6], aux = saved relu6 output */
    /* the other entries of ACTIVATIONS, athena/layers/commons.py:494-506 (the ffn activation of
     * athena/layers/transformer.py:262-270,346-354): ATHENA_ACT_UNARY + k applies function k,
     * ATHENA_ACT_MUL_DUNARY + k multiplies by its derivative at aux = the saved pre-activation.
     * k: 0 relu, 1 elu, 2 selu, 3 leaky_relu (alpha 0.2), 4 sigmoid, 5 softplus, 6 softsign, 7 tanh,
     *    8 relu6 */
    ATHENA_ACT_UNARY = 16,
    ATHENA_ACT_MUL_DUNARY = 32
};
enum { ATHENA_UNARY_COUNT = 9 };

const char* athena_last_error(void);
int athena_abi_version(void);

/* Measurement hook (no counterpart in the reference; its only timing is the wall-clock sec/iter of
 * athena/utils/metric_check.py:82-91).  Between athena_timing_begin and athena_timing_end every
 * kernel the library launches carries a pair of events that receive the kernel's own begin and end
 * timestamps; athena_timing_count = launches so far in the session, athena_timing_end returns the
 * total, athena_timing_read waits for launches [first, first + count) and writes their durations in
 * milliseconds, in launch order.  Not to be used while a stream is being captured into a graph. */
int athena_timing_begin(void);
int athena_timing_count(void);
int athena_timing_end(void);
int athena_timing_read(int first, int count, float* ms);

/* ---------------------------------------------------------------------------------------------
 * Dense layers.  Replaces tf.keras.layers.Dense / tf.matmul in
 * athena/layers/attention.py:115-137,151-153,169, athena/layers/transformer.py:262-282,346-366,
 * athena/models/speech_transformer.py:102,130,151 and athena/models/mtl_seq2seq.py:62,83, and
 * their gradients (tape.gradient, athena/solver.py:96).
 *
 *   C[M,N] = epilogue(alpha * op(A)[M,K] * op(B)[K,N])
 *   epilogue(x): x += bias[n]; C_pre = x (if given); x = act(x) or x * act'(aux);
 *                x *= dropout multiplier (if drop_p > 0); if accumulate: x += C; C = x
 *   split_k > 1: partial products are added to C with fp32 atomics; C must be fp32 and
 *                zero-filled (or hold the value to accumulate onto); no bias/act/dropout.
 *   split_k = 0: the library picks the split for the shape (no bias/act/dropout).
 *                With ``workspace`` of at least athena_gemm_workspace_bytes(M,N,K,in_dtype) bytes
 *                (16-byte aligned) the partial products are stored there and added up by a second
 *                kernel in a fixed order: bit-reproducible, C need not be initialised, and C may
 *                be bf16 (the second kernel rounds once).  Without it the library zero-fills an
 *                fp32 C and uses fp32 atomics; a bf16 C is then not split.
 *   b_colsum   : trans_a && !trans_b only (a weight gradient x^T.dy): also writes
 *                b_colsum[n] = sum_k B[k,n] -- the bias gradient (tape.gradient of the Dense
 *                bias, athena/solver.py:96) -- from the B tiles the product stages anyway.
 * bf16 operands need K, lda, ldb multiples of 8 and 16-byte aligned bases; rows are read in
 * 8-element pieces, so lda >= roundup8(M) when trans_a and ldb >= roundup8(N) when !trans_b.
 */
typedef struct athena_gemm_desc {
    const void* A;
    const void* B;
    void* C;
    void* C_pre;          /* optional pre-activation copy of C (same dtype / ld) */
    const float* bias;    /* optional [N] */
    const void* aux;      /* operand of the backward epilogues, [M, ldaux] */
    const uint64_t* rng_state; /* device: {seed, step}; needed when drop_p > 0 */
    int32_t M, N, K;
    int32_t trans_a;      /* 0: A is [M,K] (lda); 1: A is [K,M] (lda) */
    int32_t trans_b;      /* 0: B is [K,N] (ldb); 1: B is [N,K] (ldb) */
    int32_t lda, ldb, ldc, ldaux;
    int32_t in_dtype;     /* dtype of A and B */
    int32_t out_dtype;    /* dtype of C and C_pre */
    int32_t aux_dtype;
    int32_t act;          /* ATHENA_ACT_* */
    int32_t accumulate;   /* C += result (single writer per element) */
    int32_t split_k;      /* >= 1, or 0 = automatic */
    float alpha;
    float drop_p;
    uint32_t rng_site;    /* distinguishes dropout sites; same site + state reproduces the mask */
    float* b_colsum;      /* optional [N], see above */
    void* workspace;      /* optional split-K scratch, see above */
    int64_t workspace_bytes;
} athena_gemm_desc;

int athena_gemm(const athena_gemm_desc* d, athena_stream_t stream);
/* ``count`` independent products, same results as ``count`` athena_gemm calls.  bf16 products with
 * one operand layout (trans_a, trans_b) and split_k all 0 or all 1 run as ONE launch (plus one
 * reduction launch); the split-K scratch of the whole group is descs[0].workspace.  This is how
 * the weight gradients of a transformer layer (all Dense kernels of athena/layers/transformer.py
 * :262-282 and athena/layers/attention.py:115-137 under tape.gradient, athena/solver.py:96) and its
 * q/k/v projections (attention.py:151-153) are issued. */
int athena_gemm_grouped(const athena_gemm_desc* descs, int count, athena_stream_t stream);

/* Weight gradients of many Dense layers in ONE launch: C_i[M_i,N_i] = A_i^T B_i (fp32, overwritten)
 * with A_i = the layer input [K_i, M_i] and B_i = the output gradient [K_i, N_i], both bf16 row-major,
 * and bsum_i[N_i] (may be NULL) = the column sums of B_i, i.e. the bias gradient.  Replaces the
 * per-variable products of tape.gradient(loss, trainable_variables) for Dense kernels and biases,
 * athena/solver.py:96 (Dense layers of athena/layers/transformer.py:262-282, attention.py:115-137,
 * speech_transformer.py:98-130, mtl_seq2seq.py:62).  Every 256x256 output tile is one workgroup
 * that runs down the whole contraction, so there is no K split, no workspace and a fixed summation
 * order.  athena_gemm_wgrad_plan checks a HOST copy of the table, fills first_tile / tiles_m, REORDERS
 * the items (tiles that share an operand are placed on one XCD, the eight XCDs get equal work) and
 * returns the number of workgroups to launch in *total_tiles; the caller then places the table in
 * device memory (it must stay valid until the launch has run) and calls athena_gemm_wgrad_table with
 * the device copy and that number. */
typedef struct athena_wgrad_item {
    const void* A;      /* bf16 [K, lda], lda % 8 == 0, lda >= roundup8(M) */
    const void* B;      /* bf16 [K, ldb], ldb % 8 == 0, ldb >= roundup8(N) */
    float* C;           /* fp32 [M, ldc] */
    float* bsum;        /* fp32 [N] or NULL */
    int32_t M, N, K;
    int32_t lda, ldb, ldc;
    int32_t first_tile, tiles_m;    /* filled by athena_gemm_wgrad_plan */
} athena_wgrad_item;
int athena_gemm_wgrad_plan(athena_wgrad_item* items_host, int count, int* total_tiles);
int athena_gemm_wgrad_table(const athena_wgrad_item* table_dev, int count, int total_tiles, athena_stream_t stream);
/* A table with few tiles leaves most of the chip idle for the length of its longest contraction (the
 * weight gradients of ONE piece of a backward pass that a data-parallel step cuts into pieces, so that
 * each piece's gradients can be exchanged while the next piece runs: Horovod's per-tensor overlap,
 * athena/solver.py:170-172).  athena_gemm_wgrad_split (host only) cuts the contractions of such a
 * table into parts: items whose K is long are replaced by ``parts`` items over consecutive row ranges
 * of A and B, each writing its fp32 partial product (and partial column sums) into ``workspace``, and
 * ``folds`` lists the sums that remain: dst[j] = sum over parts of src[part * part_stride + j], in a
 * fixed order, so the result does not depend on which part finishes first.  Call it once with
 * out_items == NULL to learn *need_floats, *out_count and *fold_count (nothing else is written), then
 * with the buffers; hand ``out_items`` to athena_gemm_wgrad_plan / _table and, behind the table, the
 * device copy of ``folds`` to athena_gemm_wgrad_fold with *fold_blocks.  A table that already fills the
 * chip (``chip_tiles`` workgroups, 0 = 256) comes back unchanged with *fold_count == 0. */
typedef struct athena_wgrad_fold {
    float* dst;             /* [n] overwritten */
    const float* src;       /* parts vectors of n floats, part_stride apart */
    int64_t n;
    int64_t part_stride;
    int32_t parts;
    int32_t first_block;    /* filled by athena_gemm_wgrad_split */
} athena_wgrad_fold;
int athena_gemm_wgrad_split(const athena_wgrad_item* items_host, int count, int chip_tiles, float* workspace,
                            int64_t workspace_floats, int64_t* need_floats, athena_wgrad_item* out_items,
                            int out_capacity, int* out_count, athena_wgrad_fold* folds, int fold_capacity,
                            int* fold_count, int* fold_blocks);
int athena_gemm_wgrad_fold(const athena_wgrad_fold* folds_dev, int count, int blocks, athena_stream_t stream);
int64_t athena_gemm_workspace_bytes(int M, int N, int K, int in_dtype);

/* out[n] = sum_m X[m,n]  (bias gradients).  out is overwritten. */
int athena_colsum(const void* X, int dtype, int M, int N, int ld, float* out, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Residual add + dropout + LayerNormalization(epsilon) and its gradient.
 * Replaces ``norm(x + dropout(sublayer))`` of athena/layers/transformer.py:305,308,384,386,387.
 *   z = a + dropout(b) ; y = gamma * (z - mean) * rstd + beta        (rows x d)
 * b may be NULL (plain LayerNorm of a).  bwd: dgamma/dbeta are overwritten; da = dL/da = dz;
 * db = dz * dropout multiplier (may be NULL when drop_p == 0: then db == da).
 */
int athena_add_layernorm_fwd(const void* a, const void* b, const float* gamma, const float* beta, float eps,
                             int rows, int d, int dtype, float drop_p, const uint64_t* rng_state,
                             uint32_t rng_site, void* z, void* y, float* mean, float* rstd,
                             athena_stream_t stream);
/* The same with the residual stream in fp32 beside the tensors products read (the reference keeps it
 * in fp32 throughout, athena/layers/transformer.py:296-310): a_f32 (may be NULL) = a in fp32, taken in its
 * place for the sum; y_f32 (may be NULL) = an fp32 copy of y for the launch that takes y as ITS a.
 * With either, mean, rstd and y come from the unrounded sum and only the stored z and y are rounded.
 * Needs d % 8 == 0, d <= 512 and 16-byte aligned operands (ATHENA_E_UNSUPPORTED otherwise). */
int athena_add_layernorm_fwd_wide(const void* a, const float* a_f32, const void* b, const float* gamma,
                                  const float* beta, float eps, int rows, int d, int dtype, float drop_p,
                                  const uint64_t* rng_state, uint32_t rng_site, void* z, void* y, float* y_f32,
                                  float* mean, float* rstd, athena_stream_t stream);
int athena_add_layernorm_bwd(const void* dy, const void* z, const float* mean, const float* rstd,
                             const float* gamma, int rows, int d, int dtype, float drop_p,
                             const uint64_t* rng_state, uint32_t rng_site, int accumulate_da, void* da,
                             void* db, float* dgamma, float* dbeta, void* workspace, int64_t workspace_bytes,
                             athena_stream_t stream);
/* With a workspace of this many bytes the column sums dgamma/dbeta are reduced through per-workgroup
 * slabs in a fixed order (reproducible); without one (NULL) fp32 atomics are used. */
int64_t athena_add_layernorm_bwd_workspace_bytes(int rows, int d);
/* Deferred column sums: athena_add_layernorm_bwd with dgamma == dbeta == NULL leaves its
 * athena_add_layernorm_bwd_slabs(rows, d) partial sums ([slab][2][d] fp32) in the workspace and
 * athena_ln_fold_batched adds up the slabs of any number of such calls in one launch (a training
 * step has one LayerNorm gradient per residual connection, tf.keras LayerNormalization of
 * athena/layers/transformer.py:286-288,366-372; folding them together saves a launch each).
 * _slabs returns 0 when d does not qualify (d % 8 != 0 or d > 512).  ``items`` is device memory. */
typedef struct athena_ln_fold_item {
    const float* slabs;   /* workspace of one deferred athena_add_layernorm_bwd call */
    float* dgamma;        /* [d] overwritten */
    float* dbeta;         /* [d] overwritten */
    int32_t nblk;         /* athena_add_layernorm_bwd_slabs(rows, d) of that call */
    int32_t d;
} athena_ln_fold_item;
int athena_add_layernorm_bwd_slabs(int rows, int d);
int athena_ln_fold_batched(const athena_ln_fold_item* items, int count, int max_d, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * The part of a post-LN transformer layer after the attention kernel, one launch per direction
 * (bf16, d_model == 256, dff a multiple of 256; anything else returns ATHENA_E_UNSUPPORTED and the
 * caller runs the separate Dense / LayerNorm entry points).
 * Replaces, in TransformerEncoderLayer.call (athena/layers/transformer.py:296-310) and
 * TransformerDecoderLayer.call (:374-388), everything but the q/k/v projections and the attention
 * itself: the output projection of MultiHeadAttention (athena/layers/attention.py:166-169),
 * ``norm1(src + dropout1(src2))``, ``linear2(dropout(activation(linear1(src))))`` with the tanh-form
 * gelu, and ``norm2(src + dropout2(src2))``:
 *   z1 = x + dropout(ctx Wo + bo)                 y1 = LayerNorm1(z1)
 *   hpre = y1 W1 + b1     h = dropout(gelu(hpre))
 *   z2 = y1 + dropout(h W2 + b2)                  y2 = LayerNorm2(z2)
 * dff == 0 stops after y1 (an attention sub-layer that is not followed by the feed-forward block).
 * Weights are the fragment-tiled bf16 copies written by athena_refresh_shadows: rows = outputs
 * (contraction over inputs) for the forward pass, rows = inputs for the backward pass.  Dropout decisions are those of athena_gemm /
 * athena_add_layernorm_fwd at the same sites: element index row * width + column of the tensor
 * the mask applies to.  Everything the backward pass reads again is written out: z1, y1, mean1,
 * rstd1, hpre, h, z2, mean2, rstd2 (and y2, the layer output).
 * Backward: given dy = dL/dy2 (dL/dy1 when dff == 0) it writes df = dL/d(h W2 + b2) and
 * dh = dL/dhpre and da = dL/d(ctx Wo + bo) (the right-hand operands of the three weight gradients;
 * their column sums are the bias gradients), dx = dL/dx through the residual path, dctx = dL/dctx,
 * and one slab [2][256] of partial dgamma | dbeta sums per workgroup and LayerNorm
 * (athena_layer_tail_workgroups(rows) slabs each; athena_ln_fold_batched adds them up). */
typedef struct athena_layer_tail_fwd_desc {
    int32_t rows, d_model, dff, reserved;
    const void* ctx;            /* [rows, 256] attention context */
    const void* x;              /* [rows, 256] residual input */
    const void* wo_t;           /* [256, 256] output projection, tiled copy with rows = outputs */
    const float* bo;
    const float* gamma1;
    const float* beta1;
    const void* w1_t;           /* first Dense, tiled copy with rows = its dff outputs */
    const float* b1;
    const void* w2_t;           /* second Dense, tiled copy with rows = its 256 outputs */
    const float* b2;
    const float* gamma2;
    const float* beta2;
    float eps, drop_p;
    const uint64_t* rng_state;
    uint32_t site_res1, site_ffn, site_res2, reserved2;
    void* z1;
    void* y1;
    float* mean1;
    float* rstd1;
    void* hpre;                 /* [rows, dff] */
    void* h;                    /* [rows, dff] */
    void* z2;
    void* y2;
    float* mean2;
    float* rstd2;
    /* optional (next_w_t[0] != NULL): next_out[m] = y2 next_w[m] + next_b[m], m = 0..2 -- the
     * q / k / v projections of the NEXT layer's self-attention (MultiHeadAttention.call,
     * athena/layers/attention.py:150-153) on this layer's output while its rows are on the CU;
     * next_w_t: [256, 256] tiled copies with rows = outputs, next_out: [rows, 256].  With dff == 0 one
     * product, index 0 only: y1 next_w[0] + next_b[0] (the q projection of the cross-attention that
     * follows a decoder's self-attention sub-layer) */
    const void* next_w_t[3];
    const float* next_b[3];
    void* next_out[3];
    /* optional: x_f32 [rows, 256] = the residual input x in fp32, read for the residual sum in place of
     * x; y_out_f32 [rows, 256] = an fp32 copy of the final LayerNorm output (y2, or y1 when dff == 0)
     * for the launch that takes this output as its residual input.  The residual stream then runs
     * through a stack of layers unrounded (athena/layers/transformer.py:296-310 keeps it in fp32). */
    const float* x_f32;
    float* y_out_f32;
} athena_layer_tail_fwd_desc;
typedef struct athena_layer_tail_bwd_desc {
    int32_t rows, d_model, dff, reserved;
    const void* dy;
    const void* z2;
    const float* mean2;
    const float* rstd2;
    const float* gamma2;
    const void* hpre;
    const void* w2;             /* second Dense, tiled copy with rows = its dff inputs */
    const void* w1;             /* first Dense, tiled copy with rows = its 256 inputs */
    const void* z1;
    const float* mean1;
    const float* rstd1;
    const float* gamma1;
    const void* wo;             /* output projection, tiled copy with rows = its inputs */
    float drop_p, reserved2;
    const uint64_t* rng_state;
    uint32_t site_res1, site_ffn, site_res2, reserved3;
    void* df;                   /* [rows, 256] */
    void* dh;                   /* [rows, dff] */
    void* da;                   /* [rows, 256] */
    void* dx;                   /* [rows, 256] */
    void* dctx;                 /* [rows, 256] */
    float* slab2;               /* [workgroups][2][256] */
    float* slab1;
    /* optional (add_dqkv != NULL): dy is taken as dy + add_dqkv (add_w[0] | add_w[1] | add_w[2])^T
     * -- the gradient that reaches this layer's output through the q / k / v projections of the
     * layer behind it (the input gradient of its three Dense layers, attention.py:150-153) added here
     * instead of by a launch of its own; add_dqkv: [rows, 768] = dq | dk | dv, add_w: [256, 256] tiled
     * copies with rows = the projections' inputs.  With dff == 0 a single product: add_dqkv is
     * [rows, 256] (the dq of a cross-attention that takes its queries from this sub-layer) and only
     * add_w[0] is read */
    const void* add_dqkv;
    const void* add_w[3];
} athena_layer_tail_bwd_desc;
int athena_layer_tail_workgroups(int rows);
int athena_layer_tail_fwd(const athena_layer_tail_fwd_desc* d, athena_stream_t stream);
int athena_layer_tail_bwd(const athena_layer_tail_bwd_desc* d, athena_stream_t stream);

/* Products with a contraction of 256 and many output columns, bf16: for c < nblock
 *   out[c][rows, 256] (row stride ldo[c]) = x[rows, 256] (row stride ldx) * W_c (+ bias[c])
 * with W_c a [256 in, 256 out] block given as w_tiled[c], its fragment-tiled copy with the block's
 * COLUMNS as rows (athena_refresh_shadows).  One launch in which a workgroup keeps 16 or 32 rows of x
 * in LDS and walks over all blocks.  Replaces, in one launch each: the key / value Dense layers of the
 * cross-attention of ALL decoder layers applied to the encoder output (attention.py:150-152 inside
 * transformer.py:374-388; 12 blocks), the q / k / v Dense layers of an attention that takes one input
 * (attention.py:150-153; 3 blocks) and the input gradient of a Dense layer with 256 outputs (the
 * backward of speech_transformer.py:95; blocks = rows of the kernel in groups of 256, the tiled copy
 * with the kernel's ROWS as rows).  bias and its entries may be NULL.  Operands 16-byte aligned, ldx and
 * ldo multiples of 8; at most ATHENA_PANEL_MAX_BLOCKS blocks. */
#define ATHENA_PANEL_MAX_BLOCKS 20
int athena_panel_gemm(const void* x, long ldx, int rows, int nblock, const void* const* w_tiled,
                      const float* const* bias, void* const* out, const long* ldo, athena_stream_t stream);
/* The other way round, a long contraction and 256 output columns, bf16:
 *   out[rows, 256] (row stride ldo) (+)= act( sum_c a[rows, 256 c .. 256 c + 255] W_c + bias )
 * for c < nchunk, a [rows, kcols] (row stride lda; kcols a multiple of 8, 256 (nchunk - 1) < kcols <=
 * 256 nchunk: a short last piece meets the ZERO rows its weight block must have there), W_c given as
 * w_tiled[c] = the start of the piece inside a fragment-tiled copy whose rows are the OUTPUT columns and
 * whose contraction length is ldw[c] (256 for a [256 x 256] matrix of its own, in_features for a piece
 * of a Dense kernel's tiled copy with the kernel's columns as rows).  act: ATHENA_ACT_NONE or
 * ATHENA_ACT_RELU6; accumulate != 0 adds to what out holds (rounded once).  Replaces the x_net Dense
 * (speech_transformer.py:95) and the sum over all decoder layers of the input gradients of the
 * cross-attention key / value Dense layers (backward of attention.py:151-152). */
int athena_panel_gemm_k(const void* a, long lda, int rows, int kcols, int nchunk, const void* const* w_tiled,
                        const long* ldw, const float* bias, int act, int accumulate, void* out, long ldo,
                        athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Multi-head scaled dot-product attention, fused (no [B,h,Tq,Tk] tensor in memory).
 * Replaces ScaledDotProductAttention.call, athena/layers/attention.py:47-70, between the head
 * split and merge of MultiHeadAttention.call (:155-167).
 *   q [B,Tq,h,dk] (token stride ldq), k/v [B,Tk,h,dk] (ldk, ldv), out [B,Tq,h,dk] (ldo)
 *   s = q.k * scale + (-1e9 if key_mask[b,j] or (causal and j > i + causal - 1))   -- the
 *   reference's additive fp32 mask -- ; p = softmax_j(s) ; out = p.v ; lse[b,h,i] = logsumexp_j(s)
 *   causal: 0 = every key is visible; c >= 1 = query i sees keys j <= i + c - 1.  c = 1 is the
 *   decoder's look-ahead mask (athena/utils/misc.py:68-90), c = look_ahead + 1 the band of a
 *   unidirectional encoder, tf.linalg.band_part(ones, -1, look_ahead) of attention.py:55-58.
 * bwd recomputes p from lse; dq/dk/dv have the layouts/strides of q/k/v and are overwritten.
 */
int athena_mha_fwd(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv,
                   const uint8_t* key_mask, int causal, int B, int h, int Tq, int Tk, int dk, int dtype,
                   float scale, void* out, int ldo, float* lse, athena_stream_t stream);
int athena_mha_bwd(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv,
                   const uint8_t* key_mask, int causal, int B, int h, int Tq, int Tk, int dk, int dtype,
                   float scale, const void* out, const void* dout, int ldo, const float* lse,
                   float* delta /* scratch [B,h,Tq] */, void* dq, void* dk_, void* dv, int lddq, int lddk,
                   int lddv, athena_stream_t stream);

/* The attention weights as a tensor: weights[b, h, i, j] = softmax_j(q_i . k_j * scale + mask), fp32
 * [B, h, Tq, Tk] -- the second return value of MultiHeadAttention.call, athena/layers/attention.py:161,171
 * (ScaledDotProductAttention.call :47-70).  Mask arguments as for athena_mha_fwd.  The training step
 * does not call it. */
int athena_mha_weights(const void* q, const void* k, int ldq, int ldk, const uint8_t* key_mask, int causal, int B,
                       int h, int Tq, int Tk, int dk, int dtype, float scale, float* weights, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Conv2D(3x3, stride 2, "same", no bias) on NHWC tensors, as implicit GEMM.
 * Replaces layers.Conv2D of athena/models/speech_transformer.py:77-84,87-94 and its gradients.
 * "same" padding with stride 2: out = ceil(in/2); pad_total = max((out-1)*2+3-in, 0);
 * pad_before = pad_total/2.
 *   fwd  : in [B,H,W,Cin] -> out [B,Ho,Wo,Cout]; ``w`` is the HWIO kernel [3][3][Cin][Cout]
 *          (w_layout 0) or its transposed copy [Cout][3][3][Cin] (w_layout 1, the fast layout
 *          for bf16); optional ``colstats`` [2*Cout] (fp64, zeroed by the call) receives the
 *          per-channel sum and sum of squares of ``out``.
 *   dgrad: dout -> din, ``w`` is the HWIO kernel [3][3][Cin][Cout]; din overwritten.
 *   dgrad: with ``relu6_out`` (the [B,H,W,Cin] relu6 activation that was this convolution's
 *          input, same dtype) the result is also multiplied by the relu6 gate [0 < relu6_out < 6],
 *          i.e. din becomes the gradient w.r.t. the pre-activation.
 *   wgrad: dw (HWIO, fp32) overwritten.  The contraction over pixels is split; with a
 *          ``workspace`` of athena_conv3x3s2_wgrad_workspace_bytes(...) bytes the partial sums
 *          are reduced in a fixed order, otherwise fp32 atomics are used.
 * bf16 needs Cin % 8 == 0 and Cout % 8 == 0 (a Cin that is not, e.g. the 1-channel fbank
 * input, goes through athena_conv3x3s2_small_cin_*).
 */
int athena_conv3x3s2_fwd(const void* in, const void* w, int w_layout, void* out, int B, int H, int W, int Cin,
                         int Cout, int dtype, double* colstats, athena_stream_t stream);
int athena_conv3x3s2_dgrad(const void* dout, const void* w_hwio, void* din, int B, int H, int W, int Cin,
                           int Cout, int dtype, const void* relu6_out, athena_stream_t stream);
int athena_conv3x3s2_wgrad(const void* in, const void* dout, float* dw_hwio, int B, int H, int W, int Cin,
                           int Cout, int dtype, void* workspace, int64_t workspace_bytes,
                           athena_stream_t stream);
int64_t athena_conv3x3s2_wgrad_workspace_bytes(int B, int H, int W, int Cin, int Cout, int dtype);
/* Direct kernels for a small number of input channels (Cin <= 4); ``in`` and ``w`` (HWIO) are
 * fp32, ``out``/``dout`` have ``dtype``. */
int athena_conv3x3s2_small_cin_fwd(const float* in, const float* w_hwio, void* out, int B, int H, int W,
                                   int Cin, int Cout, int dtype, double* colstats, athena_stream_t stream);
int athena_conv3x3s2_small_cin_wgrad(const float* in, const void* dout, float* dw_hwio, int B, int H, int W,
                                     int Cin, int Cout, int dtype, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * First front-end layer fused: Conv2D(3x3, stride 2, same, ONE input channel) ->
 * BatchNormalization (training: batch statistics) -> relu6.  Replaces the first
 * Conv2D/BatchNormalization/ReLU(max_value=6) triple of athena/models/speech_transformer.py:72-84
 * and its gradient.  The pre-activation tensor is never stored: with one input channel its batch
 * statistics follow in closed form from 9 + 81 moments of the input.
 *   stats : moments (fp64, athena_conv1_moments_len() elements: 9 tap sums, then the 9x9 tap
 *           products, then scratch for the per-workgroup partial sums; the backward pass reads the
 *           first 90) and colstats[2*Cout] (sum, sum of squares of the pre-activations; feed
 *           athena_bn_finalize).
 *   fwd   : out[B,Ho,Wo,Cout] = relu6(BN(conv(in))).  infer = 0: s0 = mean_rstd [2*Cout];
 *           infer = 1: s0 = moving mean, s1 = moving variance.  A bf16 ``out`` never rounds a
 *           value below 6 up to 6, so [0 < out < 6] is the exact relu6 gate.
 *   bwd   : g = gradient w.r.t. the BN output, already multiplied by the relu6 gate (see
 *           athena_conv3x3s2_dgrad) when relu6_out is NULL; otherwise g is the gradient w.r.t. the
 *           relu6 output and the gate [0 < relu6_out < 6] is applied while g is read (relu6_out =
 *           the forward result, same dtype).  With ``beta`` (may be NULL) as well, bf16 and Cout % 64 == 0
 *           the gate is worked out again from in / w / mean_rstd / gamma / beta -- the forward pass's own
 *           arithmetic, so the same gate -- and relu6_out is not read: half the memory traffic.
 *           Writes dw (HWIO [9][Cout]), dgamma, dbeta.  ``workspace`` needs
 *           athena_conv1_bn_bwd_workspace_bytes(Cout) bytes.
 * Cout must be 8 * a divisor of 256. */
int64_t athena_conv1_moments_len(void);
int athena_conv1_bn_stats(const float* in, const float* w_hwio, int B, int H, int W, int Cout, double* moments,
                          double* colstats, athena_stream_t stream);
int athena_conv1_bn_relu6_fwd(const float* in, const float* w_hwio, const float* s0, const float* s1,
                              const float* gamma, const float* beta, float eps, int infer, int B, int H, int W,
                              int Cout, int dtype, void* out, athena_stream_t stream);
int64_t athena_conv1_bn_bwd_workspace_bytes(int Cout);
int athena_conv1_bn_bwd(const float* in, const void* g, const void* relu6_out, const float* w_hwio,
                        const double* moments,
                        const float* mean_rstd, const float* gamma, const float* beta, int B, int H, int W, int Cout,
                        int dtype, void* workspace, int64_t workspace_bytes, float* dw_hwio, float* dgamma,
                        float* dbeta, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * BatchNormalization (training mode, channels last) fused with relu6.
 * Replaces layers.BatchNormalization() + tf.nn.relu6, athena/models/speech_transformer.py:85-86,95-97.
 *   finalize: from colstats {sum, sumsq} over ``rows`` rows: mean, biased var; writes
 *             mean_rstd[0:C] = mean, [C:2C] = 1/sqrt(var+eps); moving_mean/var updated with
 *             ``momentum`` (moving_var with the unbiased variance) when not NULL.
 *   apply   : y = relu6(gamma*(x-mean)*rstd+beta)
 *   bwd     : dy' = dy*[0 < gamma*xhat+beta < 6] (gate recomputed from x); dgamma = sum dy'*xhat; dbeta = sum dy';
 *             dx = gamma*rstd*(dy' - dbeta/rows - xhat*dgamma/rows)
 *             (two kernels: reduce into fp64 scratch [2C], then apply; dgamma/dbeta overwritten)
 */
int athena_bn_finalize(const double* colstats, long rows, int C, float eps, float momentum, float* mean_rstd,
                       float* moving_mean, float* moving_var, athena_stream_t stream);
int athena_bn_relu6_apply(const void* x, const float* mean_rstd, const float* gamma, const float* beta,
                          long rows, int C, int dtype, void* y, athena_stream_t stream);
int athena_bn_relu6_infer(const void* x, const float* moving_mean, const float* moving_var, const float* gamma,
                          const float* beta, float eps, long rows, int C, int dtype, void* y,
                          athena_stream_t stream);
/* scratch: athena_bn_relu6_bwd_scratch_bytes(rows, C) bytes, 16-byte aligned (fp64 totals [2C] followed
 * by one fp32 slab [2C] of partial sums per 512 rows; no atomics, fixed summation order) */
int64_t athena_bn_relu6_bwd_scratch_bytes(long rows, int C);
int athena_bn_relu6_bwd(const void* dy, const void* x, const float* mean_rstd, const float* gamma,
                        const float* beta, long rows, int C, int dtype, void* scratch, int64_t scratch_bytes,
                        void* dx, float* dgamma, float* dbeta, athena_stream_t stream);
/* The same three without the relu6: layers.BatchNormalization() after each recurrent layer,
 * athena/models/deep_speech.py:80.  athena_bn_colstats collects {sum, sumsq} [2C] in fp64 over the rows
 * of a stored tensor (what the convolution epilogues collect on the fly). */
int athena_bn_colstats(const void* x, long rows, int C, int dtype, double* colstats, athena_stream_t stream);
int athena_bn_apply(const void* x, const float* mean_rstd, const float* gamma, const float* beta, long rows, int C,
                    int dtype, void* y, athena_stream_t stream);
int athena_bn_infer(const void* x, const float* moving_mean, const float* moving_var, const float* gamma,
                    const float* beta, float eps, long rows, int C, int dtype, void* y, athena_stream_t stream);
int athena_bn_bwd(const void* dy, const void* x, const float* mean_rstd, const float* gamma, const float* beta,
                  long rows, int C, int dtype, void* scratch, int64_t scratch_bytes, void* dx, float* dgamma,
                  float* dbeta, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Conv2D with any kernel size and strides, "same" padding, NHWC, no bias, and its gradients.
 * Replaces layers.Conv2D(kernel_size=(41, 11), strides=(2, 2)) and (21, 11) / (2, 1) of
 * athena/models/deep_speech.py:49-66 under the forward pass and tape.gradient (athena/solver.py:96).
 *   in [B,H,W,Cin], w_hwio [KH,KW,Cin,Cout], out [B,Ho,Wo,Cout] with Ho = ceil(H/sh), Wo = ceil(W/sw)
 *   (athena_conv2d_out_shape); Cin and Cout multiples of 8, at most 1024 taps.
 *   fwd   : colstats (may be NULL) receives {sum, sumsq} per output channel in fp64 for BatchNorm
 *   dgrad : relu6_out (may be NULL) = the relu6 output this convolution read: its gate masks din
 *   wgrad : dw_hwio fp32, overwritten; with a workspace of athena_conv2d_wgrad_workspace_bytes bytes
 *           the split partial sums are added in a fixed order, without it by fp32 atomics
 * A layer with fewer than 8 input channels (the model's first, one channel) is run as athena_im2col
 * followed by athena_gemm: col [B*Ho*Wo, ldcol] with col[r][tap*Cin + ci] and zeros in the padding
 * columns up to ldcol; its weight gradient is athena_gemm with trans_a over the same matrix. */
int athena_conv2d_out_shape(int H, int W, int KH, int KW, int sh, int sw, int* Ho, int* Wo);
int athena_conv2d_fwd(const void* in, const void* w_hwio, void* out, int B, int H, int W, int Cin, int Cout, int KH,
                      int KW, int sh, int sw, int dtype, double* colstats, athena_stream_t stream);
int athena_conv2d_dgrad(const void* dout, const void* w_hwio, void* din, int B, int H, int W, int Cin, int Cout,
                        int KH, int KW, int sh, int sw, int dtype, const void* relu6_out, athena_stream_t stream);
int64_t athena_conv2d_wgrad_workspace_bytes(int B, int H, int W, int Cin, int Cout, int KH, int KW, int sh, int sw,
                                            int dtype);
int athena_conv2d_wgrad(const void* in, const void* dout, float* dw_hwio, int B, int H, int W, int Cin, int Cout,
                        int KH, int KW, int sh, int sw, int dtype, void* workspace, int64_t workspace_bytes,
                        athena_stream_t stream);
int athena_im2col(const void* in, int in_dtype, void* col, int col_dtype, int ldcol, int B, int H, int W, int Cin,
                  int KH, int KW, int sh, int sw, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * The serial part of a recurrent layer: tf.keras.layers.RNN(cell=[GRUCell | LSTMCell](H),
 * return_sequences=True), athena/models/deep_speech.py:75-79 with athena/layers/commons.py:486-491,
 * forward and under tape.gradient (athena/solver.py:96).  cell: 0 = GRU (reset_after, gates z r h),
 * 1 = LSTM (gates i f c o); G = 3 or 4.  The input projection x W + b of all steps, and the weight
 * gradients from dxw / dhu_ext, are ordinary GEMMs done by the caller.  All arrays batch-major:
 *   xw [B,T,G*H]; u [H,G*H] recurrent kernel; u_t [G*H,H] its transposed copy (bf16 only, may be NULL:
 *   with it a step is one launch -- product and gates together -- instead of a GEMM and a gate kernel;
 *   the backward pass does the same from u alone); b_rec [G*H] fp32 recurrent bias (GRU) or NULL;
 *   hs_ext [B,T+1,H] hidden states, slot 0 = zero initial state; cs_ext [B,T+1,H] fp32 LSTM cell state;
 *   y [B,T,H] = h[t]; gates [B,T,G*H] activated gates; rh [B,T,H] GRU recurrent candidate part;
 *   dxw [B,T,G*H] gradient at x W + b; dhu_ext [B,T+1,G*H] gradient at h[t-1] U (+ b_rec), slot T zero:
 *     dU = hs_ext^T dhu_ext over all B*(T+1) rows, db_rec = column sums of dhu_ext.
 * workspace: athena_rnn_workspace_bytes(cell, B, H) bytes, 16-byte aligned.  H multiple of 8. */
int64_t athena_rnn_workspace_bytes(int cell, int B, int H);
int athena_rnn_fwd(int cell, const void* xw, const void* u, const void* u_t, const float* b_rec, void* hs_ext,
                   float* cs_ext, void* y, void* gates, void* rh, int B, int T, int H, int dtype, void* workspace,
                   int64_t workspace_bytes, athena_stream_t stream);
int athena_rnn_bwd(int cell, const void* dy, const void* u, const void* hs_ext, const float* cs_ext,
                   const void* gates, const void* rh, void* dxw, void* dhu_ext, int B, int T, int H, int dtype,
                   void* workspace, int64_t workspace_bytes, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Labels and key masks of one training step, in one launch.  Replaces insert_sos_in_labels and
 * insert_eos_in_labels (athena/utils/misc.py:32-34,50-57), compute_logit_length
 * (athena/models/speech_transformer.py:156-162) and the padding halves of create_multihead_mask
 * (athena/utils/misc.py:68-90):
 *   y0[b]   = [sos, labels[b]...]                          [B, U+1] int32
 *   tgt[b]  = labels[b] ++ [0], eos added at label_len[b]  [B, U+1] int32
 *   y_mask  = (y0 == 0)                                    [B, U+1] uint8 (1 = masked key)
 *   logit_len[b] = ceil(ceil(input_len[b] / 2) / 2)        [B] int32
 *   x_mask[b,t]  = (t >= logit_len[b])                     [B, Tp] uint8
 */
int athena_prepare_labels(const int32_t* labels, const int32_t* label_len, const int32_t* input_len, int B, int U,
                          int Tp, int sos, int eos, int32_t* y0, int32_t* tgt, uint8_t* y_mask, int32_t* logit_len,
                          uint8_t* x_mask, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Positional encoding / embedding front ends.
 *   add_pe_dropout: y[b,t,:] = dropout(x[b,t,:]*xscale + pe[t,:])   (PositionalEncoding + Dropout,
 *                   athena/layers/commons.py:35-41, speech_transformer.py:103-104)
 *   embed_fwd     : y[b,l,:] = dropout(E[ids[b,l],:]*xscale + pe[l,:]) (Embedding + scaled PE +
 *                   Dropout, speech_transformer.py:110-112)
 *   embed_bwd     : dE[v,:] = sum over the tokens (b,l) with ids[b,l] == v of dy[b,l,:]*mult*xscale: every
 *                   row of dE [V, d] is written (zero where no token has the id), nothing is added to
 *                   what dE held, and the order of the additions depends on the ids alone (token order;
 *                   a row that more than 48 tokens point at is summed in four contiguous parts)
 *   dropout_bwd   : dx = dy * mult * xscale * [0 < relu6_out < 6]  (relu6_out may be NULL: no gate)
 */
int athena_add_pe_dropout(const void* x, const float* pe, int B, int T, int d, int dtype, float xscale,
                          float drop_p, const uint64_t* rng_state, uint32_t rng_site, void* y,
                          athena_stream_t stream);
int athena_dropout_bwd(const void* dy, long n, int dtype, float xscale, float drop_p,
                       const uint64_t* rng_state, uint32_t rng_site, const void* relu6_out, void* dx,
                       athena_stream_t stream);
int athena_embed_fwd(const float* table, const int32_t* ids, const float* pe, int B, int L, int d, int V,
                     int dtype, float xscale, float drop_p, const uint64_t* rng_state, uint32_t rng_site,
                     void* y, athena_stream_t stream);
int athena_embed_bwd(const void* dy, const int32_t* ids, int B, int L, int d, int V, int dtype, float xscale,
                     float drop_p, const uint64_t* rng_state, uint32_t rng_site, float* dtable,
                     athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * CTC loss and its gradient.  Replaces tf.nn.ctc_loss(labels dense, logits batch-major,
 * blank_index) of athena/loss.py:38-45 (per-sample losses; the caller takes the mean, :46) and
 * its registered gradient.
 *   logits [B,T,V] (row stride ldl >= V, ldl % 4 == 0; fp32 or bf16), labels [B,U] int32
 *   zero-padded, label_len / logit_len [B] int32.
 *   fwd: loss[b] = -log p(labels_b | logits_b[:logit_len_b]); the workspace keeps the row
 *        logsumexp and the state posterior of every row (a list of U + 1 floats) for bwd.
 *        Three launches: one workgroup per row (logsumexp, arg-max, the emissions of the 2U+1
 *        lattice states gathered into a table), one workgroup per sample (alpha and beta
 *        recursions on probabilities in double precision, rescaled by powers of two), one wave per
 *        row (posterior) and sample (loss).  Alignments that do not fit
 *        (logit_len < label_len + repeats) follow TensorFlow's dense branch, whose initial and
 *        final state vectors hold log(1e-307) instead of log 0: a finite loss of about 7e2 and the
 *        gradient of the leaked paths over the whole padded label row.  label_len is clamped to
 *        [0, U].  2U+1 > 1024 returns ATHENA_E_UNSUPPORTED.  argmax (may be NULL): [B*T] int32,
 *        the first class holding the maximum of each row t < logit_len_b (rows beyond get 0) -- the greedy path the CTCAccuracy metric decodes, athena/metrics.py:121-132,
 *        taken from the pass that reads the row anyway.
 *   bwd: grad[b,t,v] = host_scale * grad_scale[0] * (softmax(logits[b,t])[v] - occupancy[b,t,v]),
 *        zero for t >= logit_len_b and for the padding columns v in [V, ldl).  grad_scale is one
 *        fp32 scalar on the device (the upstream gradient) or NULL (= 1).
 *   fwd_bwd: both at once for a caller that knows the factor of the gradient when it asks for the
 *        loss (tf.GradientTape over a loss whose weight is a constant, athena/solver.py:94-97 with
 *        athena/models/mtl_seq2seq.py:95): loss, argmax and workspace as fwd, and
 *        grad = grad_scale * (softmax - occupancy) as bwd would leave it.  The logits are read once:
 *        the row launch writes grad_scale * softmax while it holds the row, the last launch writes
 *        the few columns of each row that have an occupancy.  athena_ctc_loss_bwd may still follow
 *        on the same workspace.
 * workspace: athena_ctc_workspace_bytes(B,T,U) bytes, 16-byte aligned, the same buffer for both calls.
 */
size_t athena_ctc_workspace_bytes(int B, int T, int U);
int athena_ctc_loss_fwd(const void* logits, int logits_dtype, int ldl, const int32_t* labels,
                        const int32_t* label_len, const int32_t* logit_len, int B, int T, int V, int U, int blank,
                        float* loss, int32_t* argmax, void* workspace, size_t workspace_bytes,
                        athena_stream_t stream);
int athena_ctc_loss_bwd(const void* logits, int logits_dtype, int ldl, const int32_t* labels,
                        const int32_t* label_len, const int32_t* logit_len, int B, int T, int V, int U, int blank,
                        const float* grad_scale, float host_scale, void* grad, int grad_dtype, void* workspace,
                        size_t workspace_bytes, athena_stream_t stream);
int athena_ctc_loss_fwd_bwd(const void* logits, int logits_dtype, int ldl, const int32_t* labels,
                            const int32_t* label_len, const int32_t* logit_len, int B, int T, int V, int U,
                            int blank, float* loss, int32_t* argmax, float grad_scale, void* grad, int grad_dtype,
                            void* workspace, size_t workspace_bytes, athena_stream_t stream);

/* x[0..n) *= upstream[0] / expected, unless upstream[0] == expected (then every workgroup leaves after
 * reading the scalar).  The backward pass of a loss whose gradient was written in the forward pass
 * with the factor it expected (athena_ctc_loss_fwd_bwd) calls this with the upstream gradient it
 * really received (the grads argument of tape.gradient, athena/solver.py:96); n % 4 == 0, x 16-byte
 * aligned, expected != 0. */
int athena_rescale_unless(void* x, long n, int dtype, const float* upstream, float expected,
                          athena_stream_t stream);

/* athena_ctc_loss_fwd without a workspace argument.  No counterpart in the reference: it is for
 * callers that cannot allocate device memory (a stream under HIP graph capture, a serving loop, a
 * harness that forbids hipMalloc) and want the per-sample losses and the greedy path only.  The
 * workspace is a 16 MiB device array inside the library (one copy per GPU, held until the process
 * ends); athena_ctc_workspace_bytes(B,T,U) beyond that returns ATHENA_E_UNSUPPORTED.  The call
 * allocates and frees nothing.  All calls on one GPU share the array: calls that overlap in time on
 * one GPU (different streams) race, calls on one stream are safe.  The first call on a GPU asks
 * the runtime for the array's address and should come before any graph capture.  The lattices stay
 * in the array, so there is no matching bwd: take athena_ctc_loss_fwd / _bwd for gradients. */
int athena_ctc_loss_fwd_static(const void* logits, int logits_dtype, int ldl, const int32_t* labels,
                               const int32_t* label_len, const int32_t* logit_len, int B, int T, int V, int U,
                               int blank, float* loss, int32_t* argmax, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Label-smoothed softmax cross-entropy over decoder positions and its gradient.
 * Replaces Seq2SeqSparseCategoricalCrossentropy.__call__, athena/loss.py:63-80, after
 * insert_eos_in_labels (the caller passes ``targets`` [rows] = labels ++ eos, 0 = padding).
 *   y = (1-ls)*onehot(target) + ls/V
 *   fwd: row_loss[r] = -sum_v y*log_softmax(logits[r]) * [target_r != 0]; lse[r] kept for bwd
 *   bwd: grad[r,v] = host_scale * grad_scale[0] * (softmax[v] - y[v]) * [target_r != 0]
 */
int athena_ce_loss_fwd(const void* logits, int logits_dtype, int ldl, const int32_t* targets, int rows, int V,
                       float label_smoothing, float* row_loss, float* lse, athena_stream_t stream);
int athena_ce_loss_bwd(const void* logits, int logits_dtype, int ldl, const int32_t* targets, int rows, int V,
                       float label_smoothing, const float* lse, const float* grad_scale, float host_scale,
                       void* grad, int grad_dtype, athena_stream_t stream);

/* out[g] = scale * sum_i x[g*group + i] (the batch mean of tf.reduce_mean, athena/loss.py:46,79-80). */
int athena_group_sum(const float* x, int ngroups, int group, float scale, float* out, athena_stream_t stream);

/* out[0] = sum_i weights[i] * terms[i][0] for n <= 8 scalars on the device (``terms``: host array of
 * device pointers, ``weights``: host floats): the total loss of a multi-task model,
 * mtl_weight * main + (1 - mtl_weight) * extra (athena/models/mtl_seq2seq.py:95), as one launch. */
int athena_weighted_sum(const float* const* terms, const float* weights, int n, float* out, athena_stream_t stream);

/* out[r] = argmax_v logits[r, v] (first maximum), for the accuracy metrics
 * (athena/metrics.py:103,127). */
int athena_argmax_rows(const void* logits, int dtype, int ldl, int rows, int V, int32_t* out,
                       athena_stream_t stream);

/* Accuracy scoring of a batch on the device: per utterance the Levenshtein distance (tf.edit_distance,
 * normalize=False) between a hypothesis read off arg-max ids [B, L] (row stride ld_ids) and the
 * non-zero entries of labels [B, U]; errors are added to counts[0] and the number of non-zero labels
 * to counts[1] (64-bit integer adds, so the sums do not depend on the order of the utterances), and
 * written per utterance to per_utt [B, 2] when that is not null (either may be null, not both).
 * mode 0 = CTCAccuracy.__call__, athena/metrics.py:118-132 (tf.nn.ctc_greedy_decoder: ids of the
 *          first hyp_len[b] frames, repeats merged, `special` = the blank class dropped);
 * mode 1 = Seq2SeqSparseCategoricalAccuracy.__call__, athena/metrics.py:101-106 with validate_seqs,
 *          athena/utils/misc.py:98-126 (ids before the first `special` = eos, zeros dropped; with
 *          eos == 0 only the zeros are dropped); hyp_len is not read.
 * Both feed CharactorAccuracy.update_state, athena/metrics.py:73-89.  L <= 4095. */
int athena_seq_errors(const int32_t* ids, int ld_ids, const int32_t* hyp_len, const int32_t* labels, int B, int L,
                      int U, int mode, int special, int32_t* per_utt, uint64_t* counts, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Optimizer: per-tensor clip_by_norm + Adam with the warm-up schedule, on flat buffers.
 * Replaces BaseSolver.clip_by_norm + optimizer.apply_gradients, athena/solver.py:78-87,97-98,
 * tf.keras.optimizers.Adam and WarmUpLearningSchedule, athena/utils/learning_rate.py:52-86.
 *   seg_offsets [nseg+1] (int64, device): tensor i occupies [seg_offsets[i], seg_offsets[i+1]).
 *   step (int64, device): optimizer.iterations before the update; incremented by the call.
 *   lr = k*decay_rate^(step//decay_steps)*d_model^-0.5*min(step^-0.5, step*warmup^-1.5)
 *   g *= clip/max(||g||_2, clip) per tensor (clip <= 0: no clipping); Adam with t = step+1.
 *   norms: scratch [nseg] fp32.  lr_out (optional, device fp32) receives the lr used.
 */
typedef struct athena_adam_cfg {
    float beta1, beta2, eps, clip_norm;
    float d_model, warmup_steps, k, decay_steps, decay_rate;
    float grad_scale; /* multiplies every gradient first (1/world_size after a summing all-reduce) */
    /* schedule 0: the warm-up schedule above (WarmUpLearningSchedule, athena/utils/learning_rate.py:52-58);
     * schedule 1: ExponentialDecayLearningRateSchedule (learning_rate.py:112-117):
     *   lr = clamp(initial_lr * decay_rate^((step - start_decay_steps) // decay_steps), final_lr, initial_lr),
     *   the factor being 1 before start_decay_steps */
    float schedule, initial_lr, start_decay_steps, final_lr;
} athena_adam_cfg;
int athena_clip_adam_step(float* params, const float* grads, float* m, float* v, long n,
                          const int64_t* seg_offsets, int nseg, float* norms, int64_t* step,
                          const athena_adam_cfg* cfg, float* lr_out, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Masked-predictive-coding loss.  Replaces MPCLoss.__call__, athena/loss.py:83-105 (used by
 * MaskedPredictCoding.get_loss, athena/models/masked_pc.py:138-151): the L1 distance between the
 * model output and the unmasked features, counted where the masked input is exactly 0 and the
 * frame lies inside the utterance, summed over the feature axis:
 *   row_loss[b,t] = [t < logit_len[b]] * sum_c [masked_input[b,t,c] == 0] * |target[b,t,c] - logits[b,t,c]|
 * (the loss is mean(row_loss) over all B * Tp rows, taken by the caller, e.g. athena_group_sum).
 * logits fp32 [B*Tp, ldl] (ldl >= N), target and masked_input fp32 [B*Tp, N] -- the [B, T, dim, ch]
 * feature tensors read as [B, T/4, 4*dim*ch].  bwd writes grad [B*Tp, ldl] (fp32 or bf16, padding
 * columns zeroed) = -sign(target - logits) * grad_scale[0] * host_scale on the counted elements. */
int athena_mpc_loss_fwd(const float* logits, int ldl, const float* target, const float* masked_input,
                        const int32_t* logit_len, int B, int Tp, int N, float* row_loss, athena_stream_t stream);
int athena_mpc_loss_bwd(const float* logits, int ldl, const float* target, const float* masked_input,
                        const int32_t* logit_len, int B, int Tp, int N, const float* grad_scale,
                        float host_scale, void* grad, int grad_dtype, athena_stream_t stream);

/* Refresh bf16 shadows of 2-D fp32 weights after an optimizer step.  For each of ``nmat``
 * matrices (descriptor table on the device, 9 int64 each: src offset in ``params``, rows, cols,
 * offset and leading dimension of the row-major bf16 copy [rows][cols] in ``shadow``, offset and
 * leading dimension of the transposed copy [cols][rows], and the offsets of the two fragment-tiled
 * copies read by athena_layer_tail_fwd / _bwd or -1 for none), writes all copies.  Padding columns
 * (leading dimension > width) are left untouched.  Tiled copies need rows and cols multiples of 32
 * and the 4-element alignment of the vector path; a tiled copy is rows * cols elements in blocks of
 * 512: block (nb, kb) holds 16 rows x 32 contraction indices, element 8 * lane + e = row
 * 16 nb + (lane & 15), contraction index 32 kb + 8 (lane >> 4) + e, blocks nb-major; the first
 * copy takes the matrix' rows as rows and contracts over its columns, the second the other way. */
int athena_refresh_shadows(const float* params, void* shadow, const int64_t* table, int nmat,
                           const int64_t* tile_prefix /*[nmat+1] cumulative 32x32 tile counts*/,
                           long total_tiles, athena_stream_t stream);

/* rng_state[1] += 1 (advance the dropout stream once per step). */
int athena_advance_rng(uint64_t* rng_state, athena_stream_t stream);

/* Elementwise helpers: dst = cast(src) ; y = a*x + b*y on fp32 buffers. */
int athena_cast(const void* src, int src_dtype, void* dst, int dst_dtype, long n, athena_stream_t stream);
int athena_axpby(float a, const void* x, float b, void* y, long n, int dtype, athena_stream_t stream);

/* Up to ATHENA_COPY_MANY_MAX byte-wise copies dst[i] <- src[i] (bytes[i] each, regions must not overlap)
 * in ONE launch: the batch tensors going into the buffers a recorded step reads, and the metric
 * tensors going to pinned host memory after it (the reference hands the batch to the compiled
 * step as arguments, athena/solver.py:77-92, and reads the metric tensors back eagerly,
 * athena/metrics.py:118-132).  Pointers are device-accessible addresses (device memory or pinned
 * host memory). */
#define ATHENA_COPY_MANY_MAX 8
int athena_copy_many(const void* const* src, void* const* dst, const long* bytes, int n, athena_stream_t stream);

/* ---------------------------------------------------------------------------------------------
 * Paged key / value cache in 8 bits, for decoding.  The reference runs its decoder over the whole
 * history at every step (SpeechTransformer.time_propagate, athena/models/speech_transformer.py:164-194)
 * and keeps nothing; these entry points let a step compute its newest rows only.
 *
 * The cache of one attention layer, ``num_blocks`` blocks of ``block_size`` (16, 32, 64 or 128) tokens:
 *   k_codes int8 [num_blocks][hk][block_size][width]   k_scale fp32 [num_blocks][hk]
 *   v_codes int8 [num_blocks][hk][width][block_size]   v_scale fp32 [num_blocks][hk]
 * An element stands for code * scale, scales are not negative.  width is 32, 64 or 128; heads of dk <= width columns use the first
 * dk, the others hold zeros.  Codes start on 16 bytes.  Place p of the cache is token p % block_size of block
 * p / block_size; num_blocks * block_size < 2^31, table_width * block_size < 2^31 - 512.
 *
 * athena_kv_plan: the blocks and places of the next new_rows[b] tokens of every request.  lens[b] tokens are
 * cached already, in the blocks tables[b * ld_tables + 0 ...] (table_width entries a request);
 * free_blocks[0 .. free_count[0]) is a stack of free blocks.  new_rows[b] < 0 marks a finished request: its
 * blocks are put on top of the stack (in request and table order) before any are taken, and its length
 * becomes 0.  Entries beyond those lens needs are filled from the top of the stack, in request order.
 * Written: cu_rows [B + 1] (rows of the requests one behind the other; request b has rows
 * cu_rows[b] .. cu_rows[b + 1]), slots [rows] (the place of each row; -1 behind the last row), positions
 * [rows] (a row's index in its sequence; 0 behind the last row), the new table entries, the returned blocks,
 * lens_out [B] and free_count_out [1] (each may be the input itself), and status [4]: {blocks missing,
 * requests with a negative length or longer than their table, rows missing, returned blocks beyond
 * free_capacity}.  A plan that does not fit leaves a status that is not zero and changes nothing: no rows
 * (cu_rows 0, slots -1), lens_out = lens, free_count_out = free_count.  ``work``: int32 [3 * B + 3].
 * A block belongs to one request; B at least 1. */
typedef struct {
    const int32_t *lens, *new_rows;
    int32_t *tables, *free_blocks;
    const int32_t* free_count;
    int32_t *cu_rows, *slots, *positions, *lens_out, *free_count_out, *status, *work;
    int64_t ld_tables;
    int32_t table_width, free_capacity, B, block_size, rows, reserved;
} athena_kv_plan_desc;
int athena_kv_plan(const athena_kv_plan_desc* d, athena_stream_t stream);

/* Keys and values of N rows into their places.  Row t: k[t * ldk + head * ldk_head + c], c < dk; a slot
 * outside [0, num_blocks * block_size) skips its row.  Rows of one block stand one behind the other (as
 * athena_kv_plan lays them out; skipped rows may stand between them); of two rows for one place the later
 * stays.  The scale of a block and head is the largest
 * magnitude written so far / 127: it only grows, and the codes in front of the new ones are then brought to
 * the grown scale (round half to even of code * old / new); a run that begins at a block's first place
 * begins the block again, whatever its scale was.  Codes are round half to even of x / scale.  A value that
 * is not finite makes its block's scale NaN: the block then stands for NaN until it is begun again.
 * N up to 2^30 - 64; ldk and ldv 0 to 2^22 - 1, hk up to 65535. */
typedef struct {
    const void *k, *v;
    const int32_t* slots;
    int8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    int64_t ldk, ldk_head, ldv, ldv_head;
    int32_t dtype, N, num_blocks, hk, block_size, dk, width, reserved;
} athena_kv8_append_desc;
int athena_kv8_append(const athena_kv8_append_desc* d, athena_stream_t stream);

/* Attention over the cache: out[t, head] = sum_j softmax_j(scale * q[t, head] . k_j) v_j over the cached
 * tokens of t's sequence.  Sequence b has lens[b] tokens (its new ones included) and the query rows
 * cu_rows[b] .. cu_rows[b + 1] of q, its last tokens; cu_rows null: one row per sequence.  causal: row i of
 * n sees the tokens j <= lens[b] - n + i.  Query head i reads kv head i / (h / hk).  A row that sees nothing
 * gives zeros (lse -inf).  Table entries outside [0, num_blocks) hold no tokens; lengths are cut at
 * table_width * block_size, rows at N; rows that belong to no sequence are left as they were.
 * max_rows: the largest number of rows of a sequence (it shapes the launch and the workspace; a number below the truth makes the call
 * slower, results differ by the order of their sums only).
 * Rounding, besides that of the result: scores and sums in fp32; queries in fp16 (fp32 queries in two such numbers) raised so that
 * columns down to 2^-31 of a row's largest keep a bf16 number's bits and fp32 ones 22 bits down to 2^-17; probability times value
 * scale, relative to the row's largest, in 11 bits down to 2^-29 (fp32 queries: 22 down to 2^-18), fewer further down and
 * nothing below 2^-40.
 * lse: fp32 [N][h], natural logarithm of the sum of exponentials, or null.
 * ld_tables may be 0: every sequence then reads the same blocks.
 * ``workspace``: athena_kv8_attention_workspace_bytes of the same descriptor (0: none is needed; its pointers are
 * not looked at, and a table of fewer than 1024 places never needs one). */
typedef struct {
    const void* q;
    const int8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    const int32_t *tables, *lens, *cu_rows;
    void* out;
    float* lse;
    void* workspace;
    int64_t workspace_bytes, ldq, ldq_head, ldo, ldo_head, ld_tables;
    int32_t dtype, num_blocks, block_size, width, table_width, B, max_rows, N, h, hk, dk, causal;
    float scale, reserved;
} athena_kv8_attention_desc;
int64_t athena_kv8_attention_workspace_bytes(const athena_kv8_attention_desc* d);
int athena_kv8_attention(const athena_kv8_attention_desc* d, athena_stream_t stream);

/* Penalties, biases and a grammar mask on the logits of a decoding step, between the output layer and the
 * search (the reference adds scorers to log-probabilities on the host, athena/tools/beam_search.py:120-150).
 * With c = occurrences of class v in history[r, 0 .. history_len[r]) (history_len null: L; ids outside
 * [0, V) count nowhere):
 *   x = logit;  c > 0: x = x > 0 ? x / repetition[r] : x * repetition[r];  x -= frequency[r] c + presence[r];
 *   x += bias[r * ld_bias + v] + sum of bias_values[r, j] over bias_ids[r, j] == v;
 *   -inf unless bit v % 32 of word v / 32 of allowed[r * ld_allowed + ...] is set.
 * Any of history, repetition, presence, frequency, bias, bias_ids (nb = 0), allowed may be null.  ld_bias and
 * ld_allowed may be 0 (one row for all).  R up to 65535, L and nb up to 2^30.  out has the type of the logits and may be the logits. */
typedef struct {
    const void* logits;
    void* out;
    const int32_t *history, *history_len, *bias_ids, *allowed;
    const float *repetition, *presence, *frequency, *bias, *bias_values;
    int64_t ldl, ldo, ld_history, ld_bias, ld_bias_ids, ld_bias_values, ld_allowed;
    int32_t dtype, R, V, L, nb, reserved;
} athena_logits_desc;
int athena_logits_process(const athena_logits_desc* d, athena_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* ATHENA_HIP_H */
