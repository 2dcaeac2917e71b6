/* fwn_rows.h - C ABI of the row permutation passes either side of the mesh transformer's layer
 * loop, fused with the layer norms next to them (same library as fwn_attn.h).
 *
 * The reference sorts the mesh nodes along a Hilbert curve so that the k-hop mask has fewer
 * live tiles: it gathers the node features with the permutation before the 24 layers and
 * scatters them back after the final norm (patch.py:274-276, 288-292). Each of those is one
 * extra pass over [batch, n, channels] per step. Here the gather is fused with the first
 * block's layer norm and the scatter with the final layer norm and its per-member affine, so
 * the permutation costs no pass of its own.
 *
 * Conventions (as in fwn_attn.h): status codes and fwn_last_error(); launchers validate on the
 * host, enqueue on `stream`, allocate nothing and keep no pointer. Tensors are contiguous
 * [batch, n, channels] in the dtype of the descriptor; statistics are computed in float32.
 * `perm` is a device array of n int64 that must be a permutation of 0..n-1. An entry outside
 * [0, n) yields a zero row (gather) or is dropped (scatter); repeated entries make the scatter
 * write one row twice in an unspecified order. Neither touches memory outside the tensors.
 */
#ifndef FWN_ROWS_H_
#define FWN_ROWS_H_

#include <stdint.h>

#include "fwn_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FWN_ROWS_MAX_CHANNELS 4096

typedef struct fwn_rows_desc {
  int32_t batch;
  int32_t n;         /* rows (mesh nodes) per batch member */
  int32_t channels;  /* features per row: a multiple of 8, at most FWN_ROWS_MAX_CHANNELS */
  int32_t dtype;     /* fwn_dtype of x and of every output */
  float eps;         /* layer-norm epsilon, added to the biased variance */
} fwn_rows_desc;

/* x_out[b, i, :] = x[b, perm[i], :] and, when norm_out is not NULL,
 * norm_out[b, i, :] = (x_out[b, i, :] - mean) / sqrt(var + eps) over the channels (a layer norm
 * without scale or offset). Replaces jnp.take(node_features, perm, axis=1) before the layer
 * loop (patch.py:274-276) fused with the first block's st.layernorm(x, create_scale=False,
 * create_offset=False) (patch.py:244). x and x_out must not overlap. */
int fwn_rows_gather_norm_launch(const fwn_rows_desc* d, const void* x, const int64_t* perm,
                                void* x_out, void* norm_out, void* stream);

/* out[b, perm[i], :] = layer_norm(x[b, i, :]) * mul[b, :] + add[b, :], with mul and add float32
 * [batch, channels] (NULL means 1 and 0). Replaces the final st.layernorm, the per-member
 * affine that LinearNormConditioning applies to it (its scale and offset come from the
 * conditioning vector, computed by the caller) and jnp.take(x, argsort(perm), axis=1)
 * (patch.py:288-292). x and out must not overlap. */
int fwn_rows_norm_scatter_launch(const fwn_rows_desc* d, const void* x, const int64_t* perm,
                                 const float* mul, const float* add, void* out, void* stream);

/* out[b, i, :] = layer_norm(x[b, i, :]) * mul[b, :] + add[b, :] (mul and add float32
 * [batch, channels], NULL meaning 1 and 0): the block's conditioned layer norm in one pass, the
 * fwn_rows_norm_scatter_launch pass without a permutation. Replaces
 * norm_conditioning_layer(st.layernorm(x, create_scale=False, create_offset=False)) in front of
 * the attention and of the feed-forward of every block (patch.py:240-244, 250-251), whose
 * LinearNormConditioning scale and offset the caller evaluates from the conditioning vector.
 * x and out must not overlap. */
int fwn_rows_norm_affine_launch(const fwn_rows_desc* d, const void* x, const float* mul,
                                const float* add, void* out, void* stream);

/* sum[b, i, :] = x[b, i, :] + y[b, i, :] (added in float32, rounded once to the dtype) and
 * out[b, i, :] = layer_norm(sum[b, i, :]) * mul[b, :] + add[b, :]: the block's residual add
 * fused with the conditioned layer norm that reads its result. Replaces `x = x + mha(...)`
 * followed by the feed-forward's norm_conditioning_layer(st.layernorm(x)), and the feed-forward
 * residual followed by the next block's conditioned layer norm (patch.py:240-253). sum may be x
 * or y itself (an in-place residual update) or disjoint from both; out must not overlap x, y or
 * sum. */
int fwn_rows_add_norm_affine_launch(const fwn_rows_desc* d, const void* x, const void* y,
                                    const float* mul, const float* add, void* sum, void* out,
                                    void* stream);

/* The conditioning of `count` (1 to FWN_COND_MAX) norms from one conditioning vector: for norm l, with
 * weight[l] a contiguous [2 * channels, cond_size] matrix and bias[l] of 2 * channels entries, both
 * in `dtype` as cond [batch, cond_size],
 *   mul[l, b, c] = 1 + weight[l][c, :] . cond[b, :] + bias[l][c]
 *   add[l, b, c] = weight[l][channels + c, :] . cond[b, :] + bias[l][channels + c]
 * in float32, the affine the norm passes take (LinearNormConditioning's projections, which the
 * reference evaluates norm by norm, patch.py:240-253, 288-292). mul and add are float32 [count,
 * batch, channels]. weight and bias are host arrays of device pointers, read before returning. */
#define FWN_COND_MAX 64
int fwn_cond_affine_launch(int32_t count, int32_t batch, int32_t channels, int32_t cond_size, int32_t dtype,
                           const void* cond, const void* const* weight, const void* const* bias, float* mul,
                           float* add, void* stream);

/* Backward of the passes above: for every row i of x (the rows a pass normalised, with xhat their
 * layer norm and rstd its 1 / sqrt(var + eps), recomputed from x),
 *
 *   g[b, i, :]  = rstd (gm - mean(gm) - xhat mean(gm xhat)) + g_res[b, i, :],  gm = g_norm mul
 *   g_mul[b, :] = sum over i of g_norm xhat,   g_add[b, :] = sum over i of g_norm
 *
 * computed in float32; g is written to gx in the dtype. g_norm (NULL: zeros) is the gradient of
 * the norm's output, g_res (NULL: zeros) that of the sum or copy x itself also went to, mul as in
 * the forward (NULL: 1). g_mul and g_add (float32 [batch, channels]) are written when both are
 * non-NULL; that needs fwn_rows_norm_bwd_workspace_size bytes of workspace (16-byte aligned), used
 * until the launch's stream work is done, and none otherwise. The sums run in a fixed order.
 * With perm, `perm_rows` says what it permutes:
 *   FWN_ROWS_PERM_GRAD: row i's g_norm is row perm[i] of the tensor (backward of norm_scatter);
 *   FWN_ROWS_PERM_OUT: g is written to row perm[i] of gx (backward of gather_norm).
 * Entries of perm outside [0, n) read a zero row or drop the row. gx must not overlap the inputs. */
#define FWN_ROWS_PERM_GRAD 1
#define FWN_ROWS_PERM_OUT 2
int fwn_rows_norm_bwd_workspace_size(const fwn_rows_desc* d, uint64_t* bytes);
int fwn_rows_norm_bwd_launch(const fwn_rows_desc* d, const void* x, const int64_t* perm, int32_t perm_rows,
                             const void* g_norm, const void* g_res, const float* mul, void* gx, float* g_mul,
                             float* g_add, void* workspace, uint64_t workspace_bytes, void* stream);

/* dw[o, i] = sum over r of g[r, o] * x[r, i] and, where db is given, db[o] = sum over r of g[r, o]:
 * the gradients of y = x w^T + b with respect to w and b, as the transformer block's projections and
 * feed-forward take them (patch.py:165-177, 233-253). g is [rows, outs], x [rows, ins], dw [outs, ins],
 * db [outs], all contiguous bfloat16, 16-byte aligned; sums are float32, rounded to bfloat16 once.
 * outs and ins are positive multiples of FWN_LINEAR_UNIT, each at most FWN_LINEAR_MAX; rows >= 1.
 * The workspace (fwn_linear_wgrad_workspace_size bytes, 16-byte aligned) holds float32 partial sums;
 * its contents before the call do not matter. */
#define FWN_LINEAR_UNIT 64
#define FWN_LINEAR_MAX 16384
int fwn_linear_wgrad_workspace_size(int64_t rows, int32_t outs, int32_t ins, uint64_t* bytes);
int fwn_linear_wgrad_launch(int64_t rows, int32_t outs, int32_t ins, const void* g, const void* x, void* dw, void* db,
                            void* workspace, uint64_t workspace_bytes, void* stream);

/* Root-mean-square norm of rows, its output in the tensors' dtype or in 8 bits. Rows are `channels`
 * elements with stride 1; row i of x begins at i * x_stride elements (0: one row for all), of y likewise,
 * every other tensor is contiguous. Statistics are float32. */
#define FWN_RMS_MAX_CHANNELS 16384

typedef struct fwn_rms_desc {
  int64_t rows;
  int64_t x_stride, y_stride;
  int32_t channels;      /* 1 to FWN_RMS_MAX_CHANNELS */
  int32_t dtype;         /* fwn_dtype of x, y, sum, out and the gradients */
  int32_t weight_dtype;  /* the dtype, or FWN_F32 */
  float eps;             /* added to the mean square, finite and >= 0 */
} fwn_rms_desc;

/* With y, sum = x + y (added in float32, rounded once) and the norm is of sum as stored, else y and sum
 * are NULL and it is of x: out[i, :] = s[i, :] / sqrt(mean(s[i, :]^2) + eps) * weight (NULL: 1). sum and
 * out must not overlap each other or an input. */
int fwn_rms_norm_launch(const fwn_rms_desc* d, const void* x, const void* y, const void* weight, void* sum, void* out,
                        void* stream);

/* The same with the output in 8 bits: for the unrounded values v of a row, scale[i] = max(max |v| / 448,
 * 2^-126) and q[i, :] the OCP e4m3 codes of v * (1 / scale[i]), reciprocal and product each rounded to float32,
 * to nearest even: the codes nearest to v / scale[i], or, within 2^-23 of the middle of two, either of them. A row
 * with NaN has scale and codes NaN; one whose largest magnitude is infinite has scale infinity and NaN codes there. */
int fwn_rms_norm_q8_launch(const fwn_rms_desc* d, const void* x, const void* y, const void* weight, void* sum, uint8_t* q,
                           float* scale, void* stream);

/* q and scale of the rows of x as they are. */
int fwn_quantize_rows_launch(const fwn_rms_desc* d, const void* x, uint8_t* q, float* scale, void* stream);

/* Backward of fwn_rms_norm_launch at the contiguous rows s that were normalised (sum, or x):
 *   gx = g_sum + r (h - s r^2 mean(h s)),  h = g_out weight,  r = 1 / sqrt(mean(s^2) + eps)
 *   gw = sum over the rows of g_out s r, in weight_dtype
 * g_sum (NULL: zeros) is the gradient of sum. gx is the gradient of x and of y. gw may be NULL; with it the
 * launch needs fwn_rms_norm_bwd_workspace_size bytes of workspace (16-byte aligned), whose sums run in a
 * fixed order. gx and gw must not overlap an input or each other. */
int fwn_rms_norm_bwd_workspace_size(const fwn_rms_desc* d, uint64_t* bytes);
int fwn_rms_norm_bwd_launch(const fwn_rms_desc* d, const void* s, const void* weight, const void* g_out,
                            const void* g_sum, void* gx, void* gw, void* workspace, uint64_t workspace_bytes,
                            void* stream);

/* Dropout of rows with a residual: out[i, c] = kept(i, c) ? x[i, c] m : 0, plus residual[i, c] (NULL: 0), in float32 and
 * rounded once to the dtype. With T = p 2^16 to the nearest whole number, m = 2^16 / (2^16 - T) in float32, and channel c of row i is
 * kept if its 16 random bits are T or more: the halves, low one first, of the four words of Philox-4x32-10 (Salmon, Moraes,
 * Dror and Shaw 2011) with the seed's halves as its key and (c / 8, i, the offset's halves) as its counter. Nothing about what is kept is
 * stored; the same launch over the gradient of out, without a residual, is the gradient of x. Dropped values are zeros, whatever
 * they were. state, if not NULL, holds {seed, offset} in the GPU's memory, read when the kernel runs, and the two
 * members are not used. Rows are `channels` elements with stride 1; row i of x begins at i * x_stride elements, of residual
 * likewise, out is contiguous. out may be x or the residual where that is contiguous, and must not overlap either otherwise. */
#define FWN_DROPOUT_MAX_CHANNELS (1 << 30)

typedef struct fwn_dropout {
  double p;              /* 0 to 1 */
  uint64_t seed, offset;
  const uint64_t* state; /* 8-byte aligned, or NULL */
} fwn_dropout;

typedef struct fwn_dropout_desc {
  int64_t rows;          /* less than 2^32 */
  int64_t x_stride, r_stride;
  int32_t channels;      /* 1 to FWN_DROPOUT_MAX_CHANNELS */
  int32_t dtype;
  fwn_dropout drop;
} fwn_dropout_desc;

int fwn_dropout_launch(const fwn_dropout_desc* d, const void* x, const void* residual, void* out, void* stream);

/* The root-mean-square norms after a block and before the next one, with the block's gate, the residual's scale and dropout between them.
 * For rows x of the residual and y of the block's output,
 *   r1 = 1 / sqrt(mean(y^2) + eps),  b = gate y r1 post_weight,  s = scale x + dropout(b)
 *   r2 = 1 / sqrt(mean(s^2) + eps),  out = s r2 pre_weight
 * s is formed in float32 and stored rounded once in sum; the second norm is of the stored rows. Without post_norm r1 is 1.
 * NULL weights and a NULL gate are 1. Row i of gate [rows / gate_rows, channels] is that of the rows i gate_rows .. (i + 1)
 * gate_rows - 1: gate_rows is `rows` for one gate, 1 for a gate of x's shape, and divides rows. Rows of x and y are
 * `channels` elements with stride 1, x_stride and y_stride elements apart; every other tensor is contiguous. Outputs must not overlap each
 * other or an input. */
typedef struct fwn_sandwich_desc {
  int64_t rows;                            /* less than 2^32 */
  int64_t gate_rows;                       /* not read without a gate */
  int64_t x_stride, y_stride;
  int32_t channels;                        /* 1 to FWN_RMS_MAX_CHANNELS */
  int32_t dtype;                           /* of x, y, sum, out and their gradients */
  int32_t gate_dtype, post_dtype, pre_dtype; /* the dtype, or FWN_F32, also of the tensor's gradient */
  int32_t post_norm;                       /* 0 or 1 */
  float eps, scale;                        /* eps finite and >= 0, scale finite */
  fwn_dropout drop;                        /* p = 0: none */
} fwn_sandwich_desc;

int fwn_sandwich_norm_launch(const fwn_sandwich_desc* d, const void* x, const void* y, const void* gate, const void* post_weight,
                             const void* pre_weight, void* sum, void* out, void* stream);

/* Its backward at the contiguous rows s = sum, with a = g_out pre_weight, g = g_sum + r2 (a - s r2^2 mean(a s)) and
 * d = dropout(g):
 *   gx = scale g,  gy = r1 (c - y r1^2 mean(c y)) with c = d gate post_weight (without post_norm c)
 *   g_gate = sums of d y r1 post_weight over the rows of each row of gate
 *   g_post = sum of d gate y r1,  g_pre = sum of g_out s r2, both over the rows
 * g_sum and g_out may be NULL (zeros), and each output may be NULL (not wanted). The workspace
 * (fwn_sandwich_norm_bwd_workspace_size bytes, 16-byte aligned) is needed where one of g_gate (of more than one row each),
 * g_post and g_pre is; the query takes whether there is a gate. Sums run in a fixed order. */
int fwn_sandwich_norm_bwd_workspace_size(const fwn_sandwich_desc* d, int32_t gate, uint64_t* bytes);
int fwn_sandwich_norm_bwd_launch(const fwn_sandwich_desc* d, const void* s, const void* y, const void* gate,
                                 const void* post_weight, const void* pre_weight, const void* g_sum, const void* g_out, void* gx,
                                 void* gy, void* g_gate, void* g_post, void* g_pre, void* workspace, uint64_t workspace_bytes,
                                 void* stream);

/* Matrix product with bias, activation and residual in its epilogue:
 *   z = x weight^T + bias,  out = act(z) + residual
 * x is [rows, ins], weight [outs, ins], residual [rows, outs], with contiguous rows x_stride, w_stride and
 * r_stride elements apart (0: one row for all; at most FWN_LINEAR_STRIDE_MAX, r_stride FWN_LINEAR_ACT_MAX); bias
 * [outs], out and pre [rows, outs] are contiguous.
 * Products accumulate in float32; out, and pre (z for the backward, NULL: not stored) are rounded
 * once. bias and residual may be NULL. Every tensor is of `dtype`; float32 products keep float32's precision over
 * its whole range. No output of the launches here may overlap an input or another output. */
#define FWN_ACT_NONE 0
#define FWN_ACT_RELU 1
#define FWN_ACT_GELU 2      /* z (1 + erf(z / sqrt 2)) / 2 */
#define FWN_ACT_GELU_TANH 3 /* its tanh form */
#define FWN_ACT_SILU 4      /* z / (1 + exp(-z)) */
#define FWN_LINEAR_ACT_MAX (1 << 20) /* of ins and outs */
#define FWN_LINEAR_STRIDE_MAX (1 << 30)

typedef struct fwn_linear_desc {
  int64_t rows;
  int64_t x_stride, w_stride, r_stride;
  int32_t ins, outs; /* 1 to FWN_LINEAR_ACT_MAX */
  int32_t dtype;
  int32_t activation;
} fwn_linear_desc;

/* Workspaces hold nothing between launches and are 256-byte aligned; launches that can overlap need their
 * own. Their sizes are asked with the pointers of the launch, of which only NULL and the alignment matter. */
int fwn_linear_act_workspace_size(const fwn_linear_desc* d, const void* x, const void* weight, uint64_t* bytes);
int fwn_linear_act_launch(const fwn_linear_desc* d, const void* x, const void* weight, const void* bias,
                          const void* residual, void* out, void* pre, void* workspace, uint64_t workspace_bytes,
                          void* stream);

/* Gradients for the contiguous gradient g [rows, outs] of out: with dz = g act'(pre) (pre is read unless the
 * activation is FWN_ACT_NONE; dz is rounded to the dtype for the products),
 *   gx = dz weight [rows, ins],  gw = dz^T x [outs, ins],  gb = column sums of dz [outs]
 * each contiguous and skipped where NULL. The residual's gradient is g. Sums run in a fixed order. */
int fwn_linear_act_bwd_workspace_size(const fwn_linear_desc* d, const void* x, const void* weight, const void* g,
                                      const void* gx, const void* gw, const void* gb, uint64_t* bytes);
int fwn_linear_act_bwd_launch(const fwn_linear_desc* d, const void* x, const void* weight, const void* pre,
                              const void* g, void* gx, void* gw, void* gb, void* workspace, uint64_t workspace_bytes,
                              void* stream);

/* The forward of 8-bit operands: x and weight hold OCP e4m3 codes, z = (x weight^T) x_scale[row]
 * w_scale[column] + bias with float32 scales (fwn_rms_norm_q8_launch, fwn_quantize_rows_launch). The
 * descriptor's dtype is that of bias, residual and out. With FWN_F32, and of up to 32 rows, products are added in
 * float32. With FWN_BF16 the e4m3 matrix units add them, eight at a time as multiples of 2^-13 of the largest one's
 * power of two: off by less than 2^-10 of the sum of their magnitudes (random sums: 1.4e-5 of the rows' norms). */
int fwn_linear_act_q8_workspace_size(const fwn_linear_desc* d, const uint8_t* x, const uint8_t* weight, uint64_t* bytes);
int fwn_linear_act_q8_launch(const fwn_linear_desc* d, const uint8_t* x, const float* x_scale, const uint8_t* weight,
                             const float* w_scale, const void* bias, const void* residual, void* out,
                             void* workspace, uint64_t workspace_bytes, void* stream);

/* Weights of 4 bits with a scale for each group of FWN_Q4_GROUP inputs (the 4-bit format of the OCP microscaling
 * specification): w[o, i] = value(code) 2^(scale - 127), the code's top bit the sign, the others 0, 0.5, 1, 1.5, 2, 3, 4 and 6. With
 * groups = ceil(ins / FWN_Q4_GROUP), codes are [outs, 16 groups] bytes, 16-byte aligned, the even input of a pair in the low
 * half; scales are [outs, groups], 255 meaning NaN. Codes past ins are not used. A weight of 2^128 or more is infinite.
 *
 * fwn_quantize_q4_launch: the codes and scales of rows of x, x_stride elements apart. A group's scale is the least power of two
 * of which its largest magnitude is at most seven (beyond six is cut to six), its codes the nearest ones, middles to even codes.
 * Groups with NaN or infinities have the scale NaN. Codes past ins are zeros. */
#define FWN_Q4_GROUP 32
int fwn_quantize_q4_launch(int64_t rows, int32_t ins, int64_t x_stride, int32_t dtype, const void* x, uint8_t* codes,
                           uint8_t* scales, void* stream);

/* fwn_linear_act_launch with such a weight, without pre; w_stride is not read. Products are exact and added in float32 (float32
 * x as in fwn_linear_act_launch). */
int fwn_linear_act_q4_workspace_size(const fwn_linear_desc* d, const void* x, const uint8_t* scales, uint64_t* bytes);
int fwn_linear_act_q4_launch(const fwn_linear_desc* d, const void* x, const uint8_t* codes, const uint8_t* scales,
                             const void* bias, const void* residual, void* out, void* workspace, uint64_t workspace_bytes,
                             void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* FWN_ROWS_H_ */
