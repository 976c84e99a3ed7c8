/*
 * msda_b200 -- C ABI of the operators that stand beside deformable attention
 * in a transformer layer: rotary positions over several axes, (residual and)
 * layer norm, and masked attention for training and for single tokens.
 *
 * Conventions are those of msda_b200.h: device pointers, sizes and a
 * cudaStream_t passed as void*; the caller allocates every buffer, including
 * workspaces; every call returns an msda_status and leaves its message in
 * msda_last_error(); nothing synchronises with the host. Small tables
 * (strides, axis sizes) are HOST arrays, read before the call returns. dtype
 * codes are msda_dtype's.
 */
#ifndef MSDA_LAYER_B200_H_
#define MSDA_LAYER_B200_H_

#include "msda_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Type of rotary positions. */
typedef enum msda_position_type {
  MSDA_POSITION_F32 = 0,
  MSDA_POSITION_I32 = 1,
  MSDA_POSITION_I64 = 2
} msda_position_type;

/* How the frequencies of several axes are laid over the channels: each axis
 * has a ladder of its own in its own block of channels, or all axes take
 * sections of one ladder over the rotated channels. */
#define MSDA_ROTARY_LADDER_AXIS 0
#define MSDA_ROTARY_LADDER_SHARED 1
/* Which channels form a pair: k and k + n/2 of a ladder's n channels, or
 * neighbours 2k and 2k + 1. */
#define MSDA_ROTARY_PAIRING_HALF 0
#define MSDA_ROTARY_PAIRING_INTERLEAVED 1
#define MSDA_ROTARY_MAX_AXES 8
#define MSDA_ROTARY_MAX_HEAD_DIM 512

/*
 * Rotary positions over several axes, on the query and key heads in one call.
 *   query (B, S, H, D), key (B, S, Hkv, D), dtype; channels contiguous,
 *   strides of (B, S, H) in elements; key may be null with Hkv = 0.
 *   positions (B, S, A), (S, A)-contiguous, batch stride in elements (0: the
 *   same for every item).
 *   query_out, key_out: contiguous, dtype.
 * axis_dims[a] (even, A of them) channels turn with axis a; channels past
 * their sum pass through. Pair k of a ladder of n channels turns by
 * position * base^(-2k/n), formed to about twice fp32's precision, so that
 * long positions lose nothing. inverse != 0 turns back: the gradient.
 * Whole-number positions are read as fp32: exact below 2^24.
 */
MSDA_API int msda_rotary(const void* query, const void* key, const void* positions, void* query_out,
                         void* key_out, int64_t batch, int64_t seq, int32_t num_heads,
                         int32_t num_key_heads, int32_t head_dim, const int64_t* query_strides,
                         const int64_t* key_strides, int64_t position_batch_stride,
                         int32_t position_type, int32_t num_axes, const int32_t* axis_dims,
                         double base, int32_t ladder, int32_t pairing, int32_t inverse,
                         int32_t dtype, void* stream);

#define MSDA_LAYER_NORM_MAX_WIDTH (1 << 20)

/*
 * y = (h - mean(h)) / sqrt(var(h) + eps) * weight + bias over rows of C
 * channels, h = x (+ residual), in fp32 and rounded once.
 *   x, residual (nullable): rows of `width` contiguous elements at row strides
 *   in elements; y, sum_out (nullable: h rounded): contiguous, dtype.
 *   weight, bias: nullable, `param_dtype` (dtype, or MSDA_DTYPE_F32).
 *   mean, rstd: (rows,) fp32, nullable together; the backward wants them.
 * width <= MSDA_LAYER_NORM_MAX_WIDTH.
 */
MSDA_API int msda_layer_norm_forward(const void* x, const void* residual, const void* weight,
                                     const void* bias, void* y, void* sum_out, float* mean,
                                     float* rstd, int64_t rows, int64_t width, int64_t x_stride,
                                     int64_t residual_stride, float eps, int32_t dtype,
                                     int32_t param_dtype, void* stream);

/* Bytes of workspace msda_layer_norm_backward needs for the weight's and the
 * bias's gradients (0 for sizes that it refuses). */
MSDA_API size_t msda_layer_norm_backward_workspace_size(int64_t rows, int64_t width);

/*
 * Gradients of msda_layer_norm_forward: grad_x (that of the residual too,
 * contiguous, dtype), grad_weight and grad_bias (param_dtype, nullable).
 *   grad_y: row stride in elements; grad_sum (nullable): contiguous, the
 *   gradient of sum_out, added to grad_x.
 * The column sums are formed in fp32 in an order fixed by the sizes: results
 * are bitwise reproducible.
 */
MSDA_API int msda_layer_norm_backward(const void* x, const void* residual, const void* weight,
                                      const float* mean, const float* rstd, const void* grad_y,
                                      const void* grad_sum, void* grad_x, void* grad_weight,
                                      void* grad_bias, void* workspace, size_t workspace_bytes,
                                      int64_t rows, int64_t width, int64_t x_stride,
                                      int64_t residual_stride, int64_t grad_stride, int32_t dtype,
                                      int32_t param_dtype, void* stream);

#define MSDA_ATTENTION_MAX_HEAD_DIM 256

/*
 * Masked attention.
 *   query, out (B, Sq, H, D); key, value (B, Sk, Hkv, D), H a multiple of Hkv;
 *   dtype; channels contiguous, strides of (B, S, H) in elements for the
 *   inputs; out and the gradients contiguous. lse: (B, H, Sq) fp32.
 *
 * With length_b = key_lengths[b] (clamped to [0, Sk]) or Sk, query i stands at
 * place = length_b - Sq + i. It sees key j if j < length_b, and
 *   - with causal: j <= place, or j < prefix_lengths[b] where given;
 *   - with documents: neither id is negative (padding), and the ids agree or
 *     the key's is shared_document (-1: none).
 * Scores: s = scale q.k; s = softcap tanh(s / softcap) (softcap from 2^-100 to
 * 2^100, or 0: not); s -= distance_slopes[h] |place - j|. A query that sees no
 * key gets zeros, an lse of -inf and no gradient. Keys past length_b and of
 * negative documents are never read into a result, whatever they hold; a key
 * that other queries see must be finite. The rows of query and grad_out of a query that sees no key
 * may hold anything too.
 *
 * At most 65535 items, 4096 heads, 2^22 queries and 2^30 keys, 2^22 in the
 * backward; where the type is fp32 or a row is not of up to 128 channels in whole
 * 16-byte vectors, 65535 x 64 for 2^22.
 */
typedef struct msda_attention_args {
  const void *query, *key, *value;
  void* out;   /* forward: written; backward: the forward's */
  /* What rounding took from out, in its layout (16-bit types), nullable: with
   * it the backward's row sums grad_out . out are those of the unrounded out,
   * which matters to rows that see few keys. Written by the forward, read by
   * the backward. */
  void* out_residue;
  float* lse;  /* forward: written, nullable; backward: the forward's */
  const void* grad_out; /* backward */
  void *grad_query, *grad_key, *grad_value;
  int64_t batch, num_queries, num_keys;
  int32_t num_heads, num_key_heads, head_dim, dtype;
  int64_t query_strides[3], key_strides[3], value_strides[3], grad_out_strides[3];
  float scale, softcap;
  const float* distance_slopes;                     /* (H,), nullable */
  const int32_t *query_documents, *key_documents;   /* (B, Sq), (B, Sk); nullable together */
  const int32_t *prefix_lengths, *key_lengths;      /* (B,), nullable; prefix needs causal */
  int32_t shared_document, causal;
  void* workspace;
  size_t workspace_bytes;
} msda_attention_args;

/* Bytes of workspace the forward (backward = 0) or backward needs; 0 also for
 * arguments that the call refuses. */
MSDA_API size_t msda_attention_workspace_size(const msda_attention_args* args, int32_t backward);
/* Attention, and its gradients. Sums are formed in an order fixed by the
 * sizes: results are bitwise reproducible. */
MSDA_API int msda_attention_forward(const msda_attention_args* args, void* stream);
MSDA_API int msda_attention_backward(const msda_attention_args* args, void* stream);
/* The tensor-core kernels' waits are bounded: one that gives up (a fault of
 * the hardware or of this library) leaves NaN in the outputs and is counted.
 * Reads the current device's count; synchronises with it. */
MSDA_API int msda_attention_gave_up(int32_t* count);

#ifdef __cplusplus
}
#endif

#endif /* MSDA_LAYER_B200_H_ */
