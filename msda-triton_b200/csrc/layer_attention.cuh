// Masked attention: what its kernels share (parameters, masks, scores).
//
//   x_ij = scale q_i . k_j;  x = cap tanh(x / cap);  x -= slope_h |place_i - j|
//   p_ij = exp(x_ij - lse_i) where query i sees key j, else 0;  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij g_i;  ds_ij = p_ij (g_i . v_j - g_i . o_i) (1 - tanh^2) scale
//   dq_i = sum_j ds_ij k_j;  dk_j = sum_i ds_ij q_i
//
// Query i stands at place_i = length - Sq + i among the keys. Exponents are
// taken to base 2: scores carry a factor log2(e). A row that sees no key gives
// zeros, lse = -inf and no gradient.
#pragma once

#include <cfloat>

#include "msda_abi.cuh"
#include "msda_common.cuh"
#include "msda_layer_b200.h"

namespace msda {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kDocTile = 128;  // tokens one entry of the document summary stands for

// Documents of a tile of kDocTile tokens: those that are no padding lie in
// [low, high] (low > high: all padding); `padded`: some are padding; `shared`:
// some key is of the shared document.
struct DocTile {
  int low, high, padded, shared;
};

struct AttnParams {
  const void *q, *k, *v, *go;
  void *o, *dq, *dk, *dv;
  void* residue;                       // what rounding took from o (16-bit types), nullable
  float *lse, *delta;  // (B, H, Sq)
  int64_t qs[3], ks[3], vs[3], gs[3];  // strides of (B, S, H) in elements
  const float* slopes;                  // (H,), nullable
  const int *qdoc, *kdoc;               // (B, Sq), (B, Sk), nullable together
  const int *prefix, *klen;             // (B,), nullable
  const DocTile *qtile, *ktile;         // (B, ceil(S / kDocTile))
  int B, Sq, Sk, H, Hkv, D;
  float scale, cap;  // cap 0: none
  int shared, causal;  // shared -1: none
  int splits;          // parts of the keys; above 1 the parts' results go to part_o, part_ml
  float* part_o;       // (splits, B, H, Sq, D)
  float2* part_ml;     // (splits, B, H, Sq): maximum (base 2) and sum
  int kv_parts;        // parts of a key head's query heads in its gradient; above 1 the sums go to part_kv
  float* part_kv;      // (kv_parts, 2, B, Sk, Hkv, D): dv's parts and dk's
};

// A part's sums of dv, or of dk.
__device__ __forceinline__ float* kv_part(const AttnParams& p, int part, bool keys) {
  return p.part_kv + (part * 2 + (keys ? 1 : 0)) * ((int64_t)p.B * p.Sk * p.Hkv * p.D);
}

__device__ __forceinline__ int attn_length(const AttnParams& p, int b) {
  if (!p.klen) return p.Sk;
  return min(max(__ldg(p.klen + b), 0), p.Sk);
}

// What a query row sees: keys j < limit, of its document where there are any.
struct RowView {
  int limit, place, doc;
};

__device__ __forceinline__ RowView row_view(const AttnParams& p, int b, int i, int length) {
  RowView r;
  r.place = length - p.Sq + i;
  r.limit = length;
  r.doc = 0;
  if (p.causal) {
    const int before = max(r.place + 1, p.prefix ? __ldg(p.prefix + b) : 0);
    r.limit = max(0, min(length, before));
  }
  if (i >= p.Sq) {
    r.limit = 0;
  } else if (p.qdoc) {
    r.doc = __ldg(p.qdoc + (int64_t)b * p.Sq + i);
    if (r.doc < 0) r.limit = 0;
  }
  return r;
}

// Largest limit of the rows [i0, i1) (limits grow with the row).
__device__ __forceinline__ int rows_limit(const AttnParams& p, int b, int i1, int length) {
  if (!p.causal) return length;
  const int before = max(length - p.Sq + min(i1, p.Sq), p.prefix ? __ldg(p.prefix + b) : 0);
  return max(0, min(length, before));
}

// First query that may see key j0 or a later one below j1.
__device__ __forceinline__ int first_query(const AttnParams& p, int b, int j0, int length) {
  if (!p.causal) return 0;
  if (p.prefix && __ldg(p.prefix + b) > j0) return 0;
  return min(p.Sq, max(0, j0 - length + p.Sq));
}

__device__ __forceinline__ bool same_document(int qdoc, int kdoc, int shared) {
  return kdoc >= 0 && (kdoc == qdoc || kdoc == shared);
}

// Whether no query of one tile sees a key of the other by their documents.
__device__ __forceinline__ bool tiles_apart(const DocTile& q, const DocTile& k) {
  if (q.low > q.high || k.low > k.high) return true;
  return !k.shared && (q.high < k.low || q.low > k.high);
}

// Whether every query of one tile sees every key of the other by their documents.
__device__ __forceinline__ bool tiles_agree(const DocTile& q, const DocTile& k, int shared) {
  return !q.padded && !k.padded && q.low == q.high && k.low == k.high && (q.low == k.low || k.low == shared);
}

// tanh, to about 2e-7 relative: near zero an odd polynomial (fitted to the
// least relative error on |x| < 0.75: 3.3e-8), beyond it the exponential, whose
// cancellation near zero would cost digits.
constexpr float kTanhSmall = 0.75f;

__device__ __forceinline__ float tanh_small(float x) {
  const float y = x * x;
  float r = -0.004769488703459501f;
  r = fmaf(r, y, 0.019664911553263664f);
  r = fmaf(r, y, -0.0533902570605278f);
  r = fmaf(r, y, 0.13326521217823029f);
  r = fmaf(r, y, -0.3333306908607483f);
  return fmaf(r * y, x, x);
}

__device__ __forceinline__ float tanh_large(float x) {
  const float e = exp2f(-2.0f * kLog2e * fabsf(x));
  return copysignf(__fdividef(1.0f - e, 1.0f + e), x);
}

__device__ __forceinline__ float tanh_of(float x) { return fabsf(x) < kTanhSmall ? tanh_small(x) : tanh_large(x); }

// v rounded to T, and what the rounding took.
template <typename T>
__device__ __forceinline__ void put_output(const AttnParams& p, int64_t at, float v) {
  const T r = from_f32<T>(v);
  static_cast<T*>(p.o)[at] = r;
  if (p.residue) static_cast<T*>(p.residue)[at] = from_f32<T>(v - to_f32(r));
}

// The score's constants for one head, in base 2.
struct ScoreForm {
  float scale2;  // scale * log2(e)
  float cap2, inv_cap;  // cap * log2(e), scale / cap
  float slope2;
};

__device__ __forceinline__ ScoreForm score_form(const AttnParams& p, int h) {
  ScoreForm f;
  f.scale2 = p.scale * kLog2e;
  f.cap2 = p.cap * kLog2e;
  f.inv_cap = p.cap != 0.0f ? p.scale / p.cap : 0.0f;
  f.slope2 = p.slopes ? __ldg(p.slopes + h) * kLog2e : 0.0f;
  return f;
}

// Keys [first, last) of part `split` of the keys below `limit`: the same
// multiple of 64 keys for every part.
__device__ __forceinline__ void split_range(int limit, int splits, int split, int& first, int& last) {
  const int part = ((limit + splits - 1) / splits + 63) / 64 * 64;
  first = (int)min((int64_t)limit, (int64_t)part * split);
  last = min(limit, first + part);
}

// Launches (each returns the launch's error).
cudaError_t attn_documents_launch(const AttnParams& p, DocTile* qtile, DocTile* ktile, cudaStream_t st);
// Any type, head size and stride. token: few queries, the keys in p.splits parts,
// which attn_combine_launch joins where there are more than one.
cudaError_t attn_tf32_forward(const AttnParams& p, int dtype, bool token, cudaStream_t st);
cudaError_t attn_tf32_backward(const AttnParams& p, int dtype, cudaStream_t st);
// The form for single tokens: 16-bit types in the tensor-core kernels' layout.
cudaError_t attn_token_forward(const AttnParams& p, int dtype, cudaStream_t st);
// Tensor-core kernels: 16-bit types, D a multiple of 8 up to 128, rows that
// start on 16 bytes at strides of whole 16 bytes. 0 or a cudaError_t; -1 where a
// tensor map could not be made.
int attn_tc_forward(const AttnParams& p, int dtype, cudaStream_t st);
int attn_tc_backward(const AttnParams& p, int dtype, cudaStream_t st);
// Waits of the tensor-core kernels that gave up so far (reads device memory).
cudaError_t attn_tc_gave_up(int* count);
cudaError_t attn_kv_sum_launch(const AttnParams& p, int dtype, cudaStream_t st);
cudaError_t attn_combine_launch(const AttnParams& p, int dtype, cudaStream_t st);

}  // namespace msda
