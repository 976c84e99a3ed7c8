// Masked attention on the fp32 pipes: fp32 inputs, whose products the tensor
// cores would round, and head sizes, strides and alignments that their loads
// do not take.
//
// Tiles lie channel-major in shared memory ([channel][token]), so that both
// kinds of product read 16 bytes at a time: x = a . b over channels, with
// RM x 4 products a thread and step, and acc = x . c over tokens, four tokens a
// step. A warp owns whole rows (2 groups of RM rows, 16 threads across), so row
// sums are shuffles and a row's probabilities never leave the warp. Bound by
// the FMA pipes: 12 floats loaded for 32 multiply-adds in the first product.
#include "layer_attention.cuh"

namespace msda {
namespace {

constexpr int kThreads = 128;
constexpr int kCols = 64;        // columns of a tile: keys, or queries in the key gradient
constexpr int kLd = kCols + 4;   // row pitch of a 64-token tile

// rows [r0, r0 + n) of a (S, D) slice, channel-major; rows that `keep` rejects
// and channels from D to DP are zero.
template <typename T, int DP, typename Keep>
__device__ __forceinline__ void load_tile(float* dst, int ld, int n, const T* base, int64_t stride, int64_t r0, int D,
                                          bool vec, Keep keep) {
  const int row = threadIdx.x % n;
  const bool in = keep(row);
  const T* src = base + (r0 + row) * stride;
  for (int d = (threadIdx.x / n) * 4; d < DP; d += kThreads / n * 4) {
    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in) {
      if (vec && d + 4 <= D) {
        load_vec<T, 4>(src + d, f);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < D) f[i] = to_f32(src[d + i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[(d + i) * ld + row] = f[i];
  }
}

template <int DP, int RM>
struct Tile {
  static constexpr int kRows = 8 * RM;
  static constexpr int kLdr = kRows + 4;
  static constexpr int DC = DP / 16;
  static constexpr int kRowFloats = DP * kLdr, kColFloats = DP * kLd, kProbFloats = kRows * kLd;

  static __device__ __forceinline__ int row_group() { return threadIdx.x / 16; }
  static __device__ __forceinline__ int col_group() { return threadIdx.x % 16; }

  // x[r][c] = sum_d a[d][row r] b[d][column c]
  static __device__ __forceinline__ void scores(const float* a, const float* b, float (&x)[RM][4]) {
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) x[r][c] = 0.0f;
    const float* ap = a + row_group() * RM;
    const float* bp = b + col_group() * 4;
#pragma unroll 4
    for (int d = 0; d < DP; ++d) {
      float u[RM];
#pragma unroll
      for (int r = 0; r < RM; r += 4) {
        const float4 f = *reinterpret_cast<const float4*>(ap + d * kLdr + r);
        u[r] = f.x, u[r + 1] = f.y, u[r + 2] = f.z, u[r + 3] = f.w;
      }
      const float4 v = *reinterpret_cast<const float4*>(bp + d * kLd);
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        x[r][0] = fmaf(u[r], v.x, x[r][0]);
        x[r][1] = fmaf(u[r], v.y, x[r][1]);
        x[r][2] = fmaf(u[r], v.z, x[r][2]);
        x[r][3] = fmaf(u[r], v.w, x[r][3]);
      }
    }
  }

  // A warp's rows of x to shared memory, for `gather`.
  static __device__ __forceinline__ void spread(float* prob, const float (&x)[RM][4]) {
    __syncwarp();
#pragma unroll
    for (int r = 0; r < RM; ++r)
      *reinterpret_cast<float4*>(prob + (row_group() * RM + r) * kLd + col_group() * 4) =
          make_float4(x[r][0], x[r][1], x[r][2], x[r][3]);
    __syncwarp();
  }

  // acc[r][c] += sum_j prob[row r][j] t[channel col_group + 16 c][j]
  static __device__ __forceinline__ void gather(const float* prob, const float* t, float (&acc)[RM][DC]) {
#pragma unroll 1
    for (int j = 0; j < kCols; j += 4) {
      float4 x[RM];
#pragma unroll
      for (int r = 0; r < RM; ++r) x[r] = *reinterpret_cast<const float4*>(prob + (row_group() * RM + r) * kLd + j);
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const float4 v = *reinterpret_cast<const float4*>(t + (col_group() + 16 * c) * kLd + j);
#pragma unroll
        for (int r = 0; r < RM; ++r) {
          acc[r][c] = fmaf(x[r].x, v.x, acc[r][c]);
          acc[r][c] = fmaf(x[r].y, v.y, acc[r][c]);
          acc[r][c] = fmaf(x[r].z, v.z, acc[r][c]);
          acc[r][c] = fmaf(x[r].w, v.w, acc[r][c]);
        }
      }
    }
  }

  // f(row, channel, r, c) of the thread's part of the rows [r0, rows) and channels below D.
  template <typename F>
  static __device__ __forceinline__ void each(int r0, int rows, int D, F f) {
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      const int i = r0 + row_group() * RM + r;
      if (i >= rows) continue;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (col_group() + 16 * c < D) f(i, col_group() + 16 * c, r, c);
    }
  }
};

__device__ __forceinline__ float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// The score in base 2 and the cap's tanh (0 without one).
__device__ __forceinline__ float score2(const AttnParams& p, const ScoreForm& f, float s, int far, float& t) {
  t = 0.0f;
  float x = s * f.scale2;
  if (p.cap != 0.0f) {
    t = tanh_of(s * f.inv_cap);
    x = t * f.cap2;
  }
  if (p.slopes) x = fmaf(-f.slope2, (float)abs(far), x);
  return x;
}

template <typename T>
__device__ __forceinline__ bool can_vec(const void* p, const int64_t (&s)[3], int D) {
  return D % 4 == 0 && (reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T))) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

__device__ __forceinline__ bool key_padded(const AttnParams& p, int b, int j, int length) {
  return j >= length || (p.kdoc && __ldg(p.kdoc + (int64_t)b * p.Sk + j) < 0);
}

__device__ __forceinline__ bool skip_tiles(const AttnParams& p, int b, int i0, int j0) {
  if (!p.kdoc) return false;
  const int nq = (p.Sq + kDocTile - 1) / kDocTile, nk = (p.Sk + kDocTile - 1) / kDocTile;
  return tiles_apart(p.qtile[(int64_t)b * nq + i0 / kDocTile], p.ktile[(int64_t)b * nk + j0 / kDocTile]);
}

// PACK: the rows are Sq x (H / Hkv) pairs of a query and one of the heads that
// share a key head (a few queries over a long cache), and the keys are split.
template <typename T, int DP, int RM, bool PACK>
__global__ void __launch_bounds__(kThreads) attn_simt_fwd_kernel(const AttnParams p) {
  using G = Tile<DP, RM>;
  extern __shared__ float4 smem4[];
  float* qt = reinterpret_cast<float*>(smem4);
  float* kt = qt + G::kRowFloats;
  float* vt = kt + G::kColFloats;
  float* prob = vt + G::kColFloats;
  const int group = p.H / p.Hkv, b = blockIdx.z, hk = PACK ? blockIdx.y : blockIdx.y / group;
  const int pack = PACK ? group : 1, h0 = PACK ? hk * group : blockIdx.y;
  const int rows = p.Sq * pack;
  const int split = PACK ? blockIdx.x % p.splits : 0;
  const int tile = PACK ? blockIdx.x / p.splits : gridDim.x - 1 - blockIdx.x;  // long causal rows first
  const int r0 = tile * G::kRows;
  const int length = attn_length(p, b);
  int first = 0, limit = rows_limit(p, b, (r0 + G::kRows + pack - 1) / pack, length);
  if (PACK) split_range(limit, p.splits, split, first, limit);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  const bool kvec = can_vec<T>(p.k, p.ks, p.D), vvec = can_vec<T>(p.v, p.vs, p.D);
  if constexpr (PACK) {
    // One row at a time: neighbours are heads, then queries.
    for (int at = threadIdx.x; at < G::kRows * DP; at += kThreads) {
      const int r = at / DP, d = at % DP, i = (r0 + r) / pack, h = h0 + (r0 + r) % pack;
      qt[d * G::kLdr + r] = r0 + r < rows && d < p.D
          ? to_f32(static_cast<const T*>(p.q)[b * p.qs[0] + i * p.qs[1] + h * p.qs[2] + d]) : 0.0f;
    }
  } else {
    load_tile<T, DP>(qt, G::kLdr, G::kRows, static_cast<const T*>(p.q) + b * p.qs[0] + h0 * p.qs[2], p.qs[1], r0, p.D,
                     can_vec<T>(p.q, p.qs, p.D), [&](int r) { return r0 + r < p.Sq; });
  }
  RowView row[RM];
  ScoreForm f = score_form(p, h0);
  float slope[RM], m[RM], l[RM], acc[RM][G::DC], mul[RM];
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const int at = r0 + G::row_group() * RM + r;
    row[r] = row_view(p, b, at / pack, length);
    slope[r] = PACK && p.slopes ? __ldg(p.slopes + h0 + at % pack) * kLog2e : f.slope2;
    m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < G::DC; ++c) acc[r][c] = 0.0f;
  }
  for (int j0 = first; j0 < limit; j0 += kCols) {
    if (!PACK && skip_tiles(p, b, r0, j0)) continue;
    __syncthreads();
    const auto keep = [&](int r) { return !key_padded(p, b, j0 + r, length); };
    load_tile<T, DP>(kt, kLd, kCols, k, p.ks[1], j0, p.D, kvec, keep);
    load_tile<T, DP>(vt, kLd, kCols, v, p.vs[1], j0, p.D, vvec, keep);
    __syncthreads();
    float x[RM][4];
    G::scores(qt, kt, x);
    int kd[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int j = j0 + G::col_group() * 4 + c;
      kd[c] = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
    }
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      float top = -INFINITY, t;
      f.slope2 = slope[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + G::col_group() * 4 + c;
        const bool seen = j < row[r].limit && (!PACK || j < limit) &&
                          (!p.kdoc || same_document(row[r].doc, kd[c], p.shared));
        x[r][c] = seen ? score2(p, f, x[r][c], row[r].place - j, t) : -INFINITY;
        top = fmaxf(top, x[r][c]);
      }
      top = fmaxf(m[r], max16(top));
      const float base = top == -INFINITY ? 0.0f : top;
      const float keep_old = exp2f(m[r] - base);
      m[r] = top;
      float s = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[r][c] = exp2f(x[r][c] - base);
        s += x[r][c];
      }
      l[r] = fmaf(l[r], keep_old, s);
#pragma unroll
      for (int c = 0; c < G::DC; ++c) acc[r][c] *= keep_old;
    }
    G::spread(prob, x);
    G::gather(prob, vt, acc);
  }
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const float s = sum16(l[r]);
    mul[r] = s > 0.0f ? 1.0f / s : (s == 0.0f ? 0.0f : s);
    const int at = r0 + G::row_group() * RM + r;
    if (at >= rows) continue;
    const int64_t out = ((int64_t)b * p.H + h0 + at % pack) * p.Sq + at / pack;
    if constexpr (PACK) {
      const int64_t part = (int64_t)split * p.B * p.H * p.Sq + out;
      if (G::col_group() == 0) p.part_ml[part] = make_float2(m[r], s);
#pragma unroll
      for (int c = 0; c < G::DC; ++c) {
        const int d = G::col_group() + 16 * c;
        if (d < p.D) p.part_o[part * p.D + d] = acc[r][c];
      }
    } else if (p.lse && G::col_group() == 0) {
      p.lse[out] = s == 0.0f ? -INFINITY : (m[r] + log2f(s)) * kLn2;
    }
  }
  if constexpr (!PACK)
    G::each(r0, p.Sq, p.D, [&](int i, int d, int r, int c) {
      put_output<T>(p, (((int64_t)b * p.Sq + i) * p.H + h0) * p.D + d, acc[r][c] * mul[r]);
    });
}

// dq, and delta_i = g_i . o_i for the key gradient that follows.
template <typename T, int DP, int RM>
__global__ void __launch_bounds__(kThreads) attn_simt_dq_kernel(const AttnParams p) {
  using G = Tile<DP, RM>;
  extern __shared__ float4 smem4[];
  float* qt = reinterpret_cast<float*>(smem4);
  float* gt = qt + G::kRowFloats;
  float* kt = gt + G::kRowFloats;
  float* vt = kt + G::kColFloats;
  float* prob = vt + G::kColFloats;
  __shared__ float delta_s[G::kRows];
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hkv);
  const int i0 = (gridDim.x - 1 - blockIdx.x) * G::kRows;
  const int length = attn_length(p, b);
  const int limit = rows_limit(p, b, i0 + G::kRows, length);
  const ScoreForm f = score_form(p, h);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  const bool kvec = can_vec<T>(p.k, p.ks, p.D), vvec = can_vec<T>(p.v, p.vs, p.D);
  const auto in = [&](int r) { return row_view(p, b, i0 + r, length).limit > 0; };
  load_tile<T, DP>(qt, G::kLdr, G::kRows, static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2], p.qs[1], i0, p.D,
                   can_vec<T>(p.q, p.qs, p.D), in);
  load_tile<T, DP>(gt, G::kLdr, G::kRows, static_cast<const T*>(p.go) + b * p.gs[0] + h * p.gs[2], p.gs[1], i0, p.D,
                   can_vec<T>(p.go, p.gs, p.D), in);
  __syncthreads();
  if (threadIdx.x < G::kRows) {
    const int i = i0 + threadIdx.x;
    float s = 0.0f;
    if (i < p.Sq) {
      const int64_t at = (((int64_t)b * p.Sq + i) * p.H + h) * p.D;
      const T *o = static_cast<const T*>(p.o) + at, *low = p.residue ? static_cast<const T*>(p.residue) + at : nullptr;
      for (int d = 0; d < p.D; ++d)
        s = fmaf(to_f32(o[d]) + (low ? to_f32(low[d]) : 0.0f), gt[d * G::kLdr + threadIdx.x], s);
      p.delta[((int64_t)b * p.H + h) * p.Sq + i] = s;
    }
    delta_s[threadIdx.x] = s;
  }
  __syncthreads();
  RowView row[RM];
  float lse2[RM], delta[RM], acc[RM][G::DC];
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const int i = i0 + G::row_group() * RM + r;
    row[r] = row_view(p, b, i, length);
    lse2[r] = i < p.Sq ? p.lse[((int64_t)b * p.H + h) * p.Sq + i] * kLog2e : 0.0f;
    delta[r] = delta_s[G::row_group() * RM + r];
#pragma unroll
    for (int c = 0; c < G::DC; ++c) acc[r][c] = 0.0f;
  }
  for (int j0 = 0; j0 < limit; j0 += kCols) {
    if (skip_tiles(p, b, i0, j0)) continue;
    __syncthreads();
    const auto keep = [&](int r) { return !key_padded(p, b, j0 + r, length); };
    load_tile<T, DP>(kt, kLd, kCols, k, p.ks[1], j0, p.D, kvec, keep);
    load_tile<T, DP>(vt, kLd, kCols, v, p.vs[1], j0, p.D, vvec, keep);
    __syncthreads();
    float x[RM][4], dp[RM][4];
    G::scores(qt, kt, x);
    G::scores(gt, vt, dp);
    int kd[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int j = j0 + G::col_group() * 4 + c;
      kd[c] = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
    }
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + G::col_group() * 4 + c;
        const bool seen = j < row[r].limit && (!p.kdoc || same_document(row[r].doc, kd[c], p.shared));
        float t;
        const float e = exp2f(score2(p, f, x[r][c], row[r].place - j, t) - lse2[r]);
        x[r][c] = seen ? e * (dp[r][c] - delta[r]) * fmaf(-t, t, 1.0f) * p.scale : 0.0f;
      }
    G::spread(prob, x);
    G::gather(prob, kt, acc);
  }
  G::each(i0, p.Sq, p.D, [&](int i, int d, int r, int c) {
    static_cast<T*>(p.dq)[(((int64_t)b * p.Sq + i) * p.H + h) * p.D + d] = from_f32<T>(acc[r][c]);
  });
}

// dk and dv of a tile of keys: every query of every head that shares them, in
// a fixed order.
template <typename T, int DP, int RM>
__global__ void __launch_bounds__(kThreads) attn_simt_dkv_kernel(const AttnParams p) {
  using G = Tile<DP, RM>;
  extern __shared__ float4 smem4[];
  float* kt = reinterpret_cast<float*>(smem4);
  float* vt = kt + G::kRowFloats;
  float* qt = vt + G::kRowFloats;
  float* gt = qt + G::kColFloats;
  float* prob = gt + G::kColFloats;
  __shared__ float lse_s[kCols], delta_s[kCols];
  __shared__ RowView view_s[kCols];
  const int hk = blockIdx.y, b = blockIdx.z, group = p.H / p.Hkv;
  const int j0 = blockIdx.x * G::kRows;
  const int length = attn_length(p, b);
  const auto keep = [&](int r) { return !key_padded(p, b, j0 + r, length); };
  load_tile<T, DP>(kt, G::kLdr, G::kRows, static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2], p.ks[1], j0, p.D,
                   can_vec<T>(p.k, p.ks, p.D), keep);
  load_tile<T, DP>(vt, G::kLdr, G::kRows, static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2], p.vs[1], j0, p.D,
                   can_vec<T>(p.v, p.vs, p.D), keep);
  float dk[RM][G::DC], dv[RM][G::DC];
  int kd[RM];
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const int j = j0 + G::row_group() * RM + r;
    kd[r] = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
#pragma unroll
    for (int c = 0; c < G::DC; ++c) dk[r][c] = dv[r][c] = 0.0f;
  }
  const bool qvec = can_vec<T>(p.q, p.qs, p.D), gvec = can_vec<T>(p.go, p.gs, p.D);
  const int first = j0 < length ? first_query(p, b, j0, length) / kCols * kCols : p.Sq;
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    const ScoreForm f = score_form(p, h);
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T* go = static_cast<const T*>(p.go) + b * p.gs[0] + h * p.gs[2];
    for (int i0 = first; i0 < p.Sq; i0 += kCols) {
      if (skip_tiles(p, b, i0, j0)) continue;
      __syncthreads();
      if (threadIdx.x < kCols) {
        const int i = i0 + threadIdx.x;
        const int64_t at = ((int64_t)b * p.H + h) * p.Sq + i;
        view_s[threadIdx.x] = row_view(p, b, i, length);
        lse_s[threadIdx.x] = i < p.Sq ? p.lse[at] * kLog2e : 0.0f;
        delta_s[threadIdx.x] = i < p.Sq ? p.delta[at] : 0.0f;
      }
      const auto in = [&](int r) { return row_view(p, b, i0 + r, length).limit > 0; };
      load_tile<T, DP>(qt, kLd, kCols, q, p.qs[1], i0, p.D, qvec, in);
      load_tile<T, DP>(gt, kLd, kCols, go, p.gs[1], i0, p.D, gvec, in);
      __syncthreads();
      float x[RM][4], dp[RM][4];
      G::scores(kt, qt, x);
      G::scores(vt, gt, dp);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int col = G::col_group() * 4 + c;
        const RowView row = view_s[col];
        const float lse2 = lse_s[col], delta = delta_s[col];
#pragma unroll
        for (int r = 0; r < RM; ++r) {
          const int j = j0 + G::row_group() * RM + r;
          const bool seen = j < row.limit && (!p.kdoc || same_document(row.doc, kd[r], p.shared));
          float t;
          const float e = exp2f(score2(p, f, x[r][c], row.place - j, t) - lse2);
          x[r][c] = seen ? e : 0.0f;
          dp[r][c] = seen ? e * (dp[r][c] - delta) * fmaf(-t, t, 1.0f) * p.scale : 0.0f;
        }
      }
      G::spread(prob, x);
      G::gather(prob, gt, dv);
      G::spread(prob, dp);
      G::gather(prob, qt, dk);
    }
  }
  G::each(j0, p.Sk, p.D, [&](int j, int d, int r, int c) {
    const int64_t at = (((int64_t)b * p.Sk + j) * p.Hkv + hk) * p.D + d;
    static_cast<T*>(p.dk)[at] = from_f32<T>(dk[r][c]);
    static_cast<T*>(p.dv)[at] = from_f32<T>(dv[r][c]);
  });
}

// Documents of each tile of kDocTile queries or keys: a warp a tile.
__global__ void __launch_bounds__(128) attn_documents_kernel(const AttnParams p, DocTile* qtile, DocTile* ktile) {
  const int nq = (p.Sq + kDocTile - 1) / kDocTile, nk = (p.Sk + kDocTile - 1) / kDocTile;
  const int64_t warp = (int64_t)blockIdx.x * 4 + threadIdx.x / 32, total = (int64_t)p.B * (nq + nk);
  if (warp >= total) return;
  const int b = (int)(warp / (nq + nk));
  int tile = (int)(warp % (nq + nk));
  const bool keys = tile >= nq;
  if (keys) tile -= nq;
  const int S = keys ? attn_length(p, b) : p.Sq;  // keys past their length are padding
  const int* doc = keys ? p.kdoc + (int64_t)b * p.Sk : p.qdoc + (int64_t)b * p.Sq;
  int low = INT32_MAX, high = -1, pad = 0, shared = 0;
  for (int t = threadIdx.x % 32; t < kDocTile; t += 32) {
    const int at = tile * kDocTile + t;
    const int d = at < S ? __ldg(doc + at) : -1;
    if (d < 0) {
      pad = 1;
    } else {
      low = min(low, d), high = max(high, d);
      shared |= d == p.shared;
    }
  }
  low = __reduce_min_sync(kFullMask, low), high = __reduce_max_sync(kFullMask, high);
  pad = __any_sync(kFullMask, pad), shared = __any_sync(kFullMask, shared);
  if (threadIdx.x % 32 == 0) {
    DocTile out{low, high, pad, shared};
    (keys ? ktile + (int64_t)b * nk : qtile + (int64_t)b * nq)[tile] = out;
  }
}

template <typename T, int DP, int RM, bool PACK>
cudaError_t fwd(const AttnParams& p, cudaStream_t st) {
  using G = Tile<DP, RM>;
  constexpr int smem = (G::kRowFloats + 2 * G::kColFloats + G::kProbFloats) * 4;
  static std::atomic<uint64_t> set{0};
  cudaError_t e = abi::allow_smem(attn_simt_fwd_kernel<T, DP, RM, PACK>, smem, set);
  if (e != cudaSuccess) return e;
  const int rows = PACK ? p.Sq * (p.H / p.Hkv) : p.Sq;
  const dim3 grid((rows + G::kRows - 1) / G::kRows * p.splits, PACK ? p.Hkv : p.H, p.B);
  attn_simt_fwd_kernel<T, DP, RM, PACK><<<grid, kThreads, smem, st>>>(p);
  return cudaGetLastError();
}

template <typename T, int DP, int RMQ, int RMK>
cudaError_t bwd(const AttnParams& p, cudaStream_t st) {
  using Q = Tile<DP, RMQ>;
  using K = Tile<DP, RMK>;
  constexpr int smem_q = (2 * Q::kRowFloats + 2 * Q::kColFloats + Q::kProbFloats) * 4;
  constexpr int smem_k = (2 * K::kRowFloats + 2 * K::kColFloats + K::kProbFloats) * 4;
  static std::atomic<uint64_t> set_q{0}, set_k{0};
  cudaError_t e = abi::allow_smem(attn_simt_dq_kernel<T, DP, RMQ>, smem_q, set_q);
  if (e == cudaSuccess) e = abi::allow_smem(attn_simt_dkv_kernel<T, DP, RMK>, smem_k, set_k);
  if (e != cudaSuccess) return e;
  attn_simt_dq_kernel<T, DP, RMQ><<<dim3((p.Sq + Q::kRows - 1) / Q::kRows, p.H, p.B), kThreads, smem_q, st>>>(p);
  attn_simt_dkv_kernel<T, DP, RMK><<<dim3((p.Sk + K::kRows - 1) / K::kRows, p.Hkv, p.B), kThreads, smem_k, st>>>(p);
  return cudaGetLastError();
}

// Rows a thread holds (8, or 4 where the accumulators or tiles would not fit).
template <typename T>
cudaError_t fwd_t(const AttnParams& p, cudaStream_t st) {
  if (p.splits > 1) {
    if (p.D <= 32) return fwd<T, 32, 4, true>(p, st);
    if (p.D <= 64) return fwd<T, 64, 4, true>(p, st);
    if (p.D <= 128) return fwd<T, 128, 4, true>(p, st);
    return fwd<T, 256, 4, true>(p, st);
  }
  if (p.D <= 32) return fwd<T, 32, 8, false>(p, st);
  if (p.D <= 64) return fwd<T, 64, 8, false>(p, st);
  if (p.D <= 128) return fwd<T, 128, 8, false>(p, st);
  return fwd<T, 256, 4, false>(p, st);
}

template <typename T>
cudaError_t bwd_t(const AttnParams& p, cudaStream_t st) {
  if (p.D <= 32) return bwd<T, 32, 8, 8>(p, st);
  if (p.D <= 64) return bwd<T, 64, 8, 8>(p, st);
  if (p.D <= 128) return bwd<T, 128, 8, 4>(p, st);
  return bwd<T, 256, 4, 4>(p, st);
}

}  // namespace

cudaError_t attn_simt_forward(const AttnParams& p, int dtype, cudaStream_t st) {
  if (dtype == MSDA_DTYPE_F32) return fwd_t<float>(p, st);
  return dtype == MSDA_DTYPE_F16 ? fwd_t<__half>(p, st) : fwd_t<__nv_bfloat16>(p, st);
}

cudaError_t attn_simt_backward(const AttnParams& p, int dtype, cudaStream_t st) {
  if (dtype == MSDA_DTYPE_F32) return bwd_t<float>(p, st);
  return dtype == MSDA_DTYPE_F16 ? bwd_t<__half>(p, st) : bwd_t<__nv_bfloat16>(p, st);
}

cudaError_t attn_documents_launch(const AttnParams& p, DocTile* qtile, DocTile* ktile, cudaStream_t st) {
  const int64_t tiles = (int64_t)p.B * ((p.Sq + kDocTile - 1) / kDocTile + (p.Sk + kDocTile - 1) / kDocTile);
  attn_documents_kernel<<<(unsigned)((tiles + 3) / 4), 128, 0, st>>>(p, qtile, ktile);
  return cudaGetLastError();
}

}  // namespace msda
