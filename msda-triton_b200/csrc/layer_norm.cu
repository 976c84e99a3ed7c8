// Layer norm with an optional residual, forward and backward
// (msda_layer_norm_* of include/msda_layer_b200.h).
//
//   h = x + r,  mu = mean(h),  s = 1 / sqrt(mean((h - mu)^2) + eps),  y = (h - mu) s w + b
//   dh = s (gw - mean(gw) - z mean(gw z)) (+ dsum),  z = (h - mu) s,  gw = g w
//   dw = sum_rows g z,  db = sum_rows g
//
// The mean that is kept for the backward is rounded, which shows where a row lies
// many deviations from zero: both directions take out what is left of the centred
// row's own mean.
//
// Bound by HBM: a row is read once, kept in registers by the threads that
// share it (a warp up to 512 channels, 128 to 512 threads up to 8192), and
// written once; the variance is taken about the mean, from the registers. Rows
// are dealt to a grid that fits the GPU, so that a thread keeps its channels'
// weights, and in the backward their gradients' running sums, in registers from
// row to row, and the next row's loads are in flight while a row is reduced.
// Longer rows are bound by the latency of their sums over the CTA, so that these
// go together, two in the forward and three in the backward. (Staging rows in shared
// memory by bulk copies was slower: 20000 x 1000 bf16 forward 91 us for 29.) Rows
// wider than 8192 are read again from L2 for each step. Each CTA leaves one partial row of the two column sums; a second
// kernel adds the partial rows in a fixed order.
//
// 88892 x 256 bf16 with a residual: forward 28 us (137 MB, 4.8 TB/s; three quarters
// of the issue slots are taken, by the sums' shuffles), backward 42 us (182 MB, 4.3
// TB/s: it waits for its loads, with two CTAs an SM at 115 registers) and 5 us for
// the columns. 2500 x 8192 fp32 with a residual: 45 and 63 us (5.5 and 5.2 TB/s);
// 4095 x 5001 fp32, one element a load since rows start at any element: 51 and 88 us
// (3.2 and 2.8 TB/s); wider, 2000 x 20000 bf16 with a residual, a scalar a load and
// rows read again for each step: 142 us, and 209 with 117 for the columns.
#include <algorithm>

#include "msda_abi.cuh"
#include "msda_common.cuh"
#include "msda_layer_b200.h"

namespace msda {
namespace {

constexpr int kNormThreads = 256;
constexpr int kRegisterWidth = 8192;  // widest row held in registers
constexpr int kWideThreads = 1024;    // a CTA of the wider rows' kernels
constexpr int kNormSms = 148;         // grids and workspaces go by this, not by the device

struct NormParams {
  const void *x, *residual, *weight, *bias, *grad_y, *grad_sum;
  void *y, *sum_out, *grad_x;
  float *mean, *rstd;
  float *partial;  // [2][gridDim.x][width]: weight's and bias's column sums
  float *rest;     // (rows,): what the wide rows' kept means leave, in deviations; with columns only
  int64_t rows, x_stride, residual_stride, grad_stride;
  int32_t width;
  int32_t param_f32;  // weight and bias are fp32, not T
  int32_t want_columns;
  float eps;
};

// A weight or bias. The loads are volatile: the pointer is null, or the channel
// past the end, where the caller's condition keeps them from running, and the
// compiler may not move them ahead of it.
template <typename T>
__device__ __forceinline__ float param_at(const void* p, int f32, int c) {
  if (f32 || sizeof(T) == 4) {
    float v;
    asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(static_cast<const float*>(p) + c));
    return v;
  }
  unsigned short bits;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(bits) : "l"(static_cast<const T*>(p) + c));
  return to_f32(*reinterpret_cast<const T*>(&bits));
}

// Sums of N values over the TPR threads that share a row, the same in each of
// them. `red`: N values for each warp of the CTA in each of two buffers, which
// consecutive calls take in turn, so that one barrier a call is enough.
template <int TPR, int N, int M>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[M][32], int buffer) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(kFullMask, v[n], o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) red[buffer][n][threadIdx.x >> 5] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = red[buffer][n][threadIdx.x & (TPR / 32 - 1)];
#pragma unroll
    for (int o = TPR / 64; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(kFullMask, v[n], o);
  }
}

// The same for three values, as the backward wants them: the first two exchanges
// leave a quarter of a warp with each value, 6 shuffles for 15.
template <int TPR>
__device__ __forceinline__ void row_sums_of_three(float (&v)[3], float (*red)[3][32], int buffer) {
  const int lane = threadIdx.x & 31;
  const bool upper = lane & 16, odd = lane & 8;
  float a = upper ? v[2] : v[0], b = upper ? 0.0f : v[1];
  a += __shfl_xor_sync(kFullMask, upper ? v[0] : v[2], 16);
  b += __shfl_xor_sync(kFullMask, upper ? v[1] : 0.0f, 16);
  float c = odd ? b : a;
  c += __shfl_xor_sync(kFullMask, odd ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(kFullMask, c, o);
  if constexpr (TPR == 32) {
#pragma unroll
    for (int n = 0; n < 3; ++n) v[n] = __shfl_sync(kFullMask, c, n * 8);
  } else {
    constexpr int W = TPR / 32;
    if ((lane & 7) == 0 && lane < 24) red[buffer][lane >> 3][threadIdx.x >> 5] = c;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      if constexpr (W <= 8) {
        v[n] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w += 4) {
          const float4 q = *reinterpret_cast<const float4*>(&red[buffer][n][w]);
          v[n] += (q.x + q.y) + (q.z + q.w);
        }
      } else {
        v[n] = red[buffer][n][threadIdx.x & (W - 1)];
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) v[n] += __shfl_xor_sync(kFullMask, v[n], o);
      }
    }
  }
}

// A row's variance from its mean square and what its mean left. The rounding of the
// two can leave less than nothing of a constant row far from zero.
__device__ __forceinline__ float variance(float square, float rest) {
  const float v = fmaf(-rest, rest, square);
  return v < 0.0f ? 0.0f : v;
}

// TPR threads share a row, NV vectors of VEC channels each.
template <typename T, int VEC, int NV, int TPR>
struct RowTile {
  static constexpr int E = VEC * NV;
  using Raw = typename Pack<T, VEC>::Raw;

  static __device__ __forceinline__ int column(int v) { return (v * TPR + (int)(threadIdx.x % TPR)) * VEC; }
  static __device__ __forceinline__ bool inside(int e, int width) { return column(e / VEC) < width; }

  // A row still packed (zeros past its end, or if there is none).
  static __device__ __forceinline__ void fetch(const void* base, int64_t at, int width, bool any, Raw (&raw)[NV]) {
    const T* p = static_cast<const T*>(base) + at;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      raw[v] = Raw{};
      if (any && column(v) < width) raw[v] = load_raw<T, VEC>(p + column(v));
    }
  }

  static __device__ __forceinline__ void unpack(const Raw (&raw)[NV], float (&f)[E]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float e[VEC];
      unpack_raw<T, VEC>(raw[v], e);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[v * VEC + i] = e[i];
    }
  }

  static __device__ __forceinline__ void add(const Raw (&raw)[NV], float (&f)[E]) {
    float g[E];
    unpack(raw, g);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] += g[e];
  }

  static __device__ __forceinline__ void store(void* base, int64_t at, int width, const float (&f)[E]) {
    T* p = static_cast<T*>(base) + at;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = f[v * VEC + i];
      if (column(v) < width) store_vec<T, VEC>(p + column(v), e);
    }
  }

  static __device__ __forceinline__ void params(const void* base, int f32, int width, float none, float (&f)[E]) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = column(v) + i;
        f[v * VEC + i] = none;
        if (base && c < width) f[v * VEC + i] = param_at<T>(base, f32, c);
      }
  }

};

// A CTA's threads, and the rows that it works on at once.
template <int TPR>
__host__ __device__ constexpr int norm_threads() {
  return TPR == 32 ? kNormThreads : TPR;
}
template <int TPR>
__host__ __device__ constexpr int norm_rows() {
  return TPR == 32 ? kNormThreads / 32 : 1;
}

// Rows of 16 channels a thread and more than a warp have no registers left for
// the next row in the backward.
template <int TPR, int E, bool BWD>
__host__ __device__ constexpr bool norm_ahead() {
  return !(BWD && TPR > 32 && E > 8);
}

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(norm_threads<TPR>()) norm_fwd_kernel(const NormParams p) {
  using R = RowTile<T, VEC, NV, TPR>;
  constexpr int E = R::E;
  __shared__ float red[2][2][32];
  const int width = p.width;
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * norm_rows<TPR>();
  int64_t row = (int64_t)blockIdx.x * norm_rows<TPR>() + (TPR == 32 ? threadIdx.x / 32 : 0);
  typename R::Raw next[NV], more[NV];
  R::fetch(p.x, row * p.x_stride, width, row < p.rows, next);
  R::fetch(p.residual, row * p.residual_stride, width, row < p.rows && p.residual, more);
  float w[E], b[E];
  R::params(p.weight, p.param_f32, width, 1.0f, w);
  R::params(p.bias, p.param_f32, width, 0.0f, b);
  for (; row < p.rows; row += step) {
    float h[E];
    R::unpack(next, h);
    if (p.residual) R::add(more, h);
    R::fetch(p.x, (row + step) * p.x_stride, width, row + step < p.rows, next);
    if (p.residual) R::fetch(p.residual, (row + step) * p.residual_stride, width, row + step < p.rows, more);
    if (p.sum_out) R::store(p.sum_out, row * width, width, h);
    float sum[1] = {0.0f}, s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) sum[0] += h[e];
    row_sums<TPR>(sum, red, 0);
    const float mean = sum[0] * inv;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] = R::inside(e, width) ? h[e] - mean : 0.0f;
      s[0] += h[e];
      s[1] = fmaf(h[e], h[e], s[1]);
    }
    row_sums<TPR>(s, red, 1);
    const float rest = s[0] * inv;
    const float rstd = rsqrtf(variance(s[1] * inv, rest) + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = fmaf((h[e] - rest) * rstd, w[e], b[e]);
    R::store(p.y, row * width, width, h);
    if (p.mean && threadIdx.x % TPR == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

// CTAs of 256 threads of the backward that an SM has room for, which the compiler is
// held to (10000 x 1537 bf16: 66 us without, 42 us) and the grid goes by.
__host__ __device__ constexpr int norm_bwd_ctas(int vec) { return vec > 1 ? 3 : 2; }

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(norm_threads<TPR>(), TPR == 256 ? norm_bwd_ctas(VEC) : 1) norm_bwd_kernel(const NormParams p) {
  using R = RowTile<T, VEC, NV, TPR>;
  constexpr int E = R::E, kRows = norm_rows<TPR>();
  constexpr bool kAhead = norm_ahead<TPR, E, true>();
  __shared__ __align__(16) float red[2][3][32];
  const int width = p.width;
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + (TPR == 32 ? threadIdx.x / 32 : 0);
  typename R::Raw next[NV], more[NV], grad[NV];
  float mean = 0.0f, rstd = 0.0f;
  const auto fetch = [&](int64_t r, bool any) {
    R::fetch(p.x, r * p.x_stride, width, any, next);
    R::fetch(p.grad_y, r * p.grad_stride, width, any, grad);
    if (p.residual) R::fetch(p.residual, r * p.residual_stride, width, any, more);
    if (any) mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
  };
  if (kAhead) fetch(row, row < p.rows);
  float w[E], dw[E], db[E];
  R::params(p.weight, p.param_f32, width, 1.0f, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  int turn = 0;
  for (; row < p.rows; row += step, turn ^= 1) {
    if (!kAhead) fetch(row, true);
    float h[E], g[E];
    R::unpack(next, h);
    R::unpack(grad, g);
    if (p.residual) R::add(more, h);
    const float mu = mean, rs = rstd;
    if (kAhead) fetch(row + step, row + step < p.rows);
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] = R::inside(e, width) ? (h[e] - mu) * rs : 0.0f;
      const float gw = g[e] * w[e];
      db[e] += g[e];
      dw[e] = fmaf(g[e], h[e], dw[e]);
      s[0] += gw;
      s[1] = fmaf(gw, h[e], s[1]);
      s[2] += h[e];
    }
    row_sums_of_three<TPR>(s, red, turn);
    // z = h - rest, in what has been summed with h too.
    const float rest = s[2] * inv, c2 = fmaf(-rest, s[0], s[1]) * inv, c1 = fmaf(-rest, c2, s[0] * inv);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dw[e] = fmaf(-rest, g[e], dw[e]);
      g[e] = (g[e] * w[e] - c1 - h[e] * c2) * rs;
    }
    if (p.grad_sum) {
      typename R::Raw sum[NV];
      R::fetch(p.grad_sum, row * width, width, true, sum);
      R::add(sum, g);
    }
    R::store(p.grad_x, row * width, width, g);
  }
  if (!p.want_columns) return;
  float* out = p.partial + (int64_t)blockIdx.x * width;
  const int64_t second = (int64_t)gridDim.x * width;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (R::inside(e, width)) {
        const int c = R::column(e / VEC) + e % VEC;
        out[c] = dw[e];
        out[second + c] = db[e];
      }
  } else {
    // The CTA's warps add their sums in turn, in shared memory.
    __shared__ float sum[2][32 * E];
    for (int r = 0; r < kRows; ++r) {
      if ((int)(threadIdx.x / 32) == r) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int at = e * 32 + (threadIdx.x & 31);
          sum[0][at] = r ? sum[0][at] + dw[e] : dw[e];
          sum[1][at] = r ? sum[1][at] + db[e] : db[e];
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 32 * E; i += kNormThreads) {
      const int e = i / 32, lane = i & 31;
      const int c = ((e / VEC) * 32 + lane) * VEC + e % VEC;
      if (c < width) {
        out[c] = sum[0][i];
        out[second + c] = sum[1][i];
      }
    }
  }
}

// Rows wider than the registers hold: one CTA a row, a scalar a thread.
template <typename T>
__device__ __forceinline__ float wide_at(const NormParams& p, int64_t row, int c) {
  const float h = to_f32(__ldg(static_cast<const T*>(p.x) + row * p.x_stride + c));
  return p.residual ? h + to_f32(__ldg(static_cast<const T*>(p.residual) + row * p.residual_stride + c)) : h;
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_fwd_kernel(const NormParams p) {
  __shared__ float red[2][2][32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float sum[1] = {0.0f}, s[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) sum[0] += wide_at<T>(p, row, c);
    row_sums<kWideThreads>(sum, red, 0);
    const float mean = sum[0] * inv;
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) {
      const float d = wide_at<T>(p, row, c) - mean;
      s[0] += d;
      s[1] = fmaf(d, d, s[1]);
    }
    row_sums<kWideThreads>(s, red, 1);
    const float rest = s[0] * inv, rstd = rsqrtf(variance(s[1] * inv, rest) + p.eps);
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) {
      const float h = wide_at<T>(p, row, c);
      const float w = p.weight ? param_at<T>(p.weight, p.param_f32, c) : 1.0f;
      const float b = p.bias ? param_at<T>(p.bias, p.param_f32, c) : 0.0f;
      static_cast<T*>(p.y)[row * p.width + c] = from_f32<T>(fmaf((h - mean - rest) * rstd, w, b));
      if (p.sum_out) static_cast<T*>(p.sum_out)[row * p.width + c] = from_f32<T>(h);
    }
    if (p.mean && threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_bwd_kernel(const NormParams p) {
  __shared__ __align__(16) float red[2][3][32];
  const float inv = 1.0f / (float)p.width;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    const T* g = static_cast<const T*>(p.grad_y) + row * p.grad_stride;
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) {
      const float gw = to_f32(__ldg(g + c)) * (p.weight ? param_at<T>(p.weight, p.param_f32, c) : 1.0f);
      const float z = (wide_at<T>(p, row, c) - mean) * rstd;
      s[0] += gw;
      s[1] = fmaf(gw, z, s[1]);
      s[2] += z;
    }
    row_sums_of_three<kWideThreads>(s, red, turn);
    turn ^= 1;
    const float rest = s[2] * inv, c2 = fmaf(-rest, s[0], s[1]) * inv, c1 = fmaf(-rest, c2, s[0] * inv);
    if (p.want_columns && threadIdx.x == 0) p.rest[row] = rest;
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) {
      const float gw = to_f32(__ldg(g + c)) * (p.weight ? param_at<T>(p.weight, p.param_f32, c) : 1.0f);
      float d = (gw - c1 - (wide_at<T>(p, row, c) - mean) * rstd * c2) * rstd;
      if (p.grad_sum) d += to_f32(__ldg(static_cast<const T*>(p.grad_sum) + row * p.width + c));
      static_cast<T*>(p.grad_x)[row * p.width + c] = from_f32<T>(d);
    }
  }
}

// The wide rows' column sums: a thread a column, rows dealt to blockIdx.y.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_wide_columns_kernel(const NormParams p) {
  const int c = blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= p.width) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float g = to_f32(__ldg(static_cast<const T*>(p.grad_y) + row * p.grad_stride + c));
    db += g;
    dw = fmaf(g, (wide_at<T>(p, row, c) - __ldg(p.mean + row)) * __ldg(p.rstd + row) - __ldg(p.rest + row), dw);
  }
  p.partial[(int64_t)blockIdx.y * p.width + c] = dw;
  p.partial[((int64_t)gridDim.y + blockIdx.y) * p.width + c] = db;
}

// Column sums of the partial rows: a CTA takes 32 columns of one of the two
// gradients; its warps take every 32nd row and are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_columns_kernel(const float* partial, int rows, int width, void* grad_weight,
                                                            void* grad_bias, int param_f32) {
  __shared__ float tile[32][33];
  void* out = blockIdx.y ? grad_bias : grad_weight;
  if (!out) return;
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const float* p = partial + (int64_t)blockIdx.y * rows * width + c;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int r = warp; r < rows; r += 32) s += __ldcg(p + (int64_t)r * width);
  }
  tile[warp][lane] = s;
  __syncthreads();
  s = tile[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
  const int cc = blockIdx.x * 32 + warp;
  if (lane == 0 && cc < width) {
    if (param_f32) static_cast<float*>(out)[cc] = s;
    else static_cast<T*>(out)[cc] = from_f32<T>(s);
  }
}

using namespace abi;

struct NormShape {
  int vec, nv, tpr;
};

// Threads a row and channels a thread by the width alone: 8 channels, or 16
// where a warp (up to 512) or 512 threads (up to 8192) hold the row with them. A
// barrier for each sum costs more than the threads bring, forward and backward: 40000
// x 512 bf16 27 and 42 us by warps, 37 and 69 us by 128 threads; 20000 x 768 bf16 23
// and 31 us by 128 threads, 38 and 57 us by 256; 10000 x 2048 bf16 25 and 44 us by
// 256, 45 and 59 us by 512. (The slower side's backward had two sums a row, not three.)
int norm_threads_of(int64_t width) { return width <= 512 ? 32 : width <= 1024 ? 128 : width <= 2048 ? 256 : 512; }
int norm_channels_of(int64_t width) { return width <= 8 * norm_threads_of(width) ? 8 : 16; }

// The vector is the widest of 16 bytes, 4 bytes and one element that the
// width, the strides and the buffers allow.
NormShape norm_shape(int64_t width, int es, int64_t unit) {
  const int v16 = 16 / es, v4 = 4 / es;
  NormShape s;
  s.vec = unit % v16 == 0 ? v16 : unit % v4 == 0 ? v4 : 1;
  s.tpr = norm_threads_of(width);
  s.nv = width <= 32 && s.vec == 1 ? 1 : norm_channels_of(width) / s.vec;
  return s;
}

// Most CTAs of a backward, each of which leaves a partial row. (Of the four an SM by
// warps two are resident; grids of two were not measured.)
int64_t norm_backward_most(int64_t width) {
  if (width > kRegisterWidth) return kNormSms * 2;
  return kNormSms * (norm_threads_of(width) <= 256 ? 4 : norm_channels_of(width) == 8 ? 2 : 1);
}

int norm_grid(int64_t rows, const NormShape& s, bool backward, int64_t width) {
  const bool warps = s.tpr == 32;
  const int64_t ctas = warps ? (rows + kNormThreads / 32 - 1) / (kNormThreads / 32) : rows;
  const int64_t most = backward ? (s.tpr == 256 ? kNormSms * norm_bwd_ctas(s.vec) : norm_backward_most(width))
                                : kNormSms * (width > kRegisterWidth ? 2 : 2048 / (warps ? kNormThreads : s.tpr));
  return (int)(ctas < most ? ctas : most);
}

template <typename T>
cudaError_t norm_launch(const NormParams& p, const NormShape& s, bool backward, int grid, cudaStream_t st) {
  if (p.width > kRegisterWidth) {
    if (!backward) {
      norm_wide_fwd_kernel<T><<<grid, kWideThreads, 0, st>>>(p);
    } else {
      norm_wide_bwd_kernel<T><<<grid, kWideThreads, 0, st>>>(p);
      if (p.want_columns)
        norm_wide_columns_kernel<T><<<dim3((p.width + kNormThreads - 1) / kNormThreads, grid), kNormThreads, 0, st>>>(p);
    }
    return cudaGetLastError();
  }
#define MSDA_NORM(VEC_, NV_, TPR_)                                                                  \
  if (s.vec == VEC_ && s.nv == NV_ && s.tpr == TPR_) {                                              \
    if (backward) norm_bwd_kernel<T, VEC_, NV_, TPR_><<<grid, norm_threads<TPR_>(), 0, st>>>(p);    \
    else norm_fwd_kernel<T, VEC_, NV_, TPR_><<<grid, norm_threads<TPR_>(), 0, st>>>(p);             \
    return cudaGetLastError();                                                                      \
  }
#define MSDA_NORM_VEC(VEC_)                                                                         \
  MSDA_NORM(VEC_, 8 / (VEC_), 32) MSDA_NORM(VEC_, 16 / (VEC_), 32) MSDA_NORM(VEC_, 8 / (VEC_), 128) \
  MSDA_NORM(VEC_, 8 / (VEC_), 256) MSDA_NORM(VEC_, 8 / (VEC_), 512) MSDA_NORM(VEC_, 16 / (VEC_), 512)
  MSDA_NORM_VEC(16 / (int)sizeof(T))
  if constexpr (sizeof(T) == 2) {
    MSDA_NORM_VEC(2)
  }
  MSDA_NORM(1, 1, 32)
  MSDA_NORM_VEC(1)
#undef MSDA_NORM_VEC
#undef MSDA_NORM
  return cudaErrorInvalidConfiguration;
}

int check_norm(const char* fn, int64_t rows, int64_t width, int32_t dtype, int32_t param_dtype) {
  if (elem_size(dtype) == 0) return fail(MSDA_ERR_UNSUPPORTED, "%s: unsupported dtype code %d (0=f32, 1=f16, 2=bf16)", fn, dtype);
  if (param_dtype != dtype && param_dtype != MSDA_DTYPE_F32)
    return fail(MSDA_ERR_UNSUPPORTED, "%s: weights are of the rows' dtype or fp32 (got code %d)", fn, param_dtype);
  if (rows < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: negative number of rows", fn);
  if (rows > (int64_t(1) << 40)) return fail(MSDA_ERR_UNSUPPORTED, "%s: too many rows", fn);
  if (width < 1 || width > MSDA_LAYER_NORM_MAX_WIDTH)
    return fail(MSDA_ERR_UNSUPPORTED, "%s: width=%lld outside [1, %d]", fn, (long long)width, MSDA_LAYER_NORM_MAX_WIDTH);
  return MSDA_OK;
}

// What every row's start and length is a multiple of, in elements (up to 16 bytes).
struct Unit {
  int es;
  int64_t unit;
  Unit(int es_, int64_t width) : es(es_), unit(16 / es_) { length(width); }
  void length(int64_t n) {
    while (unit > 1 && n % unit) unit >>= 1;
  }
  void buffer(const void* p) {
    while (unit > 1 && !aligned(p, unit * es)) unit >>= 1;
  }
  void rows(const void* p, int64_t n, int64_t stride) {
    if (!p) return;
    buffer(p);
    if (n > 1) length(stride < 0 ? -stride : stride);
  }
};

}  // namespace
}  // namespace msda

extern "C" {

int msda_layer_norm_forward(const void* x, const void* residual, const void* weight, const void* bias, void* y,
                            void* sum_out, float* mean, float* rstd, int64_t rows, int64_t width, int64_t x_stride,
                            int64_t residual_stride, float eps, int32_t dtype, int32_t param_dtype, void* stream) {
  using namespace msda;
  const char* fn = "msda_layer_norm_forward";
  if (int rc = check_norm(fn, rows, width, dtype, param_dtype)) return rc;
  if (!(eps >= 0)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", fn);
  if (x_stride < 0 || residual_stride < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  if (rows == 0) return succeed();
  if (!x || !y || !mean != !rstd) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  const int es = elem_size(dtype), pes = elem_size(param_dtype);
  const void* buffers[] = {x, residual, y, sum_out};
  for (const void* b : buffers)
    if (!aligned(b, es)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  if (!aligned(weight, pes) || !aligned(bias, pes) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  Unit u(es, width);
  u.rows(x, rows, x_stride);
  u.rows(residual, rows, residual_stride);
  u.rows(y, rows, width);
  u.rows(sum_out, rows, width);
  NormParams p = {};
  p.x = x, p.residual = residual, p.weight = weight, p.bias = bias, p.y = y, p.sum_out = sum_out;
  p.mean = mean, p.rstd = rstd;
  p.rows = rows, p.width = (int32_t)width, p.x_stride = x_stride, p.residual_stride = residual_stride, p.eps = eps;
  p.param_f32 = param_dtype == MSDA_DTYPE_F32;
  const NormShape s = norm_shape(width, es, u.unit);
  const int grid = norm_grid(rows, s, false, width);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == MSDA_DTYPE_F32   ? norm_launch<float>(p, s, false, grid, st)
                  : dtype == MSDA_DTYPE_F16 ? norm_launch<__half>(p, s, false, grid, st)
                                            : norm_launch<__nv_bfloat16>(p, s, false, grid, st);
  if (e != cudaSuccess) return cuda_fail(e, "layer norm launch");
  return succeed();
}

size_t msda_layer_norm_backward_workspace_size(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > MSDA_LAYER_NORM_MAX_WIDTH) return 0;
  const size_t columns = 2 * (size_t)std::min(rows, msda::norm_backward_most(width)) * (size_t)width;
  return sizeof(float) * (columns + (width > msda::kRegisterWidth ? (size_t)rows : 0));
}

int msda_layer_norm_backward(const void* x, const void* residual, const void* weight, const float* mean,
                             const float* rstd, const void* grad_y, const void* grad_sum, void* grad_x,
                             void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                             int64_t rows, int64_t width, int64_t x_stride, int64_t residual_stride,
                             int64_t grad_stride, int32_t dtype, int32_t param_dtype, void* stream) {
  using namespace msda;
  const char* fn = "msda_layer_norm_backward";
  if (int rc = check_norm(fn, rows, width, dtype, param_dtype)) return rc;
  if (x_stride < 0 || residual_stride < 0 || grad_stride < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  const int es = elem_size(dtype), pes = elem_size(param_dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool columns = grad_weight || grad_bias;
  if (!aligned(grad_weight, pes) || !aligned(grad_bias, pes))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  if (rows == 0) {
    void* out[2] = {grad_weight, grad_bias};
    for (void* o : out)
      if (o)
        if (cudaError_t e = cudaMemsetAsync(o, 0, (size_t)width * pes, st)) return cuda_fail(e, "layer norm zero-fill");
    return succeed();
  }
  if (!x || !mean || !rstd || !grad_y || !grad_x) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  const void* buffers[] = {x, residual, grad_y, grad_sum, grad_x};
  for (const void* b : buffers)
    if (!aligned(b, es)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  if (!aligned(weight, pes) || !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(workspace, 4))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  const size_t need = msda_layer_norm_backward_workspace_size(rows, width);
  if (columns && (!workspace || workspace_bytes < need))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, needs %zu", fn, workspace ? workspace_bytes : 0, need);
  Unit u(es, width);
  u.rows(x, rows, x_stride);
  u.rows(residual, rows, residual_stride);
  u.rows(grad_y, rows, grad_stride);
  u.rows(grad_sum, rows, width);
  u.rows(grad_x, rows, width);
  NormParams p = {};
  p.x = x, p.residual = residual, p.weight = weight, p.grad_y = grad_y, p.grad_sum = grad_sum, p.grad_x = grad_x;
  p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.partial = static_cast<float*>(workspace);
  if (columns) p.rest = p.partial + 2 * std::min(rows, norm_backward_most(width)) * width;
  p.rows = rows, p.width = (int32_t)width, p.x_stride = x_stride, p.residual_stride = residual_stride;
  p.grad_stride = grad_stride;
  p.param_f32 = param_dtype == MSDA_DTYPE_F32, p.want_columns = columns;
  const NormShape s = norm_shape(width, es, u.unit);
  const int grid = norm_grid(rows, s, true, width);
  cudaError_t e = dtype == MSDA_DTYPE_F32   ? norm_launch<float>(p, s, true, grid, st)
                  : dtype == MSDA_DTYPE_F16 ? norm_launch<__half>(p, s, true, grid, st)
                                            : norm_launch<__nv_bfloat16>(p, s, true, grid, st);
  if (e == cudaSuccess && columns) {
    const dim3 g((unsigned)((width + 31) / 32), 2);
    if (dtype == MSDA_DTYPE_F32)
      e = launch_ex(norm_columns_kernel<float>, g, dim3(1024), 0, st, true, p.partial, grid, p.width, grad_weight, grad_bias, p.param_f32);
    else if (dtype == MSDA_DTYPE_F16)
      e = launch_ex(norm_columns_kernel<__half>, g, dim3(1024), 0, st, true, p.partial, grid, p.width, grad_weight, grad_bias, p.param_f32);
    else
      e = launch_ex(norm_columns_kernel<__nv_bfloat16>, g, dim3(1024), 0, st, true, p.partial, grid, p.width, grad_weight, grad_bias, p.param_f32);
  }
  if (e != cudaSuccess) return cuda_fail(e, "layer norm backward launch");
  return succeed();
}

}  // extern "C"
