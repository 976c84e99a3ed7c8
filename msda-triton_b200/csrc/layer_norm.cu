// Layer norm with an optional residual, forward and backward
// (msda_layer_norm_* of include/msda_layer_b200.h).
//
//   h = x + r,  mu = mean(h),  s = 1 / sqrt(mean((h - mu)^2) + eps),  y = (h - mu) s w + b
//   dh = s (gw - mean(gw) - z mean(gw z)) (+ dsum),  z = (h - mu) s,  gw = g w
//   dw = sum_rows g z,  db = sum_rows g
//
// Bound by HBM: a row is read once, kept in registers by the threads that
// share it (a warp up to 1024 channels, 256 threads up to 8192), and written
// once; the variance is taken about the mean, from the registers. Wider rows
// are read again from L2 for each of these steps. Rows are dealt to a grid that fits the GPU, so that a thread keeps
// its channels' weights, and in the backward their gradients' running sums,
// in registers from row to row. Each CTA leaves one partial row of the two
// column sums; a second kernel adds the partial rows in a fixed order.
#include "msda_abi.cuh"
#include "msda_common.cuh"
#include "msda_layer_b200.h"

namespace msda {
namespace {

constexpr int kNormThreads = 256;
constexpr int kRegisterWidth = 8192;  // widest row held in registers
constexpr int kWideThreads = 1024;    // a CTA of the wider rows' kernels
constexpr int kPartialRows = 296;  // most CTAs of a backward: two an SM

struct NormParams {
  const void *x, *residual, *weight, *bias, *grad_y, *grad_sum;
  void *y, *sum_out, *grad_x;
  float *mean, *rstd;
  float *partial;  // [2][gridDim.x][width]: weight's and bias's column sums
  int64_t rows, x_stride, residual_stride, grad_stride;
  int32_t width;
  int32_t param_f32;  // weight and bias are fp32, not T
  int32_t want_columns;
  float eps;
};

template <typename T>
__device__ __forceinline__ float param_at(const void* p, int f32, int c) {
  return f32 ? __ldg(static_cast<const float*>(p) + c) : to_f32(__ldg(static_cast<const T*>(p) + c));
}

// Sum over the TPR threads that share a row, the same in each of them. `red`:
// one float for each warp of the CTA in each of a few buffers; consecutive
// calls take different ones, so that one barrier a call is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[32], int buffer) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[buffer][threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < TPR / 32 ? red[buffer][threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  }
  return v;
}

template <typename T, int VEC, int NV, int TPR>
struct RowTile {
  static constexpr int kRows = kNormThreads / TPR;  // rows a CTA works on at once
  static constexpr int E = VEC * NV;

  static __device__ __forceinline__ int column(int v) { return (v * TPR + (int)(threadIdx.x % TPR)) * VEC; }

  static __device__ __forceinline__ void load(const void* base, int64_t at, int width, float (&f)[E]) {
    const T* p = static_cast<const T*>(base) + at;
    typename Pack<T, VEC>::Raw raw[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      raw[v] = typename Pack<T, VEC>::Raw{};
      if (column(v) < width) raw[v] = load_raw<T, VEC>(p + column(v));
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float e[VEC];
      unpack_raw<T, VEC>(raw[v], e);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[v * VEC + i] = e[i];
    }
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
        f[v * VEC + i] = base && c < width ? param_at<T>(base, f32, c) : none;
      }
  }

  static __device__ __forceinline__ bool inside(int e, int width) { return column(e / VEC) < width; }
};

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_kernel(const NormParams p) {
  using R = RowTile<T, VEC, NV, TPR>;
  constexpr int E = R::E;
  __shared__ float red[3][32];
  const int width = p.width;
  const float inv = 1.0f / (float)width;
  float w[E], b[E];
  R::params(p.weight, p.param_f32, width, 1.0f, w);
  R::params(p.bias, p.param_f32, width, 0.0f, b);
  for (int64_t row = (int64_t)blockIdx.x * R::kRows + threadIdx.x / TPR; row < p.rows;
       row += (int64_t)gridDim.x * R::kRows) {
    float h[E];
    R::load(p.x, row * p.x_stride, width, h);
    if (p.residual) {
      float r[E];
      R::load(p.residual, row * p.residual_stride, width, r);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] += r[e];
    }
    if (p.sum_out) R::store(p.sum_out, row * width, width, h);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += h[e];
    const float mean = row_sum<TPR>(s, red, 0) * inv;
    // The mean's rounding is taken out again: it would show where the row
    // lies many deviations from zero.
    float rest = 0.0f;
    s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] = R::inside(e, width) ? h[e] - mean : 0.0f;
      rest += h[e];
      s = fmaf(h[e], h[e], s);
    }
    rest = row_sum<TPR>(rest, red, 1) * inv;
    const float rstd = rsqrtf(fmaf(-rest, rest, row_sum<TPR>(s, red, 2) * inv) + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = fmaf((h[e] - rest) * rstd, w[e], b[e]);
    R::store(p.y, row * width, width, h);
    if (p.mean && threadIdx.x % TPR == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_kernel(const NormParams p) {
  using R = RowTile<T, VEC, NV, TPR>;
  constexpr int E = R::E;
  __shared__ float red[3][32];
  const int width = p.width;
  const float inv = 1.0f / (float)width;
  float w[E], dw[E], db[E];
  R::params(p.weight, p.param_f32, width, 1.0f, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  for (int64_t row = (int64_t)blockIdx.x * R::kRows + threadIdx.x / TPR; row < p.rows;
       row += (int64_t)gridDim.x * R::kRows) {
    float h[E], g[E];
    R::load(p.x, row * p.x_stride, width, h);
    R::load(p.grad_y, row * p.grad_stride, width, g);
    if (p.residual) {
      float r[E];
      R::load(p.residual, row * p.residual_stride, width, r);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] += r[e];
    }
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] = R::inside(e, width) ? (h[e] - mean) * rstd : 0.0f;
      db[e] += g[e];
      dw[e] = fmaf(g[e], h[e], dw[e]);
      g[e] *= w[e];
      s1 += g[e];
      s2 = fmaf(g[e], h[e], s2);
    }
    const float c1 = row_sum<TPR>(s1, red, 0) * inv, c2 = row_sum<TPR>(s2, red, 1) * inv;
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = (g[e] - c1 - h[e] * c2) * rstd;
    if (p.grad_sum) {
      R::load(p.grad_sum, row * width, width, h);
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] += h[e];
    }
    R::store(p.grad_x, row * width, width, g);
  }
  if (!p.want_columns) return;
  float* out = p.partial + (int64_t)blockIdx.x * width;
  const int64_t second = (int64_t)gridDim.x * width;
  if constexpr (R::kRows == 1) {
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
    for (int r = 0; r < R::kRows; ++r) {
      if ((int)(threadIdx.x / TPR) == r) {
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
  __shared__ float red[3][32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float s = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) s += wide_at<T>(p, row, c);
    const float mean = row_sum<kWideThreads>(s, red, 0) * inv;
    float rest = 0.0f;
    s = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) {
      const float d = wide_at<T>(p, row, c) - mean;
      rest += d;
      s = fmaf(d, d, s);
    }
    rest = row_sum<kWideThreads>(rest, red, 1) * inv;
    const float rstd = rsqrtf(fmaf(-rest, rest, row_sum<kWideThreads>(s, red, 2) * inv) + p.eps);
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
  __shared__ float red[3][32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    const T* g = static_cast<const T*>(p.grad_y) + row * p.grad_stride;
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += kWideThreads) {
      const float gw = to_f32(__ldg(g + c)) * (p.weight ? param_at<T>(p.weight, p.param_f32, c) : 1.0f);
      s1 += gw;
      s2 = fmaf(gw, (wide_at<T>(p, row, c) - mean) * rstd, s2);
    }
    const float c1 = row_sum<kWideThreads>(s1, red, 0) * inv, c2 = row_sum<kWideThreads>(s2, red, 1) * inv;
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
    dw = fmaf(g, (wide_at<T>(p, row, c) - __ldg(p.mean + row)) * __ldg(p.rstd + row), dw);
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

// The vector is the widest of 16 bytes, 4 bytes and one element that the
// width, the strides and the buffers allow; then the fewest threads a row that
// hold it in at most 32 registers each.
NormShape norm_shape(int64_t width, int es, int64_t unit) {
  const int v16 = 16 / es, v4 = 4 / es;
  NormShape s;
  s.vec = unit % v16 == 0 ? v16 : unit % v4 == 0 ? v4 : 1;
  s.tpr = width <= 1024 ? 32 : 256;
  const int64_t vectors = (width + s.vec - 1) / s.vec;
  s.nv = next_pow2((int)((vectors + s.tpr - 1) / s.tpr));
  if (s.nv * s.vec < 8 && s.nv * s.vec > 1) s.nv = s.vec >= 8 ? 1 : 8 / s.vec;
  return s;
}

int norm_grid(int64_t rows, const NormShape& s, bool backward) {
  const int64_t per_cta = kNormThreads / s.tpr;
  const int64_t ctas = (rows + per_cta - 1) / per_cta;
  // Forward: as many CTAs as can be resident; backward: two an SM, since
  // each leaves a partial row.
  const int64_t most = backward ? kPartialRows : (int64_t)sm_count() * 8;
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
#define MSDA_NORM(VEC_, NV_, TPR_)                                                                      \
  if (s.vec == VEC_ && s.nv == NV_ && s.tpr == TPR_) {                                                  \
    if (backward) norm_bwd_kernel<T, VEC_, NV_, TPR_><<<grid, kNormThreads, 0, st>>>(p);                     \
    else norm_fwd_kernel<T, VEC_, NV_, TPR_><<<grid, kNormThreads, 0, st>>>(p);                              \
    return cudaGetLastError();                                                                          \
  }
#define MSDA_NORM_TPR(VEC_, NV_) MSDA_NORM(VEC_, NV_, 32) MSDA_NORM(VEC_, NV_, 256)
  if constexpr (sizeof(T) == 2) {
    MSDA_NORM_TPR(8, 1)
    MSDA_NORM_TPR(8, 2)
    MSDA_NORM_TPR(8, 4)
    MSDA_NORM_TPR(2, 4)
    MSDA_NORM_TPR(2, 8)
    MSDA_NORM_TPR(2, 16)
  } else {
    MSDA_NORM_TPR(4, 2)
    MSDA_NORM_TPR(4, 4)
    MSDA_NORM_TPR(4, 8)
  }
  MSDA_NORM(1, 1, 32)
  MSDA_NORM_TPR(1, 8)
  MSDA_NORM_TPR(1, 16)
  MSDA_NORM_TPR(1, 32)
#undef MSDA_NORM_TPR
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
  const int grid = norm_grid(rows, s, false);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == MSDA_DTYPE_F32   ? norm_launch<float>(p, s, false, grid, st)
                  : dtype == MSDA_DTYPE_F16 ? norm_launch<__half>(p, s, false, grid, st)
                                            : norm_launch<__nv_bfloat16>(p, s, false, grid, st);
  if (e != cudaSuccess) return cuda_fail(e, "layer norm launch");
  return succeed();
}

size_t msda_layer_norm_backward_workspace_size(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > MSDA_LAYER_NORM_MAX_WIDTH) return 0;
  return sizeof(float) * 2 * (size_t)(rows < msda::kPartialRows ? rows : msda::kPartialRows) * (size_t)width;
}

int msda_layer_norm_backward(const void* x, const void* residual, const void* weight, const float* mean,
                             const float* rstd, const void* grad_y, const void* grad_sum, void* grad_x,
                             void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                             int64_t rows, int64_t width, int64_t x_stride, int64_t residual_stride,
                             int64_t grad_stride, int32_t dtype, int32_t param_dtype, void* stream) {
  using namespace msda;
  const char* fn = "msda_layer_norm_backward";
  if (int rc = check_norm(fn, rows, width, dtype, param_dtype)) return rc;
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
  p.rows = rows, p.width = (int32_t)width, p.x_stride = x_stride, p.residual_stride = residual_stride;
  p.grad_stride = grad_stride;
  p.param_f32 = param_dtype == MSDA_DTYPE_F32, p.want_columns = columns;
  const NormShape s = norm_shape(width, es, u.unit);
  const int grid = norm_grid(rows, s, true);
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
