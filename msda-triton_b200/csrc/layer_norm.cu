// Layer norm with an optional residual, forward and backward
// (msda_layer_norm_* of include/msda_layer_b200.h).
//
//   h = x + r,  mu = mean(h),  s = 1 / sqrt(mean((h - mu)^2) + eps),  y = (h - mu) s w + b
//   dh = s (gw - mean(gw) - z mean(gw z)) (+ dsum),  z = (h - mu) s,  gw = g w
//   dw = sum_rows g z,  db = sum_rows g
//
// Bound by HBM: a row is read once, kept in registers by the threads that
// share it, and written once; the variance is taken about the mean, from the
// registers. Rows are dealt to a grid that fits the GPU, so that a thread keeps
// its channels' weights, and in the backward their gradients' running sums, in
// registers from row to row. What matters is how many bytes are in flight:
//   - up to 512 channels a warp has a row, and loads the next one while it
//     reduces this one;
//   - up to 8192 channels a CTA has a row, and bulk copies bring the next ones
//     to a ring in shared memory. (With the rows in registers alone, 256 to 1024
//     threads each, the backward of 4095 x 5001 in fp32 took 92 to 117 us.)
//   - wider rows are read again from L2 for each step.
// Each CTA leaves one partial row of the two column sums; a second kernel adds
// the partial rows in a fixed order.
#include <algorithm>

#include "msda_abi.cuh"
#include "msda_common.cuh"
#include "layer_tcgen05.cuh"
#include "msda_layer_b200.h"

namespace msda {
namespace {

constexpr int kNormThreads = 256;
constexpr int kWarpWidth = 512;       // widest row of a warp
constexpr int kRegisterWidth = 8192;  // widest row of a CTA
constexpr int kWideThreads = 1024;    // a CTA of the wider rows' kernels
constexpr int kNormSms = 148;         // grids and workspaces go by this, not by the device

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

  // The same from shared memory.
  static __device__ __forceinline__ void staged(const char* row, int width, Raw (&raw)[NV]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      raw[v] = Raw{};
      if (column(v) < width) raw[v] = *reinterpret_cast<const Raw*>(row + column(v) * (int)sizeof(T));
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

  // A row h = x (+ r) to y, its mean and reciprocal deviation. scale(e, z): the
  // normalised channel with its weight and bias.
  template <typename Scale>
  static __device__ __forceinline__ void normalise(const NormParams& p, int64_t row, float (&h)[E], float (*red)[32], float inv,
                                                   Scale scale) {
    const int width = p.width;
    if (p.sum_out) store(p.sum_out, row * width, width, h);
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
      h[e] = inside(e, width) ? h[e] - mean : 0.0f;
      rest += h[e];
      s = fmaf(h[e], h[e], s);
    }
    rest = row_sum<TPR>(rest, red, 1) * inv;
    const float rstd = rsqrtf(fmaf(-rest, rest, row_sum<TPR>(s, red, 2) * inv) + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = scale(e, (h[e] - rest) * rstd);
    store(p.y, row * width, width, h);
    if (p.mean && threadIdx.x % TPR == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }

  // The gradient of row h = x (+ r) from g, and the column sums' share.
  template <typename Weight>
  static __device__ __forceinline__ void differentiate(const NormParams& p, int64_t row, float mean, float rstd, float (&h)[E],
                                                       float (&g)[E], float (&dw)[E], float (&db)[E], float (*red)[32], float inv,
                                                       Weight weight) {
    const int width = p.width;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] = inside(e, width) ? (h[e] - mean) * rstd : 0.0f;
      db[e] += g[e];
      dw[e] = fmaf(g[e], h[e], dw[e]);
      g[e] *= weight(e);
      s1 += g[e];
      s2 = fmaf(g[e], h[e], s2);
    }
    const float c1 = row_sum<TPR>(s1, red, 0) * inv, c2 = row_sum<TPR>(s2, red, 1) * inv;
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = (g[e] - c1 - h[e] * c2) * rstd;
    if (p.grad_sum) {
      Raw sum[NV];
      fetch(p.grad_sum, row * width, width, true, sum);
      add(sum, g);
    }
    store(p.grad_x, row * width, width, g);
  }
};

// A warp a row.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_kernel(const NormParams p) {
  using R = RowTile<T, VEC, NV, 32>;
  constexpr int E = R::E;
  const int width = p.width;
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * (kNormThreads / 32);
  int64_t row = (int64_t)blockIdx.x * (kNormThreads / 32) + threadIdx.x / 32;
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
    R::normalise(p, row, h, nullptr, inv, [&](int e, float z) { return fmaf(z, w[e], b[e]); });
  }
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_kernel(const NormParams p) {
  using R = RowTile<T, VEC, NV, 32>;
  constexpr int E = R::E, kRows = kNormThreads / 32;
  const int width = p.width;
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / 32;
  typename R::Raw next[NV], more[NV], grad[NV];
  R::fetch(p.x, row * p.x_stride, width, row < p.rows, next);
  R::fetch(p.grad_y, row * p.grad_stride, width, row < p.rows, grad);
  R::fetch(p.residual, row * p.residual_stride, width, row < p.rows && p.residual, more);
  float mean = 0.0f, rstd = 0.0f;
  if (row < p.rows) mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
  float w[E], dw[E], db[E];
  R::params(p.weight, p.param_f32, width, 1.0f, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  for (; row < p.rows; row += step) {
    float h[E], g[E];
    R::unpack(next, h);
    R::unpack(grad, g);
    if (p.residual) R::add(more, h);
    const float mu = mean, rs = rstd;
    const bool again = row + step < p.rows;
    R::fetch(p.x, (row + step) * p.x_stride, width, again, next);
    R::fetch(p.grad_y, (row + step) * p.grad_stride, width, again, grad);
    if (p.residual) R::fetch(p.residual, (row + step) * p.residual_stride, width, again, more);
    if (again) mean = __ldg(p.mean + row + step), rstd = __ldg(p.rstd + row + step);
    R::differentiate(p, row, mu, rs, h, g, dw, db, nullptr, inv, [&](int e) { return w[e]; });
  }
  if (!p.want_columns) return;
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
  float* out = p.partial + (int64_t)blockIdx.x * width;
  const int64_t second = (int64_t)gridDim.x * width;
  for (int i = threadIdx.x; i < 32 * E; i += kNormThreads) {
    const int e = i / 32, lane = i & 31;
    const int c = ((e / VEC) * 32 + lane) * VEC + e % VEC;
    if (c < width) {
      out[c] = sum[0][i];
      out[second + c] = sum[1][i];
    }
  }
}

// A CTA a row, from a ring of staged rows. A slot holds the row of each input
// (x, gradient, residual) with the 16-byte pieces that its ends lie in; the last
// piece of a row after which the buffer may end is left out, and loaded apart.
struct NormSlots {
  const char* base[3];
  int64_t stride[3];  // bytes
  int inputs, slots, slot_row;  // slot_row: bytes of one input's row in a slot
};

__device__ __forceinline__ void stage_row(const NormSlots& s, char* slot, uint64_t* bar, int64_t row, int bytes, bool last) {
  uint32_t total = 0;
  for (int i = 0; i < s.inputs; ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(s.base[i] + row * s.stride[i]), end = at + bytes;
    const uintptr_t low = at & ~uintptr_t(15), high = last ? end & ~uintptr_t(15) : (end + 15) & ~uintptr_t(15);
    if (high > low) total += (uint32_t)(high - low);
  }
  tc::bar_expect(bar, total);
  for (int i = 0; i < s.inputs; ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(s.base[i] + row * s.stride[i]), end = at + bytes;
    const uintptr_t low = at & ~uintptr_t(15), high = last ? end & ~uintptr_t(15) : (end + 15) & ~uintptr_t(15);
    if (high > low)
      asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   ::"r"(tc::smem_u32(slot + i * s.slot_row)), "l"(low), "r"((uint32_t)(high - low)), "r"(tc::smem_u32(bar))
                   : "memory");
  }
}

// CTAs an SM that the ring is laid out for.
template <int E, bool BWD>
constexpr int staged_resident() {
  return E == 32 ? (BWD ? 1 : 2) : E == 16 ? (BWD ? 2 : 3) : (BWD ? 3 : 4);
}

template <typename T, int VEC, int NV, bool BWD>
__global__ void __launch_bounds__(kNormThreads, (staged_resident<VEC * NV, BWD>()))
    norm_staged_kernel(const NormParams p, const NormSlots s) {
  using R = RowTile<T, VEC, NV, kNormThreads>;
  constexpr int E = R::E, kMost = 8;
  extern __shared__ __align__(128) char ring[];
  __shared__ uint64_t full[kMost];
  __shared__ float red[3][32];
  __shared__ int abort_flag;
  const int width = p.width, bytes = width * (int)sizeof(T);
  const float inv = 1.0f / (float)width;
  float* ws = reinterpret_cast<float*>(ring + s.slots * s.inputs * s.slot_row);  // weights, then biases
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < s.slots; ++i) tc::bar_init(&full[i], 1);
    tc::fence_async_smem();
  }
  // Whether the buffer may end with this row.
  const auto last = [&](int64_t row) {
    bool l = row + 1 == p.rows;
    for (int i = 0; i < s.inputs; ++i) l = l || s.stride[i] < bytes;
    return l;
  };
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 0; i < s.slots; ++i) {
      const int64_t row = blockIdx.x + (int64_t)i * gridDim.x;
      if (row < p.rows) stage_row(s, ring + i * s.inputs * s.slot_row, &full[i], row, bytes, last(row));
    }
  float w[E], b[BWD ? 1 : E], dw[BWD ? E : 1], db[BWD ? E : 1];
  constexpr bool kHold = E == 8;  // the parameters in registers; else in shared memory
  if constexpr (kHold) {
    R::params(p.weight, p.param_f32, width, 1.0f, w);
    if constexpr (!BWD) R::params(p.bias, p.param_f32, width, 0.0f, b);
  } else {
    for (int c = threadIdx.x; c < width; c += kNormThreads) {
      ws[c] = 1.0f;
      if (p.weight) ws[c] = param_at<T>(p.weight, p.param_f32, c);
      if constexpr (!BWD) {
        ws[width + c] = 0.0f;
        if (p.bias) ws[width + c] = param_at<T>(p.bias, p.param_f32, c);
      }
    }
    __syncthreads();
  }
  if constexpr (BWD) {
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  }
  int n = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, ++n) {
    const int at = n % s.slots;
    char* slot = ring + at * s.inputs * s.slot_row;
    float mean = 0.0f, rstd = 0.0f;
    if constexpr (BWD) mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    bool ok = tc::bar_wait(&full[at], (n / s.slots) & 1, &abort_flag);
    // Where an input's row starts in the slot.
    const auto from = [&](int i) { return slot + i * s.slot_row + (reinterpret_cast<uintptr_t>(s.base[i] + row * s.stride[i]) & 15); };
    if (last(row)) {  // the pieces left out
      for (int i = 0; i < s.inputs; ++i) {
        const T* src = reinterpret_cast<const T*>(s.base[i] + row * s.stride[i]);
        const uintptr_t start = reinterpret_cast<uintptr_t>(src), cut = (start + bytes) & ~uintptr_t(15);
        const int c = (cut > start ? (int)((cut - start) / sizeof(T)) : 0) + threadIdx.x;
        if (c < width) reinterpret_cast<T*>(from(i))[c] = src[c];
      }
      __syncthreads();
    }
    typename R::Raw raw[NV];
    float h[E];
    R::staged(from(0), width, raw);
    R::unpack(raw, h);
    if (p.residual) {
      R::staged(from(BWD ? 2 : 1), width, raw);
      R::add(raw, h);
    }
    if constexpr (BWD) {
      float g[E];
      R::staged(from(1), width, raw);
      R::unpack(raw, g);
      if (!ok) mean = NAN;
      R::differentiate(p, row, mean, rstd, h, g, dw, db, red, inv, [&](int e) {
        if constexpr (kHold) return w[e];
        return ws[min(R::column(e / VEC) + e % VEC, width - 1)];
      });
    } else {
      if (!ok) h[0] = NAN;
      R::normalise(p, row, h, red, inv, [&](int e, float z) {
        if constexpr (kHold) return fmaf(z, w[e], b[e]);
        const int c = min(R::column(e / VEC) + e % VEC, width - 1);
        return fmaf(z, ws[c], ws[width + c]);
      });
    }
    // Every thread has read the slot: all have come to the row's sums since.
    const int64_t later = row + (int64_t)s.slots * gridDim.x;
    if (threadIdx.x == 0 && later < p.rows && ok) {
      tc::fence_async_smem();
      stage_row(s, slot, &full[at], later, bytes, last(later));
    }
  }
  if constexpr (BWD) {
    if (!p.want_columns) return;
    float* out = p.partial + (int64_t)blockIdx.x * width;
    const int64_t second = (int64_t)gridDim.x * width;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (R::inside(e, width)) {
        const int c = R::column(e / VEC) + e % VEC;
        out[c] = dw[e];
        out[second + c] = db[e];
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
  int vec, nv;
  bool staged, wide;
};

// Channels a thread of a CTA's row: 8, or more where that does not hold it.
int staged_channels(int64_t width) { return width <= 8 * kNormThreads ? 8 : width <= 16 * kNormThreads ? 16 : 32; }

// The vector is the widest of 16 bytes, 4 bytes and one element that the
// width, the strides and the buffers allow. `whole`: the inputs' buffers start on
// 16 bytes, as staging takes them.
NormShape norm_shape(int64_t width, int es, int64_t unit, bool whole) {
  const int v16 = 16 / es, v4 = 4 / es;
  NormShape s;
  s.vec = unit % v16 == 0 ? v16 : unit % v4 == 0 ? v4 : 1;
  s.staged = width > kWarpWidth && width <= kRegisterWidth && whole;
  s.wide = width > kWarpWidth && !s.staged;
  if (s.staged) s.nv = staged_channels(width) / s.vec;
  else s.nv = width <= 32 && s.vec == 1 ? 1 : (width <= 256 ? 8 : 16) / s.vec;
  return s;
}

// Most CTAs of a backward, each of which leaves a partial row.
int64_t norm_backward_most(int64_t width) {
  if (width <= kWarpWidth) return kNormSms * (width <= 256 ? 4 : 2);
  if (width > kRegisterWidth) return kNormSms * 2;
  const int e = staged_channels(width);
  return kNormSms * (e == 8 ? staged_resident<8, true>() : e == 16 ? staged_resident<16, true>() : staged_resident<32, true>());
}

int norm_grid(int64_t rows, const NormShape& s, bool backward, int64_t width) {
  const int64_t per_cta = s.staged || s.wide ? 1 : kNormThreads / 32;
  const int64_t ctas = (rows + per_cta - 1) / per_cta;
  int64_t most = norm_backward_most(width);
  if (!backward) {
    const int e = staged_channels(width);
    most = kNormSms * (s.wide ? 2 : !s.staged ? 8 : e == 8 ? staged_resident<8, false>() : e == 16 ? staged_resident<16, false>()
                                                                                                    : staged_resident<32, false>());
  }
  return (int)(ctas < most ? ctas : most);
}

template <typename T, int VEC, int NV, bool BWD>
cudaError_t staged_launch(const NormParams& p, int grid, cudaStream_t st) {
  constexpr int E = VEC * NV;
  NormSlots s = {};
  int n = 0;
  const auto input = [&](const void* base, int64_t stride) {
    s.base[n] = static_cast<const char*>(base);
    s.stride[n++] = stride * (int64_t)sizeof(T);
  };
  input(p.x, p.x_stride);
  if (BWD) input(p.grad_y, p.grad_stride);
  if (p.residual) input(p.residual, p.residual_stride);
  s.inputs = n;
  s.slot_row = (p.width * (int)sizeof(T) + 15) / 16 * 16 + 16;
  // The ring takes what the CTA's share of an SM's shared memory leaves.
  const int room = 220 * 1024 / staged_resident<E, BWD>() - 2048 - (E == 8 ? 0 : (BWD ? 4 : 8) * p.width);
  s.slots = std::min(8, room / (s.inputs * s.slot_row));
  if (s.slots < 1) s.slots = 1;
  const int smem = s.slots * s.inputs * s.slot_row + (E == 8 ? 0 : (BWD ? 4 : 8) * p.width);
  static std::atomic<uint64_t> set{0};
  cudaError_t e = allow_smem(norm_staged_kernel<T, VEC, NV, BWD>, 220 * 1024, set);
  if (e != cudaSuccess) return e;
  norm_staged_kernel<T, VEC, NV, BWD><<<grid, kNormThreads, smem, st>>>(p, s);
  return cudaGetLastError();
}

template <typename T>
cudaError_t norm_launch(const NormParams& p, const NormShape& s, bool backward, int grid, cudaStream_t st) {
  if (s.wide) {
    if (!backward) {
      norm_wide_fwd_kernel<T><<<grid, kWideThreads, 0, st>>>(p);
    } else {
      norm_wide_bwd_kernel<T><<<grid, kWideThreads, 0, st>>>(p);
      if (p.want_columns)
        norm_wide_columns_kernel<T><<<dim3((p.width + kNormThreads - 1) / kNormThreads, grid), kNormThreads, 0, st>>>(p);
    }
    return cudaGetLastError();
  }
#define MSDA_NORM(VEC_, NV_)                                                                 \
  if (!s.staged && s.vec == VEC_ && s.nv == NV_) {                                           \
    if (backward) norm_bwd_kernel<T, VEC_, NV_><<<grid, kNormThreads, 0, st>>>(p);           \
    else norm_fwd_kernel<T, VEC_, NV_><<<grid, kNormThreads, 0, st>>>(p);                    \
    return cudaGetLastError();                                                               \
  }
#define MSDA_NORM_STAGED(VEC_, NV_)                                                          \
  if (s.staged && s.vec == VEC_ && s.nv == NV_)                                              \
    return backward ? staged_launch<T, VEC_, NV_, true>(p, grid, st) : staged_launch<T, VEC_, NV_, false>(p, grid, st);
#define MSDA_NORM_VEC(VEC_)                                                                  \
  MSDA_NORM(VEC_, 8 / (VEC_)) MSDA_NORM(VEC_, 16 / (VEC_)) MSDA_NORM_STAGED(VEC_, 8 / (VEC_)) \
  MSDA_NORM_STAGED(VEC_, 16 / (VEC_)) MSDA_NORM_STAGED(VEC_, 32 / (VEC_))
  MSDA_NORM_VEC(16 / (int)sizeof(T))
  if constexpr (sizeof(T) == 2) {
    MSDA_NORM_VEC(2)
  }
  MSDA_NORM(1, 1)
  MSDA_NORM_VEC(1)
#undef MSDA_NORM_VEC
#undef MSDA_NORM_STAGED
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
  const NormShape s = norm_shape(width, es, u.unit, aligned(x, 16) && aligned(residual, 16));
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
  return sizeof(float) * 2 * (size_t)std::min(rows, msda::norm_backward_most(width)) * (size_t)width;
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
  p.rows = rows, p.width = (int32_t)width, p.x_stride = x_stride, p.residual_stride = residual_stride;
  p.grad_stride = grad_stride;
  p.param_f32 = param_dtype == MSDA_DTYPE_F32, p.want_columns = columns;
  const NormShape s = norm_shape(width, es, u.unit, aligned(x, 16) && aligned(residual, 16) && aligned(grad_y, 16));
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
