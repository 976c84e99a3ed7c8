// Rotary positions over several axes (msda_rotary of include/msda_layer_b200.h).
//
//   a' = a cos t - b sin t,  b' = a sin t + b cos t,  t = position[axis] * base^(-2k/n)
//
// for the pair (a, b) of channels that the ladder's step k turns. The kernel
// is bound by HBM: each head vector is read once and written once. A CTA takes
// a few tokens, forms the cosines and sines of their pairs once in shared
// memory, and turns every query and key head of those tokens with them, 16
// bytes a thread at a time, two items in flight. Query and key of 4 x 22223
// tokens, 16 heads of 32 bf16 channels in all (182 MB) take 38 us, 4.8 TB/s; of 2 x
// 16384 tokens, 40 heads of 128 (671 MB), 110 us interleaved, 6.1 TB/s, 131 us by
// halves, 5.1 TB/s. What is above the bytes' time is the items' index arithmetic,
// the cosines, of which a token's 16 serve only 16 heads in the first case, and the
// last wave of CTAs. (Four items in flight: 138 us by halves, at fewer CTAs an SM;
// one: 44 us in the first case.)
#include <cmath>

#include "msda_abi.cuh"
#include "msda_common.cuh"
#include "msda_layer_b200.h"

namespace msda {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kMaxPairs = MSDA_ROTARY_MAX_HEAD_DIM / 2;
constexpr int kMaxCached = 1024;  // cosine / sine pairs a CTA holds (8 KB)
constexpr int kMaxTokens = 128;   // tokens a CTA holds

struct RotaryTable {
  // Frequencies in turns per unit of position, as the sum of two fp32 numbers.
  float hi[kMaxPairs];
  float lo[kMaxPairs];
  uint16_t first[kMaxPairs], second[kMaxPairs];  // the pair's channels
  uint8_t axis[kMaxPairs];
};

struct RotaryParams {
  const void* x[2];  // query, key
  void* y[2];
  const void* positions;
  int64_t stride[2][3];  // (B, S, H) of query and key
  int64_t position_batch_stride;
  int64_t tokens;  // B * S
  uint32_t seq;
  int32_t heads[2], D, pairs, num_axes, position_type, tokens_per_cta, items, all_heads;
  uint32_t items_magic, heads_magic, pairs_magic;  // ceil(2^32 / d): n / d = umulhi(n, magic) for n * d < 2^32
  float sign;
};

__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d, uint32_t magic) {
  return d == 1 ? n : __umulhi(n, magic);
}

__device__ __forceinline__ float position_at(const RotaryParams& p, int64_t at) {
  if (p.position_type == MSDA_POSITION_F32) return __ldg(static_cast<const float*>(p.positions) + at);
  if (p.position_type == MSDA_POSITION_I32) return (float)__ldg(static_cast<const int*>(p.positions) + at);
  return (float)__ldg(static_cast<const long long*>(p.positions) + at);
}

// A thread's item: VP pairs, or as many bytes of the channels that pass
// through. HALF: the pairs' first and second channels are VP contiguous
// elements each; else they are 2 VP contiguous elements (read one by one for
// VP = 0, which stands for one pair without alignment).
template <typename T, int VP, bool HALF>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p,
                                                                const __grid_constant__ RotaryTable table) {
  constexpr int N = VP == 0 ? 1 : VP;                   // pairs an item
  constexpr int W = HALF ? N : (VP == 0 ? 1 : 2 * VP);  // elements a load
  constexpr bool TWO = HALF || VP == 0;                 // an item is two loads
  constexpr int U = 2;                                  // items in flight a thread
  using Raw = typename Pack<T, W>::Raw;
  __shared__ __align__(16) float2 turn[kMaxCached];
  __shared__ int64_t from[3][kMaxTokens];  // the tokens' rows of query and key, and their positions
  // The table, which lanes read at places of their own: constant memory would
  // serve these one after the other (4 x 8000 tokens, 12 heads of 74 fp32 channels
  // on three axes: 226 us for 79).
  __shared__ float2 frequency[kMaxPairs];
  __shared__ ushort2 channels[kMaxPairs];
  __shared__ uint8_t axis[kMaxPairs];
  for (int k = threadIdx.x; k < p.pairs; k += kRotaryThreads) {
    frequency[k] = make_float2(table.hi[k], table.lo[k]);
    channels[k] = make_ushort2(table.first[k], table.second[k]);
    axis[k] = table.axis[k];
  }
  const int64_t token0 = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int count = (int)min((int64_t)p.tokens_per_cta, p.tokens - token0);
  if ((int)threadIdx.x < count) {
    const int t = threadIdx.x;
    const int64_t b = (token0 + t) / p.seq, s = token0 + t - b * p.seq;
    from[0][t] = b * p.stride[0][0] + s * p.stride[0][1];
    from[1][t] = b * p.stride[1][0] + s * p.stride[1][1];
    from[2][t] = b * p.position_batch_stride + s * p.num_axes;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (uint32_t)(count * p.pairs); i += kRotaryThreads) {
    const uint32_t t = quotient(i, p.pairs, p.pairs_magic);
    const int k = i - t * p.pairs;
    const float pos = position_at(p, from[2][t] + axis[k]);
    // pos * frequency exactly, as h + l; whole turns leave h without a rounding.
    const float2 freq = frequency[k];
    const float f = freq.x, h = pos * f, l = fmaf(pos, f, -h);
    const float turns = (h - rintf(h)) + fmaf(pos, freq.y, l);
    float sn, cs;
    sincospif(2.0f * turns, &sn, &cs);
    turn[i] = make_float2(cs, sn * p.sign);
  }
  __syncthreads();
  const int pair_items = p.pairs / N;
  const uint32_t work = (uint32_t)count * p.all_heads * p.items;
  for (uint32_t i0 = threadIdx.x; i0 < work; i0 += U * kRotaryThreads) {
    Raw first[U], second[U];
    T* y[U];
    int at[U], apart[U];  // pair in `turn` (-1: passes through), the second load's distance
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * kRotaryThreads;
      y[u] = nullptr;
      if (i >= work) continue;
      const uint32_t row = quotient(i, p.items, p.items_magic);
      const int item = (int)(i - row * p.items);
      const uint32_t t = quotient(row, p.all_heads, p.heads_magic);
      uint32_t h = row - t * p.all_heads;
      const int which = h >= (uint32_t)p.heads[0];
      if (which) h -= p.heads[0];
      int c = 2 * p.pairs + (item - pair_items) * W;
      at[u] = -1, apart[u] = 0;
      if (item < pair_items) {
        const int k = item * N;
        at[u] = t * p.pairs + k;
        if constexpr (TWO) c = channels[k].x, apart[u] = channels[k].y - c;
        else c = 2 * k;
      }
      const T* x = static_cast<const T*>(p.x[which]) + from[which][t] + h * p.stride[which][2] + c;
      y[u] = static_cast<T*>(p.y[which]) + ((token0 + t) * p.heads[which] + h) * (int64_t)p.D + c;
      first[u] = load_raw<T, W>(x);
      if (TWO && at[u] >= 0) second[u] = load_raw<T, W>(x + apart[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!y[u]) continue;
      if (at[u] < 0) {
        *reinterpret_cast<Raw*>(y[u]) = first[u];
        continue;
      }
      float2 cs[N];
      if constexpr (N > 1) {  // `at` is a multiple of N
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float4 r = *reinterpret_cast<const float4*>(turn + at[u] + j);
          cs[j] = make_float2(r.x, r.y), cs[j + 1] = make_float2(r.z, r.w);
        }
      } else {
        cs[0] = turn[at[u]];
      }
      float a[W];
      unpack_raw<T, W>(first[u], a);
      if constexpr (TWO) {
        float d[W];
        unpack_raw<T, W>(second[u], d);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float2 r = cs[j];
          const float v = a[j] * r.x - d[j] * r.y;
          d[j] = a[j] * r.y + d[j] * r.x;
          a[j] = v;
        }
        store_vec<T, W>(y[u], a);
        store_vec<T, W>(y[u] + apart[u], d);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float2 r = cs[j];
          const float v = a[2 * j] * r.x - a[2 * j + 1] * r.y;
          a[2 * j + 1] = a[2 * j] * r.y + a[2 * j + 1] * r.x;
          a[2 * j] = v;
        }
        store_vec<T, W>(y[u], a);
      }
    }
  }
}

using namespace abi;

template <typename T>
cudaError_t rotary_launch(const RotaryParams& p, const RotaryTable& t, int vp, bool half, unsigned grid,
                          cudaStream_t st) {
#define MSDA_ROTARY(VP_, HALF_)                                              \
  if (vp == VP_ && half == HALF_) {                                          \
    rotary_kernel<T, VP_, HALF_><<<grid, kRotaryThreads, 0, st>>>(p, t);     \
    return cudaGetLastError();                                               \
  }
  if constexpr (sizeof(T) == 2) {
    MSDA_ROTARY(8, true)
    MSDA_ROTARY(4, false)
  }
  MSDA_ROTARY(4, true)
  MSDA_ROTARY(2, true)
  MSDA_ROTARY(1, true)
  MSDA_ROTARY(2, false)
  MSDA_ROTARY(1, false)
  MSDA_ROTARY(0, false)
#undef MSDA_ROTARY
  return cudaErrorInvalidConfiguration;
}

uint32_t magic_of(uint32_t d) { return d <= 1 ? 0 : (uint32_t)(((uint64_t(1) << 32) + d - 1) / d); }

}  // namespace
}  // namespace msda

extern "C" int msda_rotary(const void* query, const void* key, const void* positions, void* query_out,
                           void* key_out, int64_t batch, int64_t seq, int32_t num_heads,
                           int32_t num_key_heads, int32_t head_dim, const int64_t* query_strides,
                           const int64_t* key_strides, int64_t position_batch_stride,
                           int32_t position_type, int32_t num_axes, const int32_t* axis_dims, double base,
                           int32_t ladder, int32_t pairing, int32_t inverse, int32_t dtype, void* stream) {
  using namespace msda;
  using namespace msda::abi;
  const char* fn = "msda_rotary";
  const int es = elem_size(dtype);
  if (es == 0) return fail(MSDA_ERR_UNSUPPORTED, "%s: unsupported dtype code %d (0=f32, 1=f16, 2=bf16)", fn, dtype);
  if (position_type < MSDA_POSITION_F32 || position_type > MSDA_POSITION_I64)
    return fail(MSDA_ERR_UNSUPPORTED, "%s: unsupported position type %d", fn, position_type);
  if (batch < 0 || seq < 0 || num_heads < 1 || num_key_heads < 0)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch, seq >= 0, num_heads >= 1, num_key_heads >= 0)", fn);
  if ((int64_t)num_heads + num_key_heads > 65535)
    return fail(MSDA_ERR_UNSUPPORTED, "%s: more than 65535 query and key heads", fn);
  if (head_dim < 1 || head_dim > MSDA_ROTARY_MAX_HEAD_DIM)
    return fail(MSDA_ERR_UNSUPPORTED, "%s: head_dim=%d outside [1, %d]", fn, head_dim, MSDA_ROTARY_MAX_HEAD_DIM);
  if (seq > (int64_t(1) << 31) - 1 || (seq > 0 && batch > (int64_t(1) << 40) / seq))
    return fail(MSDA_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  if (num_axes < 1 || num_axes > MSDA_ROTARY_MAX_AXES || !axis_dims)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: num_axes must be in [1, %d]", fn, MSDA_ROTARY_MAX_AXES);
  if (!(base > 0) || !std::isfinite(base)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: base must be positive", fn);
  if ((ladder != MSDA_ROTARY_LADDER_AXIS && ladder != MSDA_ROTARY_LADDER_SHARED) ||
      (pairing != MSDA_ROTARY_PAIRING_HALF && pairing != MSDA_ROTARY_PAIRING_INTERLEAVED))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: unknown ladder or pairing", fn);
  int64_t rotated = 0;
  for (int a = 0; a < num_axes; ++a) {
    if (axis_dims[a] < 0 || axis_dims[a] % 2)
      return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: axis_dims[%d]=%d must be even and >= 0", fn, a, axis_dims[a]);
    rotated += axis_dims[a];
  }
  if (rotated > head_dim)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: axis_dims sum to %lld, over head_dim=%d", fn, (long long)rotated, head_dim);
  if (batch == 0 || seq == 0) return succeed();
  if (!query || !query_out || !positions || !query_strides || (num_key_heads > 0 && (!key || !key_out || !key_strides)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);

  RotaryParams p = {};
  RotaryTable t;
  const bool half = pairing == MSDA_ROTARY_PAIRING_HALF;
  const double two_pi = 6.283185307179586476925286766559;
  // The vector width: what divides every offset at which an item may begin.
  int64_t unit = 8;
  auto divides = [&](int64_t v) {
    while (unit > 1 && v % unit) unit >>= 1;
  };
  int64_t start = 0;
  int k = 0;
  for (int a = 0; a < num_axes; ++a) {
    const int n = ladder == MSDA_ROTARY_LADDER_AXIS ? axis_dims[a] : (int)rotated;
    const int64_t offset = ladder == MSDA_ROTARY_LADDER_AXIS ? start : 0;
    for (int i = 0; i < axis_dims[a] / 2; ++i, ++k) {
      const int step = ladder == MSDA_ROTARY_LADDER_AXIS ? i : (int)(start / 2) + i;
      const double f = std::pow(base, -2.0 * step / n) / two_pi;
      t.hi[k] = (float)f;
      t.lo[k] = (float)(f - (double)t.hi[k]);
      t.axis[k] = (uint8_t)a;
      t.first[k] = (uint16_t)(half ? offset + step : 2 * k);
      t.second[k] = (uint16_t)(half ? offset + step + n / 2 : 2 * k + 1);
    }
    // HALF items hold pairs of one ladder: its halves' offset and size.
    if (half) divides(offset), divides(n / 2);
    start += axis_dims[a];
  }
  divides(rotated);
  divides(head_dim);
  const void* in[2] = {query, key};
  void* out[2] = {query_out, key_out};
  const int64_t* strides[2] = {query_strides, key_strides};
  p.heads[0] = num_heads;
  p.heads[1] = num_key_heads;
  for (int w = 0; w < 2 && p.heads[w] > 0; ++w) {
    p.x[w] = in[w];
    p.y[w] = out[w];
    if (!aligned(in[w], es) || !aligned(out[w], es)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
    const int64_t sizes[3] = {batch, seq, p.heads[w]};
    for (int i = 0; i < 3; ++i) {
      p.stride[w][i] = strides[w][i];
      if (sizes[i] > 1) divides(strides[w][i] < 0 ? -strides[w][i] : strides[w][i]);
    }
    while (unit > 1 && (!aligned(in[w], unit * es) || !aligned(out[w], unit * es))) unit >>= 1;
  }
  const int pos_es = position_type == MSDA_POSITION_I64 ? 8 : 4;
  if (!aligned(positions, pos_es)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned positions", fn);
  while (unit * es > 16) unit >>= 1;
  const int vp = (int)(half ? unit : unit / 2);
  const int width = half ? (int)unit : (unit < 2 ? 1 : (int)unit);
  const int per_item = vp == 0 ? 1 : vp;
  p.positions = positions;
  p.position_batch_stride = position_batch_stride;
  p.tokens = batch * seq;
  p.seq = (uint32_t)seq;
  p.D = head_dim;
  p.pairs = k;
  p.num_axes = num_axes;
  p.position_type = position_type;
  p.sign = inverse ? -1.0f : 1.0f;
  p.items = k / per_item + (head_dim - (int)rotated) / width;
  p.all_heads = num_heads + num_key_heads;
  p.items_magic = magic_of(p.items);
  p.heads_magic = magic_of(p.all_heads);
  p.pairs_magic = magic_of(p.pairs);
  // Tokens a CTA: 4096 items (16 a thread) spread the cosines' cost over the
  // heads and keep the loop busy, as long as the grid still fills the GPU twice.
  const int64_t per_token = (int64_t)p.items * p.all_heads;
  if (per_token > (int64_t(1) << 22)) return fail(MSDA_ERR_UNSUPPORTED, "%s: num_heads * head_dim too large", fn);
  int64_t tpc = 4096 / per_token;
  if (k > 0 && tpc > kMaxCached / k) tpc = kMaxCached / k;
  if (tpc > kMaxTokens) tpc = kMaxTokens;
  const int64_t fill = p.tokens / (2 * sm_count());
  if (tpc > fill) tpc = fill;
  if (tpc < 1) tpc = 1;
  p.tokens_per_cta = (int)tpc;
  const int64_t grid = (p.tokens + tpc - 1) / tpc;
  if (grid > 0x7fffffff) return fail(MSDA_ERR_UNSUPPORTED, "%s: too many tokens for one grid", fn);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == MSDA_DTYPE_F32) e = rotary_launch<float>(p, t, vp, half, (unsigned)grid, st);
  else if (dtype == MSDA_DTYPE_F16) e = rotary_launch<__half>(p, t, vp, half, (unsigned)grid, st);
  else e = rotary_launch<__nv_bfloat16>(p, t, vp, half, (unsigned)grid, st);
  if (e != cudaSuccess) return cuda_fail(e, "rotary launch");
  return succeed();
}
