// Attention of a few queries over a long cache, fp16 and bf16: the form for
// single tokens.
//
// Bound by HBM: the visible keys and values are read once. The heads that share
// a key head and the queries are packed into the 16 rows of an m16n8k16 product,
// so that shared heads cost no further reads. Each warp has a ring of its own in
// shared memory, which asynchronous copies of 16 bytes fill two steps of 16 keys
// ahead (padded keys as zeros): no barrier in the loop, and enough bytes in
// flight. (Loading straight to registers, a step at a time, read a cache of 1.3 GB
// at 3.6 TB/s.) The order of channels within a product is free as long as both
// sides agree, so a thread takes 8 neighbouring channels of a key for four k-slots
// of two products; for the values it takes a few neighbouring channels of four keys
// and pairs the keys by byte permutes. The rows' pitches keep both kinds of read
// free of bank conflicts. The keys are split over CTAs, whose parts the combining
// kernel joins. 32 streams of 16384 keys, 32 heads on 8 key heads of 128 channels
// (2.15 GB) take 357 us, 6.0 TB/s; of 4096 to 16384 keys each 276 us, 5.3 TB/s, the
// lengths' spread holding it up, and with capped scores 303 us, 4.8 TB/s, the cap's
// arithmetic too (with the softmax of rows 8.. that are empty there: 329 us).
#include "layer_attention.cuh"

namespace msda {
namespace {

constexpr int kWarps = 4;
constexpr int kStep = 16;  // keys a warp takes at once

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  Pack<T, 2> u;
  u.e[0] = from_f32<T>(a);
  u.e[1] = from_f32<T>(b);
  return u.raw;
}

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool in) {
  const int bytes = in ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

constexpr int kAhead = 3;  // slots of a warp's ring

// Pitches in bytes: of a key, an odd multiple of 64 bytes (two keys' quarters of 64
// bytes fill the banks); of a value, 16 bytes past a multiple of 64 (four pairs of
// values' first 16 bytes lie 32 bytes apart).
template <int DP>
struct Ring {
  static constexpr int kKey = DP == 32 ? 64 : DP * 2 + 64;
  static constexpr int kValue = DP * 2 + 16;
  static constexpr int kSlot = kStep * (kKey + kValue);
  static constexpr int kBytes = kWarps * kAhead * kSlot;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kWarps * 32, DP == 128 ? 2 : DP == 64 ? 3 : 4) attn_token_kernel(const AttnParams p) {
  constexpr int KC = DP / 32;               // 32-channel chunks of a key
  constexpr int VE = DP == 32 ? 4 : 8;      // neighbouring channels of a value that a thread takes
  constexpr int VC = DP / (8 * VE);         // groups of them
  constexpr int NT = DP / 8;                // output tiles of 8 channels
  using R = Ring<DP>;
  extern __shared__ __align__(128) char ring[];
  __shared__ float2 part_ml[kWarps][16];
  static_assert((kWarps - 1) * 16 * (DP + 4) * 4 <= R::kBytes, "the parts take the ring's place");
  float (*part_o)[16][DP + 4] = reinterpret_cast<float (*)[16][DP + 4]>(ring);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int group = p.H / p.Hkv, rows = p.Sq * group;
  const int tiles = (rows + 15) / 16;
  // The heads are the fast dimension: they read neighbouring bytes of the cache's
  // rows at about the same time.
  const int hk = blockIdx.x / tiles, r0 = blockIdx.x % tiles * 16, b = blockIdx.z, split = blockIdx.y;
  const bool both = rows - r0 > 8;  // rows 8.. too
  pdl_trigger();
  const int length = attn_length(p, b);
  int first, last;
  split_range(rows_limit(p, b, (min(r0 + 16, rows) + group - 1) / group, length), p.splits, split, first, last);
  const T* kb = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* vb = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  const int* kdoc = p.kdoc ? p.kdoc + (int64_t)b * p.Sk : nullptr;
  ScoreForm f = score_form(p, 0);
  RowView row[2];
  float slope[2];
  uint32_t qa[KC][2][4];  // products' left sides: rows g and g + 8, channels 8 t ... of each chunk
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + g + 8 * i, at = r / group, h = hk * group + r % group;
    const bool in = r < rows;
    row[i] = row_view(p, b, in ? at : p.Sq, length);
    slope[i] = in && p.slopes ? __ldg(p.slopes + h) * kLog2e : 0.0f;
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + at * p.qs[1] + h * p.qs[2];
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = c * 32 + t * 8;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (in && d < p.D) u = __ldg(reinterpret_cast<const uint4*>(q + d));
      qa[c][0][i] = u.x, qa[c][0][2 + i] = u.y, qa[c][1][i] = u.z, qa[c][1][2 + i] = u.w;
    }
  }
  float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;

  char* mine_ring = ring + warp * kAhead * R::kSlot;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(mine_ring);
  // A step's keys and values, 16 bytes a lane at a time; a group of copies each.
  const auto fill = [&](int j0, int slot) {
    if (j0 < last) {
      constexpr int kPieces = DP / 8;
      const uint32_t key_at = ring_at + slot * R::kSlot, value_at = key_at + kStep * R::kKey;
#pragma unroll
      for (int i = 0; i < kStep * kPieces / 32; ++i) {
        const int at = i * 32 + lane, r = at / kPieces, d = at % kPieces * 8, j = j0 + r;
        const bool in = j < last && d < p.D && (!kdoc || __ldg(kdoc + j) >= 0);
        const int64_t jj = in ? j : first;  // an address in the cache, whether read or not
        copy16(key_at + r * R::kKey + d * 2, kb + jj * p.ks[1] + (in ? d : 0), in);
        copy16(value_at + r * R::kValue + d * 2, vb + jj * p.vs[1] + (in ? d : 0), in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int start = first + warp * kStep;
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i) fill(start + i * kWarps * kStep, i);
  int slot = 0;
  for (int j0 = start; j0 < last; j0 += kWarps * kStep) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
    __syncwarp();
    // The slot that the step before has left.
    fill(j0 + (kAhead - 1) * kWarps * kStep, slot == 0 ? kAhead - 1 : slot - 1);
    const char* key_row = mine_ring + slot * R::kSlot;
    const char* value_row = key_row + kStep * R::kKey;
    slot = slot + 1 == kAhead ? 0 : slot + 1;
    uint4 kr[2][KC];
    uint32_t vr[4][VC][VE / 2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int c = 0; c < KC; ++c)
        kr[n][c] = *reinterpret_cast<const uint4*>(key_row + (g + 8 * n) * R::kKey + c * 64 + t * 16);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const char* v = value_row + (t * 2 + (n & 1) + (n >> 1) * 8) * R::kValue;
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        if constexpr (VE == 8) {
          const uint4 u = *reinterpret_cast<const uint4*>(v + c * 128 + g * 16);
          vr[n][c][0] = u.x, vr[n][c][1] = u.y, vr[n][c][2] = u.z, vr[n][c][3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(v + g * 8);
          vr[n][c][0] = u.x, vr[n][c][1] = u.y;
        }
      }
    }
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        mma16816<T>(s[n], qa[c][0], kr[n][c].x, kr[n][c].y);
        mma16816<T>(s[n], qa[c][1], kr[n][c].z, kr[n][c].w);
      }
    }
    // s[n][2 i + e]: row g + 8 i, key j0 + 8 n + 2 t + e. Rows 8.. may all be empty.
    bool small = true;  // scores well below the cap, the common case
    if (p.cap != 0.0f) {
      float big = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(s[n][i]));
      small = __all_sync(kFullMask, big * fabsf(f.inv_cap) < kTanhSmall);
    }
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + 8 * n + 2 * t + e;
        const int kd = kdoc && j < last ? __ldg(kdoc + j) : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i == 1 && !both) continue;
          float x = s[n][2 * i + e] * f.scale2;
          if (p.cap != 0.0f) {
            x = s[n][2 * i + e] * f.inv_cap;
            x = (small ? tanh_small(x) : tanh_of(x)) * f.cap2;
          }
          if (p.slopes) x = fmaf(-slope[i], (float)abs(row[i].place - j), x);
          const bool seen = j < last && j < row[i].limit && (!kdoc || same_document(row[i].doc, kd, p.shared));
          s[n][2 * i + e] = seen ? x : -INFINITY;
          top[i] = fmaxf(top[i], s[n][2 * i + e]);
        }
      }
    uint32_t pa[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !both) continue;
      top[i] = fmaxf(top[i], __shfl_xor_sync(kFullMask, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(kFullMask, top[i], 2));
      const float base = top[i] == -INFINITY ? 0.0f : top[i];
      const float old = exp2f(m[i] - base);
      m[i] = top[i];
      l[i] *= old;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float e0 = exp2f(s[n][2 * i] - base), e1 = exp2f(s[n][2 * i + 1] - base);
        l[i] += e0 + e1;
        pa[2 * n + i] = pack2<T>(e0, e1);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][2 * i] *= old;
        o[n][2 * i + 1] *= old;
      }
    }
    // Output tile (c, e): channels c * 64 + 8-wide (or 4-wide) groups' element e.
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const uint32_t pick = e & 1 ? 0x7632 : 0x5410;
        const uint32_t b0 = __byte_perm(vr[0][c][e / 2], vr[1][c][e / 2], pick);
        const uint32_t b1 = __byte_perm(vr[2][c][e / 2], vr[3][c][e / 2], pick);
        mma16816<T>(o[c * VE + e], pa, b0, b1);
      }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // Join the CTA's warps, in the ring's place.
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(kFullMask, l[i], 1);
    l[i] += __shfl_xor_sync(kFullMask, l[i], 2);
    if (t == 0) part_ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
  }
  __syncthreads();
  float all_m[2], all_l[2], mine[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    all_m[i] = -INFINITY, all_l[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all_m[i] = fmaxf(all_m[i], part_ml[w][g + 8 * i].x);
    const float base = all_m[i] == -INFINITY ? 0.0f : all_m[i];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = part_ml[w][g + 8 * i];
      all_l[i] += ml.y * exp2f(ml.x - base);
    }
    mine[i] = exp2f(m[i] - base);
  }
  // Channel of o[c * VE + e][2 i + x]: c * 64 + (2 t + x) * VE + e.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        o[n][2 * i + x] *= mine[i];
        if (warp > 0) part_o[warp - 1][g + 8 * i][n / VE * 64 + (2 * t + x) * VE + n % VE] = o[n][2 * i + x];
      }
  __syncthreads();
  if (warp > 0) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + g + 8 * i;
    if (r >= rows) continue;
    const int at = r / group, h = hk * group + r % group;
    const int64_t out = ((int64_t)b * p.H + h) * p.Sq + at;
    const int64_t part = (int64_t)split * p.B * p.H * p.Sq + out;
    const float mul = all_l[i] > 0.0f ? 1.0f / all_l[i] : (all_l[i] == 0.0f ? 0.0f : all_l[i]);
    if (t == 0) {
      if (p.splits > 1) p.part_ml[part] = make_float2(all_m[i], all_l[i]);
      else if (p.lse) p.lse[out] = all_l[i] == 0.0f ? -INFINITY : (all_m[i] + log2f(all_l[i])) * kLn2;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int d = n / VE * 64 + (2 * t + x) * VE + n % VE;
        float v = o[n][2 * i + x];
#pragma unroll
        for (int w = 0; w < kWarps - 1; ++w) v += part_o[w][g + 8 * i][d];
        if (d >= p.D) continue;
        if (p.splits > 1) p.part_o[part * p.D + d] = v;
        else put_output<T>(p, (((int64_t)b * p.Sq + at) * p.H + h) * p.D + d, v * mul);
      }
  }
}

// Joins the parts of each row (at most 64) in the parts' order: a warp a row.
template <typename T>
__global__ void __launch_bounds__(128) attn_combine_kernel(const AttnParams p) {
  pdl_wait();
  const int64_t rows = (int64_t)p.B * p.H * p.Sq;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= rows) return;
  const int lane = threadIdx.x % 32;
  // A lane has two parts' maximum and sum.
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ml[i] = make_float2(-INFINITY, 0.0f);
    if (lane + 32 * i < p.splits) ml[i] = __ldcg(&p.part_ml[(lane + 32 * i) * rows + row]);
  }
  float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
  const float base = top == -INFINITY ? 0.0f : top;
  // A part without keys has no weight, and its sums were not written.
  const float weight[2] = {ml[0].y == 0.0f ? 0.0f : exp2f(ml[0].x - base), ml[1].y == 0.0f ? 0.0f : exp2f(ml[1].x - base)};
  float total = 0.0f, acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float w = __shfl_sync(kFullMask, s < 32 ? weight[0] : weight[1], s & 31);
    const float sum = __shfl_sync(kFullMask, s < 32 ? ml[0].y : ml[1].y, s & 31);
    total = fmaf(sum, w, total);
    const float* o = p.part_o + (s * rows + row) * p.D;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float v = 0.0f;
      if (sum != 0.0f && lane + 32 * c < p.D) v = __ldcg(o + lane + 32 * c);
      acc[c] = fmaf(v, w, acc[c]);
    }
  }
  const float mul = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
  const int i = (int)(row % p.Sq), h = (int)(row / p.Sq % p.H);
  const int64_t b = row / p.Sq / p.H;
  const int64_t out = ((b * p.Sq + i) * p.H + h) * p.D;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < p.D) put_output<T>(p, out + lane + 32 * c, acc[c] * mul);
  if (p.lse && lane == 0) p.lse[row] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
}

// dv (blockIdx.y 0) and dk from the parts' sums, in the parts' order.
template <typename T>
__global__ void __launch_bounds__(256) attn_kv_sum_kernel(const AttnParams p) {
  const int64_t all = (int64_t)p.B * p.Sk * p.Hkv * p.D, step = (int64_t)gridDim.x * 1024;
  const float* from = kv_part(p, 0, blockIdx.y != 0);
  T* to = static_cast<T*>(blockIdx.y ? p.dk : p.dv);
  for (int64_t i0 = (int64_t)blockIdx.x * 1024 + threadIdx.x; i0 < all; i0 += step) {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int part = 0; part < p.kv_parts; ++part)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * 256 < all) sum[u] += __ldg(from + part * 2 * all + i0 + u * 256);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 256 < all) to[i0 + u * 256] = from_f32<T>(sum[u]);
  }
}

template <typename T>
cudaError_t token_t(const AttnParams& p, cudaStream_t st) {
  const int rows = p.Sq * (p.H / p.Hkv);
  const dim3 grid(p.Hkv * ((rows + 15) / 16), p.splits, p.B);
  const auto launch = [&](auto kernel, int smem, std::atomic<uint64_t>& set) {
    cudaError_t e = abi::allow_smem(kernel, smem, set);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kWarps * 32, smem, st>>>(p);
    return cudaGetLastError();
  };
  static std::atomic<uint64_t> set[3];
  if (p.D <= 32) return launch(attn_token_kernel<T, 32>, Ring<32>::kBytes, set[0]);
  if (p.D <= 64) return launch(attn_token_kernel<T, 64>, Ring<64>::kBytes, set[1]);
  return launch(attn_token_kernel<T, 128>, Ring<128>::kBytes, set[2]);
}

}  // namespace

cudaError_t attn_token_forward(const AttnParams& p, int dtype, cudaStream_t st) {
  return dtype == MSDA_DTYPE_F16 ? token_t<__half>(p, st) : token_t<__nv_bfloat16>(p, st);
}

cudaError_t attn_kv_sum_launch(const AttnParams& p, int dtype, cudaStream_t st) {
  const int64_t blocks = ((int64_t)p.B * p.Sk * p.Hkv * p.D + 1023) / 1024;
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096), 2);
  if (dtype == MSDA_DTYPE_F32) attn_kv_sum_kernel<float><<<grid, 256, 0, st>>>(p);
  else if (dtype == MSDA_DTYPE_F16) attn_kv_sum_kernel<__half><<<grid, 256, 0, st>>>(p);
  else attn_kv_sum_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t attn_combine_launch(const AttnParams& p, int dtype, cudaStream_t st) {
  const int64_t rows = (int64_t)p.B * p.H * p.Sq;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (dtype == MSDA_DTYPE_F32) return launch_ex(attn_combine_kernel<float>, grid, dim3(128), 0, st, true, p);
  if (dtype == MSDA_DTYPE_F16) return launch_ex(attn_combine_kernel<__half>, grid, dim3(128), 0, st, true, p);
  return launch_ex(attn_combine_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, true, p);
}

}  // namespace msda
