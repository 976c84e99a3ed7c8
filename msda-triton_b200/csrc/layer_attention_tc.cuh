// Masked attention on the tensor cores (tcgen05), fp16 and bf16.
//
// All tiles are 128 tokens in 128-byte swizzled shared-memory rows, brought by
// TMA (channels past the head size and tokens past the end come as zeros). The
// scores land in TMEM, one query (or key) a lane; a thread reads its row's 128
// (or 64) scores into registers, and writes the probabilities back to TMEM in 16
// bits over the scores that it has read, from where the second product takes
// them as its left side: they never pass through shared memory.
//
// Roles: one warp loads, one issues the products (one elected lane), eight warps
// do the softmax. Each wait is bounded (layer_tcgen05.cuh); a kernel whose wait
// gave up leaves NaN in its outputs.
#pragma once

#include "layer_attention.cuh"
#include "layer_tcgen05.cuh"

namespace msda {
namespace tc {

// What the scores of a kernel's instance go through.
constexpr int kCapped = 1, kSloped = 2, kGrouped = 4;  // cap; distance bias; documents

constexpr int kSoftmaxThreads = 256;
constexpr int kThreads = kSoftmaxThreads + 128;  // two warpgroups of softmax, one of the other roles
constexpr int kLoadWarp = 8, kMmaWarp = 9;

// The launch has 168 registers a thread; the softmax takes what the other
// warpgroup leaves: 256 x 216 + 128 x 72 = 384 x 168.
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
__device__ __forceinline__ void leave_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

template <typename T> struct IsBf16 { static constexpr bool value = false; };
template <> struct IsBf16<__nv_bfloat16> { static constexpr bool value = true; };

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  if constexpr (IsBf16<T>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two fp32 values in a register pair: one instruction does both.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return f2_pack(lo, hi); }
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A row's largest value: four chains.
template <int N>
__device__ __forceinline__ float row_max(const float (&s)[N]) {
  float m[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int c = 0; c < N; c += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max3(m[i], s[c + i], s[c + 4 + i]);
  return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

// s <- tanh(inv_cap s) by an odd polynomial, two columns an instruction. (The cap
// comes in as the scores' factor, further on: powers of inv_cap worked into the
// coefficients would leave fp32's range where the cap is wide.)
template <int K, int N>
__device__ __forceinline__ void cap_polynomial(const ScoreForm& f, const float (&poly)[K], float (&s)[N]) {
  const uint64_t inv = pair_of(f.inv_cap, f.inv_cap);
  uint64_t a[K];
#pragma unroll
  for (int i = 0; i < K; ++i) a[i] = pair_of(poly[i], poly[i]);
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    const uint64_t x = pair_mul(pair_of(s[c], s[c + 1]), inv), y = pair_mul(x, x);
    uint64_t r = a[K - 1];
#pragma unroll
    for (int i = K - 2; i >= 0; --i) r = f2_fma(r, y, a[i]);
    f2_unpack(f2_fma(pair_mul(x, y), r, x), s[c], s[c + 1]);
  }
}

// Scores of a thread's row as shares of the cap. Scores well below the cap, the
// common case, go by a polynomial: below a quarter of it (2 terms, 4.9e-7
// relative at most), below three quarters (tanh_small's 5 terms), else one by one.
template <int N>
__device__ __forceinline__ void cap_scores(const ScoreForm& f, float (&s)[N]) {
  float top[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < N; c += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i] = max3_abs(top[i], s[c + i], s[c + 4 + i]);
  const float big = fmaxf(max3(top[0], top[1], top[2]), top[3]) * fabsf(f.inv_cap);
  if (__all_sync(kFullMask, big < 0.25f)) {
    const float poly[2] = {-0.33324572443962097f, 0.12876421213150024f};
    cap_polynomial(f, poly, s);
  } else if (__all_sync(kFullMask, big < kTanhSmall)) {
    const float poly[5] = {-0.3333306908607483f, 0.13326521217823029f, -0.0533902570605278f, 0.019664911553263664f,
                           -0.004769488703459501f};
    cap_polynomial(f, poly, s);
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] = tanh_of(s[c] * f.inv_cap);
  }
}

// What documents say of a block of query tiles (bit t: tile t) and a key tile.
struct TileState {
  uint8_t apart;  // no query of the tile sees a key
  uint8_t agree;  // documents hide nothing
  bool skip;      // apart from every tile of the block
  bool padded;    // some keys are padding: their rows must be cleared
};

// rows: [i0, i0 + n * 128), n <= 2; keys: tile j.
__device__ __forceinline__ TileState tile_state(const AttnParams& p, int b, int i0, int n, int j, int length) {
  TileState s{0, 3, false, (j + 1) * kTileTokens > length && length < p.Sk};
  if (!p.kdoc) return s;
  const int nq = (p.Sq + kDocTile - 1) / kDocTile, nk = (p.Sk + kDocTile - 1) / kDocTile;
  const DocTile k = p.ktile[(int64_t)b * nk + j];
  s.apart = 3, s.agree = 0;
  for (int t = 0; t < n && i0 / kDocTile + t < nq; ++t) {
    const DocTile q = p.qtile[(int64_t)b * nq + i0 / kDocTile + t];
    if (!tiles_apart(q, k)) s.apart &= ~(1 << t);
    if (tiles_agree(q, k, p.shared)) s.agree |= 1 << t;
  }
  s.skip = s.apart == 3;
  s.padded = s.padded || k.padded;
  return s;
}

// Which of the keys k0 ... (32 a word) a thread's query sees by its document: a
// ballot for each document among the warp's queries, of which there are few.
template <int W>
__device__ __forceinline__ void document_masks(const AttnParams& p, const int* kdoc, int k0, int doc, uint32_t (&mask)[W]) {
  const int lane = threadIdx.x % 32;
  int mine[W];
#pragma unroll
  for (int w = 0; w < W; ++w) mine[w] = k0 + w * 32 + lane < p.Sk ? __ldg(kdoc + k0 + w * 32 + lane) : -1;
  for (uint32_t todo = kFullMask; todo;) {
    const int d = __shfl_sync(kFullMask, doc, __ffs(todo) - 1);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t seen = __ballot_sync(kFullMask, same_document(d, mine[w], p.shared));
      if (doc == d) mask[w] = seen;
    }
    todo &= ~__ballot_sync(kFullMask, doc == d);
  }
}

// Parities of the barriers that say a ring's stage has been cleared, one for each
// stage: a stage is not filled again before its products are done, so that none of
// these can end two phases ahead of the wait for the first. (One barrier for all
// stages could: the ring's tiles may be loaded and cleared before the issuing
// thread looks at it, and its parity stands as if nothing had come.)
struct StagePhases {
  uint32_t bits = 0;
  __device__ __forceinline__ uint32_t next(int stage) {
    const uint32_t parity = bits >> stage & 1;
    bits ^= 1u << stage;
    return parity;
  }
};

// Clears the rows of a tile that `keep` rejects (a warp): 0 x NaN is NaN, and a
// product over tokens would spread what padding holds.
template <int DP, typename Keep>
__device__ __forceinline__ void clear_rows(char* tile, Keep keep) {
  for (int r = threadIdx.x % 32; r < kTileTokens; r += 32) {
    if (keep(r)) continue;
#pragma unroll
    for (int c = 0; c < (DP + kChunk - 1) / kChunk; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(tile + c * kChunkBytes + r * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncwarp();
}

// Key tile j's rows that are no padding.
struct KeyRows {
  const int* doc;  // nullable
  int first, length;
  __device__ __forceinline__ bool operator()(int r) const {
    return first + r < length && (!doc || __ldg(doc + first + r) >= 0);
  }
};

// The steps that a block of queries goes through: its key tiles, or with STEP 64
// their halves, less what the limit or the documents leave out. Every role walks
// them by itself.
template <int STEP, bool DOCS>
struct KeySteps {
  int j, half, n;  // key tile, its half, the tile's number among those visited
  int tiles, halves;  // key tiles below the limit; halves of the last of them
  bool done;
  TileState state;

  __device__ __forceinline__ void seek(const AttnParams& p, int b, int i0, int rows, int length) {
    if constexpr (!DOCS) {
      done = j >= tiles;
      state = TileState{0, 3, false, j * kTileTokens + kTileTokens > length && length < p.Sk};
    } else {
      for (;; ++j) {
        done = j >= tiles;
        if (done) return;
        state = tile_state(p, b, i0, rows, j, length);
        if (!state.skip) return;
      }
    }
  }
  __device__ __forceinline__ KeySteps(const AttnParams& p, int b, int i0, int rows, int limit, int length)
      : j(0), half(0), n(0), tiles((limit + kTileTokens - 1) / kTileTokens), halves(STEP == 128 || (limit - 1) % kTileTokens < 64 ? 1 : 2) {
    seek(p, b, i0, rows, length);
  }
  __device__ __forceinline__ int count() const { return STEP == 128 || j + 1 == tiles ? halves : 2; }
  __device__ __forceinline__ void next_tile(const AttnParams& p, int b, int i0, int rows, int length) {
    half = 0, ++j, ++n;
    seek(p, b, i0, rows, length);
  }
  __device__ __forceinline__ void advance(const AttnParams& p, int b, int i0, int rows, int length) {
    if (half + 1 == count()) next_tile(p, b, i0, rows, length);
    else half = 1;
  }
};

// ---------------------------------------------------------------------------
// Forward: 256 queries of a head a CTA, as two tiles of 128 that take turns: while
// one tile's rows are exponentiated the tensor cores work on the other's products.
// Above 64 channels a step is 128 keys, 2 x 1024 cycles of products, and on the
// 16-a-cycle exponential units 2 x 1024 cycles too; the sums take half of TMEM,
// one CTA an SM. Up to 64 channels the exponentials are the bound, and what
// counts is that warps are there to keep them busy: steps of 64 keys and half of
// TMEM let two CTAs share an SM, four warps for each of its schedulers. (Two
// buffers of 64 keys a tile with one CTA took 606 us and 544 us for 8192 x 16
// heads of 128 and of 32 channels: products of 64 columns run at half rate, and
// two warps left the exponential units idle for half of the time.)
// bf16, 8192 tokens on 16 heads, without a mask / causal: 128 channels 518 us (1062
// TFLOP/s) / 260 us, bound by products and exponentials that do not cover one
// another wholly; 64 channels 415 / 212 us, 32 channels 382 / 194 us, bound by the
// exponential units (of which the cap's tanh, a polynomial, takes none: causal and
// capped at 128 channels 343 us).
// ---------------------------------------------------------------------------
template <int DP>
struct FwdShape {
  static constexpr int kTile = tile_bytes<DP>();
  static constexpr int kStages = 4;
  static constexpr int kSmem = 1024 + (2 + kStages) * kTile;
  static constexpr int kStep = DP > 64 ? 128 : 64;
  static constexpr int kCtas = DP > 64 ? 1 : 2;
  // With 128 scores a thread the softmax takes registers from the other roles'
  // warpgroup.
  static constexpr bool kSplit = DP > 64;
  static constexpr int kThreads = kSplit ? tc::kThreads : kSoftmaxThreads + 64;
  static constexpr int kColumns = DP > 64 ? 512 : 256;
};

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(FwdShape<DP>::kThreads, FwdShape<DP>::kCtas)
    attn_tc_fwd_kernel(const AttnParams p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
  using Shape = FwdShape<DP>;
  constexpr bool DOCS = (MODE & kGrouped) != 0;
  constexpr int NS = Shape::kStages, STEP = Shape::kStep, OUT = 2 * STEP;  // OUT: first TMEM column of the sums
  extern __shared__ char raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  char* sq = smem;
  char* ring = smem + 2 * Shape::kTile;  // slots: a visited tile's keys, then its values
  __shared__ uint64_t q_full, kv_full[NS], kv_empty[NS], s_full[2], p_full[2], o_full[2], cleared[NS / 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  volatile int* abort = &abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, hk = h / (p.H / p.Hkv);
  const int i0 = (gridDim.y - 1 - blockIdx.y) * 2 * kTileTokens;  // long causal rows first
  const int length = attn_length(p, b);
  const int limit = rows_limit(p, b, i0 + 2 * kTileTokens, length);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    bar_init(&q_full, 1);
    for (int i = 0; i < NS / 2; ++i) bar_init(&cleared[i], 1);
    for (int i = 0; i < NS; ++i) bar_init(&kv_full[i], 1), bar_init(&kv_empty[i], 1);
    for (int t = 0; t < 2; ++t) bar_init(&s_full[t], 1), bar_init(&p_full[t], 4), bar_init(&o_full[t], 1);
    fence_async_smem();
  }
  if (warp == kMmaWarp) tmem_alloc<Shape::kColumns>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp < kLoadWarp) {
    if constexpr (Shape::kSplit) take_registers();
    const int t = warp / 4, i = i0 + threadIdx.x;  // tile and query of this thread
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;
    const uint32_t s_at = tmem + lanes + t * STEP, o_at = tmem + lanes + OUT + t * DP;
    const RowView row = row_view(p, b, i, length);
    const ScoreForm f = score_form(p, h);
    const int* kdoc = p.kdoc ? p.kdoc + (int64_t)b * p.Sk : nullptr;
    float m = -INFINITY, l = 0.0f;  // in base 2; m trails the maximum by at most kSlack
    constexpr float kSlack = 8.0f;
    bool ok = true;
    int u = 0;
    for (KeySteps<STEP, DOCS> at(p, b, i0, 2, limit, length); !at.done && ok; at.advance(p, b, i0, 2, length), ++u) {
      ok = warp_wait(&s_full[t], u & 1, abort);
      if (!ok) break;
      fence_after();
      if (DOCS && (at.state.apart >> t & 1)) {  // the step is the other tile's: no probabilities
        const uint32_t none[16] = {};
#pragma unroll
        for (int c = 0; c < STEP / 2; c += 16) tmem_store16(s_at + c, none);
        tmem_wait_store();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&p_full[t]);
        continue;
      }
      float s[STEP];
#pragma unroll
      for (int c = 0; c < STEP; c += 32) tmem_load32(s_at + c, s + c);
      tmem_wait_load();
      const int j0 = at.j * kTileTokens + at.half * 64;
      float factor = f.scale2;
      {
        if constexpr ((MODE & kCapped) != 0) {
          cap_scores(f, s);
          factor = f.cap2;
        }
        if constexpr ((MODE & kSloped) != 0) {
          const float far = (float)(row.place - j0);
#pragma unroll
          for (int c = 0; c < STEP; ++c) s[c] = fmaf(-f.slope2, fabsf(far - (float)c), s[c] * factor);
          factor = 1.0f;
        }
      }
      const int seen = row.limit - j0;
      if (!__all_sync(kFullMask, seen >= STEP)) {
#pragma unroll
        for (int c = 0; c < STEP; ++c) s[c] = c < seen ? s[c] : -INFINITY;
      }
      if (DOCS && !(at.state.agree >> t & 1)) {
        uint32_t mask[STEP / 32];
        document_masks(p, kdoc, j0, row.doc, mask);
#pragma unroll
        for (int c = 0; c < STEP; ++c) s[c] = mask[c / 32] >> (c % 32) & 1 ? s[c] : -INFINITY;
      }
      if (factor <= 0.0f) {  // a negative scale: its own factor now, so that the largest score is the largest value
#pragma unroll
        for (int c = 0; c < STEP; ++c) s[c] = s[c] == -INFINITY ? -INFINITY : s[c] * factor;
        factor = 1.0f;
      }
      const float top = row_max(s) * factor;
      // The reference maximum moves only when a row has grown by 2^8 past it, so
      // that the sums in TMEM are seldom rescaled; 2^8 is far from overflow.
      if (__any_sync(kFullMask, top > m + kSlack)) {
        const float next = fmaxf(m, top);
        const float old = next == -INFINITY ? 1.0f : ex2(m - next);
        m = next;
        l *= old;
        if (u > 0) {
          // The scores came after the product of the step before: the sums rest.
#pragma unroll 1
          for (int c = 0; c < DP; c += 8) {
            float o[8];
            tmem_load8(o_at + c, o);
            tmem_wait_load();
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] *= old;
            tmem_store8(o_at + c, reinterpret_cast<uint32_t*>(o));
          }
        }
      }
      const float base = m == -INFINITY ? 0.0f : -m;
      const uint64_t factor2 = pair_of(factor, factor), base2 = pair_of(base, base);
      uint64_t sum0 = 0, sum1 = 0;  // pairs of zeros
#pragma unroll
      for (int from = 0; from < STEP; from += 32) {
        uint32_t packed[16];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const float* x = s + from + 2 * c;
          float e0, e1, e2, e3;
          f2_unpack(f2_fma(pair_of(x[0], x[1]), factor2, base2), e0, e1);
          f2_unpack(f2_fma(pair_of(x[2], x[3]), factor2, base2), e2, e3);
          e0 = ex2(e0), e1 = ex2(e1), e2 = ex2(e2), e3 = ex2(e3);
          sum0 = pair_add(sum0, pair_of(e0, e1)), sum1 = pair_add(sum1, pair_of(e2, e3));
          packed[c] = pack_pair<T>(e0, e1);
          packed[c + 1] = pack_pair<T>(e2, e3);
        }
        tmem_store16(s_at + from / 2, packed);
      }
      tmem_wait_store();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&p_full[t]);
      float part[4];
      f2_unpack(sum0, part[0], part[1]);
      f2_unpack(sum1, part[2], part[3]);
      l += (part[0] + part[1]) + (part[2] + part[3]);
    }
    if (ok && u > 0) ok = warp_wait(&o_full[t], 0, abort);
    fence_after();
    const float mul = !ok ? NAN : l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    const int64_t at = (((int64_t)b * p.Sq + i) * p.H + h) * p.D;
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
      float o[32];
      if (u > 0) {
        tmem_load32(o_at + c, o);
        tmem_wait_load();
      }
      if (i < p.Sq) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (c + e >= p.D) continue;
          uint4 high, low;
          uint32_t* hi = reinterpret_cast<uint32_t*>(&high);
          uint32_t* lo = reinterpret_cast<uint32_t*>(&low);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float a = u > 0 ? o[e + 2 * x] * mul : mul, d = u > 0 ? o[e + 2 * x + 1] * mul : mul;
            hi[x] = pack_pair<T>(a, d);
            Pack<T, 2> v;
            v.raw = hi[x];
            lo[x] = pack_pair<T>(a - to_f32(v.e[0]), d - to_f32(v.e[1]));
          }
          *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + at + c + e) = high;
          if (p.residue) *reinterpret_cast<uint4*>(static_cast<T*>(p.residue) + at + c + e) = low;
        }
      }
    }
    if (i < p.Sq && p.lse)
      p.lse[((int64_t)b * p.H + h) * p.Sq + i] = !ok ? NAN : l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    fence_before();
  } else {
    if constexpr (Shape::kSplit) leave_registers();
    if (warp == kLoadWarp) {
    const int* kdoc = p.kdoc ? p.kdoc + (int64_t)b * p.Sk : nullptr;
    int n = 0;  // ring slots filled
    bool ok = true;
    if (limit > 0) {
      if (lane == 0) {
        bar_expect(&q_full, 2 * Shape::kTile);
        tma_tile<DP>(sq, &qmap, &q_full, h, i0, b);
        tma_tile<DP>(sq + Shape::kTile, &qmap, &q_full, h, i0 + kTileTokens, b);
      }
      for (KeySteps<STEP, DOCS> at(p, b, i0, 2, limit, length); !at.done && ok; at.next_tile(p, b, i0, 2, length)) {
        for (int kv = 0; kv < 2 && ok; ++kv, ++n) {
          const int slot = n % NS;
          if (n >= NS) ok = warp_wait(&kv_empty[slot], (n / NS - 1) & 1, abort);
          if (!ok) break;
          if (lane == 0) {
            bar_expect(&kv_full[slot], Shape::kTile);
            tma_tile<DP>(ring + slot * Shape::kTile, kv ? &vmap : &kmap, &kv_full[slot], hk, at.j * kTileTokens, b);
          }
          __syncwarp();
          if (kv && at.state.padded) {  // padded keys' values are cleared before their product
            ok = warp_wait(&kv_full[slot], (n / NS) & 1, abort);
            clear_rows<DP>(ring + slot * Shape::kTile, KeyRows{kdoc, at.j * kTileTokens, length});
            if (lane == 0) bar_arrive(&cleared[slot / 2]);
          }
        }
      }
      // Copies in flight end before the CTA does.
      warp_wait(&q_full, 0, abort);
      for (int i = max(0, n - NS); i < n; ++i) warp_wait(&kv_full[i % NS], (i / NS) & 1, abort);
    }
    } else if (warp == kMmaWarp && elect_one()) {
    // One thread issues: with its whole warp in step, the waits and elections
    // between the products cost more than the products of small heads.
    constexpr uint32_t ds = instr_desc<IsBf16<T>::value>(STEP, false), dv = instr_desc<IsBf16<T>::value>(DP, true);
    constexpr uint64_t kHalfTile = 64 * 128 >> 4, kSlot = Shape::kTile >> 4;
    const uint64_t q_desc = by_channels(smem_u32(sq)), k_desc = by_channels(smem_u32(ring)), v_desc = by_tokens(smem_u32(ring));
    bool ok = limit == 0 || bar_wait(&q_full, 0, abort);
    KeySteps<STEP, DOCS> at(p, b, i0, 2, limit, length);
    int slot = 0;  // of the tile's keys; its values': the next
    uint32_t phase = 0, turn = 0;
    StagePhases cleared_phase;
    const auto scores = [&](int t, uint64_t k) {
      product_channels<DP>(tmem + t * STEP, q_desc + t * kSlot, k, ds);
      commit(&s_full[t]);
    };
    if (!at.done && ok) {
      ok = bar_wait(&kv_full[0], 0, abort);
      fence_after();
      if (ok) {
        scores(0, k_desc);
        scores(1, k_desc);
        if (at.count() == 1) commit(&kv_empty[0]);
      }
    }
    bool add = false;
    while (!at.done && ok) {
      const int count = at.count(), k_slot = slot, v_slot = slot + 1;
      const uint64_t v = v_desc + v_slot * kSlot;
      ok = bar_wait(&kv_full[v_slot], phase, abort);
      if (ok && at.state.padded) ok = bar_wait(&cleared[v_slot / 2], cleared_phase.next(v_slot / 2), abort);
      at.next_tile(p, b, i0, 2, length);
      slot += 2;
      if (slot == NS) slot = 0, phase ^= 1;
      // A step's values' products, each followed by the next step's scores.
      for (int half = 0; half < count && ok; ++half) {
        const bool same = half + 1 < count, more = same || !at.done;
        const uint64_t k = same ? k_desc + k_slot * kSlot + kHalfTile : k_desc + slot * kSlot;
        if (!same && more) ok = bar_wait(&kv_full[slot], phase, abort);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          ok = ok && bar_wait(&p_full[t], turn, abort);
          fence_after();
          if (!ok) break;
          product_half(tmem + OUT + t * DP, tmem + t * STEP, v + half * 4 * kTokenStep, dv, add);
          if constexpr (STEP == 128) product_half(tmem + OUT + t * DP, tmem + t * STEP + 32, v + 4 * kTokenStep, dv, true);
          if (more) scores(t, k);
          else commit(&o_full[t]);
        }
        add = true;
        turn ^= 1;
        if (!ok) break;
        if (same) commit(&kv_empty[k_slot]);
        else if (more && at.count() == 1) commit(&kv_empty[slot]);
      }
      if (ok) commit(&kv_empty[v_slot]);
    }
    if (!ok) {
      commit(&q_full);
      bar_wait(&q_full, 1, abort);
    }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    tmem_free<Shape::kColumns>(tmem);
  }
}

// ---------------------------------------------------------------------------
// Backward, in two kernels without atomics: dq by tiles of 128 queries (which
// also leaves delta_i = g_i . o_i), then dk and dv by tiles of 128 keys. Scores are
// formed in both: 7 products of a tile pair instead of 5, and a fixed order of
// sums. A step is 128 columns (keys; queries) above 64 channels, 64 up to it,
// where two CTAs share an SM's TMEM; each half of the eight warps takes half of
// the columns. The derivative goes to TMEM in 16 bits without the scale, which
// its sums get at the end: in fp16 it would cost small gradients digits.
// Rounding it costs dq and dk as much again as rounding their results does (2.4e-3
// of bf16 gradients against 1.7e-3): a second 16-bit part would take a fourth
// product and TMEM that is not there.
// bf16, 8192 tokens on 16 heads, dq / dkv without a mask: 128 channels (4 key heads)
// 748 / 1064 us (1100 and 1033 TFLOP/s counting what is formed), 64 channels 447 /
// 712 us, 32 channels 413 / 664 us; causal at 128 channels 419 / 470 us, capped
// too 442 / 542 us. Bound as the forward is: by products at 128 channels, below by
// the exponentials and the traffic of scores between TMEM and registers.
// ---------------------------------------------------------------------------
template <int DP>
struct BwdShape {
  static constexpr int kTile = tile_bytes<DP>();
  static constexpr int kSmem = 1024 + 6 * kTile;  // two tiles that stay, two stages of two
  static constexpr int kStep = DP > 64 ? 128 : 64;
  static constexpr int kCtas = DP > 64 ? 1 : 2;
  static constexpr bool kSplit = DP > 64;  // registers, as in the forward
  static constexpr int kThreads = kSplit ? tc::kThreads : kSoftmaxThreads + 64;
  static constexpr int kColumns = DP > 64 ? 512 : 256;
};

// A thread's N probabilities from its scores, in place; with a cap its
// derivative 1 - tanh^2 in t2. far(c): places between query and key; lse(c, ..):
// minus the log-sum-exp, to base 2, of columns c and c + 1, and of c + 2 and c + 3.
template <int MODE, int N, typename Far, typename Lse>
__device__ __forceinline__ void probabilities(const AttnParams& p, const ScoreForm& f, float (&s)[N], float (&t2)[MODE & kCapped ? N : 2],
                                              Far far, Lse lse) {
  float factor = f.scale2;
  {
    if constexpr ((MODE & kCapped) != 0) {
      cap_scores(f, s);
      const uint64_t less = pair_of(-1.0f, -1.0f), one = pair_of(1.0f, 1.0f);
#pragma unroll
      for (int c = 0; c < N; c += 2) {
        const uint64_t x = pair_of(s[c], s[c + 1]);
        f2_unpack(f2_fma(pair_mul(x, x), less, one), t2[c], t2[c + 1]);
      }
      factor = f.cap2;
    }
    if constexpr ((MODE & kSloped) != 0) {
#pragma unroll
      for (int c = 0; c < N; ++c) s[c] = fmaf(-f.slope2, fabsf(far(c)), s[c] * factor);
      factor = 1.0f;
    }
  }
  const uint64_t factor2 = pair_of(factor, factor);
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    uint64_t l0, l1;
    lse(c, l0, l1);
    f2_unpack(f2_fma(pair_of(s[c], s[c + 1]), factor2, l0), s[c], s[c + 1]);
    f2_unpack(f2_fma(pair_of(s[c + 2], s[c + 3]), factor2, l1), s[c + 2], s[c + 3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[c + e] = ex2(s[c + e]);
  }
}

template <int N>
__device__ __forceinline__ void multiply(float (&s)[N], const float (&t)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 2) f2_unpack(pair_mul(pair_of(s[c], s[c + 1]), pair_of(t[c], t[c + 1])), s[c], s[c + 1]);
}

// dp <- s (dp - delta); delta(c, ..): minus the columns' row sums, as lse above.
// `clean`: masked columns (s = 0) stay 0 whatever dp holds there.
template <int N, typename Delta>
__device__ __forceinline__ void derivatives(const float (&s)[N], float (&dp)[N], bool clean, Delta delta) {
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    uint64_t d0, d1;
    delta(c, d0, d1);
    f2_unpack(pair_mul(pair_add(pair_of(dp[c], dp[c + 1]), d0), pair_of(s[c], s[c + 1])), dp[c], dp[c + 1]);
    f2_unpack(pair_mul(pair_add(pair_of(dp[c + 2], dp[c + 3]), d1), pair_of(s[c + 2], s[c + 3])), dp[c + 2], dp[c + 3]);
  }
  if (clean) {
#pragma unroll
    for (int c = 0; c < N; ++c) dp[c] = s[c] == 0.0f ? 0.0f : dp[c];
  }
}

template <int N>
__device__ __forceinline__ void load_row(uint32_t at, float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 32) tmem_load32(at + c, v + c);
  tmem_wait_load();
}

// N values of a thread's row to TMEM in 16 bits, and word of it to `bar`.
template <typename T, int N>
__device__ __forceinline__ void store_row(uint32_t at, const float (&v)[N], uint64_t* bar) {
#pragma unroll
  for (int from = 0; from < N; from += 32) {
    uint32_t packed[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) packed[c] = pack_pair<T>(v[from + 2 * c], v[from + 2 * c + 1]);
    tmem_store16(at + from / 2, packed);
  }
  tmem_wait_store();
  fence_before();
  __syncwarp();
  if (threadIdx.x % 32 == 0) bar_arrive(bar);
}

// COLS columns of a thread's row of a sum in TMEM, times mul, to global memory.
template <typename T, int COLS>
__device__ __forceinline__ void write_row(T* out, bool in, uint32_t at, int first, int D, float mul, bool any) {
#pragma unroll
  for (int c = 0; c < COLS; c += 32) {
    float o[32];
    if (any) {
      tmem_load32(at + c, o);
      tmem_wait_load();
    }
    if (!in) continue;
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      if (first + c + e >= D) continue;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int x = 0; x < 8; x += 4) {
          float4 v = make_float4(mul - mul, mul - mul, mul - mul, mul - mul);
          if (any) v = make_float4(o[e + x] * mul, o[e + x + 1] * mul, o[e + x + 2] * mul, o[e + x + 3] * mul);
          *reinterpret_cast<float4*>(out + c + e + x) = v;
        }
        continue;
      }
      uint4 v;
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        w[x] = any ? pack_pair<T>(o[e + 2 * x] * mul, o[e + 2 * x + 1] * mul) : pack_pair<T>(mul - mul, mul - mul);
      *reinterpret_cast<uint4*>(out + c + e) = v;
    }
  }
}

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(BwdShape<DP>::kThreads, BwdShape<DP>::kCtas)
    attn_tc_dq_kernel(const AttnParams p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap gmap) {
  using Shape = BwdShape<DP>;
  constexpr bool DOCS = (MODE & kGrouped) != 0;
  constexpr int STEP = Shape::kStep, N = STEP / 2;
  extern __shared__ char raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  char *sq = smem, *sg = smem + Shape::kTile, *ring = smem + 2 * Shape::kTile;  // stage: key tile, value tile
  __shared__ uint64_t q_full, kv_full[2], kv_empty[2], s_full[2], dp_full, dp_empty, ds_full[2], done, cleared[2];
  __shared__ float delta_part[2][kTileTokens];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  volatile int* abort = &abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, hk = h / (p.H / p.Hkv);
  const int i0 = (gridDim.y - 1 - blockIdx.y) * kTileTokens;
  const int length = attn_length(p, b);
  const int limit = rows_limit(p, b, i0 + kTileTokens, length);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    bar_init(&q_full, 1), bar_init(&done, 1), bar_init(&dp_full, 1);
    for (int i = 0; i < 2; ++i) bar_init(&kv_full[i], 1), bar_init(&kv_empty[i], 1), bar_init(&s_full[i], 1), bar_init(&cleared[i], 1);
    bar_init(&dp_empty, kSoftmaxThreads / 32);
    for (int i = 0; i < 2; ++i) bar_init(&ds_full[i], kSoftmaxThreads / 32);
    fence_async_smem();
  }
  if (warp == kMmaWarp) tmem_alloc<Shape::kColumns>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  // Two buffers of scores, whose place the derivative takes; dp; dq.
  const uint32_t tmem = tmem_slot, dp_at = tmem + 2 * STEP, dq_at = tmem + 3 * STEP;

  if (warp < kLoadWarp) {
    if constexpr (Shape::kSplit) take_registers();
    const int half = warp / 4, r = threadIdx.x % kTileTokens, i = i0 + r;
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;
    const RowView row = row_view(p, b, i, length);
    const ScoreForm f = score_form(p, h);
    const int* kdoc = p.kdoc ? p.kdoc + (int64_t)b * p.Sk : nullptr;
    const bool in = i < p.Sq;
    const int64_t stat = ((int64_t)b * p.H + h) * p.Sq + i;
    // delta: each half of the warps sums every other 8 channels.
    float delta = 0.0f;
    if (in && row.limit > 0) {
      const int64_t o_at = (((int64_t)b * p.Sq + i) * p.H + h) * p.D;
      const T* o = static_cast<const T*>(p.o) + o_at;
      const T* low = p.residue ? static_cast<const T*>(p.residue) + o_at : nullptr;
      const T* g = static_cast<const T*>(p.go) + b * p.gs[0] + i * p.gs[1] + h * p.gs[2];
#pragma unroll 4
      for (int d = half * 8; d < p.D; d += 16) {
        float x[8], y[8], z[8];
        load_vec<T, 8>(o + d, x);
        load_vec<T, 8>(g + d, y);
        if (low) {
          load_vec<T, 8>(low + d, z);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] += z[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e], delta);
      }
    }
    delta_part[half][r] = delta;
    named_barrier(1, kSoftmaxThreads);
    delta = delta_part[0][r] + delta_part[1][r];
    if (in && half == 0) p.delta[stat] = delta;
    const float lse = in && row.limit > 0 ? p.lse[stat] * -kLog2e : 0.0f;
    const uint64_t lse2 = pair_of(lse, lse), delta2 = pair_of(-delta, -delta);
    bool ok = true;
    int u = 0;
    for (KeySteps<STEP, DOCS> at(p, b, i0, 1, limit, length); !at.done && ok; at.advance(p, b, i0, 1, length), ++u) {
      const int c0 = at.j * kTileTokens + at.half * 64 + half * N;  // the thread's first key
      const uint32_t s_at = tmem + lanes + (u & 1) * STEP + half * N;
      ok = warp_wait(&s_full[u & 1], (u >> 1) & 1, abort);
      if (!ok) break;
      fence_after();
      float s[N], t2[MODE & kCapped ? N : 2];
      load_row(s_at, s);
      const int seen = row.limit - c0;
      const float away = (float)(row.place - c0);
      probabilities<MODE>(p, f, s, t2, [&](int c) { return away - (float)c; }, [&](int, uint64_t& a, uint64_t& d) { a = d = lse2; });
      if constexpr ((MODE & kCapped) != 0) multiply(s, t2);
      bool masked = false;
      if (!__all_sync(kFullMask, seen >= N)) {
        masked = true;
#pragma unroll
        for (int c = 0; c < N; ++c) s[c] = c < seen ? s[c] : 0.0f;
      }
      if (DOCS && !(at.state.agree & 1)) {
        masked = true;
        uint32_t mask[N / 32];
        document_masks(p, kdoc, c0, row.doc, mask);
#pragma unroll
        for (int c = 0; c < N; ++c) s[c] = mask[c / 32] >> (c % 32) & 1 ? s[c] : 0.0f;
      }
      ok = warp_wait(&dp_full, u & 1, abort);
      if (!ok) break;
      fence_after();
      float dp[N];
      load_row(dp_at + lanes + half * N, dp);
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&dp_empty);
      derivatives(s, dp, masked, [&](int, uint64_t& a, uint64_t& d) { a = d = delta2; });
      store_row<T>(s_at, dp, &ds_full[u & 1]);
    }
    if (ok && u > 0) ok = warp_wait(&done, 0, abort);
    fence_after();
    // Each half of the warps writes half of the channels, or the first all of them
    // where half would be less than a load's 32.
    constexpr int cols = DP >= 64 ? DP / 2 : DP;
    if (half * cols < DP)
      write_row<T, cols>(static_cast<T*>(p.dq) + (((int64_t)b * p.Sq + i) * p.H + h) * p.D + half * cols, in,
                         dq_at + lanes + half * cols, half * cols, p.D, ok ? p.scale : NAN, u > 0);
    fence_before();
  } else {
    if constexpr (Shape::kSplit) leave_registers();
    if (warp == kLoadWarp) {
      if (limit > 0) {
        if (lane == 0) {
          bar_expect(&q_full, 2 * Shape::kTile);
          tma_tile<DP>(sq, &qmap, &q_full, h, i0, b);
          tma_tile<DP>(sg, &gmap, &q_full, h, i0, b);
        }
        const int* kdoc = p.kdoc ? p.kdoc + (int64_t)b * p.Sk : nullptr;
        int n = 0;
        bool ok = true;
        for (KeySteps<STEP, DOCS> at(p, b, i0, 1, limit, length); !at.done && ok; at.next_tile(p, b, i0, 1, length)) {
          const int slot = n % 2;
          if (n >= 2) ok = warp_wait(&kv_empty[slot], (n / 2 - 1) & 1, abort);
          if (!ok) break;
          char* stage = ring + slot * 2 * Shape::kTile;
          if (lane == 0) {
            bar_expect(&kv_full[slot], 2 * Shape::kTile);
            tma_tile<DP>(stage, &kmap, &kv_full[slot], hk, at.j * kTileTokens, b);
            tma_tile<DP>(stage + Shape::kTile, &vmap, &kv_full[slot], hk, at.j * kTileTokens, b);
          }
          __syncwarp();
          if (at.state.padded) {  // padded keys are cleared: dq's product goes over all of the tile's
            ok = warp_wait(&kv_full[slot], (n / 2) & 1, abort);
            clear_rows<DP>(stage, KeyRows{kdoc, at.j * kTileTokens, length});
            if (lane == 0) bar_arrive(&cleared[slot]);
          }
          ++n;
        }
        warp_wait(&q_full, 0, abort);
        for (int i = max(0, n - 2); i < n; ++i) warp_wait(&kv_full[i % 2], (i / 2) & 1, abort);
      }
    } else if (warp == kMmaWarp && elect_one()) {
      constexpr uint32_t ds = instr_desc<IsBf16<T>::value>(STEP, false), dd = instr_desc<IsBf16<T>::value>(DP, true);
      constexpr uint64_t kHalfTile = 64 * 128 >> 4, kTileDesc = Shape::kTile >> 4;
      const uint64_t q_desc = by_channels(smem_u32(sq)), g_desc = q_desc + kTileDesc, kv_desc = by_channels(smem_u32(ring));
      const uint64_t k_tokens = by_tokens(smem_u32(ring));
      bool ok = limit == 0 || bar_wait(&q_full, 0, abort);
      int u = 0, prev_slot = 0;
      StagePhases cleared_phase;
      uint64_t prev_k = 0;      // keys of the step before, whose dq is due
      bool prev_last = false;   // it was its tile's last
      // A barrier for each of the two buffers: a step's scores and dp are issued before
      // the step before is waited for, so that its derivative too may be there by then.
      const auto finish = [&]() {
        ok = bar_wait(&ds_full[(u - 1) & 1], ((u - 1) >> 1) & 1, abort);
        fence_after();
        if (!ok) return;
        product_parts<STEP>(dq_at, tmem + ((u - 1) & 1) * STEP, prev_k, dd, u > 1);
        if (prev_last) commit(&kv_empty[prev_slot]);
      };
      for (KeySteps<STEP, DOCS> at(p, b, i0, 1, limit, length); !at.done && ok; at.next_tile(p, b, i0, 1, length)) {
        const int slot = at.n & 1, count = at.count();
        ok = bar_wait(&kv_full[slot], (at.n >> 1) & 1, abort);
        if (ok && at.state.padded) ok = bar_wait(&cleared[slot], cleared_phase.next(slot), abort);
        for (int half = 0; half < count && ok; ++half, ++u) {
          // Scores into the buffer that the step before last has left, ahead of
          // the softmax of the step before.
          const uint64_t k = kv_desc + slot * 2 * kTileDesc + half * kHalfTile;
          fence_after();
          product_channels<DP>(tmem + (u & 1) * STEP, q_desc, k, ds);
          commit(&s_full[u & 1]);
          if (u > 0) ok = bar_wait(&dp_empty, (u - 1) & 1, abort);
          fence_after();
          if (!ok) break;
          product_channels<DP>(dp_at, g_desc, k + kTileDesc, ds);
          commit(&dp_full);
          if (u > 0) finish();
          prev_slot = slot, prev_k = k_tokens + slot * 2 * kTileDesc + half * 4 * kTokenStep, prev_last = half + 1 == count;
        }
      }
      if (ok && u > 0) finish();
      commit(&done);
      if (!ok) bar_wait(&done, 0, abort);
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    tmem_free<Shape::kColumns>(tmem);
  }
}

// The steps that a block of keys goes through: every head of its group, the
// tiles of queries from the first that may see it, or with STEP 64 their halves.
// state.padded: some queries of the tile may see no key at all.
template <int STEP, bool DOCS>
struct QuerySteps {
  int g, i, half, n;  // head of the group, query tile, its half, the tile's number among those visited
  int first, tiles, halves;
  bool done;
  TileState state;

  __device__ __forceinline__ void seek(const AttnParams& p, int b, int group, int kt, int length) {
    for (;;) {
      if (i >= tiles) i = first, ++g;
      done = g >= group || first >= tiles;
      if (done) return;
      if constexpr (!DOCS) {
        state = TileState{0, 3, false, p.causal && i * kTileTokens < p.Sq - length};
        return;
      } else {
        state = tile_state(p, b, i * kTileTokens, 1, kt, length);
        if (!state.skip) {
          state.padded = true;
          return;
        }
        ++i;
      }
    }
  }
  __device__ __forceinline__ QuerySteps(const AttnParams& p, int b, int group, int kt, int length)
      : g(0), half(0), n(0), tiles((p.Sq + kTileTokens - 1) / kTileTokens),
        halves(STEP == 128 || (p.Sq - 1) % kTileTokens < 64 ? 1 : 2) {
    const int j0 = kt * kTileTokens;
    first = i = j0 < length ? first_query(p, b, j0, length) / kTileTokens : tiles;
    seek(p, b, group, kt, length);
  }
  __device__ __forceinline__ int count() const { return STEP == 128 || i + 1 == tiles ? halves : 2; }
  __device__ __forceinline__ void next_tile(const AttnParams& p, int b, int group, int kt, int length) {
    half = 0, ++i, ++n;
    seek(p, b, group, kt, length);
  }
  __device__ __forceinline__ void advance(const AttnParams& p, int b, int group, int kt, int length) {
    if (half + 1 == count()) next_tile(p, b, group, kt, length);
    else half = 1;
  }
  __device__ __forceinline__ int row() const { return i * kTileTokens + half * 64; }
};

// What a key-tile thread needs of each query of a step.
template <int STEP>
struct __align__(16) QueryStats {
  float lse[STEP], delta[STEP];  // negative; lse to base 2
  int limit[STEP], place[STEP], doc[STEP];
};

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(BwdShape<DP>::kThreads, BwdShape<DP>::kCtas)
    attn_tc_dkv_kernel(const AttnParams p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap gmap) {
  using Shape = BwdShape<DP>;
  constexpr bool DOCS = (MODE & kGrouped) != 0;
  constexpr int STEP = Shape::kStep, N = STEP / 2;
  extern __shared__ char raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  char *sk = smem, *sv = smem + Shape::kTile, *ring = smem + 2 * Shape::kTile;  // stage: query tile, gradient tile
  __shared__ uint64_t k_full, q_full[2], q_empty[2], s_full, p_full, dp_full, ds_full, done, cleared[2];
  __shared__ QueryStats<STEP> stats[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  volatile int* abort = &abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int hk = blockIdx.x % p.Hkv, part = blockIdx.x / p.Hkv % p.kv_parts, b = blockIdx.x / (p.Hkv * p.kv_parts);
  const int group = p.H / p.Hkv / p.kv_parts, head0 = (hk * p.kv_parts + part) * group;  // this CTA's query heads
  const int kt = blockIdx.y, j0 = kt * kTileTokens;  // early keys, which the most causal queries see, first
  const int length = attn_length(p, b);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    bar_init(&k_full, 1), bar_init(&done, 1), bar_init(&s_full, 1), bar_init(&dp_full, 1);
    for (int i = 0; i < 2; ++i) bar_init(&q_full[i], 1), bar_init(&q_empty[i], 1), bar_init(&cleared[i], 1);
    bar_init(&p_full, kSoftmaxThreads / 32), bar_init(&ds_full, kSoftmaxThreads / 32);
    fence_async_smem();
  }
  if (warp == kMmaWarp) tmem_alloc<Shape::kColumns>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  // Scores, then probabilities; dp, then its derivative; dv; dk.
  const uint32_t tmem = tmem_slot, dp_at = tmem + STEP, dv_at = tmem + 2 * STEP, dk_at = dv_at + DP;

  if (warp < kLoadWarp) {
    if constexpr (Shape::kSplit) take_registers();
    const int half = warp / 4, r = threadIdx.x % kTileTokens, j = j0 + r;  // key of this thread
    const int c0 = half * N;
    const uint32_t lanes = (uint32_t)(warp % 4) << 21, s_at = tmem + lanes + c0;
    const int kd = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
    const bool live = j < length;
    // The queries' statistics of a step are fetched during the step before: the
    // first half of the warps has a query's log-sum-exp and row sum, the second
    // its view of the keys.
    float lse = 0.0f, delta = 0.0f;
    RowView view{};
    const auto fetch = [&](const QuerySteps<STEP, DOCS>& at) {
      if (at.done || r >= STEP) return;
      const int i = at.row() + r;
      view = row_view(p, b, i, length);
      if (half == 0) {
        const int64_t stat = ((int64_t)b * p.H + head0 + at.g) * p.Sq + i;
        lse = view.limit > 0 ? __ldg(p.lse + stat) * -kLog2e : 0.0f;
        delta = view.limit > 0 ? -__ldg(p.delta + stat) : 0.0f;
      }
    };
    bool ok = true;
    int u = 0;
    QuerySteps<STEP, DOCS> at(p, b, group, kt, length);
    fetch(at);
    // A warp whose wait gave up still comes to the others' barriers.
    while (!at.done) {
      QueryStats<STEP>& q = stats[u & 1];
      const ScoreForm f = score_form(p, head0 + at.g);
      const bool agree = at.state.agree & 1;
      // This buffer was read two steps ago: every thread has passed the barrier
      // of the step between.
      if (r < STEP) {
        if (half == 0) q.lse[r] = lse, q.delta[r] = delta;
        else q.limit[r] = view.limit, q.place[r] = view.place, q.doc[r] = view.doc;
      }
      int full;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n barrier.cta.red.and.pred q, 1, %2, p;\n selp.s32 %0, 1, 0, q;\n}"
                   : "=r"(full) : "r"((int)(r >= STEP || view.limit >= j0 + kTileTokens)), "r"(kSoftmaxThreads) : "memory");
      const bool whole = full && agree;  // every query of the step sees every key of the tile
      at.advance(p, b, group, kt, length);
      fetch(at);
      const int turn = u++ & 1;
      ok = ok && warp_wait(&s_full, turn, abort);
      if (!ok) continue;
      fence_after();
      float s[N], t2[MODE & kCapped ? N : 2];
      load_row(s_at, s);
      const auto pairs = [&](const float* from, int c, uint64_t& a, uint64_t& d) {
        const float4 v = *reinterpret_cast<const float4*>(from + c0 + c);
        a = pair_of(v.x, v.y), d = pair_of(v.z, v.w);
      };
      probabilities<MODE>(p, f, s, t2, [&](int c) { return (float)(q.place[c0 + c] - j); },
                          [&](int c, uint64_t& a, uint64_t& d) { pairs(q.lse, c, a, d); });
      if (!whole) {
#pragma unroll
        for (int c = 0; c < N; c += 4) {
          const int4 limit = *reinterpret_cast<const int4*>(q.limit + c0 + c);
          s[c] = live & (j < limit.x) ? s[c] : 0.0f;
          s[c + 1] = live & (j < limit.y) ? s[c + 1] : 0.0f;
          s[c + 2] = live & (j < limit.z) ? s[c + 2] : 0.0f;
          s[c + 3] = live & (j < limit.w) ? s[c + 3] : 0.0f;
        }
        if (DOCS && !agree) {
          // A key of the shared document is of every query's; padded queries' limit is 0.
          const bool any = kd >= 0 && kd == p.shared;
#pragma unroll
          for (int c = 0; c < N; c += 4) {
            const int4 doc = *reinterpret_cast<const int4*>(q.doc + c0 + c);
            s[c] = (any | (doc.x == kd)) ? s[c] : 0.0f;
            s[c + 1] = (any | (doc.y == kd)) ? s[c + 1] : 0.0f;
            s[c + 2] = (any | (doc.z == kd)) ? s[c + 2] : 0.0f;
            s[c + 3] = (any | (doc.w == kd)) ? s[c + 3] : 0.0f;
          }
        }
      }
      store_row<T>(s_at, s, &p_full);
      if constexpr ((MODE & kCapped) != 0) {
        // Padded keys lie in the tile as they came: a score of NaN has a derivative of NaN.
        if (!whole) {
#pragma unroll
          for (int c = 0; c < N; ++c) t2[c] = s[c] == 0.0f ? 0.0f : t2[c];
        }
        multiply(s, t2);
      }
      ok = warp_wait(&dp_full, turn, abort);
      if (!ok) continue;
      fence_after();
      float dp[N];
      load_row(dp_at + lanes + c0, dp);
      derivatives(s, dp, !whole, [&](int c, uint64_t& a, uint64_t& d) { pairs(q.delta, c, a, d); });
      store_row<T>(dp_at + lanes + c0, dp, &ds_full);
    }
    if (ok && u > 0) ok = warp_wait(&done, 0, abort);
    fence_after();
    const bool in = j < p.Sk;
    const int64_t out = (((int64_t)b * p.Sk + j) * p.Hkv + hk) * p.D;
    // The first half of the warps writes dv, the second dk.
    const uint32_t sums = (half == 0 ? dv_at : dk_at) + lanes;
    const float mul = !ok ? NAN : half == 0 ? 1.0f : p.scale;
    if (p.kv_parts > 1) write_row<float, DP>(kv_part(p, part, half != 0) + out, in, sums, 0, p.D, mul, u > 0);
    else write_row<T, DP>(static_cast<T*>(half == 0 ? p.dv : p.dk) + out, in, sums, 0, p.D, mul, u > 0);
    fence_before();
  } else {
    if constexpr (Shape::kSplit) leave_registers();
    if (warp == kLoadWarp) {
      QuerySteps<STEP, DOCS> at(p, b, group, kt, length);
      if (!at.done) {
        if (lane == 0) {
          bar_expect(&k_full, 2 * Shape::kTile);
          tma_tile<DP>(sk, &kmap, &k_full, hk, j0, b);
          tma_tile<DP>(sv, &vmap, &k_full, hk, j0, b);
        }
        int n = 0;
        bool ok = true;
        for (; !at.done && ok; at.next_tile(p, b, group, kt, length)) {
          const int slot = n % 2, h = head0 + at.g, i0 = at.i * kTileTokens;
          if (n >= 2) ok = warp_wait(&q_empty[slot], (n / 2 - 1) & 1, abort);
          if (!ok) break;
          char* stage = ring + slot * 2 * Shape::kTile;
          if (lane == 0) {
            bar_expect(&q_full[slot], 2 * Shape::kTile);
            tma_tile<DP>(stage, &qmap, &q_full[slot], h, i0, b);
            tma_tile<DP>(stage + Shape::kTile, &gmap, &q_full[slot], h, i0, b);
          }
          __syncwarp();
          if (at.state.padded) {
            // Queries that see no key (padding, an id that no key has, a place before
            // the first key) and their gradients count for nothing, whatever they hold.
            const float* lse = p.lse + ((int64_t)b * p.H + h) * p.Sq;
            uint32_t idle = 0;
#pragma unroll
            for (int x = 0; x < kTileTokens / 32; ++x) {
              const int i = i0 + x * 32 + lane;
              if (i < p.Sq && __ldg(lse + i) == -INFINITY) idle |= 1u << x;
            }
            if (__any_sync(kFullMask, idle != 0)) {
              const auto keep = [&](int r) { return !(idle >> (r / 32) & 1); };
              ok = warp_wait(&q_full[slot], (n / 2) & 1, abort);
              clear_rows<DP>(stage, keep);
              clear_rows<DP>(stage + Shape::kTile, keep);
            }
            if (lane == 0) bar_arrive(&cleared[slot]);
          }
          ++n;
        }
        warp_wait(&k_full, 0, abort);
        for (int i = max(0, n - 2); i < n; ++i) warp_wait(&q_full[i % 2], (i / 2) & 1, abort);
      }
    } else if (warp == kMmaWarp && elect_one()) {
      constexpr uint32_t ds = instr_desc<IsBf16<T>::value>(STEP, false), dd = instr_desc<IsBf16<T>::value>(DP, true);
      constexpr uint64_t kHalfTile = 64 * 128 >> 4, kTileDesc = Shape::kTile >> 4;
      const uint64_t k_desc = by_channels(smem_u32(sk)), v_desc = k_desc + kTileDesc, qg_desc = by_channels(smem_u32(ring));
      const uint64_t qg_tokens = by_tokens(smem_u32(ring));
      QuerySteps<STEP, DOCS> at(p, b, group, kt, length);
      bool ok = at.done || bar_wait(&k_full, 0, abort);
      int u = 0, prev_slot = 0;
      StagePhases cleared_phase;
      uint64_t prev_q = 0;     // queries of the step before, whose sums are due
      bool prev_last = false;  // it was its tile's last
      // dv of the step before, then this step's scores over its probabilities;
      // dk of the step before, then this step's dp over its derivative: each
      // product runs while the softmax works on the other half.
      const auto add_dv = [&]() {
        ok = bar_wait(&p_full, (u - 1) & 1, abort);
        fence_after();
        if (ok) product_parts<STEP>(dv_at, tmem, prev_q + kTileDesc, dd, u > 1);
      };
      const auto add_dk = [&]() {
        ok = ok && bar_wait(&ds_full, (u - 1) & 1, abort);
        fence_after();
        if (!ok) return;
        product_parts<STEP>(dk_at, dp_at, prev_q, dd, u > 1);
        if (prev_last) commit(&q_empty[prev_slot]);
      };
      for (; !at.done && ok; at.next_tile(p, b, group, kt, length)) {
        const int slot = at.n & 1, count = at.count();
        ok = bar_wait(&q_full[slot], (at.n >> 1) & 1, abort);
        if (ok && at.state.padded) ok = bar_wait(&cleared[slot], cleared_phase.next(slot), abort);
        for (int half = 0; half < count && ok; ++half, ++u) {
          const uint64_t q = qg_desc + slot * 2 * kTileDesc + half * kHalfTile;
          if (u > 0) add_dv();
          if (!ok) break;
          fence_after();
          product_channels<DP>(tmem, k_desc, q, ds);
          commit(&s_full);
          if (u > 0) add_dk();
          if (!ok) break;
          product_channels<DP>(dp_at, v_desc, q + kTileDesc, ds);
          commit(&dp_full);
          prev_slot = slot, prev_q = qg_tokens + slot * 2 * kTileDesc + half * 4 * kTokenStep, prev_last = half + 1 == count;
        }
      }
      if (ok && u > 0) {
        add_dv();
        add_dk();
      }
      commit(&done);
      if (!ok) bar_wait(&done, 0, abort);
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    tmem_free<Shape::kColumns>(tmem);
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
bool make_map(CUtensorMap* map, const void* base, bool bf16, int64_t D, int64_t H, int64_t S, int64_t B, const int64_t (&strides)[3]);

template <typename T, int DP, int MODE>
cudaError_t launch_fwd(const AttnParams& p, const CUtensorMap (&m)[4], cudaStream_t st) {
  using Shape = FwdShape<DP>;
  static std::atomic<uint64_t> set{0};
  cudaError_t e = abi::allow_smem(attn_tc_fwd_kernel<T, DP, MODE>, Shape::kSmem, set);
  if (e != cudaSuccess) return e;
  const dim3 grid(p.H * p.B, (p.Sq + 2 * kTileTokens - 1) / (2 * kTileTokens));
  attn_tc_fwd_kernel<T, DP, MODE><<<grid, Shape::kThreads, Shape::kSmem, st>>>(p, m[0], m[1], m[2]);
  return cudaGetLastError();
}

template <typename T, int DP, int MODE>
cudaError_t launch_bwd(const AttnParams& p, const CUtensorMap (&m)[4], cudaStream_t st) {
  using Shape = BwdShape<DP>;
  static std::atomic<uint64_t> set_q{0}, set_k{0};
  cudaError_t e = abi::allow_smem(attn_tc_dq_kernel<T, DP, MODE>, Shape::kSmem, set_q);
  if (e == cudaSuccess) e = abi::allow_smem(attn_tc_dkv_kernel<T, DP, MODE>, Shape::kSmem, set_k);
  if (e != cudaSuccess) return e;
  const auto tiles = [](int n) { return (unsigned)((n + kTileTokens - 1) / kTileTokens); };
  attn_tc_dq_kernel<T, DP, MODE><<<dim3(p.H * p.B, tiles(p.Sq)), Shape::kThreads, Shape::kSmem, st>>>(p, m[0], m[1], m[2], m[3]);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  attn_tc_dkv_kernel<T, DP, MODE><<<dim3(p.Hkv * p.kv_parts * p.B, tiles(p.Sk)), Shape::kThreads, Shape::kSmem, st>>>(p, m[0], m[1], m[2], m[3]);
  return cudaGetLastError();
}

template <typename T, int MODE>
cudaError_t launch_by_size(const AttnParams& p, const CUtensorMap (&m)[4], bool backward, cudaStream_t st) {
  if (p.D <= 32) return backward ? launch_bwd<T, 32, MODE>(p, m, st) : launch_fwd<T, 32, MODE>(p, m, st);
  if (p.D <= 64) return backward ? launch_bwd<T, 64, MODE>(p, m, st) : launch_fwd<T, 64, MODE>(p, m, st);
  return backward ? launch_bwd<T, 128, MODE>(p, m, st) : launch_fwd<T, 128, MODE>(p, m, st);
}

template <typename T>
int run(const AttnParams& p, bool backward, cudaStream_t st) {
  constexpr bool bf16 = IsBf16<T>::value;
  CUtensorMap m[4];
  if (!make_map(&m[0], p.q, bf16, p.D, p.H, p.Sq, p.B, p.qs) || !make_map(&m[1], p.k, bf16, p.D, p.Hkv, p.Sk, p.B, p.ks) ||
      !make_map(&m[2], p.v, bf16, p.D, p.Hkv, p.Sk, p.B, p.vs) ||
      (backward && !make_map(&m[3], p.go, bf16, p.D, p.H, p.Sq, p.B, p.gs)))
    return -1;
  switch ((p.cap != 0.0f ? kCapped : 0) | (p.slopes ? kSloped : 0) | (p.kdoc ? kGrouped : 0)) {
    case 0: return (int)launch_by_size<T, 0>(p, m, backward, st);
    case 1: return (int)launch_by_size<T, 1>(p, m, backward, st);
    case 2: return (int)launch_by_size<T, 2>(p, m, backward, st);
    case 3: return (int)launch_by_size<T, 3>(p, m, backward, st);
    case 4: return (int)launch_by_size<T, 4>(p, m, backward, st);
    case 5: return (int)launch_by_size<T, 5>(p, m, backward, st);
    case 6: return (int)launch_by_size<T, 6>(p, m, backward, st);
    default: return (int)launch_by_size<T, 7>(p, m, backward, st);
  }
}

}  // namespace tc
}  // namespace msda
