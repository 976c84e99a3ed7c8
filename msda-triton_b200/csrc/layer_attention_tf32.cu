// Masked attention in 32 bits, and of 16-bit heads, strides and alignments that
// the tensor-core kernels of layer_attention_tc.cuh do not take.
//
// The products run on the tensor cores by register fragments (m16n8k8, tf32 in,
// fp32 sums): an fp32 number is the sum of two tf32 numbers to 2^-22 of its size,
//   x y = xh yh + xh yl + xl yh  (+ xl yl, below 2^-20 x y),
// three products for one, at 92 TFLOP/s a bound above the 72 of the FMA pipes.
// 16-bit inputs are tf32 numbers as they stand: their scores need one product,
// probabilities with values two. (On the FMA pipes, with 8 x 4 sums a thread, a
// training step of 2 x 1500 tokens, 8 heads of 128 channels took 5.8 ms.)
//
// A CTA has 64 rows (queries; keys in their gradient), 16 a warp, in one group of
// four warps or two that share the work of a step of 32 or 64 columns (keys between
// them in the forward and in dq, products in the key gradient). Steps come by
// asynchronous copies, in the forward into the other of two slots; elsewhere the
// SM's other CTAs cover them. All tiles lie as rows of DP + 4 floats: four
// words past a multiple of 32, so that the fragments of both kinds of product (over
// channels, by ldmatrix; over tokens, word by word) are free of bank conflicts. The
// second product takes the probabilities from the first one's registers: its eight
// k-slots are the tokens in the order 0 2 4 6 1 3 5 7, in which a thread has them.
//
// fp32, 2 x 1201 tokens, 8 heads of 32 channels, causal with prefixes: forward 79
// us, dq 106 us, dk and dv 145 us, 26 to 29 TFLOP/s of products formed; 2 x 1500
// tokens, 8 heads of 128: forward 585 us, 31 TFLOP/s, a training step 2.2 ms, 38
// TFLOP/s. Bound by what stands around the products, the splitting of fragments and
// their waits (the tensor pipe is a quarter to a third active), and at these sizes by
// CTAs that fill the GPU one and a third times.
#include "layer_attention.cuh"

namespace msda {
namespace {

constexpr int kThreads = 128;      // forward: a warp has 16 rows
constexpr int kBwdThreads = 256;  // backward: two groups of four warps
constexpr int kRows = 64;  // rows of a CTA, 16 a warp
constexpr int kCols = 32;  // columns of a step

template <int DP>
struct Pitch {
  static constexpr int kFloats = DP + 4;
  static constexpr int kRowTile = kRows * kFloats, kColTile = kCols * kFloats;
};

// x cut to a tf32 number, and what is left of it, rounded to one (the product cuts
// the bits below): 2^-22 of x at most is lost, to either side. (Cut as well, the
// second part would lose 2^-21, always towards zero: twice the error of a gradient.)
__device__ __forceinline__ void split(float x, uint32_t& high, uint32_t& low) {
  high = __float_as_uint(x) & 0xffffe000u;
  low = __float_as_uint(x - __uint_as_float(high)) + 0x1000u;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// d = a b (+ c)
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2,
                                    float c3) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// A fragment in its two parts; EXACT: it is of tf32 numbers.
template <bool EXACT, int N>
__device__ __forceinline__ void parts(const uint32_t (&x)[N], uint32_t (&high)[N], uint32_t (&low)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (EXACT) high[i] = x[i], low[i] = 0;
    else split(__uint_as_float(x[i]), high[i], low[i]);
  }
}

// d[n] += a b[n] over 8 k-slots for N tiles at a time, whose products take turns in
// the pipe, the small ones first. The tensor cores cut their running sum, which
// over the steps of a long sum would cost several digits: d begins at zero every
// second step, and `join` adds it to the long sum, rounded. `rest`: what is left of
// b past its two parts, or nothing (WHOLE).
template <bool EXACT_A, bool EXACT_B, bool WHOLE, int N>
__device__ __forceinline__ void products(float (&d)[N][4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const uint32_t (&bh)[N][2],
                                         const uint32_t (&bl)[N][2], const uint32_t (&rest)[WHOLE ? N : 1][2]) {
  if constexpr (WHOLE) {
#pragma unroll
    for (int n = 0; n < N; ++n) mma(d[n], ah, rest[n][0], rest[n][1], d[n][0], d[n][1], d[n][2], d[n][3]);
  }
  if constexpr (!EXACT_A) {
#pragma unroll
    for (int n = 0; n < N; ++n) mma(d[n], al, bh[n][0], bh[n][1], d[n][0], d[n][1], d[n][2], d[n][3]);
  }
  if constexpr (!EXACT_B) {
#pragma unroll
    for (int n = 0; n < N; ++n) mma(d[n], ah, bl[n][0], bl[n][1], d[n][0], d[n][1], d[n][2], d[n][3]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) mma(d[n], ah, bh[n][0], bh[n][1], d[n][0], d[n][1], d[n][2], d[n][3]);
}

template <int N>
__device__ __forceinline__ void clear(float (&d)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.0f;
}

template <int N>
__device__ __forceinline__ void join(float (*c)[4], const float (&d)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[n][i] += d[n][i];
}

// c[n] = a (16 rows) . b (columns 8 n ...)^T over channels below D.
template <int DP, int NT, bool EXACT>
__device__ __forceinline__ void scores(const float* a, const float* b, int D, float (&c)[NT][4]) {
  constexpr int P = Pitch<DP>::kFloats;
  const int lane = threadIdx.x % 32;
  // Matrices of 8 rows x 4 channels: a's rows 0.. and 8.., then four channels on;
  // b's columns 0.. with both groups of channels, then columns 8...
  const uint32_t a_at = (uint32_t)__cvta_generic_to_shared(a + (lane % 16) * P + lane / 16 * 4);
  const uint32_t b_at = (uint32_t)__cvta_generic_to_shared(b + (lane % 8 + lane / 16 * 8) * P + lane / 8 % 2 * 4);
  clear(c);
  const uint32_t none[1][2] = {{0, 0}};
  // Two steps of 8 channels at a time (tiles are padded with zeros).
  const int pairs = (D + 15) / 16;
#pragma unroll 1
  for (int k = 0; k < pairs; ++k) {
    float d[NT][4];
    clear(d);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t x[4], ah[4], al[4], y[(NT + 1) / 2][4], bh[NT][2], bl[NT][2];
      ldmatrix4(x, a_at + k * 64 + half * 32);
#pragma unroll
      for (int n = 0; n < NT; n += 2) ldmatrix4(y[n / 2], b_at + n * 8 * P * 4 + k * 64 + half * 32);
      parts<EXACT>(x, ah, al);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t z[2] = {y[n / 2][n % 2 * 2], y[n / 2][n % 2 * 2 + 1]};
        parts<EXACT>(z, bh[n], bl[n]);
      }
      products<EXACT, EXACT, false, NT>(d, ah, al, bh, bl, none);
    }
    join(c, d);
  }
}

// out += p (16 x 8 NT, in the layout of `scores`) . t over tokens; EXACT: t is of
// tf32 numbers. WHOLE: t's last bits too, by a fourth product, so that a
// probability of 1 gives the value itself (and the row's gradient, g . v - g . o,
// nothing). W channels of rows of DP.
template <int DP, int W, int NT, bool EXACT, bool WHOLE>
__device__ __forceinline__ void gather(const float (&p)[NT][4], const float* t, float (&out)[W / 8][4]) {
  constexpr int P = Pitch<DP>::kFloats, N = W < 32 ? W / 8 : 4;
  constexpr bool REST = WHOLE && !EXACT;
  const int lane = threadIdx.x % 32;
  const float* at = t + lane % 4 * 2 * P + lane / 4;
  constexpr int PAIR = NT < 2 ? 1 : 2;  // tiles of 8 tokens that are summed before they join
#pragma unroll
  for (int n0 = 0; n0 < NT; n0 += PAIR) {
    uint32_t ah[PAIR][4], al[PAIR][4];
#pragma unroll
    for (int m = 0; m < PAIR; ++m) {
      // Row g: tokens 2 t and 2 t + 1 are slots t and t + 4.
      const float* q = p[n0 + m];
      const uint32_t x[4] = {__float_as_uint(q[0]), __float_as_uint(q[2]), __float_as_uint(q[1]), __float_as_uint(q[3])};
      parts<false>(x, ah[m], al[m]);
    }
#pragma unroll
    for (int d = 0; d < W / 8; d += N) {
      float c[N][4];
      clear(c);
#pragma unroll
      for (int m = 0; m < PAIR; ++m) {
        uint32_t bh[N][2], bl[N][2], rest[REST ? N : 1][2];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float* z = at + (n0 + m) * 8 * P + (d + i) * 8;
          const uint32_t y[2] = {__float_as_uint(z[0]), __float_as_uint(z[P])};
          parts<EXACT>(y, bh[i], bl[i]);
          if constexpr (REST) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              rest[i][e] = __float_as_uint(__uint_as_float(y[e]) - __uint_as_float(bh[i][e]) - __uint_as_float(bl[i][e] & 0xffffe000u));
          }
        }
        products<false, EXACT, REST, N>(c, ah[m], al[m], bh, bl, rest);
      }
      join(out + d, c);
    }
  }
}

// Rows r0 + [0, n) of a (S, D) slice to shared memory; rows that `keep` rejects
// and channels from D on are zeros. fp32 by asynchronous copies. `vec`: 16 bytes
// at a time.
template <typename T, int DP, int THREADS = kThreads, typename Keep>
__device__ __forceinline__ void load_rows(float* to, int n, const T* base, int64_t stride, int r0, int D, bool vec, Keep keep) {
  constexpr int P = Pitch<DP>::kFloats;
  if (sizeof(T) == 4 && vec) {
    for (int i = threadIdx.x; i < n * (DP / 4); i += THREADS) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      const bool in = d < D && keep(r);
      const T* from = in ? base + (int64_t)(r0 + r) * stride + d : base;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + r * P + d)),
                   "l"(from), "r"(in ? 16 : 0) : "memory");
    }
  } else if (sizeof(T) == 2 && vec) {
    for (int i = threadIdx.x; i < n * (DP / 4); i += THREADS) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (d < D && keep(r)) load_vec<T, 4>(base + (int64_t)(r0 + r) * stride + d, f);
      *reinterpret_cast<float4*>(to + r * P + d) = make_float4(f[0], f[1], f[2], f[3]);
    }
  } else {
    for (int i = threadIdx.x; i < n * DP; i += THREADS) {
      const int r = i / DP, d = i % DP;
      float f = 0.0f;
      if (d < D && keep(r)) f = to_f32(__ldg(base + (int64_t)(r0 + r) * stride + d));
      to[r * P + d] = f;
    }
  }
}

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows in pieces of 4 channels: 16 bytes of fp32, 8 of a 16-bit type.
template <typename T>
__device__ __forceinline__ bool can_vec(const void* p, const int64_t (&s)[3], int D) {
  return D % 4 == 0 && (reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T))) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
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

__device__ __forceinline__ bool key_padded(const AttnParams& p, int b, int j, int length) {
  return j >= length || (p.kdoc && __ldg(p.kdoc + (int64_t)b * p.Sk + j) < 0);
}

__device__ __forceinline__ bool skip_tiles(const AttnParams& p, int b, int i0, int j0) {
  if (!p.kdoc) return false;
  const int nq = (p.Sq + kDocTile - 1) / kDocTile, nk = (p.Sk + kDocTile - 1) / kDocTile;
  return tiles_apart(p.qtile[(int64_t)b * nq + i0 / kDocTile], p.ktile[(int64_t)b * nk + j0 / kDocTile]);
}

__device__ __forceinline__ float max4(float v) {
  v = fmaxf(v, __shfl_xor_sync(kFullMask, v, 1));
  return fmaxf(v, __shfl_xor_sync(kFullMask, v, 2));
}
__device__ __forceinline__ float sum4(float v) {
  v += __shfl_xor_sync(kFullMask, v, 1);
  return v + __shfl_xor_sync(kFullMask, v, 2);
}

__device__ __forceinline__ float inverse(float s) { return s > 0.0f ? 1.0f / s : (s == 0.0f ? 0.0f : s); }

// Scores of a warp's 16 rows and 8 NT columns to probabilities, with the rows'
// running maximum and sum; what the rows' sums have to be multiplied by in `old`.
// column(n, e): the key of tile n's column 2 t + e. `whole`: every row sees every
// column.
template <int NT, typename Far>
__device__ __forceinline__ void softmax_step(const AttnParams& p, const ScoreForm (&f)[2], const RowView (&row)[2], float (&s)[NT][4],
                                             const int (&kd)[NT][2], int j0, int end, bool whole, Far column, float (&m)[2], float (&l)[2],
                                             float (&old)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float top = -INFINITY, t;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + column(n, e);
        const bool seen = whole || (j < end && j < row[i].limit && (!p.kdoc || same_document(row[i].doc, kd[n][e], p.shared)));
        s[n][2 * i + e] = seen ? score2(p, f[i], s[n][2 * i + e], row[i].place - j, t) : -INFINITY;
        top = fmaxf(top, s[n][2 * i + e]);
      }
    top = fmaxf(m[i], max4(top));
    const float base = top == -INFINITY ? 0.0f : top;
    old[i] = ex2(m[i] - base);
    m[i] = top;
    l[i] *= old[i];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][2 * i + e] = ex2(s[n][2 * i + e] - base);
        l[i] += s[n][2 * i + e];
      }
  }
}

// Slots of the forward's ring: with one, three CTAs of 128 channels share an SM,
// and cover one another's copies (2 x 1500 tokens, 8 heads: 872 us with two).
template <int DP>
__host__ __device__ constexpr int forward_slots() {
  return DP == 128 ? 1 : 2;
}

// Groups of four warps that have 32 keys of a step each: two up to 64 channels,
// whose sums are joined at the end. (With one, 2 x 1201 tokens on 8 heads of 32
// channels took 112 us: 304 CTAs of four warps leave the schedulers idle.)
template <int DP>
__host__ __device__ constexpr int forward_groups() {
  return DP <= 64 ? 2 : 1;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads * forward_groups<DP>(), DP <= 64 ? 2 : DP == 128 ? 3 : 1) attn_tf32_fwd_kernel(const AttnParams p) {
  constexpr int NT = kCols / 8;
  constexpr bool EXACT = sizeof(T) == 2;
  constexpr int SLOTS = forward_slots<DP>(), GROUPS = forward_groups<DP>(), COLS = kCols * GROUPS, THREADS = kThreads * GROUPS;
  constexpr int kTile = COLS * Pitch<DP>::kFloats;
  using S = Pitch<DP>;
  extern __shared__ __align__(16) float smem[];
  float *qs = smem, *ring = smem + S::kRowTile;  // slots: keys, then values
  const int side = threadIdx.x / kThreads, warp = threadIdx.x / 32 % 4, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, hk = h / (p.H / p.Hkv);
  const int i0 = (gridDim.y - 1 - blockIdx.y) * kRows;  // long causal rows first
  const int length = attn_length(p, b);
  const int limit = rows_limit(p, b, i0 + kRows, length);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  const bool kvec = can_vec<T>(p.k, p.ks, p.D), vvec = can_vec<T>(p.v, p.vs, p.D);
  const auto next = [&](int j) {
    while (j < limit && skip_tiles(p, b, i0, j)) j += COLS;
    return j;
  };
  const auto fill = [&](int j, int slot) {
    if (j < limit) {
      const auto keep = [&](int r) { return !key_padded(p, b, j + r, length); };
      load_rows<T, DP, THREADS>(ring + slot * 2 * kTile, COLS, k, p.ks[1], j, p.D, kvec, keep);
      load_rows<T, DP, THREADS>(ring + (slot * 2 + 1) * kTile, COLS, v, p.vs[1], j, p.D, vvec, keep);
    }
    copies_done();
  };
  load_rows<T, DP, THREADS>(qs, kRows, static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2], p.qs[1], i0, p.D,
                   can_vec<T>(p.q, p.qs, p.D), [&](int r) { return i0 + r < p.Sq; });
  int j0 = next(0);
  fill(j0, 0);
  const ScoreForm f[2] = {score_form(p, h), score_form(p, h)};
  RowView row[2];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, out[DP / 8][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) row[i] = row_view(p, b, i0 + warp * 16 + g + 8 * i, length);
#pragma unroll
  for (int d = 0; d < DP / 8; ++d) out[d][0] = out[d][1] = out[d][2] = out[d][3] = 0.0f;
  const auto column = [&](int n, int e) { return side * kCols + n * 8 + 2 * t + e; };
  for (int slot = 0; j0 < limit; slot ^= SLOTS - 1) {
    const int j1 = next(j0 + COLS);
    if constexpr (SLOTS == 2) {
      fill(j1, slot ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    const float* ks = ring + slot * 2 * kTile + side * S::kColTile;
    float s[NT][4], old[2];
    scores<DP, NT, EXACT>(qs + warp * 16 * S::kFloats, ks, p.D, s);
    int kd[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + column(n, e);
        kd[n][e] = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
      }
    const bool whole = !p.kdoc && __all_sync(kFullMask, j0 + COLS <= min(row[0].limit, row[1].limit));
    softmax_step<NT>(p, f, row, s, kd, j0, limit, whole, column, m, l, old);
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) {
      out[d][0] *= old[0], out[d][1] *= old[0];
      out[d][2] *= old[1], out[d][3] *= old[1];
    }
    gather<DP, DP, NT, EXACT, true>(s, ks + kTile, out);
    __syncthreads();
    if constexpr (SLOTS == 1) fill(j1, 0);
    j0 = j1;
  }
  l[0] = sum4(l[0]), l[1] = sum4(l[1]);
  if constexpr (GROUPS == 2) {
    // The second group's parts take the queries' and the ring's place.
    copies_wait<0>();
    __syncthreads();
    float* ml = ring;
    if (side == 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = warp * 16 + g + 8 * i;
        if (t == 0) ml[2 * r] = m[i], ml[2 * r + 1] = l[i];
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
          *reinterpret_cast<float2*>(qs + r * S::kFloats + d * 8 + 2 * t) = make_float2(out[d][2 * i], out[d][2 * i + 1]);
      }
    }
    __syncthreads();
    if (side == 1) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = warp * 16 + g + 8 * i;
      const float other = ml[2 * r], top = fmaxf(m[i], other), base = top == -INFINITY ? 0.0f : top;
      const float w0 = ex2(m[i] - base), w1 = ex2(other - base);
      m[i] = top;
      l[i] = fmaf(l[i], w0, ml[2 * r + 1] * w1);
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        const float2 o = *reinterpret_cast<const float2*>(qs + r * S::kFloats + d * 8 + 2 * t);
        out[d][2 * i] = fmaf(out[d][2 * i], w0, o.x * w1);
        out[d][2 * i + 1] = fmaf(out[d][2 * i + 1], w0, o.y * w1);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float sum = l[i], mul = inverse(sum);
    const int r = i0 + warp * 16 + g + 8 * i;
    if (r >= p.Sq) continue;
    if (p.lse && t == 0)
      p.lse[((int64_t)b * p.H + h) * p.Sq + r] = sum == 0.0f ? -INFINITY : (m[i] + log2f(sum)) * kLn2;
    const int64_t at = (((int64_t)b * p.Sq + r) * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (d * 8 + 2 * t + e < p.D) put_output<T>(p, at + d * 8 + 2 * t + e, out[d][2 * i + e] * mul);
  }
}

// A few queries over long keys: the rows are 16 pairs of a query and one of the
// heads that share a key head, and a warp has 8 of the 32 keys of a step.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attn_tf32_token_kernel(const AttnParams p) {
  constexpr bool EXACT = sizeof(T) == 2;
  using S = Pitch<DP>;
  extern __shared__ __align__(16) float smem[];
  __shared__ float2 part_ml[4][16];
  float *qs = smem, *ring = smem + 16 * S::kFloats;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int group = p.H / p.Hkv, rows = p.Sq * group, tiles = (rows + 15) / 16;
  const int hk = blockIdx.x / tiles, r0 = blockIdx.x % tiles * 16, b = blockIdx.z, part = blockIdx.y;
  pdl_trigger();
  const int length = attn_length(p, b);
  int first, last;
  split_range(rows_limit(p, b, (min(r0 + 16, rows) + group - 1) / group, length), p.splits, part, first, last);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  const bool kvec = can_vec<T>(p.k, p.ks, p.D), vvec = can_vec<T>(p.v, p.vs, p.D);
  const auto fill = [&](int j, int slot) {
    if (j < last) {
      const auto keep = [&](int r) { return j + r < last && !key_padded(p, b, j + r, length); };
      load_rows<T, DP>(ring + slot * 2 * S::kColTile, kCols, k, p.ks[1], j, p.D, kvec, keep);
      load_rows<T, DP>(ring + (slot * 2 + 1) * S::kColTile, kCols, v, p.vs[1], j, p.D, vvec, keep);
    }
    copies_done();
  };
  for (int i = threadIdx.x; i < 16 * DP; i += kThreads) {
    const int r = r0 + i / DP, d = i % DP, at = r / group, h = hk * group + r % group;
    float x = 0.0f;
    if (r < rows && d < p.D) x = to_f32(static_cast<const T*>(p.q)[b * p.qs[0] + at * p.qs[1] + h * p.qs[2] + d]);
    qs[i / DP * S::kFloats + d] = x;
  }
  fill(first, 0);
  ScoreForm f[2];
  RowView row[2];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, out[DP / 8][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + g + 8 * i;
    row[i] = row_view(p, b, r < rows ? r / group : p.Sq, length);
    f[i] = score_form(p, r < rows ? hk * group + r % group : 0);
  }
#pragma unroll
  for (int d = 0; d < DP / 8; ++d) out[d][0] = out[d][1] = out[d][2] = out[d][3] = 0.0f;
  const auto column = [&](int, int e) { return warp * 8 + 2 * t + e; };
  int slot = 0;
  for (int j0 = first; j0 < last; j0 += kCols, slot ^= 1) {
    fill(j0 + kCols, slot ^ 1);
    copies_wait<1>();
    __syncthreads();
    const float* ks = ring + slot * 2 * S::kColTile + warp * 8 * S::kFloats;
    float s[1][4], old[2];
    scores<DP, 1, EXACT>(qs, ks, p.D, s);
    int kd[1][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = j0 + column(0, e);
      kd[0][e] = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
    }
    softmax_step<1>(p, f, row, s, kd, j0, last, false, column, m, l, old);
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) {
      out[d][0] *= old[0], out[d][1] *= old[0];
      out[d][2] *= old[1], out[d][3] *= old[1];
    }
    gather<DP, DP, 1, EXACT, true>(s, ks + S::kColTile, out);
    __syncthreads();
  }
  copies_wait<0>();
  __syncthreads();
  // The warps' parts, in the ring's place.
  float (*sum)[16][S::kFloats] = reinterpret_cast<float (*)[16][S::kFloats]>(ring);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] = sum4(l[i]);
    if (t == 0) part_ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) sum[warp][g + 8 * i][d * 8 + 2 * t + e] = out[d][2 * i + e];
  }
  __syncthreads();
  for (int r = warp; r < 16 && r0 + r < rows; r += 4) {
    float top = -INFINITY, total = 0.0f, w[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) top = fmaxf(top, part_ml[x][r].x);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      w[x] = exp2f(part_ml[x][r].x - base);
      total = fmaf(part_ml[x][r].y, w[x], total);
    }
    const int at = (r0 + r) / group, h = hk * group + (r0 + r) % group;
    const int64_t o = ((int64_t)b * p.H + h) * p.Sq + at, po = (int64_t)part * p.B * p.H * p.Sq + o;
    if (lane == 0) {
      if (p.splits > 1) p.part_ml[po] = make_float2(top, total);
      else if (p.lse) p.lse[o] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
    }
    for (int d = lane; d < p.D; d += 32) {
      float x = 0.0f;
#pragma unroll
      for (int y = 0; y < 4; ++y) x = fmaf(sum[y][r][d], w[y], x);
      if (p.splits > 1) p.part_o[po * p.D + d] = x;
      else put_output<T>(p, (((int64_t)b * p.Sq + at) * p.H + h) * p.D + d, x * inverse(total));
    }
  }
}

// Warp w of either group, which have the same 16 rows.
__device__ __forceinline__ void pair_sync(int w) { asm volatile("bar.sync %0, 64;" ::"r"(w + 1) : "memory"); }
__device__ __forceinline__ void pair_arrive(int w) { asm volatile("bar.arrive %0, 64;" ::"r"(w + 1) : "memory"); }

// z x, z being p (1 - tanh^2) >= 0 or, of a key that a row does not see, -0.
__device__ __forceinline__ float times_seen(float z, float x) { return __float_as_uint(z) == 0x80000000u ? 0.0f : z * x; }

// dq, and delta_i = g_i . o_i for the key gradient that follows. Each group of four
// warps has half of a step's keys; their sums are added at the end.
template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, DP <= 128 ? 2 : 1) attn_tf32_dq_kernel(const AttnParams p) {
  constexpr int COLS = DP <= 64 ? 2 * kCols : kCols, NT = COLS / 16, kTile = COLS * Pitch<DP>::kFloats;
  constexpr bool EXACT = sizeof(T) == 2;
  using S = Pitch<DP>;
  extern __shared__ __align__(16) float smem[];
  float *qs = smem, *gs = smem + S::kRowTile, *ring = smem + 2 * S::kRowTile;
  __shared__ float delta_s[kRows];
  const int side = threadIdx.x / 128, warp = threadIdx.x / 32 % 4, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, hk = h / (p.H / p.Hkv);
  const int i0 = (gridDim.y - 1 - blockIdx.y) * kRows;
  const int length = attn_length(p, b);
  const int limit = rows_limit(p, b, i0 + kRows, length);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  const bool kvec = can_vec<T>(p.k, p.ks, p.D), vvec = can_vec<T>(p.v, p.vs, p.D);
  const auto next = [&](int j) {
    while (j < limit && skip_tiles(p, b, i0, j)) j += COLS;
    return j;
  };
  const auto fill = [&](int j) {
    if (j < limit) {
      const auto keep = [&](int r) { return !key_padded(p, b, j + r, length); };
      load_rows<T, DP, kBwdThreads>(ring, COLS, k, p.ks[1], j, p.D, kvec, keep);
      load_rows<T, DP, kBwdThreads>(ring + kTile, COLS, v, p.vs[1], j, p.D, vvec, keep);
    }
    copies_done();
  };
  const auto in = [&](int r) { return row_view(p, b, i0 + r, length).limit > 0; };
  load_rows<T, DP, kBwdThreads>(qs, kRows, static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2], p.qs[1], i0, p.D,
                   can_vec<T>(p.q, p.qs, p.D), in);
  load_rows<T, DP, kBwdThreads>(gs, kRows, static_cast<const T*>(p.go) + b * p.gs[0] + h * p.gs[2], p.gs[1], i0, p.D,
                   can_vec<T>(p.go, p.gs, p.D), in);
  // delta from the outputs, which take the ring's 64 rows, by the arithmetic that
  // forms g . v: where a row sees one key the two cancel.
  for (int i = threadIdx.x; i < kRows * DP; i += kBwdThreads) {
    const int r = i / DP, d = i % DP;
    float o = 0.0f;
    if (d < p.D && in(r)) {
      const int64_t at = (((int64_t)b * p.Sq + i0 + r) * p.H + h) * p.D + d;
      o = to_f32(static_cast<const T*>(p.o)[at]);
      if (p.residue) o += to_f32(static_cast<const T*>(p.residue)[at]);
    }
    ring[r * S::kFloats + d] = o;
  }
  copies_done();
  copies_wait<0>();
  __syncthreads();
  if (side == 0) {
    float c[2][4];
    scores<DP, 2, false>(gs + warp * 16 * S::kFloats, ring + warp * 16 * S::kFloats, p.D, c);
    if (t == g / 2) {
      delta_s[warp * 16 + g] = g & 1 ? c[0][1] : c[0][0];
      delta_s[warp * 16 + g + 8] = g & 1 ? c[1][3] : c[1][2];
    }
  }
  __syncthreads();
  if (threadIdx.x < kRows && i0 + threadIdx.x < p.Sq)
    p.delta[((int64_t)b * p.H + h) * p.Sq + i0 + threadIdx.x] = delta_s[threadIdx.x];
  int j0 = next(0);
  fill(j0);
  copies_wait<0>();
  __syncthreads();
  const ScoreForm f = score_form(p, h);
  RowView row[2];
  float lse2[2], delta[2], dq[DP / 8][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = warp * 16 + g + 8 * i;
    row[i] = row_view(p, b, i0 + r, length);
    lse2[i] = i0 + r < p.Sq ? p.lse[((int64_t)b * p.H + h) * p.Sq + i0 + r] * kLog2e : 0.0f;
    delta[i] = delta_s[r];
  }
#pragma unroll
  for (int d = 0; d < DP / 8; ++d) dq[d][0] = dq[d][1] = dq[d][2] = dq[d][3] = 0.0f;
  while (j0 < limit) {
    const bool whole = !p.kdoc && __all_sync(kFullMask, j0 + COLS <= min(row[0].limit, row[1].limit));
    const float* ks = ring + side * (COLS / 2) * S::kFloats;
    float s[NT][4], dp[NT][4];
    scores<DP, NT, EXACT>(qs + warp * 16 * S::kFloats, ks, p.D, s);
    scores<DP, NT, EXACT>(gs + warp * 16 * S::kFloats, ks + kTile, p.D, dp);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + side * (COLS / 2) + n * 8 + 2 * t + e;
        const int kd = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool seen = whole || (j < row[i].limit && (!p.kdoc || same_document(row[i].doc, kd, p.shared)));
          float th;
          const float x = ex2(score2(p, f, s[n][2 * i + e], row[i].place - j, th) - lse2[i]);
          s[n][2 * i + e] = seen ? x * (dp[n][2 * i + e] - delta[i]) * fmaf(-th, th, 1.0f) : 0.0f;
        }
      }
    gather<DP, DP, NT, EXACT, false>(s, ks, dq);
    __syncthreads();
    j0 = next(j0 + COLS);
    fill(j0);
    copies_wait<0>();
    __syncthreads();
  }
  // The second group's sums go through the queries' place.
  if (side == 1) {
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float2*>(qs + (warp * 16 + g + 8 * i) * S::kFloats + d * 8 + 2 * t) = make_float2(dq[d][2 * i], dq[d][2 * i + 1]);
  }
  __syncthreads();
  if (side == 1) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i0 + warp * 16 + g + 8 * i;
    if (r >= p.Sq) continue;
    T* to = static_cast<T*>(p.dq) + (((int64_t)b * p.Sq + r) * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) {
      const float2 other = *reinterpret_cast<const float2*>(qs + (warp * 16 + g + 8 * i) * S::kFloats + d * 8 + 2 * t);
      const int c = d * 8 + 2 * t;
      if (c < p.D) to[c] = from_f32<T>((dq[d][2 * i] + other.x) * p.scale);
      if (c + 1 < p.D) to[c + 1] = from_f32<T>((dq[d][2 * i + 1] + other.y) * p.scale);
    }
  }
}

// dk and dv of 64 keys: every query of every head that shares them, in a fixed
// order. One group of four warps forms the probabilities and has dv, the other
// forms g . v and has dk: two products each, and 16 sums a thread and step handed
// over within a pair of warps.
template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, DP <= 128 ? 2 : 1) attn_tf32_dkv_kernel(const AttnParams p) {
  constexpr int NT = kCols / 8;
  constexpr bool EXACT = sizeof(T) == 2;
  using S = Pitch<DP>;
  extern __shared__ __align__(16) float smem[];
  float *ks = smem, *vs = smem + S::kRowTile, *qs = smem + 2 * S::kRowTile, *gs = qs + S::kColTile;
  float4* mid = reinterpret_cast<float4*>(gs + S::kColTile) + threadIdx.x % 128;  // a pair of warps' p (1 - tanh^2)
  __shared__ float lse_s[kCols], delta_s[kCols];
  __shared__ RowView view_s[kCols];
  const bool keys = threadIdx.x >= 128;  // this group has dk
  const int warp = threadIdx.x / 32 % 4, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int hk = blockIdx.x % p.Hkv, part = blockIdx.x / p.Hkv % p.kv_parts, b = blockIdx.x / (p.Hkv * p.kv_parts);
  const int group = p.H / p.Hkv / p.kv_parts, head0 = (hk * p.kv_parts + part) * group;  // this CTA's query heads
  const int j0 = blockIdx.y * kRows;
  const int length = attn_length(p, b);
  const auto keep = [&](int r) { return !key_padded(p, b, j0 + r, length); };
  load_rows<T, DP, kBwdThreads>(ks, kRows, static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2], p.ks[1], j0, p.D,
                   can_vec<T>(p.k, p.ks, p.D), keep);
  load_rows<T, DP, kBwdThreads>(vs, kRows, static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2], p.vs[1], j0, p.D,
                   can_vec<T>(p.v, p.vs, p.D), keep);
  float out[DP / 8][4];
  clear(out);
  int kd[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = j0 + warp * 16 + g + 8 * i;
    kd[i] = p.kdoc && j < length ? __ldg(p.kdoc + (int64_t)b * p.Sk + j) : 0;
  }
  const bool qvec = can_vec<T>(p.q, p.qs, p.D), gvec = can_vec<T>(p.go, p.gs, p.D);
  const int first = j0 < length ? first_query(p, b, j0, length) / kCols * kCols : p.Sq;
  for (int x = 0; x < group; ++x) {
    const int h = head0 + x;
    const ScoreForm f = score_form(p, h);
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
      // A query that sees no key counts for nothing, whatever its rows hold.
      const float* lse = p.lse + ((int64_t)b * p.H + h) * p.Sq + i0;
      const auto in = [&](int r) { return i0 + r < p.Sq && __ldg(lse + r) != -INFINITY; };
      load_rows<T, DP, kBwdThreads>(qs, kCols, static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2], p.qs[1], i0, p.D, qvec, in);
      load_rows<T, DP, kBwdThreads>(gs, kCols, static_cast<const T*>(p.go) + b * p.gs[0] + h * p.gs[2], p.gs[1], i0, p.D, gvec, in);
      copies_done();
      copies_wait<0>();
      __syncthreads();
      float s[NT][4];
      scores<DP, NT, EXACT>((keys ? vs : ks) + warp * 16 * S::kFloats, keys ? gs : qs, p.D, s);
      if (keys) {
        pair_sync(warp);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 z = mid[n * 128];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float delta = delta_s[n * 8 + 2 * t + e];
            s[n][e] = times_seen(e ? z.y : z.x, s[n][e] - delta);
            s[n][2 + e] = times_seen(e ? z.w : z.z, s[n][2 + e] - delta);
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float z[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = n * 8 + 2 * t + e;
            const RowView row = view_s[c];
            const float lse2 = lse_s[c];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int j = j0 + warp * 16 + g + 8 * i;
              const bool seen = j < row.limit && (!p.kdoc || same_document(row.doc, kd[i], p.shared));
              float th;
              const float y = ex2(score2(p, f, s[n][2 * i + e], row.place - j, th) - lse2);
              s[n][2 * i + e] = seen ? y : 0.0f;
              z[2 * i + e] = seen ? y * fmaf(-th, th, 1.0f) : -0.0f;
            }
          }
          mid[n * 128] = make_float4(z[0], z[1], z[2], z[3]);
        }
        pair_arrive(warp);
      }
      gather<DP, DP, NT, EXACT, false>(s, keys ? qs : gs, out);
    }
  }
  T* to = static_cast<T*>(keys ? p.dk : p.dv);
  float* sums = p.kv_parts > 1 ? kv_part(p, part, keys) : nullptr;
  const float mul = keys ? p.scale : 1.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = j0 + warp * 16 + g + 8 * i;
    if (j >= p.Sk) continue;
    const int64_t at = (((int64_t)b * p.Sk + j) * p.Hkv + hk) * p.D;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = d * 8 + 2 * t + e;
        if (c >= p.D) continue;
        if (p.kv_parts > 1) sums[at + c] = out[d][2 * i + e] * mul;
        else to[at + c] = from_f32<T>(out[d][2 * i + e] * mul);
      }
  }
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

template <typename K>
cudaError_t launch(K kernel, dim3 grid, int threads, int floats, std::atomic<uint64_t>& set, const AttnParams& p, cudaStream_t st) {
  cudaError_t e = abi::allow_smem(kernel, floats * 4, set);
  if (e != cudaSuccess) return e;
  kernel<<<grid, threads, floats * 4, st>>>(p);
  return cudaGetLastError();
}

unsigned row_tiles(int n) { return (unsigned)((n + kRows - 1) / kRows); }

template <typename T, int DP>
cudaError_t forward(const AttnParams& p, bool token, cudaStream_t st) {
  using S = Pitch<DP>;
  static std::atomic<uint64_t> set[2];
  if (token) {
    const int rows = p.Sq * (p.H / p.Hkv);
    return launch(attn_tf32_token_kernel<T, DP>, dim3(p.Hkv * ((rows + 15) / 16), p.splits, p.B), kThreads,
                  16 * S::kFloats + 4 * S::kColTile, set[0], p, st);
  }
  return launch(attn_tf32_fwd_kernel<T, DP>, dim3(p.H * p.B, row_tiles(p.Sq)), kThreads * forward_groups<DP>(),
                S::kRowTile + 2 * forward_slots<DP>() * forward_groups<DP>() * S::kColTile, set[1], p, st);
}

template <typename T, int DP>
cudaError_t backward(const AttnParams& p, cudaStream_t st) {
  using S = Pitch<DP>;
  static std::atomic<uint64_t> set[2];
  constexpr int floats = 2 * S::kRowTile + 2 * S::kColTile, wide = DP <= 64 ? floats + 2 * S::kColTile : floats;
  cudaError_t e = launch(attn_tf32_dq_kernel<T, DP>, dim3(p.H * p.B, row_tiles(p.Sq)), kBwdThreads, wide, set[0], p, st);
  if (e == cudaSuccess)
    e = launch(attn_tf32_dkv_kernel<T, DP>, dim3(p.Hkv * p.kv_parts * p.B, row_tiles(p.Sk)), kBwdThreads, floats + 128 * kCols / 2, set[1], p, st);
  return e;
}

template <typename T>
cudaError_t forward_by_size(const AttnParams& p, bool token, cudaStream_t st) {
  if (p.D <= 32) return forward<T, 32>(p, token, st);
  if (p.D <= 64) return forward<T, 64>(p, token, st);
  if (p.D <= 128) return forward<T, 128>(p, token, st);
  return forward<T, 256>(p, token, st);
}

template <typename T>
cudaError_t backward_by_size(const AttnParams& p, cudaStream_t st) {
  if (p.D <= 32) return backward<T, 32>(p, st);
  if (p.D <= 64) return backward<T, 64>(p, st);
  if (p.D <= 128) return backward<T, 128>(p, st);
  return backward<T, 256>(p, st);
}

}  // namespace

cudaError_t attn_tf32_forward(const AttnParams& p, int dtype, bool token, cudaStream_t st) {
  if (dtype == MSDA_DTYPE_F32) return forward_by_size<float>(p, token, st);
  return dtype == MSDA_DTYPE_F16 ? forward_by_size<__half>(p, token, st) : forward_by_size<__nv_bfloat16>(p, token, st);
}

cudaError_t attn_tf32_backward(const AttnParams& p, int dtype, cudaStream_t st) {
  if (dtype == MSDA_DTYPE_F32) return backward_by_size<float>(p, st);
  return dtype == MSDA_DTYPE_F16 ? backward_by_size<__half>(p, st) : backward_by_size<__nv_bfloat16>(p, st);
}

cudaError_t attn_documents_launch(const AttnParams& p, DocTile* qtile, DocTile* ktile, cudaStream_t st) {
  const int64_t tiles = (int64_t)p.B * ((p.Sq + kDocTile - 1) / kDocTile + (p.Sk + kDocTile - 1) / kDocTile);
  attn_documents_kernel<<<(unsigned)((tiles + 3) / 4), 128, 0, st>>>(p, qtile, ktile);
  return cudaGetLastError();
}

}  // namespace msda
