// Building blocks of the tensor-core attention kernels: mbarriers with bounded
// waits, TMA tile loads, tcgen05 descriptors, products and TMEM access.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace msda {
namespace tc {

constexpr int kChunk = 64;              // 16-bit channels of a 128-byte shared-memory row
constexpr int kTileTokens = 128;        // tokens of a tile
constexpr int kChunkBytes = kTileTokens * 128;  // one chunk of a tile

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// One lane of a whole warp, always the same: it issues the products and their
// commits. (With a test of the lane number instead, the compiler does not know
// that a single thread runs, and a product cost about 100 cycles to issue.)
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(pred));
  return pred != 0;
}

// --- mbarriers -------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

// Waits of this translation unit's kernels that gave up since the library was loaded.
static __device__ int g_gave_up;

// Waits for the phase of this parity to end; after kWaitTries tries (each of
// which the hardware suspends for up to about a microsecond) or when another
// role has given up, sets *abort and returns false.
constexpr int kWaitTries = 1 << 22;
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  for (int i = 0; i < kWaitTries; ++i) {
    if (bar_try(bar, parity)) return true;
    if ((i & 255) == 255 && *abort) return false;
  }
  *abort = 1;
  atomicAdd(&g_gave_up, 1);
  return false;
}

// The same answer for all of a warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, abort));
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// --- TMA ---------------------------------------------------------------------
// A box of 64 channels x 1 head x 128 tokens x 1 item of a (B, S, H, D) tensor.
__device__ __forceinline__ void tma_box(void* dst, const CUtensorMap* map, uint64_t* bar, int channel, int head, int token,
                                        int item) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(channel), "r"(head), "r"(token), "r"(item), "r"(smem_u32(bar))
      : "memory");
}

// All the chunks of a tile of DP channels.
template <int DP>
__device__ __forceinline__ void tma_tile(char* dst, const CUtensorMap* map, uint64_t* bar, int head, int token, int item) {
#pragma unroll
  for (int c = 0; c < (DP + kChunk - 1) / kChunk; ++c)
    tma_box(dst + c * kChunkBytes, map, bar, c * kChunk, head, token, item);
}

template <int DP>
__host__ __device__ constexpr int tile_bytes() {
  return (DP + kChunk - 1) / kChunk * kChunkBytes;
}

// --- tcgen05 -----------------------------------------------------------------
// Shared-memory operand descriptors of tiles in 128-byte swizzled rows (one
// token a row, 8 rows an atom of 1024 bytes). `lead` is the distance between
// 64-channel chunks where the channels are the product's outer dimension.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}

// A tile as an operand whose contracted dimension is its channels, or its tokens.
__device__ __forceinline__ uint64_t by_channels(uint32_t tile) { return smem_desc(tile, 16); }
__device__ __forceinline__ uint64_t by_tokens(uint32_t tile) { return smem_desc(tile, kChunkBytes); }

// What 16 channels, or 16 tokens, further on adds to the descriptor.
constexpr uint64_t kTokenStep = 16 * 128 >> 4;
__host__ __device__ constexpr uint64_t channel_offset(int k) { return (uint64_t)((k / 4) * kChunkBytes + (k % 4) * 32) >> 4; }

// 128 x N product of 16-bit inputs with fp32 sums; outer_b: B's tokens are the
// contracted dimension.
template <bool BF16>
__host__ __device__ constexpr uint32_t instr_desc(int n, bool tokens_b) {
  return 1u << 4 | (BF16 ? 1u : 0u) << 7 | (BF16 ? 1u : 0u) << 10 | (tokens_b ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 |
         (128u >> 4) << 24;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

// d = a . b^T over DP channels of two tiles (by_channels).
template <int DP>
__device__ __forceinline__ void product_channels(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) mma_ss(d, a + channel_offset(k), b + channel_offset(k), idesc, k > 0);
}

// d (128 x DP) += p . t over 64 tokens of a tile (by_tokens): p 16-bit in TMEM.
__device__ __forceinline__ void product_half(uint32_t d, uint32_t p, uint64_t t, uint32_t idesc, bool add) {
#pragma unroll
  for (int k = 0; k < 4; ++k) mma_ts(d, p + k * 8, t + k * kTokenStep, idesc, add || k > 0);
}

// The same over N tokens, p in two parts: the first half of the tokens from
// column p, the others from column p + N / 2.
template <int N>
__device__ __forceinline__ void product_parts(uint32_t d, uint32_t p, uint64_t t, uint32_t idesc, bool add) {
#pragma unroll
  for (int k = 0; k < N / 16; ++k)
    mma_ts(d, p + (k < N / 32 ? k * 8 : N / 2 + (k - N / 32) * 8), t + k * kTokenStep, idesc, add || k > 0);
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS) : "memory");
}

// 32 columns of the warp's 32 lanes: a row a thread.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr) : "memory");
}

// The same for 8 columns.
__device__ __forceinline__ void tmem_load8(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

}  // namespace tc
}  // namespace msda
