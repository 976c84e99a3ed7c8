// C ABI of masked attention (declared in include/msda_layer_b200.h): argument
// checks, the choice of kernel and the workspace's layout.
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "layer_attention.cuh"

namespace msda {
namespace tc {

int run_f16(const AttnParams& p, bool backward, cudaStream_t st);
int run_bf16(const AttnParams& p, bool backward, cudaStream_t st);
cudaError_t gave_up_f16(int* count);
cudaError_t gave_up_bf16(int* count);

// The map of a (B, S, H, D) tensor by boxes of 64 channels x 1 head x 128 tokens
// in 128-byte swizzled rows; what lies outside comes as zeros.
bool make_map(CUtensorMap* map, const void* base, bool bf16, int64_t D, int64_t H, int64_t S, int64_t B,
              const int64_t (&strides)[3]) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode) return false;
  const cuuint64_t size[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)S, (cuuint64_t)B};
  const int64_t from[3] = {strides[2], strides[1], strides[0]};
  cuuint64_t stride[3];
  // A dimension of one element may have any stride; 16 bytes stand for it.
  for (int i = 0; i < 3; ++i) stride[i] = size[i + 1] > 1 ? (cuuint64_t)from[i] * 2 : 16;
  const cuuint32_t box[4] = {64, 1, 128, 1}, step[4] = {1, 1, 1, 1};
  const auto run = [&] {
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), size,
                  stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = run();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
    // A thread that has not used its device so far (autograd's, when the memory comes
    // from a cache) has no context: the runtime would bind it at its first launch.
    int device;
    if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return false;
    r = run();
  }
  return r == CUDA_SUCCESS;
}

}  // namespace tc

int attn_tc_forward(const AttnParams& p, int dtype, cudaStream_t st) {
  return dtype == MSDA_DTYPE_F16 ? tc::run_f16(p, false, st) : tc::run_bf16(p, false, st);
}

int attn_tc_backward(const AttnParams& p, int dtype, cudaStream_t st) {
  return dtype == MSDA_DTYPE_F16 ? tc::run_f16(p, true, st) : tc::run_bf16(p, true, st);
}

cudaError_t attn_tc_gave_up(int* count) {
  int a = 0, b = 0;
  cudaError_t e = tc::gave_up_f16(&a);
  if (e == cudaSuccess) e = tc::gave_up_bf16(&b);
  *count = a + b;
  return e;
}

}  // namespace msda

namespace {

using namespace msda;
using namespace msda::abi;

constexpr int kMaxSplits = 64;
constexpr int kMaxRows = 1 << 22;  // queries, and keys that have a gradient

enum class Path { kAny, kToken, kTensor };

// 16-byte loads of 8 channels: the tensor-core kernels' layout.
bool rows_of_16(const void* p, const int64_t (&s)[3], const int64_t (&n)[3]) {
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8)) return false;
  return aligned(p, 16);
}

bool tensor_layout(const msda_attention_args* a, bool backward) {
  if (a->dtype == MSDA_DTYPE_F32 || a->head_dim % 8 || a->head_dim > 128) return false;
  const int64_t nq[3] = {a->batch, a->num_queries, a->num_heads}, nk[3] = {a->batch, a->num_keys, a->num_key_heads};
  return rows_of_16(a->query, a->query_strides, nq) && rows_of_16(a->key, a->key_strides, nk) &&
         rows_of_16(a->value, a->value_strides, nk) && aligned(a->out, 16) && aligned(a->out_residue, 16) &&
         (!backward || (rows_of_16(a->grad_out, a->grad_out_strides, nq) && aligned(a->grad_query, 16) &&
                        aligned(a->grad_key, 16) && aligned(a->grad_value, 16)));
}

// Refusals by type and sizes, which the workspace's size goes by too.
int check_sizes(const char* fn, const msda_attention_args* a, bool backward) {
  if (!a) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null arguments", fn);
  if (elem_size(a->dtype) == 0) return fail(MSDA_ERR_UNSUPPORTED, "%s: unsupported dtype code %d (0=f32, 1=f16, 2=bf16)", fn, a->dtype);
  if (a->batch < 0 || a->num_queries < 0 || a->num_keys < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (a->num_heads < 1 || a->num_key_heads < 1 || a->num_heads % a->num_key_heads)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: num_heads=%d must be a multiple of num_key_heads=%d", fn, a->num_heads, a->num_key_heads);
  if (a->head_dim < 1 || a->head_dim > MSDA_ATTENTION_MAX_HEAD_DIM)
    return fail(MSDA_ERR_UNSUPPORTED, "%s: head_dim=%d outside [1, %d]", fn, a->head_dim, MSDA_ATTENTION_MAX_HEAD_DIM);
  if (a->batch > 65535 || a->num_heads > 4096 || a->num_queries > kMaxRows || a->num_keys > (backward ? kMaxRows : 1 << 30))
    return fail(MSDA_ERR_UNSUPPORTED, "%s: sizes exceed batch 65535, 4096 heads, 2^22 queries or 2^30 keys (2^22 in the backward)", fn);
  // The other kernels' grids have a tile of 64 rows for each of y's 65535 steps.
  if (!tensor_layout(a, backward) && (a->num_queries > 65535 * 64 || (backward && a->num_keys > 65535 * 64)))
    return fail(MSDA_ERR_UNSUPPORTED, "%s: more than %d rows of fp32, or of a layout without 16-byte rows of up to 128 channels", fn,
                65535 * 64);
  return MSDA_OK;
}

int check(const char* fn, const msda_attention_args* a, bool backward) {
  if (int rc = check_sizes(fn, a, backward)) return rc;
  if (!std::isfinite(a->scale) || !std::isfinite(a->softcap) || a->softcap < 0)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: scale must be finite, softcap finite and >= 0", fn);
  // Beyond, the cap to base 2 or its inverse leaves 32 bits.
  if (a->softcap != 0 && (a->softcap < 0x1p-100f || a->softcap > 0x1p100f || !std::isfinite(a->scale / a->softcap)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: softcap=%g outside [2^-100, 2^100], or scale / softcap not finite", fn, (double)a->softcap);
  if (!a->query_documents != !a->key_documents)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: documents of queries and keys come together", fn);
  if (a->prefix_lengths && !a->causal) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: prefix_lengths needs causal", fn);
  if (a->batch == 0) return MSDA_OK;
  const int es = elem_size(a->dtype);
  if (a->num_queries > 0 && (!a->query || !a->out)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (a->num_keys > 0 && (!a->key || !a->value)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  const void* data[] = {a->query, a->key, a->value, a->out, a->out_residue, a->grad_out, a->grad_query, a->grad_key, a->grad_value};
  for (const void* p : data)
    if (!aligned(p, es)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  const void* words[] = {a->lse, a->distance_slopes, a->query_documents, a->key_documents, a->prefix_lengths, a->key_lengths};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: misaligned buffer", fn);
  if (backward) {
    if (a->num_queries > 0 && (!a->lse || !a->grad_out || !a->grad_query))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
    if (a->num_keys > 0 && (!a->grad_key || !a->grad_value)) return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  }
  return MSDA_OK;
}

struct Plan {
  Path path = Path::kAny;
  bool few = false;  // few query rows
  int splits = 1;
  int64_t q_tiles = 0, k_tiles = 0;  // document summary entries
  int kv_parts = 1;
  size_t delta = 0, part_ml = 0, part_o = 0, part_kv = 0, bytes = 0;  // byte offsets, after the summary; total
};

// Whether the few-rows kernels, whose CTAs split the keys of 16 query rows (queries
// x heads that share a key head), are the faster ones. Both walk over the same keys,
// so their times compare by tiles of 16 rows against waves of the other kernel's
// CTAs. Measured over 8192 keys, few-rows / other kernel: 1 x 8 heads of 64 16-bit
// channels 128 rows 59 / 139 us, 512 rows 139 / 133 us; 8 x 32 heads on 8 of 128
// channels 64 rows 262 / 283 us, 128 rows 432 / 285 us; fp32, 1 x 8 heads of 64
// channels 512 rows 454 / 718 us; 8 x 32 on 8 of 128 channels 128 rows 1719 / 2637
// us, 256 rows 3368 / 2638 us. Over few keys in one wave the start counts: 10 / 7 us
// over 100 keys of 128 channels, 3.7 / 4.8 us over 10 of 32. (Over 300 random
// calls the rule's choice takes 1.5% more time than the better one.) Documents, of
// which the other kernels skip tiles, leave the single tokens' 64 rows.
bool few_rows_faster(const msda_attention_args* a, bool tensor) {
  const int64_t rows = a->num_queries * (a->num_heads / a->num_key_heads), heads = a->batch * a->num_heads;
  const int64_t tiles = a->batch * a->num_key_heads * ((rows + 15) / 16);
  if (a->query_documents && rows > 64) return false;
  if (!tensor) return tiles <= std::max<int64_t>(300, 2 * heads * ((a->num_queries + 63) / 64));
  const bool narrow = a->head_dim <= 64;
  const int64_t room = sm_count() * (narrow ? 2 : 1), waves = (heads * ((a->num_queries + 255) / 256) + room - 1) / room;
  if (waves == 1 && a->num_keys < (narrow ? 256 : 512)) return narrow && rows <= 16;
  return narrow ? tiles + 90 <= 350 * waves : tiles + 100 <= 215 * waves;
}

// Parts of the query heads that share a key head, each on CTAs of its own in the key
// gradient: as many as divide them evenly and leave at most two waves of CTAs. The
// parts' fp32 sums are joined by a kernel of their own. Together, causal, in one part
// / so: 1 x 4096 tokens, 8 bf16 heads of 64 channels on one key head 639 / 98 us; 16
// heads of 128 on 4 key heads 236 / 143 us (without a mask, where one part fills the
// GPU evenly, 258 / 269 us); fp32, 1 x 1500, 8 heads of 64 on 2 812 / 229 us.
int kv_parts_of(const msda_attention_args* a, bool tensor) {
  const int64_t group = a->num_heads / a->num_key_heads, rows = tensor ? 128 : 64;
  const int64_t room = sm_count() * ((tensor ? a->head_dim <= 64 : a->head_dim <= 128) ? 2 : 1);
  const int64_t ctas = a->batch * a->num_key_heads * ((a->num_keys + rows - 1) / rows);
  int64_t n = ctas > 0 ? std::min(group, 2 * room / ctas) : 1;
  while (n > 1 && group % n) --n;
  return n < 1 ? 1 : (int)n;
}

Plan plan_of(const msda_attention_args* a, bool backward) {
  Plan p;
  const int64_t group = a->num_heads / a->num_key_heads, rows = a->num_queries * group;
  const bool tensor = tensor_layout(a, backward);
  if (tensor && a->num_keys > 0) p.path = Path::kTensor;
  p.few = !backward && few_rows_faster(a, tensor);
  if (p.few) {
    if (tensor) p.path = Path::kToken;
    // Parts of at least 2048 keys (512 for the slower kernel of 32 bits), up to 16
    // CTAs an SM, so that streams of different lengths even out; of at least 128
    // keys where that leaves fewer than 2 CTAs an SM. With at least 512 and 2048
    // keys, 32 heads on 8 of 128 16-bit channels: 4 streams of 4096 to 16384 keys 69
    // and 44 us, 8 of up to 8192 58 and 46 us, 32 of 16384 377 and 366 us; fp32, 16
    // of up to 8192 on 8 heads of 64 channels 129 and 184 us. (At 32 and 64 16-bit
    // channels, where 2048 keys are a quarter and half of the bytes, not measured.)
    const int64_t tiles = (rows + 15) / 16;
    const int64_t ctas = std::max<int64_t>(1, a->batch * a->num_key_heads * tiles);
    const int64_t even = std::min<int64_t>(16 * sm_count() / ctas, a->num_keys / (tensor ? 2048 : 512));
    const int64_t fill = std::min<int64_t>(2 * sm_count() / ctas, (a->num_keys + 127) / 128);
    const int64_t s = std::min<int64_t>(std::max(even, fill), kMaxSplits);
    p.splits = s < 1 ? 1 : (int)s;
  }
  size_t at = 0;
  const bool documents = a->query_documents && !p.few;
  if (documents) {
    p.q_tiles = a->batch * ((a->num_queries + kDocTile - 1) / kDocTile);
    p.k_tiles = a->batch * ((a->num_keys + kDocTile - 1) / kDocTile);
    at = align256((p.q_tiles + p.k_tiles) * sizeof(DocTile));
  }
  const size_t all = (size_t)a->batch * a->num_heads * a->num_queries;
  if (backward) {
    p.delta = at;
    at += align256(all * 4);
    p.kv_parts = kv_parts_of(a, tensor);
    if (p.kv_parts > 1) {
      p.part_kv = at;
      at += align256((size_t)p.kv_parts * 2 * a->batch * a->num_keys * a->num_key_heads * a->head_dim * 4);
    }
  }
  if (p.splits > 1) {
    p.part_ml = at;
    at += align256(all * p.splits * 8);
    p.part_o = at;
    at += align256(all * p.splits * a->head_dim * 4);
  }
  p.bytes = at;
  return p;
}

void copy3(int64_t (&to)[3], const int64_t (&from)[3]) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

AttnParams params_of(const msda_attention_args* a, const Plan& plan) {
  AttnParams p = {};
  p.q = a->query, p.k = a->key, p.v = a->value, p.go = a->grad_out;
  p.o = a->out, p.residue = a->dtype == MSDA_DTYPE_F32 ? nullptr : a->out_residue, p.dq = a->grad_query, p.dk = a->grad_key, p.dv = a->grad_value;
  p.lse = a->lse;
  copy3(p.qs, a->query_strides);
  copy3(p.ks, a->key_strides);
  copy3(p.vs, a->value_strides);
  copy3(p.gs, a->grad_out_strides);
  p.slopes = a->distance_slopes;
  p.qdoc = a->query_documents, p.kdoc = a->key_documents;
  p.prefix = a->prefix_lengths, p.klen = a->key_lengths;
  p.B = (int)a->batch, p.Sq = (int)a->num_queries, p.Sk = (int)a->num_keys;
  p.H = a->num_heads, p.Hkv = a->num_key_heads, p.D = a->head_dim;
  p.scale = a->scale, p.cap = a->softcap;
  p.shared = a->shared_document < 0 ? -1 : a->shared_document;
  p.causal = a->causal != 0;
  p.splits = plan.splits;
  char* ws = static_cast<char*>(a->workspace);
  if (plan.q_tiles + plan.k_tiles > 0) {
    p.qtile = reinterpret_cast<DocTile*>(ws);
    p.ktile = p.qtile + plan.q_tiles;
  }
  p.delta = reinterpret_cast<float*>(ws + plan.delta);
  p.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
  p.kv_parts = plan.kv_parts;
  p.part_kv = reinterpret_cast<float*>(ws + plan.part_kv);
  return p;
}

int check_workspace(const char* fn, const msda_attention_args* a, const Plan& plan) {
  if (plan.bytes && (!a->workspace || a->workspace_bytes < plan.bytes || !aligned(a->workspace, 16)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes (16-byte aligned), needs %zu", fn,
                a->workspace ? a->workspace_bytes : 0, plan.bytes);
  return MSDA_OK;
}

cudaError_t documents(const AttnParams& p, const Plan& plan, cudaStream_t st) {
  if (plan.q_tiles + plan.k_tiles == 0) return cudaSuccess;
  return attn_documents_launch(p, const_cast<DocTile*>(p.qtile), const_cast<DocTile*>(p.ktile), st);
}

}  // namespace

extern "C" {

size_t msda_attention_workspace_size(const msda_attention_args* a, int32_t backward) {
  if (check_sizes("msda_attention_workspace_size", a, backward != 0) || a->batch == 0 || a->num_queries == 0) return 0;
  return plan_of(a, backward != 0).bytes;
}

int msda_attention_forward(const msda_attention_args* a, void* stream) {
  const char* fn = "msda_attention_forward";
  if (int rc = check(fn, a, false)) return rc;
  if (a->batch == 0 || a->num_queries == 0) return succeed();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Plan plan = plan_of(a, false);
  if (int rc = check_workspace(fn, a, plan)) return rc;
  const AttnParams p = params_of(a, plan);
  cudaError_t e = documents(p, plan, st);
  if (e == cudaSuccess && plan.path == Path::kTensor) {
    const int rc = attn_tc_forward(p, a->dtype, st);
    if (rc < 0) return fail(MSDA_ERR_CUDA, "%s: no tensor map for these sizes and strides", fn);
    e = (cudaError_t)rc;
  } else if (e == cudaSuccess) {
    e = plan.path == Path::kToken ? attn_token_forward(p, a->dtype, st) : attn_tf32_forward(p, a->dtype, plan.few, st);
  }
  if (e == cudaSuccess && plan.splits > 1) e = attn_combine_launch(p, a->dtype, st);
  if (e != cudaSuccess) return cuda_fail(e, "attention launch");
  return succeed();
}

int msda_attention_gave_up(int32_t* count) {
  if (!count) return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_attention_gave_up: null pointer argument");
  int n = 0;
  const cudaError_t e = attn_tc_gave_up(&n);
  if (e != cudaSuccess) return cuda_fail(e, "attention status");
  *count = n;
  return succeed();
}

int msda_attention_backward(const msda_attention_args* a, void* stream) {
  const char* fn = "msda_attention_backward";
  if (int rc = check(fn, a, true)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->batch == 0) return succeed();
  if (a->num_queries == 0 || a->num_keys == 0) {
    const size_t row = (size_t)a->batch * a->head_dim * elem_size(a->dtype);
    cudaError_t e = cudaSuccess;
    if (a->num_queries > 0) e = cudaMemsetAsync(a->grad_query, 0, row * a->num_queries * a->num_heads, st);
    if (e == cudaSuccess && a->num_keys > 0) e = cudaMemsetAsync(a->grad_key, 0, row * a->num_keys * a->num_key_heads, st);
    if (e == cudaSuccess && a->num_keys > 0) e = cudaMemsetAsync(a->grad_value, 0, row * a->num_keys * a->num_key_heads, st);
    if (e != cudaSuccess) return cuda_fail(e, "attention zero-fill");
    return succeed();
  }
  const Plan plan = plan_of(a, true);
  if (int rc = check_workspace(fn, a, plan)) return rc;
  const AttnParams p = params_of(a, plan);
  cudaError_t e = documents(p, plan, st);
  if (e == cudaSuccess && plan.path == Path::kTensor) {
    const int rc = attn_tc_backward(p, a->dtype, st);
    if (rc < 0) return fail(MSDA_ERR_CUDA, "%s: no tensor map for these sizes and strides", fn);
    e = (cudaError_t)rc;
  } else if (e == cudaSuccess) {
    e = attn_tf32_backward(p, a->dtype, st);
  }
  if (e == cudaSuccess && plan.kv_parts > 1) e = attn_kv_sum_launch(p, a->dtype, st);
  if (e != cudaSuccess) return cuda_fail(e, "attention backward launch");
  return succeed();
}

}  // extern "C"
