// The tensor-core attention kernels for bf16.
#include "layer_attention_tc.cuh"

namespace msda {
namespace tc {

int run_bf16(const AttnParams& p, bool backward, cudaStream_t st) { return run<__nv_bfloat16>(p, backward, st); }

cudaError_t gave_up_bf16(int* count) { return cudaMemcpyFromSymbol(count, g_gave_up, sizeof(int)); }

}  // namespace tc
}  // namespace msda
