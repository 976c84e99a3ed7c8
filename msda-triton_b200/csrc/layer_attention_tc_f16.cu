// The tensor-core attention kernels for fp16.
#include "layer_attention_tc.cuh"

namespace msda {
namespace tc {

int run_f16(const AttnParams& p, bool backward, cudaStream_t st) { return run<__half>(p, backward, st); }

cudaError_t gave_up_f16(int* count) { return cudaMemcpyFromSymbol(count, g_gave_up, sizeof(int)); }

}  // namespace tc
}  // namespace msda
