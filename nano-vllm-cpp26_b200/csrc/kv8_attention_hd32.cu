// The mma.sync attention over the 8-bit paged cache at head_dim 32 (a file each, so
// that they compile side by side).
#include "kv8_attention.cuh"

namespace nvllm {

template cudaError_t launch_kv8_rows<32>(const Kv8AttnParams&, const Kv8Work&, bool, int32_t,
                                          cudaStream_t);

}  // namespace nvllm
