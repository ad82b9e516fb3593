// The prefill kernel over the 8-bit cache (quantized_prefill_umma.cuh) for bfloat16 queries.

#include "quantized_prefill_umma.cuh"

namespace nvj {

int launch_quantized_prefill_bf16(const QtParams& p, int head_dim, int tiles, int most_tiles, cudaStream_t stream) {
  return launch_quantized_prefill_type<__nv_bfloat16>(p, head_dim, tiles, most_tiles, stream);
}

}  // namespace nvj
