// The prefill kernel over the 8-bit cache (quantized_prefill_umma.cuh) for float32 queries.

#include "quantized_prefill_umma.cuh"

namespace nvj {

int launch_quantized_prefill_f32(const QtParams& p, int head_dim, int tiles, int most_tiles, cudaStream_t stream) {
  return launch_quantized_prefill_type<float>(p, head_dim, tiles, most_tiles, stream);
}

}  // namespace nvj
