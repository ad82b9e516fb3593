// The tcgen05 kernel over the 8-bit cache (quantized_umma.cuh) for f16 queries.

#include "quantized_umma.cuh"

namespace nvj {

int launch_quantized_umma_f16(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int head_dim,
                               int ranges, cudaStream_t stream) {
  return launch_quantized_umma_shape<__half>(k_map, v_map, a, p, head_dim, ranges, stream);
}

}  // namespace nvj
