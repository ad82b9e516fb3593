// Selection of blocks: tensor-core tiles over f16 bounds, f16 queries (block_select.cuh).

#include "block_select.cuh"

namespace nvj {

int launch_block_select_f16(const SelectParams& p, cudaStream_t stream) { return launch_block_select_dims<__half, 1>(p, stream); }

}  // namespace nvj
