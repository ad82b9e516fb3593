// Selection of blocks: tensor-core tiles over bf16 bounds (block_select.cuh); queries of another type as two terms.

#include "block_select.cuh"

namespace nvj {

int launch_block_select_bf16(const SelectParams& p, cudaStream_t stream) {
  return p.q_dtype == NVJ_BF16 ? launch_block_select_dims<__nv_bfloat16, 1>(p, stream) : launch_block_select_dims<__nv_bfloat16, 2>(p, stream);
}

}  // namespace nvj
