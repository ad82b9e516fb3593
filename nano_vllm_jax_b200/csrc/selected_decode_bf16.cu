// Decode attention over selected blocks: the tensor-core form for bf16 caches (selected_decode.cuh).

#include "selected_decode.cuh"

namespace nvj {

int launch_selected_bf16(const SelectedParams& p, cudaStream_t stream) { return launch_selected_dims<__nv_bfloat16>(p, p.q_dtype == NVJ_BF16, stream); }

}  // namespace nvj
