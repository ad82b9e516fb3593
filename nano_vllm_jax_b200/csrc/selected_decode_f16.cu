// Decode attention over selected blocks: the tensor-core form for f16 caches (selected_decode.cuh).

#include "selected_decode.cuh"

namespace nvj {

int launch_selected_f16(const SelectedParams& p, cudaStream_t stream) { return launch_selected_dims<__half>(p, p.q_dtype == NVJ_F16, stream); }

}  // namespace nvj
