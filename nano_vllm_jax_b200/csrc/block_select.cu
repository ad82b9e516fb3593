// Selection of the blocks of a row that its attention is to read (block_select.cuh): the form on the CUDA cores, and the C entry.

#include "block_select.cuh"

namespace nvj {

template <typename C>
static int launch_block_select_lanes(const SelectParams& p, cudaStream_t stream) {
  return p.d > 128 ? launch_block_select<C, 0, 2, 1>(p, stream) : launch_block_select<C, 0, 1, 1>(p, stream);
}

}  // namespace nvj

extern "C" int nvj_select_blocks(const void* q, int q_dtype, const void* k_bounds, int cache_dtype, int64_t num_blocks, int block_size,
                                 int num_kv_heads, int head_dim, int num_q_heads, const int32_t* block_tables, int table_width,
                                 const int32_t* seq_lens, const int32_t* positions, int rows, int width, int budget, int first, int last,
                                 int32_t* selected, int32_t* status, nvj_stream_t stream) {
  using namespace nvj;
  if (rows < 0 || width < 0 || table_width < 0 || num_blocks < 0 || block_size < 1 || num_kv_heads < 1 || num_q_heads < 1 ||
      num_q_heads % num_kv_heads != 0 || budget < 1 || first < 0 || last < 0 || (long long)first + last > budget)
    return NVJ_ERR_INVALID_ARGUMENT;
  if (q_dtype < NVJ_BF16 || q_dtype > NVJ_F32 || cache_dtype < NVJ_BF16 || cache_dtype > NVJ_F32 || head_dim < 8 || head_dim > 256 ||
      head_dim % 8 != 0 || num_kv_heads > 1024 || block_size > 65536)
    return NVJ_ERR_UNSUPPORTED;
  if ((long long)rows * width == 0) return NVJ_OK;
  if (table_width > kBsMostColumns || (long long)table_width * block_size > 0x7fffffffLL || (long long)rows * width > 0x7fffffffLL / 8)
    return NVJ_ERR_TOO_LARGE;
  if (!q || !k_bounds || !seq_lens || !selected || !status || (table_width > 0 && !block_tables)) return NVJ_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k_bounds)) return NVJ_ERR_INVALID_ARGUMENT;
  SelectParams p{};
  p.q = q;
  p.bounds = k_bounds;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.positions = positions;
  p.out = selected;
  p.status = status;
  p.num_blocks = num_blocks;
  p.q_dtype = q_dtype;
  p.cache_dtype = cache_dtype;
  p.rows = rows;
  p.width = width;
  p.table_width = table_width;
  p.block_size = block_size;
  p.hkv = num_kv_heads;
  p.groups = num_q_heads / num_kv_heads;
  p.d = head_dim;
  p.budget = budget;
  p.first = first;
  p.last = last;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // tensor-core tiles where bounds and queries are exact in terms of the cache's type: all queries over bf16 bounds, f16 ones over f16
  if (p.groups <= 16 && num_blocks > 0) {
    if (cache_dtype == NVJ_BF16) return launch_block_select_bf16(p, s);
    if (cache_dtype == NVJ_F16 && q_dtype == NVJ_F16) return launch_block_select_f16(p, s);
  }
  if (cache_dtype == NVJ_BF16) return launch_block_select_lanes<__nv_bfloat16>(p, s);
  if (cache_dtype == NVJ_F16) return launch_block_select_lanes<__half>(p, s);
  return launch_block_select_lanes<float>(p, s);
}
