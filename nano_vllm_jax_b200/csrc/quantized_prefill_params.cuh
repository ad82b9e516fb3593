// What the prefill kernel over the 8-bit cache is given (quantized_prefill_umma.cuh), and the types of query it is built for.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace nvj {

constexpr int kQtMostSplits = 8;   // CTAs that share a tile's keys, at most
constexpr int kQtSplitTiles = 3;   // tiles of 64 keys for each of them, at least
constexpr int kQtFlush = 64;       // tiles after which the sums are emptied

struct QtParams {
  const void* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* kv_lens;
  const int32_t* positions;
  const int32_t* query_start_loc;
  float* out;
  float* flush;  // nullable scratch for the sums of clusters' CTAs: [kv head][CTA][128 rows][head_dim]
  int32_t* status;
  long long num_blocks, flush_bytes;
  int rows, table_width, block_size, num_kv_heads, groups, token_bucket, skip_single, splits;
  float scale_log2;
};

// `tiles`: how many tiles of 128 query rows the batch has per kv head, as far as the caller knows; `most_tiles`: how many it can have.
int launch_quantized_prefill_bf16(const QtParams& p, int head_dim, int tiles, int most_tiles, cudaStream_t stream);
int launch_quantized_prefill_f16(const QtParams& p, int head_dim, int tiles, int most_tiles, cudaStream_t stream);
int launch_quantized_prefill_f32(const QtParams& p, int head_dim, int tiles, int most_tiles, cudaStream_t stream);

}  // namespace nvj
