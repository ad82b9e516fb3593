// What the tcgen05 kernel over the 8-bit cache is given (quantized_umma.cuh), and the types of query it is built for.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nvj {

struct DecodeParams;
struct UmmaCut;

struct QuParams {
  const void* q;
  const float* k_scale;
  const float* v_scale;
  const int32_t* positions;        // nullable: [rows, width], packed: per token
  const int32_t* query_start_loc;  // packed: rows of one query token
  float* out;
  float* part_acc;  // [2 * ranges][hcts][tile_columns][head_dim]
  float* part_ml;   // [2 * ranges][hcts][tile_columns][2]
  UmmaCut* cuts;    // [ranges]
  int width, columns, groups, num_q_heads, num_kv_heads;
  int unit, unit_log2;  // keys per box: the largest of 16, 32 and 64 that divides a block
  int column_tiles, tile_columns, hcts;  // hcts = num_kv_heads * column_tiles
  float scale_log2;
};

int launch_quantized_umma_bf16(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int head_dim,
                               int ranges, cudaStream_t stream);
int launch_quantized_umma_f16(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int head_dim,
                              int ranges, cudaStream_t stream);
int launch_quantized_umma_f32(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int head_dim,
                              int ranges, cudaStream_t stream);

}  // namespace nvj
