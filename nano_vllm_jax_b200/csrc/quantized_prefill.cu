// Ragged packed prefill attention over the 8-bit paged cache: the entry point and its routes.
//
//   * Rows of a single query token go to the decode kernel, which spreads a row over SMs.
//   * The model's shape with bf16 queries: the rows' blocks are written out once as bf16 (exact: a scale is a power of two) into
//     pages of a scratch cache, and the tcgen05 tiles of the bf16 cache run over it (paged_prefill_umma2.cu).  Writing out moves 5 bytes
//     per number, once per call: 6 us for 3.6k keys, 1% of a prompt's time.
//   * Every other head layout, block size and query type: quantized_prefill_umma.cuh, which converts the numbers on their way into shared memory,
//     for every 128 query rows anew (the pages' batches would take it 29.7 us instead of 28.7 for 512 tokens of three rows behind 1024, 135
//     instead of 108 for a prompt of 4096; 41.5 instead of 45.6 for 256 tokens behind 4000).

#include "quantized_kv.cuh"
#include "quantized_prefill_params.cuh"

namespace nvj {

int prefill_over_pages(const void* q, const void* k_pages, const void* v_pages, long long pages, const int32_t* page_tables, int table_width,
                       const int32_t* kv_lens, const int32_t* positions, const int32_t* query_start_loc, int rows, int token_bucket, float scale,
                       float* out, int32_t* status, void* workspace, size_t workspace_bytes, int part, int tile_pairs, cudaStream_t stream);

int paged_decode_quantized(const void* q, int q_dtype, const void* k_cache_layer, const void* v_cache_layer, const float* k_scale, const float* v_scale,
                           int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int num_q_heads, const int32_t* block_tables,
                           int table_width, const int32_t* seq_lens, const int32_t* positions, const int32_t* query_start_loc, int rows, int width,
                           int tokens, float scale, float* out, int32_t* status, void* workspace, size_t workspace_bytes, int form,
                           nvj_stream_t stream);

// ---- pages of a scratch bf16 cache ----------------------------------------------------------------------------------------------
struct QUnpackParams {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* kv_lens;
  const int32_t* positions;
  const int32_t* query_start_loc;
  char* k_pages;  // page row * table_width + b: block b of the row
  char* v_pages;
  int32_t* page_tables;
  int32_t* status;
  long long num_blocks;
  int rows, table_width, skip_single, token_bucket;
};

// Grid (x: blocks of a row in strides, y: rows); the model's shape, 16 tokens of 2 heads of 256: a thread four pieces of 16 numbers, two of K and two
// of V, of one head.  The block's id is asked for together with the row's length: two trips to memory in a row.  A block whose id is outside
// the pool has no page, and the tiles leave its keys out; the rows behind the last key that a token sees, which hold anything, become zeros.
__global__ void __launch_bounds__(256) quantized_unpack_kernel(QUnpackParams p) {
  constexpr int kRow = 512, kBlock = 16 * kRow;  // bytes of a token, and of a block
  pdl_wait();
  pdl_release();
  const int row = blockIdx.y;
  const int len = p.kv_lens[row], from = p.query_start_loc[row], end = p.query_start_loc[row + 1], to = end < p.token_bucket ? end : p.token_bucket;
  const bool skip = to <= from || from < 0 || (p.skip_single && end - from == 1);
  // Keys that a token sees: all of the row's where its last token stands at their end, as nearly always; else the tokens are looked at.
  int seen = len;
  if (!skip && p.positions[to - 1] + 1 < len) {
    __shared__ int most;
    if (threadIdx.x == 0) most = 0;
    __syncthreads();
    int mine = 0;
    for (int i = from + threadIdx.x; i < to; i += 256) mine = max(mine, p.positions[i] < len ? p.positions[i] + 1 : len);
    atomicMax(&most, __reduce_max_sync(kFullMask, mine));
    __syncthreads();
    seen = most;
  }
  const int head = (threadIdx.x * 16 % kRow) / 256, token = threadIdx.x * 16 / kRow;  // of the first piece; the second is eight tokens on
  for (int b = blockIdx.x; b < p.table_width; b += gridDim.x) {
    const long long page = (long long)row * p.table_width + b;
    const int id = p.block_tables[page];
    if (threadIdx.x == 0) p.page_tables[page] = (int)page;
    const int left = len - b * 16;  // tokens of the row from this block on
    if (skip || left <= 0) continue;
    const bool ok = id >= 0 && id < p.num_blocks;
    if (!ok && threadIdx.x == 0) {
      atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      p.page_tables[page] = -1;
    }
    uint4 w[4];
    const int left_seen = seen - b * 16;
    float unit[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (ok && token + 8 * (i & 1) < left)
        w[i] = ld_stream_u4((i < 2 ? p.k_cache : p.v_cache) + (long long)id * kBlock + (i & 1) * (kBlock / 2) + threadIdx.x * 16);
    }
    if (ok) {
      unit[0] = p.k_scale[(long long)id * 2 + head];
      unit[1] = p.v_scale[(long long)id * 2 + head];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (token + 8 * (i & 1) >= left_seen) w[i] = make_uint4(0, 0, 0, 0);
      const uint32_t in[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      const float u = unit[i >> 1];
      uint32_t out[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = q_float2(q_half2(in[k])), y = q_float2(q_half2_high(in[k]));
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * u, x.y * u), hi = __floats2bfloat162_rn(y.x * u, y.y * u);
        out[2 * k] = *reinterpret_cast<const uint32_t*>(&lo);
        out[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&hi);
      }
      uint4* at = reinterpret_cast<uint4*>((i < 2 ? p.k_pages : p.v_pages) + 2 * (page * kBlock + (i & 1) * (kBlock / 2) + threadIdx.x * 16));
      at[0] = make_uint4(out[0], out[1], out[2], out[3]);
      at[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
}

// Tiles of 128 query rows per kv head: full ones, and one that is not per row.
static long long quantized_prefill_most_tiles(int rows, int token_bucket, int groups) {
  return (long long)token_bucket * groups / 128 + (rows < token_bucket ? rows : token_bucket) + 1;
}
// ... and as many as there are, by the caller's number of 64-token tiles (negative: not known).
static long long quantized_prefill_tiles(int rows, int token_bucket, int groups, int tile_pairs) {
  const long long most = quantized_prefill_most_tiles(rows, token_bucket, groups) - 1;
  const long long told = tile_pairs < 0 ? most : ((long long)tile_pairs * (groups + groups % 2) + 1) / 2;
  return told < 1 ? 1 : told < most ? told : most;
}

// Whether a call's rows are written out as bf16 pages for the tcgen05 tiles.
static bool quantized_unpacks(int q_dtype, int block_size, int num_kv_heads, int head_dim, int num_q_heads, float scale) {
  return q_dtype == NVJ_BF16 && block_size == 16 && num_kv_heads == 2 && head_dim == 256 && num_q_heads == 8 && scale > 0.f;
}
// Pages of at most 1 GiB; a batch with more table room than that has its numbers converted tile by tile.
constexpr long long kQMostPages = 32768;  // (rows among them: the grid's y)


// Bytes of a batch's pages, 0 where there are none.
static size_t quantized_page_bytes(int q_dtype, int rows, int table_width, int block_size, int num_kv_heads, int head_dim, int num_q_heads, float scale) {
  const long long pages = (long long)rows * table_width;
  if (pages <= 0 || pages > kQMostPages || !quantized_unpacks(q_dtype, block_size, num_kv_heads, head_dim, num_q_heads, scale)) return 0;
  return (size_t)(pages * 2 * block_size * num_kv_heads * head_dim * 2 + (pages * 4 + 255) / 256 * 256);
}
}  // namespace nvj

// The scratch serves the decode kernel's partials and then the pages, or the sums that clusters empty behind kQtFlush tiles, one launch behind the other.
extern "C" size_t nvj_paged_prefill_quantized_workspace_bytes(int q_dtype, int rows, int table_width, int block_size, int num_kv_heads,
                                                              int head_dim, int num_q_heads, float scale, int single_rows, int token_bucket, int tile_pairs) {
  using namespace nvj;
  if (rows <= 0 || table_width <= 0 || token_bucket <= 0 || num_q_heads <= 0 || !quantized_cache_shape_ok(block_size, num_kv_heads, head_dim) ||
      num_q_heads % num_kv_heads != 0)
    return 0;
  const int groups = num_q_heads / num_kv_heads;
  const long long tiles = quantized_prefill_tiles(rows, token_bucket, groups, tile_pairs) * num_kv_heads;
  const long long splits = 148 / tiles < kQtMostSplits ? 148 / tiles : kQtMostSplits;
  size_t sums = 0;
  if (splits > 1 && (long long)table_width * block_size > 2LL * kQtFlush * 64)
    sums = (size_t)(quantized_prefill_most_tiles(rows, token_bucket, groups) * splits * num_kv_heads * 128 * head_dim * 4);
  const size_t partials =
      single_rows == 0 ? 0 : nvj_paged_decode_quantized_workspace_bytes(rows, 1, table_width, block_size, num_kv_heads, head_dim, num_q_heads, 0);
  const size_t pages = quantized_page_bytes(q_dtype, rows, table_width, block_size, num_kv_heads, head_dim, num_q_heads, scale);
  if (pages > 0) sums = pages;
  return sums > partials ? sums : partials;
}

extern "C" int nvj_paged_prefill_quantized(const void* q, int q_dtype, const void* k_cache_layer, const void* v_cache_layer,
                                           const float* k_scale, const float* v_scale, int64_t num_blocks, int block_size,
                                           int num_kv_heads, int head_dim, int num_q_heads, const int32_t* block_tables, int table_width,
                                           const int32_t* kv_lens, const int32_t* positions, const int32_t* query_start_loc, int rows,
                                           int token_bucket, float scale, float* out, int32_t* status, void* workspace,
                                           size_t workspace_bytes, int single_rows, int tile_pairs, nvj_stream_t stream) {
  using namespace nvj;
  if (rows < 0 || token_bucket < 0 || table_width < 0 || num_blocks < 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (q_dtype < NVJ_BF16 || q_dtype > NVJ_F32 || !quantized_cache_shape_ok(block_size, num_kv_heads, head_dim)) return NVJ_ERR_UNSUPPORTED;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (token_bucket == 0) return NVJ_OK;
  if (!q || !out || !status || !query_start_loc || !positions || !k_cache_layer || !v_cache_layer || !k_scale || !v_scale)
    return NVJ_ERR_INVALID_ARGUMENT;
  if (rows > 0 && (!kv_lens || (table_width > 0 && !block_tables))) return NVJ_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache_layer) || !aligned16(v_cache_layer)) return NVJ_ERR_INVALID_ARGUMENT;
  if ((long long)table_width * block_size > 0x7fffffffLL - 65536 || (long long)token_bucket * num_q_heads > 0x7fffffffLL - 65536)
    return NVJ_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int skip_single = single_rows != 0;
  if (skip_single && rows > 0) {
    const int rc = paged_decode_quantized(q, q_dtype, k_cache_layer, v_cache_layer, k_scale, v_scale, num_blocks, block_size, num_kv_heads, head_dim,
                                          num_q_heads, block_tables, table_width, kv_lens, positions, query_start_loc, rows, 1, token_bucket, scale, out,
                                          status, workspace, workspace_bytes, 0, stream);
    if (rc != NVJ_OK) return rc;
  }
  const size_t needed = quantized_page_bytes(q_dtype, rows, table_width, block_size, num_kv_heads, head_dim, num_q_heads, scale);
  if (needed > 0 && workspace && workspace_bytes >= needed && aligned16(workspace)) {
    const long long pages = (long long)rows * table_width, page_bytes = 2LL * block_size * num_kv_heads * head_dim;
    QUnpackParams u{};
    u.k_cache = static_cast<const uint8_t*>(k_cache_layer);
    u.v_cache = static_cast<const uint8_t*>(v_cache_layer);
    u.k_scale = k_scale;
    u.v_scale = v_scale;
    u.block_tables = block_tables;
    u.kv_lens = kv_lens;
    u.positions = positions;
    u.query_start_loc = query_start_loc;
    u.k_pages = static_cast<char*>(workspace);
    u.v_pages = u.k_pages + pages * page_bytes;
    u.page_tables = reinterpret_cast<int32_t*>(u.v_pages + pages * page_bytes);
    u.status = status;
    u.num_blocks = num_blocks;
    u.rows = rows;
    u.table_width = table_width;
    u.skip_single = skip_single;
    u.token_bucket = token_bucket;
    const int across = (148 * 8 + rows - 1) / rows;
    if (launch_after(quantized_unpack_kernel, dim3(across < table_width ? across : table_width, rows), dim3(256), 0, s, u) != cudaSuccess)
      return NVJ_ERR_LAUNCH;
    // (with no rows of one token the key ranges may be split; part 3 asks for that by a workspace, and writes nothing there)
    const int rc = prefill_over_pages(q, u.k_pages, u.v_pages, pages, u.page_tables, table_width, kv_lens, positions, query_start_loc, rows, token_bucket,
                                      scale, out, status, skip_single ? nullptr : workspace, skip_single ? 0 : workspace_bytes, skip_single ? 2 : 3,
                                      tile_pairs, s);
    if (rc != NVJ_ERR_UNSUPPORTED) return rc;  // (without a tensor-map encoder)
  }
  QtParams p{};
  p.q = q;
  p.k_cache = static_cast<const uint8_t*>(k_cache_layer);
  p.v_cache = static_cast<const uint8_t*>(v_cache_layer);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.kv_lens = kv_lens;
  p.positions = positions;
  p.query_start_loc = query_start_loc;
  p.out = out;
  p.status = status;
  p.num_blocks = num_blocks;
  p.rows = rows;
  p.table_width = table_width;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.groups = num_q_heads / num_kv_heads;
  p.token_bucket = token_bucket;
  p.skip_single = skip_single;
  p.scale_log2 = scale * 1.4426950408889634f;
  if (workspace && aligned16(workspace)) {
    p.flush = static_cast<float*>(workspace);
    p.flush_bytes = (long long)workspace_bytes;
  }
  const long long most = quantized_prefill_most_tiles(rows, token_bucket, p.groups), tiles = quantized_prefill_tiles(rows, token_bucket, p.groups, tile_pairs);
  if (most > 0x7fffffffLL) return NVJ_ERR_TOO_LARGE;
  if (q_dtype == NVJ_BF16) return launch_quantized_prefill_bf16(p, head_dim, (int)tiles, (int)most, s);
  if (q_dtype == NVJ_F16) return launch_quantized_prefill_f16(p, head_dim, (int)tiles, (int)most, s);
  return launch_quantized_prefill_f32(p, head_dim, (int)tiles, (int)most, s);
}
