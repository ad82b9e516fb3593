// The layout of a packed step, made on the device from its rows' lengths: blocks taken from a free list into the rows' block tables,
// then position, row, slot of every token and the step's query_start_loc, lengths and the list's new head.
//
//   need[r]  = ceil((cached[r] + new[r]) / bs) - ceil(cached[r] / bs)
//   first[r] = head + need[0] + .. + need[r - 1]          block_tables[r][ceil(cached[r] / bs) + j] = free_blocks[first[r] + j]
//   qsl[r]   = new[0] + .. + new[r - 1]                   token qsl[r] + t: position cached[r] + t, slot from the table entry
//
// One launch.  Every CTA adds up the lengths itself (thread i the rows 32 at a time of its share, then a scan over the threads'
// sums), which costs a CTA one trip to memory for up to a few thousand rows and spares a grid-wide wait, and keeps both
// prefixes in shared memory; then it writes its share of the tokens and of the rows.  A token's row is found by bisection there.
// A slot comes from the free list or from the old part of the table, never from an entry that another CTA is writing, so no
// order between CTAs is needed.
// The kernel is bound by latency (two dependent trips) up to ~10^5 tokens; 12 bytes per token are written.

#include "nvj_common.cuh"

namespace nvj {

struct LayoutParams {
  const int32_t* cached_lens;
  const int32_t* new_lens;
  int32_t* block_tables;
  const int32_t* free_blocks;
  const int32_t* free_head;
  int32_t* positions;
  int32_t* token_row_ids;
  int32_t* slot_mapping;
  int32_t* query_start_loc;
  int32_t* seq_lens;
  int32_t* free_head_out;
  int32_t* status;
  int rows, table_width, block_size, free_count, token_bucket;
};

constexpr int kLayoutThreads = 512;

// Row r's cached and new tokens; a row that its table has no room for, or a negative length, is flagged and gets nothing.
__device__ __forceinline__ int2 layout_row(const LayoutParams& p, int r, int* bad) {
  int c = p.cached_lens[r], n = p.new_lens[r];
  if (c < 0 || n < 0 || (long long)c + n > (long long)p.table_width * p.block_size) {
    *bad = 1;
    n = 0;
    const long long most = (long long)p.table_width * p.block_size;
    c = c < 0 ? 0 : (c > most ? (int)most : c);
  }
  return make_int2(c, n);
}
__device__ __forceinline__ int layout_blocks(int tokens, int bs) { return (int)(((long long)tokens + bs - 1) / bs); }

__global__ void __launch_bounds__(kLayoutThreads) packed_layout_kernel(LayoutParams p) {
  pdl_wait();
  pdl_release();
  extern __shared__ int layout_smem[];
  int* qsl = layout_smem;               // [rows + 1]
  int* first = layout_smem + p.rows + 1;  // [rows + 1], from 0
  __shared__ int2 sums[kLayoutThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = *p.free_head;
  const int per = (p.rows + kLayoutThreads - 1) / kLayoutThreads;  // consecutive rows of a thread
  int bad = 0;
  int2 mine = make_int2(0, 0);
  for (int k = 0; k < per; ++k) {
    const int r = tid * per + k;
    if (r < p.rows) {
      const int2 cn = layout_row(p, r, &bad);
      mine.x += cn.y;
      mine.y += layout_blocks(cn.x + cn.y, p.block_size) - layout_blocks(cn.x, p.block_size);
    }
  }
  int2 upto = mine;  // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(kFullMask, upto.x, o), b = __shfl_up_sync(kFullMask, upto.y, o);
    if (lane >= o) upto.x += a, upto.y += b;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  if (p.rows == 0 && tid == 0) qsl[0] = first[0] = 0;
  int2 at = make_int2(upto.x - mine.x, upto.y - mine.y);
  for (int w = 0; w < warp; ++w) at.x += sums[w].x, at.y += sums[w].y;
  for (int k = 0; k < per; ++k) {
    const int r = tid * per + k;
    if (r < p.rows) {
      int unused = 0;
      const int2 cn = layout_row(p, r, &unused);
      qsl[r] = at.x;
      first[r] = at.y;
      at.x += cn.y;
      at.y += layout_blocks(cn.x + cn.y, p.block_size) - layout_blocks(cn.x, p.block_size);
    }
    if (r == p.rows - 1) qsl[p.rows] = at.x, first[p.rows] = at.y;
  }
  __syncthreads();
  const int total = qsl[p.rows];
  const long long threads = (long long)gridDim.x * kLayoutThreads, me = (long long)blockIdx.x * kLayoutThreads + tid;
  // An id from the list, -1 past its end (a slot or table entry that the kernels downstream flag and skip).
  auto taken = [&](long long k) {
    const long long i = (long long)head + k;
    return i >= 0 && i < p.free_count ? p.free_blocks[i] : -1;
  };
  if (blockIdx.x == 0) {
    for (int r = tid; r <= p.rows; r += kLayoutThreads) p.query_start_loc[r] = qsl[r];
    if (tid == 0) {
      *p.free_head_out = head + first[p.rows];
      if (total > p.token_bucket) bad = 1;
      if (first[p.rows] > 0 && (head < 0 || (long long)head + first[p.rows] > p.free_count)) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
    }
    if (bad) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
  }
  for (long long i = me; i < p.token_bucket; i += threads) {
    int row = 0, position = 0, slot = -1;
    if (i < total) {
      int lo = 0, hi = p.rows - 1;  // the last row with qsl[row] <= i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (qsl[mid] <= i) lo = mid;
        else hi = mid - 1;
      }
      row = lo;
      int unused = 0;
      const int c = layout_row(p, row, &unused).x, held = layout_blocks(c, p.block_size);
      position = c + (int)(i - qsl[row]);
      const int b = position / p.block_size;
      const int id = b < held ? p.block_tables[(long long)row * p.table_width + b] : taken(first[row] + (b - held));
      slot = id < 0 ? -1 : id * p.block_size + (position - b * p.block_size);
    }
    p.positions[i] = position;
    p.token_row_ids[i] = row;
    p.slot_mapping[i] = slot;
  }
  for (long long r = me; r < p.rows; r += threads) {
    int unused = 0;
    const int2 cn = layout_row(p, (int)r, &unused);
    p.seq_lens[r] = cn.x + cn.y;
  }
  // the new table entries, one per thread: entry k of all of them belongs to the last row with first[row] <= k
  for (long long k = me; k < first[p.rows]; k += threads) {
    int lo = 0, hi = p.rows - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    int unused = 0;
    const int held = layout_blocks(layout_row(p, lo, &unused).x, p.block_size);
    p.block_tables[(long long)lo * p.table_width + held + (int)(k - first[lo])] = taken(k);
  }
}

constexpr int kLayoutMaxRows = 16384;  // two prefixes of so many rows in shared memory

}  // namespace nvj

extern "C" int nvj_build_packed_layout(const int32_t* cached_lens, const int32_t* new_lens, int rows, int32_t* block_tables,
                                       int table_width, int block_size, const int32_t* free_blocks, int free_count,
                                       const int32_t* free_head, int token_bucket, int32_t* positions, int32_t* token_row_ids,
                                       int32_t* slot_mapping, int32_t* query_start_loc, int32_t* seq_lens, int32_t* free_head_out,
                                       int32_t* status, nvj_stream_t stream) {
  using namespace nvj;
  if (rows < 0 || table_width < 0 || block_size <= 0 || free_count < 0 || token_bucket < 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (rows > kLayoutMaxRows) return NVJ_ERR_TOO_LARGE;
  // (no sum of lengths or of blocks can then pass 32 bits)
  if ((long long)table_width * block_size * (rows > 0 ? rows : 1) > 0x7fffffffLL) return NVJ_ERR_TOO_LARGE;
  if (!free_head || !free_head_out || !query_start_loc || !status || free_head == free_head_out) return NVJ_ERR_INVALID_ARGUMENT;
  if (rows > 0 && (!cached_lens || !new_lens || !seq_lens || (table_width > 0 && !block_tables))) return NVJ_ERR_INVALID_ARGUMENT;
  if (free_count > 0 && !free_blocks) return NVJ_ERR_INVALID_ARGUMENT;
  if (token_bucket > 0 && (!positions || !token_row_ids || !slot_mapping)) return NVJ_ERR_INVALID_ARGUMENT;
  const int smem = 2 * (rows + 1) * (int)sizeof(int);
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) {
        return cudaFuncSetAttribute(packed_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    2 * (kLayoutMaxRows + 1) * (int)sizeof(int)) == cudaSuccess;
      }))
    return NVJ_ERR_LAUNCH;
  LayoutParams p{cached_lens, new_lens, block_tables, free_blocks, free_head, positions, token_row_ids, slot_mapping, query_start_loc,
                 seq_lens, free_head_out, status, rows, table_width, block_size, free_count, token_bucket};
  const long long work = token_bucket > rows ? token_bucket : rows;
  long long ctas = (work + kLayoutThreads - 1) / kLayoutThreads;
  ctas = ctas < 1 ? 1 : (ctas > 148 ? 148 : ctas);
  return launch_after(packed_layout_kernel, dim3((unsigned)ctas), dim3(kLayoutThreads), (size_t)smem, static_cast<cudaStream_t>(stream), p) ==
                 cudaSuccess
             ? NVJ_OK
             : NVJ_ERR_LAUNCH;
}
