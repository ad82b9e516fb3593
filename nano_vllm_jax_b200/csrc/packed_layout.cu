// The layout of a packed step, made on the device from its rows' lengths: blocks taken from a free list into the rows' block tables,
// then position, row, slot of every token and the step's query_start_loc, lengths and the list's new head.
//
//   need[r]  = ceil((cached[r] + new[r]) / bs) - ceil(cached[r] / bs)
//   first[r] = head + need[0] + .. + need[r - 1]          block_tables[r][ceil(cached[r] / bs) + j] = free_blocks[first[r] + j]
//   qsl[r]   = new[0] + .. + new[r - 1]                   token qsl[r] + t: position cached[r] + t, slot from the table entry
//
// One launch.  Every CTA adds up the lengths itself (a thread consecutive rows, then a scan over the threads' sums), which costs
// one trip to memory for up to a few thousand rows and spares a grid-wide wait, and keeps both prefixes in shared memory; then it writes
// its share of the tokens and of the rows.  A thread writes four tokens in a row: it finds the first one's row by bisection and walks on.
// A slot comes from the free list or from the old part of the table, never from an entry that another CTA is writing, so no
// order between CTAs is needed.
// Bound by latency: the launch, the trip for the lengths, the scan, the trip for the table entries, the stores (12 bytes per token): 256 rows of
// one token 5.7 us, 4096 rows of up to 63 9.8 us (3 MB: 0.4 us).

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
  // 0 <= x < 2^31 divided by the block size: (x * by >> 32) >> shift with by = floor(2^(31 + l) / block_size) + 1, l the least with
  // 2^l >= block_size, shift = l - 1 (Granlund and Montgomery); 0: block size 1.  (64-bit divisions, two or four a row: 7 of 12 us of
  // 4096 rows.)
  unsigned by;
  int shift;
};

constexpr int kLayoutThreads = 512;
constexpr int kLayoutHeld = 8;  // rows that a thread keeps in registers between the two looks at them

__device__ __forceinline__ int layout_quotient(const LayoutParams& p, int x) { return p.by ? (int)(__umulhi((unsigned)x, p.by) >> p.shift) : x; }
__device__ __forceinline__ int layout_blocks(const LayoutParams& p, int tokens) { return tokens > 0 ? layout_quotient(p, tokens - 1) + 1 : 0; }
// A row's cached and new tokens; a row that its table has no room for, or a negative length, is flagged and gets nothing.
__device__ __forceinline__ int2 layout_row(const LayoutParams& p, int c, int n, int* bad) {
  const long long most = (long long)p.table_width * p.block_size;
  if (c < 0 || n < 0 || (long long)c + n > most) {
    *bad = 1;
    n = 0;
    c = c < 0 ? 0 : (c > most ? (int)most : c);
  }
  return make_int2(c, n);
}
// The last i < n with from[i] <= x.
__device__ __forceinline__ int layout_find(const int* from, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (from[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kLayoutThreads) packed_layout_kernel(LayoutParams p) {
  extern __shared__ int layout_smem[];
  int* qsl = layout_smem;           // [rows + 1]
  int* first = qsl + p.rows + 1;    // [rows + 1], from 0
  int* cached = first + p.rows + 1;  // [rows]
  __shared__ int2 sums[kLayoutThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_release();
  const int head = *p.free_head;
  int per = (p.rows + kLayoutThreads - 1) / kLayoutThreads;  // consecutive rows of a thread
  const bool wide = per > 1 && ((reinterpret_cast<uintptr_t>(p.cached_lens) | reinterpret_cast<uintptr_t>(p.new_lens)) & 15) == 0;
  if (wide) per = (per + 3) & ~3;  // four rows per load
  int c[kLayoutHeld], n[kLayoutHeld];
  int bad = 0;
  if (wide) {
#pragma unroll
    for (int k = 0; k < kLayoutHeld; k += 4) {
      const int r = tid * per + k;
      if (k < per && r + 4 <= p.rows) {
        const int4 x = *reinterpret_cast<const int4*>(p.cached_lens + r), y = *reinterpret_cast<const int4*>(p.new_lens + r);
        c[k] = x.x; c[k + 1] = x.y; c[k + 2] = x.z; c[k + 3] = x.w;
        n[k] = y.x; n[k + 1] = y.y; n[k + 2] = y.z; n[k + 3] = y.w;
      } else {
#pragma unroll
        for (int e = k; e < k + 4; ++e) {
          const bool there = e < per && tid * per + e < p.rows;
          c[e] = there ? p.cached_lens[tid * per + e] : 0;
          n[e] = there ? p.new_lens[tid * per + e] : 0;
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kLayoutHeld; ++k) {
      const bool there = k < per && tid * per + k < p.rows;
      c[k] = there ? p.cached_lens[tid * per + k] : 0;
      n[k] = there ? p.new_lens[tid * per + k] : 0;
    }
  }
  auto fresh_blocks = [&](int2 cn) { return layout_blocks(p, cn.x + cn.y) - layout_blocks(p, cn.x); };
  int2 mine = make_int2(0, 0);
#pragma unroll
  for (int k = 0; k < kLayoutHeld; ++k) {
    if (k >= per) continue;
    const int2 cn = layout_row(p, c[k], n[k], &bad);
    mine.x += cn.y;
    mine.y += fresh_blocks(cn);
  }
  for (int k = kLayoutHeld; k < per && tid * per + k < p.rows; ++k) {
    const int2 cn = layout_row(p, p.cached_lens[tid * per + k], p.new_lens[tid * per + k], &bad);
    mine.x += cn.y;
    mine.y += fresh_blocks(cn);
  }
  int2 upto = mine;  // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(kFullMask, upto.x, o), b = __shfl_up_sync(kFullMask, upto.y, o);
    if (lane >= o) upto.x += a, upto.y += b;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  int2 at = make_int2(upto.x - mine.x, upto.y - mine.y);
#pragma unroll
  for (int w = 0; w < kLayoutThreads / 32; ++w)
    if (w < warp) at.x += sums[w].x, at.y += sums[w].y;
  if (p.rows == 0 && tid == 0) qsl[0] = first[0] = 0;
  auto leave = [&](int r, int2 cn) {
    qsl[r] = at.x;
    first[r] = at.y;
    cached[r] = cn.x;
    at.x += cn.y;
    at.y += fresh_blocks(cn);
    if (r == p.rows - 1) qsl[p.rows] = at.x, first[p.rows] = at.y;
  };
  int unused = 0;
#pragma unroll
  for (int k = 0; k < kLayoutHeld; ++k)
    if (k < per && tid * per + k < p.rows) leave(tid * per + k, layout_row(p, c[k], n[k], &unused));
  for (int k = kLayoutHeld; k < per && tid * per + k < p.rows; ++k)
    leave(tid * per + k, layout_row(p, p.cached_lens[tid * per + k], p.new_lens[tid * per + k], &unused));
  __syncthreads();
  const int total = qsl[p.rows], blocks = first[p.rows];
  const long long threads = (long long)gridDim.x * kLayoutThreads, me = (long long)blockIdx.x * kLayoutThreads + tid;
  // An id from the list, -1 past its end (a slot or table entry that the kernels downstream flag and skip, as a negative id in it is).
  auto taken = [&](long long k) {
    const long long i = (long long)head + k;
    return i >= 0 && i < p.free_count ? p.free_blocks[i] : -1;
  };
  if (blockIdx.x == 0) {
    if (tid == 0) {
      *p.free_head_out = head + blocks;
      if (total > p.token_bucket) bad = 1;
    }
    if (bad) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
  }
  const bool vector = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.token_row_ids) |
                        reinterpret_cast<uintptr_t>(p.slot_mapping)) & 15) == 0;
  for (long long i0 = 4 * me; i0 < p.token_bucket; i0 += 4 * threads) {
    int position[4], row[4], slot[4];
    int r = i0 < total ? layout_find(qsl, p.rows, (int)i0) : 0, held = 0, block = -1, id = -1;  // of the token in front
    bool begun = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long long i = i0 + e;
      position[e] = row[e] = 0;
      slot[e] = -1;
      if (i < total) {
        bool moved = !begun;
        while (i >= qsl[r + 1]) ++r, moved = true;
        if (moved) held = layout_blocks(p, cached[r]), block = -1;
        begun = true;
        row[e] = r;
        position[e] = cached[r] + (int)(i - qsl[r]);
        const int b = layout_quotient(p, position[e]);
        if (b != block) {
          block = b;
          id = b < held ? p.block_tables[(long long)r * p.table_width + b] : taken(first[r] + (b - held));
        }
        const long long at = (long long)id * p.block_size + (position[e] - b * p.block_size);
        if (id >= 0 && at <= 0x7fffffffLL) slot[e] = (int)at;  // (an id whose slots no int32 names belongs to no pool)
      }
    }
    if (vector && i0 + 4 <= p.token_bucket) {
      *reinterpret_cast<int4*>(p.positions + i0) = make_int4(position[0], position[1], position[2], position[3]);
      *reinterpret_cast<int4*>(p.token_row_ids + i0) = make_int4(row[0], row[1], row[2], row[3]);
      *reinterpret_cast<int4*>(p.slot_mapping + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e < p.token_bucket) {
          p.positions[i0 + e] = position[e];
          p.token_row_ids[i0 + e] = row[e];
          p.slot_mapping[i0 + e] = slot[e];
        }
    }
  }
  for (long long r = me; r <= p.rows; r += threads) {
    p.query_start_loc[r] = qsl[r];
    if (r < p.rows) p.seq_lens[r] = cached[r] + (qsl[r + 1] - qsl[r]);
  }
  // the new table entries: entry k of all of them belongs to the last row with first[row] <= k
  for (long long k = me; k < blocks; k += threads) {
    const int r = layout_find(first, p.rows, (int)k), id = taken(k);
    if (id < 0) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
    p.block_tables[(long long)r * p.table_width + layout_blocks(p, cached[r]) + (int)(k - first[r])] = id;
  }
}

constexpr int kLayoutMaxRows = 16384;  // two prefixes and a length of so many rows in shared memory
constexpr int layout_smem_bytes(int rows) { return (3 * rows + 2) * (int)sizeof(int); }

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
  if (rows > 0 && (seq_lens == cached_lens || seq_lens == new_lens)) return NVJ_ERR_INVALID_ARGUMENT;  // (a CTA reads them while another writes)
  if (free_count > 0 && !free_blocks) return NVJ_ERR_INVALID_ARGUMENT;
  if (token_bucket > 0 && (!positions || !token_row_ids || !slot_mapping)) return NVJ_ERR_INVALID_ARGUMENT;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) {
        return cudaFuncSetAttribute(packed_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    layout_smem_bytes(kLayoutMaxRows)) == cudaSuccess;
      }))
    return NVJ_ERR_LAUNCH;
  LayoutParams p{cached_lens, new_lens, block_tables, free_blocks, free_head, positions, token_row_ids, slot_mapping, query_start_loc,
                 seq_lens, free_head_out, status, rows, table_width, block_size, free_count, token_bucket, 0u, 0};
  if (block_size > 1) {
    int l = 0;
    while ((1ll << l) < block_size) ++l;
    p.by = (unsigned)((1ull << (31 + l)) / (unsigned)block_size + 1);
    p.shift = l - 1;
  }
  const long long work = token_bucket / 4 > rows ? token_bucket / 4 : rows;
  long long ctas = (work + kLayoutThreads - 1) / kLayoutThreads;
  ctas = ctas < 1 ? 1 : (ctas > 148 ? 148 : ctas);
  return launch_after(packed_layout_kernel, dim3((unsigned)ctas), dim3(kLayoutThreads), (size_t)layout_smem_bytes(rows), static_cast<cudaStream_t>(stream), p) ==
                 cudaSuccess
             ? NVJ_OK
             : NVJ_ERR_LAUNCH;
}
