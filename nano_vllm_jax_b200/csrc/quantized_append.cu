// Append of new K/V rows to the 8-bit paged cache (quantized_kv.cuh).
//
// A block's tokens share a scale per kv head, so the unit of work is not a token but a run: the tokens of one call that stand
// together in the batch and fall into one block.  A run's rows of K, or of V, of one kv head are taken by one warp (batches of a few tokens per
// row) or by a CTA of four (prompts): their largest magnitude, found in registers, settles the block's scale; the rows that were there are
// rescaled if it has to grow, and the new ones stored.  K and V, the heads and the runs have nothing in common, so there are no
// atomics and no second pass over memory.
// bytes = tokens * kv_heads * head_dim * 2 * (source size + 1).  Prompts are bound by HBM and, in front of it, by the chain positions -> block id ->
// scale -> stores: 16384 bf16 tokens of 2 heads of 256 11.0 us (50 MB: 7.7 us), 13 with cold caches; with a warp per run, 126 registers of held rows and so
// half of the CTAs in a second wave, a quarter more.  A decode step is launch and chain: 256 tokens 3.3 - 3.5 us.

#include "quantized_kv.cuh"

namespace nvj {

struct QAppendParams {
  const void* new_k;
  const void* new_v;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  const int32_t* positions;
  const int32_t* block_tables;
  const int32_t* token_row_ids;    // packed batches
  const int32_t* query_start_loc;  // nullable
  const int32_t* seq_lens;         // nullable: rows with seq_lens[r] <= 0 are skipped
  int32_t* status;
  long long num_blocks;
  int qsl_rows, packed, n_tokens, n_cols, table_rows, table_width, block_size, num_kv_heads;
};

// Block and offset of a position, for the block sizes that there are (a division by a number that is not known: ~25 instructions of a kernel that
// is bound by them).
__device__ __forceinline__ int q_block_of(int pos, int block_size) {
  return block_size == 48 ? (int)__umulhi((unsigned)pos >> 4, 0x55555556u) : (int)((unsigned)pos >> (31 - __clz(block_size)));
}
__device__ __forceinline__ int q_offset_of(int pos, int block_size) { return pos - q_block_of(pos, block_size) * block_size; }

// The largest magnitude of raw rows, two numbers an instruction; NaN does not count, infinity does (and is looked for then).
template <typename T>
struct QMost {
  __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
  __device__ __forceinline__ void add(const QRaw<T>& r) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[k])));
  }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct QMost<__half> {
  __half2 m = __floats2half2_rn(0.f, 0.f);
  __device__ __forceinline__ void add(const QRaw<__half>& r) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&w[k])));
  }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct QMost<float> {
  float m = 0.f;
  __device__ __forceinline__ void add(const QRaw<float>& r) {
    float x[8];
    q_floats(r, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[k]));
  }
  __device__ __forceinline__ float value() const { return m; }
};

// What a lane knows about one token of the batch: its row's place in the block table, or -1 for a token that is not written.
struct QToken {
  long long entry;  // row * table_width + block of the row
};

__device__ __forceinline__ QToken q_token(const QAppendParams& p, int i) {
  QToken t{-1};
  if (i < 0 || i >= p.n_tokens) return t;
  const int pos = p.positions[i];
  const int row = p.packed ? p.token_row_ids[i] : i / p.n_cols;
  if (p.query_start_loc) {
    if (p.packed) {
      if (i >= p.query_start_loc[p.qsl_rows]) return t;
    } else {
      if (row >= p.qsl_rows || i - row * p.n_cols >= p.query_start_loc[row + 1] - p.query_start_loc[row]) return t;
    }
  }
  if (row < 0 || row >= p.table_rows) {
    atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
    return t;
  }
  if (p.seq_lens && p.seq_lens[row] <= 0) return t;
  const int block = q_block_of(pos, p.block_size);
  if (pos < 0 || block >= p.table_width) {
    atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    return t;
  }
  t.entry = (long long)row * p.table_width + block;
  return t;
}

// One run: `n` tokens from `first` on, of table entry `entry`, by kShare warps that meet at the CTA's barrier.  kLanes lanes hold a row of
// 8 * kLanes elements; a warp takes every kShare-th step of its rows.
template <typename T, int kD, int kShare>
__device__ void q_append_run(const QAppendParams& p, int first, int n, long long entry, int head, bool is_v, int warp, int lane) {
  constexpr int kLanes = kD / 8, kRows = 32 / kLanes;  // lanes of a row, rows of a step
  constexpr int kHold = 4;                             // steps whose rows stay in registers between the two looks at them
  __shared__ float largest_of[kShare];
  const int col = (lane % kLanes) * 8, sub = warp * kRows + lane / kLanes;
  constexpr int kNext = kShare * kRows;  // rows from one step to the next
  const long long token_stride = (long long)p.num_kv_heads * kD;
  const T* src = static_cast<const T*>(is_v ? p.new_v : p.new_k) + (long long)first * token_stride + (long long)head * kD + col;
  const int id = p.block_tables[entry];
  const int steps = (n + kNext - 1) / kNext;
  QRaw<T> held[kHold];
#pragma unroll
  for (int s = 0; s < kHold; ++s)
    if (s * kNext + sub < n) held[s] = q_load8(src + (long long)(s * kNext + sub) * token_stride);
  if (id < 0 || id >= p.num_blocks) {
    if (warp == 0 && lane == 0) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
    return;
  }
  float* scale_at = (is_v ? p.v_scale : p.k_scale) + (long long)id * p.num_kv_heads + head;
  const float before = *scale_at;
  // the offsets of up to 32 tokens at a time, one per lane; whether the block begins here, and which of its rows are new
  bool begins = false;
  unsigned fresh[2] = {0u, 0u};  // offsets 0 - 31 and 32 - 63
  int my_offset = 0;             // of token first + lane
  for (int c = 0; c < n; c += 32) {
    const int o = c + lane < n ? q_offset_of(p.positions[first + c + lane], p.block_size) : -1;
    if (c == 0) my_offset = o;
    begins |= __any_sync(kFullMask, o == 0);
    fresh[0] |= __reduce_or_sync(kFullMask, o >= 0 && o < 32 ? 1u << o : 0u);
    fresh[1] |= __reduce_or_sync(kFullMask, o >= 32 ? 1u << (o - 32) : 0u);
  }
  float x[8];
  auto over_all = [&](float mine) {  // the largest of the run's
    mine = __int_as_float(__reduce_max_sync(kFullMask, __float_as_int(mine)));
    if constexpr (kShare > 1) {
      if (lane == 0) largest_of[warp] = mine;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kShare; ++w) mine = fmaxf(mine, largest_of[w]);
      __syncthreads();  // (before it is written again)
    }
    return mine;
  };
  QMost<T> most;
#pragma unroll
  for (int s = 0; s < kHold; ++s)
    if (s * kNext + sub < n) most.add(held[s]);
  for (int s = kHold; s < steps; ++s)
    if (s * kNext + sub < n) most.add(q_load8(src + (long long)(s * kNext + sub) * token_stride));
  float largest = over_all(most.value());
  if (largest == INFINITY) {  // rarely: the finite ones
    float finite = 0.f;
#pragma unroll 1
    for (int s = 0; s < steps; ++s)
      if (s * kNext + sub < n) {
        q_floats(q_load8(src + (long long)(s * kNext + sub) * token_stride), x);
        finite = q_largest(finite, x);
      }
    largest = over_all(finite);
  }
  const float wanted = q_scale_for(largest);
  const float scale = begins ? wanted : fmaxf(wanted, before);
  uint8_t* base = (is_v ? p.v_cache : p.k_cache) + ((long long)id * p.block_size * p.num_kv_heads + head) * kD + col;
  if (scale != before && warp == 0 && lane == 0) *scale_at = scale;
  if (!begins && scale > before) {  // the rows that were there, in the new unit
    const float ratio = before / scale;
    for (int o = sub; o < p.block_size; o += kNext) {
      if (fresh[o >> 5] >> (o & 31) & 1) continue;
      uint2* at = reinterpret_cast<uint2*>(base + (long long)o * token_stride);
      const uint2 w = *at;
      const float2 a = q_float2(q_half2(w.x)), b = q_float2(q_half2_high(w.x)), c = q_float2(q_half2(w.y)), d = q_float2(q_half2_high(w.y));
      *at = make_uint2(q_pack2(a.x * ratio, a.y * ratio) | q_pack2(b.x * ratio, b.y * ratio) << 16,
                       q_pack2(c.x * ratio, c.y * ratio) | q_pack2(d.x * ratio, d.y * ratio) << 16);
    }
  }
  const float inverse = 1.f / scale;
  auto store = [&](int o, const QRaw<T>& raw) {
    q_floats(raw, x);
    *reinterpret_cast<uint2*>(base + (long long)o * token_stride) =
        make_uint2(q_pack2(x[0] * inverse, x[1] * inverse) | q_pack2(x[2] * inverse, x[3] * inverse) << 16,
                   q_pack2(x[4] * inverse, x[5] * inverse) | q_pack2(x[6] * inverse, x[7] * inverse) << 16);
  };
#pragma unroll
  for (int s = 0; s < kHold; ++s) {
    const int r = s * kNext + sub, o = __shfl_sync(kFullMask, my_offset, r & 31);
    if (r < n) store(r < 32 ? o : q_offset_of(p.positions[first + r], p.block_size), held[s]);
  }
  for (int s = kHold; s < steps; ++s) {
    const int r = s * kNext + sub;
    if (r < n) store(q_offset_of(p.positions[first + r], p.block_size), q_load8(src + (long long)r * token_stride));
  }
}

// Grid x: windows of `window` tokens; the CTA takes the runs that begin in its window one behind the other.  kShare 1: a warp for each (K or V,
// head), grid y counts them in fours; 4: the CTA's warps share the runs of one.
constexpr int kQAppendWarps = 4;
template <typename T, int kD, int kShare>
__global__ void __launch_bounds__(32 * kQAppendWarps) quantized_append_kernel(QAppendParams p, int window) {
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = kShare > 1 ? (int)blockIdx.y : (int)blockIdx.y * kQAppendWarps + warp;
  const int base = blockIdx.x * window;  // first token of the window
  const int head = part >> 1;
  const bool is_v = part & 1;
  if (head >= p.num_kv_heads) return;
  if constexpr (kShare > 1) {  // a prompt: the window's rows on their way to the L2 while their places are looked up
    constexpr int kLines = kD * (int)sizeof(T) / 128;
    const char* from = static_cast<const char*>(is_v ? p.new_v : p.new_k);
    for (int i = threadIdx.x; i < window * kLines; i += 32 * kQAppendWarps) {
      const long long token = base + i / kLines;
      if (token < p.n_tokens)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(from + (token * p.num_kv_heads + head) * kD * (long long)sizeof(T) + i % kLines * 128));
    }
  }
  // lane l looks at token base - 1 + l: the one in front tells whether the window's first token begins a run
  const QToken t = q_token(p, base - 1 + lane);
  const long long in_front = __shfl_up_sync(kFullMask, t.entry, 1);
  const bool same = lane > 0 && t.entry >= 0 && t.entry == in_front;
  const unsigned chain = __ballot_sync(kFullMask, same);
  unsigned starts = __ballot_sync(kFullMask, lane > 0 && lane <= window && t.entry >= 0 && !same);
  for (; starts; starts &= starts - 1) {
    const int at = __ffs(starts) - 1;  // lane of the run's first token
    const long long entry = __shfl_sync(kFullMask, t.entry, at);
    const int first = base - 1 + at;
    const unsigned follow = at == 31 ? 0u : ~(chain >> (at + 1));  // bit j clear: token first + 1 + j is of the run
    int n = 1 + (follow ? __ffs(follow) - 1 : 32);
    if (at + n > 31) {  // the run may go on behind what the lanes have seen
      n = 32 - at;
      for (;;) {
        const unsigned more = __ballot_sync(kFullMask, q_token(p, first + n + lane).entry == entry);
        const int add = more == kFullMask ? 32 : __ffs(~more) - 1;
        n += add;
        if (add < 32) break;
      }
    }
    q_append_run<T, kD, kShare>(p, first, n, entry, head, is_v, kShare > 1 ? warp : 0, lane);
  }
}

template <typename T>
static int launch_quantized_append(const QAppendParams& p, int head_dim, cudaStream_t stream) {
  // Batches of a few tokens per row: a run per window.  Prompts: windows of 16 tokens, in which one run begins, mostly (16384 tokens when they took 14.7 us,
  // before the divisions went: a window per token 37, most of it warps that find nothing to do; windows of 31 16.5).
  const long long rows = p.packed ? p.qsl_rows : (p.n_tokens + p.n_cols - 1) / p.n_cols;
  const bool prompt = p.n_tokens > 4 * (rows > 0 ? rows : 1);
  const int window = prompt ? 16 : 1, parts = 2 * p.num_kv_heads;
  const dim3 grid((p.n_tokens + window - 1) / window, prompt ? parts : (parts + kQAppendWarps - 1) / kQAppendWarps);
  auto go = [&](auto* kernel) {
    return launch_after(kernel, grid, dim3(32 * kQAppendWarps), 0, stream, p, window) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
  };
  auto dims = [&](auto share) {
    constexpr int kShare = decltype(share)::value;
    if (head_dim == 256) return go(quantized_append_kernel<T, 256, kShare>);
    if (head_dim == 128) return go(quantized_append_kernel<T, 128, kShare>);
    return go(quantized_append_kernel<T, 64, kShare>);
  };
  return prompt ? dims(std::integral_constant<int, kQAppendWarps>{}) : dims(std::integral_constant<int, 1>{});
}

}  // namespace nvj

extern "C" int nvj_kv_append_quantized(const void* new_k, const void* new_v, int src_dtype, const int32_t* positions,
                                       const int32_t* block_tables, const int32_t* token_row_ids, int table_rows, int table_width,
                                       const int32_t* query_start_loc, int qsl_rows, const int32_t* seq_lens, int n_rows, int n_cols,
                                       void* k_cache_layer, void* v_cache_layer, float* k_scale, float* v_scale, int64_t num_blocks,
                                       int block_size, int num_kv_heads, int head_dim, int32_t* status, nvj_stream_t stream) {
  using namespace nvj;
  if (n_rows < 0 || n_cols < 0 || table_rows < 0 || table_width < 0 || qsl_rows < 0 || num_blocks < 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (src_dtype < NVJ_BF16 || src_dtype > NVJ_F32 || !quantized_cache_shape_ok(block_size, num_kv_heads, head_dim)) return NVJ_ERR_UNSUPPORTED;
  const long long n = (long long)n_rows * n_cols;
  if (n == 0) return NVJ_OK;
  if (n > 0x7fffffffLL - 64) return NVJ_ERR_TOO_LARGE;
  if (!new_k || !new_v || !positions || !block_tables || !k_cache_layer || !v_cache_layer || !k_scale || !v_scale || !status)
    return NVJ_ERR_INVALID_ARGUMENT;
  if (!aligned16(new_k) || !aligned16(new_v) || !aligned16(k_cache_layer) || !aligned16(v_cache_layer)) return NVJ_ERR_INVALID_ARGUMENT;
  if (table_rows == 0 || table_width == 0 || num_blocks == 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (token_row_ids && n_rows != 1) return NVJ_ERR_INVALID_ARGUMENT;
  QAppendParams p{};
  p.new_k = new_k;
  p.new_v = new_v;
  p.k_cache = static_cast<uint8_t*>(k_cache_layer);
  p.v_cache = static_cast<uint8_t*>(v_cache_layer);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.positions = positions;
  p.block_tables = block_tables;
  p.token_row_ids = token_row_ids;
  p.query_start_loc = query_start_loc;
  p.seq_lens = seq_lens;
  p.status = status;
  p.num_blocks = num_blocks;
  p.qsl_rows = qsl_rows;
  p.packed = token_row_ids != nullptr;
  p.n_tokens = (int)n;
  p.n_cols = n_cols;
  p.table_rows = table_rows;
  p.table_width = table_width;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (src_dtype == NVJ_BF16) return launch_quantized_append<__nv_bfloat16>(p, head_dim, s);
  if (src_dtype == NVJ_F16) return launch_quantized_append<__half>(p, head_dim, s);
  return launch_quantized_append<float>(p, head_dim, s);
}
