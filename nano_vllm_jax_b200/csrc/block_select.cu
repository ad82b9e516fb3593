// Selection of the blocks of a row that its attention is to read.
//
//   score(b) = max over the heads g of the kv head's group of  sum_d max(q_gd, 0) high_bd + min(q_gd, 0) low_bd
// which no key of block b exceeds: low and high are the bounds of its keys (rope_append.cu).  Chosen are the `first` first and the
// `last` last blocks that the token sees and, of the others, those of the highest scores; ties go to the lowest column.  A score
// that is NaN, or beyond fp32, ranks as infinity.
//
// Columns are whole numbers, so the border between chosen and left has to lie where it lies in exact arithmetic.  The scores are
// sums in fp32 whose error is bounded by eps = c * |q|_1 * (largest |bound| of the blocks), c from the number of
// roundings; with t the border's score, blocks above t + 2 eps are in and those below t - 2 eps are out whatever was rounded, and the
// few between the two are scored again in 64 bits.  Usually that is the block at the border alone, and nothing is left to decide.
//
// One thread-block cluster per query token and kv head: its warps score 16 blocks at a time and leave the scores, as ordered
// integers, in the first CTA's shared memory, which finds the border by a radix selection and writes the columns in ascending order.
// No workspace, no second launch.  Bound by the bytes of the bounds, 2 head_dim numbers per block and kv head: 1/block_size of the cache.

#include "cluster.cuh"
#include "decode_cluster.cuh"
#include "quantized_kv.cuh"

namespace nvj {

struct SelectParams {
  const void* q;
  const void* bounds;  // [num_blocks, hkv, 2, D]
  const int32_t* block_tables;
  const int32_t* seq_lens;
  const int32_t* positions;  // nullable [rows, width]
  int32_t* out;              // [rows, width, hkv, budget]
  int32_t* status;
  long long num_blocks;
  int q_dtype, cache_dtype;
  int rows, width, table_width, block_size, hkv, groups, d, budget, first, last;
};

constexpr int kBsWarps = 8, kBsThreads = 32 * kBsWarps;
constexpr int kBsBins = 2048;
constexpr int kBsMostColumns = 45056;  // of a row: their scores fit one SM's shared memory, beside the queries
constexpr int kBsMostCtas = 16;
constexpr uint32_t kBsInfinity = 0xff800000u;  // bs_key(+infinity)

// Floats as integers of the same order; NaN as infinity.
__device__ __forceinline__ uint32_t bs_key(float x) {
  if (x != x) return kBsInfinity;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bs_float(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

__device__ __forceinline__ float bs_load(const void* p, long long i, int dtype) {
  if (dtype == NVJ_F32) return static_cast<const float*>(p)[i];
  if (dtype == NVJ_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

struct BsShared {
  uint32_t hist[kBsBins];
  uint32_t scan[kBsWarps];
  uint32_t pick, above;     // radix selection: the digit and what lies above it
  uint32_t count;
  float most[kBsMostCtas * kBsWarps];  // largest |bound| that each warp of the cluster has met in a block of a finite score
  double norm[kBsWarps], low[kBsWarps], high[kBsWarps];
};

// Sum over the CTA of one number per thread; all threads get the sum of the threads in front (exclusive) and the whole.
__device__ __forceinline__ uint32_t bs_scan(uint32_t x, uint32_t* scan, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_up_sync(kFullMask, y, o);
    if (lane >= o) y += z;
  }
  if (lane == 31) scan[warp] = y;
  __syncthreads();
  uint32_t front = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kBsWarps; ++w) {
    const uint32_t s = scan[w];
    if (w < warp) front += s;
    total += s;
  }
  __syncthreads();
  return front + y - x;
}

// The `want`-th largest (from 1) of keys[begin .. end), by digits from the top; `above` = how many are larger.
__device__ uint32_t bs_nth(const uint32_t* keys, int begin, int end, uint32_t want, BsShared& s, uint32_t& above) {
  uint32_t prefix = 0, mask = 0;
  above = 0;
#pragma unroll 1
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bins = digit == 2 ? 1024 : 2048;
    for (int i = threadIdx.x; i < kBsBins; i += kBsThreads) s.hist[i] = 0;
    __syncthreads();
    for (int i = begin + threadIdx.x; i < end; i += kBsThreads) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&s.hist[k >> shift & (bins - 1)], 1u);
    }
    __syncthreads();
    // from the top: thread t holds bins [2048 - 8 (t + 1), 2048 - 8 t)
    constexpr int kEach = kBsBins / kBsThreads;
    uint32_t mine = 0, total;
    const int top = kBsBins - kEach * (int)threadIdx.x;
#pragma unroll
    for (int i = 1; i <= kEach; ++i) mine += s.hist[top - i];
    const uint32_t front = above + bs_scan(mine, s.scan, total);
    if (front < want && want <= front + mine) {
      uint32_t run = front;
      for (int i = 1; i <= kEach; ++i) {
        const uint32_t h = s.hist[top - i];
        if (want <= run + h) {
          s.pick = top - i;
          s.above = run;
          break;
        }
        run += h;
      }
    }
    __syncthreads();
    above = s.above;
    prefix |= s.pick << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    __syncthreads();
  }
  return prefix;
}

// Score of one block in 64 bits, by a warp; the same in every lane.
__device__ double bs_exact(const SelectParams& p, long long q_at, long long bounds_at, int lane) {
  double best = -INFINITY;
  for (int g = 0; g < p.groups; ++g) {
    double sum = 0.0;
    for (int d = lane; d < p.d; d += 32) {
      const float q = bs_load(p.q, q_at + (long long)g * p.d + d, p.q_dtype);
      const float low = bs_load(p.bounds, bounds_at + d, p.cache_dtype), high = bs_load(p.bounds, bounds_at + p.d + d, p.cache_dtype);
      sum += (double)q * (double)(q > 0.f ? high : low);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
    best = sum > best ? sum : best;
  }
  return best;
}

// `f(column, score in 64 bits)` by the warps of the CTA, for the columns whose key is `key`; in batches of what the list holds.
template <class F>
__device__ __forceinline__ void bs_rescore(const SelectParams& p, BsShared& s, const uint32_t* keys, const int32_t* table, long long q_at, int head,
                                           int begin, int end, uint32_t key, F&& f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int base = begin; base < end; base += kBsBins) {
    const int stop = min(end, base + kBsBins);
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int i = base + threadIdx.x; i < stop; i += kBsThreads)
      if (keys[i] == key) s.hist[atomicAdd(&s.count, 1u)] = i;
    __syncthreads();
    const int m = (int)s.count;
    for (int j = warp; j < m; j += kBsWarps) {
      const int i = (int)s.hist[j];
      f(i, bs_exact(p, q_at, ((long long)table[i] * p.hkv + head) * 2 * p.d, lane));
    }
    __syncthreads();
  }
}

// The larger of two, NaN if either is.
__device__ __forceinline__ float bs_larger(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Scores of up to 16 blocks by a warp, for any type and head_dim: a block at a time, the dims over the lanes.
__device__ void bs_score_any(const SelectParams& p, long long q_at, const int32_t* table, int head, int c0, int n, uint32_t keys_at, float& most,
                             int lane) {
  for (int c = c0; c < n && c < c0 + 16; ++c) {
    const int id = table[c];
    float best = -INFINITY, large = 0.f;
    if (id < 0 || id >= p.num_blocks) {
      if (lane == 0) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
    } else {
      const long long at = ((long long)id * p.hkv + head) * 2 * p.d;
      for (int g = 0; g < p.groups; ++g) {
        float sum = 0.f;
        for (int d = lane; d < p.d; d += 32) {
          const float q = bs_load(p.q, q_at + (long long)g * p.d + d, p.q_dtype);
          const float low = bs_load(p.bounds, at + d, p.cache_dtype), high = bs_load(p.bounds, at + p.d + d, p.cache_dtype);
          sum = fmaf(fmaxf(q, 0.f), high, sum);
          sum = fmaf(fminf(q, 0.f), low, sum);
          if (q != q) sum = q;
          large = fmaxf(large, fmaxf(fabsf(low), fabsf(high)));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
        best = bs_larger(best, sum);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) large = fmaxf(large, __shfl_xor_sync(kFullMask, large, o));
    if (best - best == 0.f) most = fmaxf(most, large);
    if (lane == 0) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(keys_at + 4 * c), "r"(bs_key(best)) : "memory");
  }
}

// The same on tensor-core tiles, for head_dim 64, 128 and 256 and up to 16 query heads of a kv head: the blocks are the rows of an mma.sync tile, the heads its
// columns, and the contraction runs over the 2 D bounds, the positive parts of the queries standing against the high ones, the negative parts against the low.
// A lane's 16 bytes of a block's bounds are its operands as they come (selected_decode.cuh); 128 dims of 16 blocks are under way in
// registers, and each piece is asked for again as soon as it has been used.
template <typename C, int kD, int kTiles, int kTerms>
struct BsTiles {
  static constexpr int kPitch = kD + 8;
  static constexpr int kHalves = kD > 128 ? kD / 128 : 1, kPieces = kD / 32 / kHalves;
  static constexpr int kQBytes = kTerms * 2 * 8 * kTiles * kPitch * 2;  // [term][sign][column][pitch]

  // The queries' parts into shared memory.
  static __device__ void stage(const SelectParams& p, long long q_at, C* qs) {
    for (int i = threadIdx.x; i < 8 * kTiles * kD; i += kBsThreads) {
      const int col = i / kD, d = i % kD;
      float x = col < p.groups ? bs_load(p.q, q_at + (long long)col * kD + d, p.q_dtype) : 0.f;
      const bool negative = x < 0.f;
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
        C h;
        if constexpr (std::is_same<C, __half>::value) h = __float2half_rn(x);
        else h = kTerms > 1 ? __float2bfloat16_rz(x) : __float2bfloat16_rn(x);  // (cut: the largest f32 numbers stay finite)
        x -= (float)h;
        qs[((term * 2 + (negative ? 1 : 0)) * 8 * kTiles + col) * kPitch + d] = h;
        qs[((term * 2 + (negative ? 0 : 1)) * 8 * kTiles + col) * kPitch + d] = C(0.f);
      }
    }
  }

  uint4 held[kPieces][2][2];  // [piece][low, high][row g, row g + 8]
  const C* at[2];             // bounds of rows g and g + 8, this lane's dims; null: no block there
  int id;                     // of column tile + lane, the tile behind the one in the registers

  __device__ void fetch_id(const int32_t* table, int c0, int n, int lane) { id = lane < 16 && c0 + lane < n ? table[c0 + lane] : -1; }
  // places of the tile whose ids are there; flags those outside the pool
  __device__ void take(const SelectParams& p, int head, int c0, int n, int lane) {
    const bool used = lane < 16 && c0 + lane < n;
    if (used && (id < 0 || id >= p.num_blocks)) {
      atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      id = -1;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int mine = __shfl_sync(kFullMask, id, (lane >> 2) + 8 * r);
      at[r] = mine < 0 ? nullptr : static_cast<const C*>(p.bounds) + ((long long)mine * p.hkv + head) * 2 * kD + 8 * (lane & 3);
    }
  }
  __device__ void ask(int piece, int half) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        held[piece][b][r] = make_uint4(0, 0, 0, 0);
        if (at[r]) held[piece][b][r] = ld_stream_u4(at[r] + b * kD + 32 * (half * kPieces + piece));
      }
  }
  static __device__ __forceinline__ void widen(uint32_t& m, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<C, __half>::value) {
        const __half2 x = __hmax2(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&w[i])));
        m = *reinterpret_cast<const uint32_t*>(&x);
      } else {
        const __nv_bfloat162 x = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&m), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
        m = *reinterpret_cast<const uint32_t*>(&x);
      }
    }
  }
  static __device__ __forceinline__ float larger(uint32_t m) {
    float2 f;
    if constexpr (std::is_same<C, __half>::value) f = q_float2(m);
    else f = bf16x2_to_float2(m);
    return fmaxf(f.x, f.y);
  }

  // All tiles from c0 on, `stride` columns apart.
  __device__ void run(const SelectParams& p, const C* qs, const int32_t* table, int head, int c0, int stride, int n, uint32_t keys_at, float& most, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float acc[kTiles][2][4];
    uint32_t large[2];
    bool there[2];
    while (c0 < n) {
      const int next = c0 + stride;
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][0][i] = acc[j][1][i] = 0.f;
      large[0] = large[1] = 0u;
      there[0] = at[0] != nullptr;
      there[1] = at[1] != nullptr;
#pragma unroll
      for (int half = 0; half < kHalves; ++half) {
        if (half == kHalves - 1) {  // what is asked for from here on is the next tile's
          take(p, head, next, n, lane);
          fetch_id(table, next + stride, n, lane);
        }
#pragma unroll
        for (int piece = 0; piece < kPieces; ++piece) {
          const uint4 low0 = held[piece][0][0], low1 = held[piece][0][1], high0 = held[piece][1][0], high1 = held[piece][1][1];
          widen(large[0], low0);
          widen(large[0], high0);
          widen(large[1], low1);
          widen(large[1], high1);
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
              const C* q = qs + ((term * 2 * kTiles + j) * 8 + g) * kPitch + 32 * (half * kPieces + piece) + 8 * t;
              const uint4 up = *reinterpret_cast<const uint4*>(q), down = *reinterpret_cast<const uint4*>(q + 8 * kTiles * kPitch);
              cm_mma<C>(acc[j][0], {high0.x, high1.x, high0.y, high1.y}, up.x, up.y);
              cm_mma<C>(acc[j][1], {low0.x, low1.x, low0.y, low1.y}, down.x, down.y);
              cm_mma<C>(acc[j][0], {high0.z, high1.z, high0.w, high1.w}, up.z, up.w);
              cm_mma<C>(acc[j][1], {low0.z, low1.z, low0.w, low1.w}, down.z, down.w);
            }
          ask(piece, half == kHalves - 1 ? 0 : half + 1);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float best = -INFINITY, m = larger(large[r]);
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (8 * j + 2 * t + i < p.groups) best = bs_larger(best, acc[j][0][2 * r + i] + acc[j][1][2 * r + i]);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          best = bs_larger(best, __shfl_xor_sync(kFullMask, best, o));
          m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        }
        if (!there[r]) best = -INFINITY;
        if (best - best == 0.f) most = fmaxf(most, m);
        const int c = c0 + g + 8 * r;
        if (t == 0 && c < n) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(keys_at + 4 * c), "r"(bs_key(best)) : "memory");
      }
      c0 = next;
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, o));
  }
};

// kD 0: any type and layout.
template <typename C, int kD, int kTiles, int kTerms>
__global__ void __launch_bounds__(kBsThreads, 2) block_select_kernel(SelectParams p, int ctas) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ BsShared s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = ctas > 1 ? (int)cl_rank() : 0;
  const int token = blockIdx.x / ctas, row = token / p.width, head = blockIdx.y;
  if (ctas > 1) cl_arrive();  // (no CTA is written to before it is there)
  pdl_wait();
  pdl_release();
  int len = p.seq_lens[row];
  if (len > (long long)p.table_width * p.block_size) {
    if (threadIdx.x == 0 && rank == 0) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    len = p.table_width * p.block_size;
  }
  if (p.positions) len = min(len - 1, p.positions[token]) + 1;
  const int n = len > 0 ? (len - 1) / p.block_size + 1 : 0;
  const int hq = p.hkv * p.groups;
  int32_t* out = p.out + ((long long)token * p.hkv + head) * p.budget;
  if (ctas > 1) cl_wait();
  if (n <= p.budget) {  // all of them
    if (rank == 0)
      for (int i = threadIdx.x; i < p.budget; i += kBsThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  const long long q_at = ((long long)token * hq + (long long)head * p.groups) * p.d;
  const uint32_t keys_at = ctas > 1 ? cl_map(keys, 0) : smem_u32(keys);

  // |q|_1, the largest of the group's heads
  if (rank == 0) {
    double mine = 0.0;
    for (int g = warp; g < p.groups; g += kBsWarps) {
      double sum = 0.0;
      for (int d = lane; d < p.d; d += 32) sum += (double)fabsf(bs_load(p.q, q_at + (long long)g * p.d + d, p.q_dtype));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
      mine = sum > mine ? sum : mine;
    }
    if (lane == 0) s.norm[warp] = mine;
  }
  float most = 0.f;
  const int c0 = (rank * kBsWarps + warp) * 16, stride = ctas * kBsWarps * 16;
  if constexpr (kD > 0) {
    using Tiles = BsTiles<C, kD, kTiles, kTerms>;
    __shared__ __align__(16) C qs[Tiles::kQBytes / 2];
    Tiles tiles;
    tiles.fetch_id(table, c0, n, lane);
    tiles.take(p, head, c0, n, lane);
#pragma unroll
    for (int piece = 0; piece < Tiles::kPieces; ++piece) tiles.ask(piece, 0);
    tiles.fetch_id(table, c0 + stride, n, lane);
    Tiles::stage(p, q_at, qs);
    __syncthreads();
    tiles.run(p, qs, table, head, c0, stride, n, keys_at, most, lane);
  } else {
    for (int c = c0; c < n; c += stride) bs_score_any(p, q_at, table, head, c, n, keys_at, most, lane);
  }
  if (lane == 0) {
    const uint32_t at = (ctas > 1 ? cl_map(s.most, 0) : smem_u32(s.most)) + 4 * (rank * kBsWarps + warp);
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(most) : "memory");
  }
  if (ctas > 1) {
    cl_sync();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // the border among the columns that are not chosen anyway
  const int begin = p.first, end = n - p.last;
  uint32_t want = p.budget - p.first - p.last, border = 0xffffffffu, take_equal = 0;
  if (want > 0) {
    uint32_t above;
    border = bs_nth(keys, begin, end, want, s, above);
    take_equal = want - above;
    const float t = bs_float(border);
    if (t - t == 0.f) {
      double norm = 0.0;
      float large = 0.f;
      for (int w = 0; w < kBsWarps; ++w) norm = s.norm[w] > norm ? s.norm[w] : norm;
      for (int w = 0; w < ctas * kBsWarps; ++w) large = fmaxf(large, s.most[w]);
      // 2 D products, their sums in trees or rows of fp32: at most 2 D roundings of 2^-24 (chains of fused multiply-adds), or D / 8 steps of the
      // tensor cores that cut 17 numbers at 2^-23 of the largest, 2.2 D * 2^-23, for each term of the queries; two terms leave 2^-16 of a query at most
      constexpr double kSlip = kTerms > 1 ? 0x1p-16 : 0.0;
      const double eps = (3.0 * kTerms * 0x1p-23 * p.d + kSlip) * norm * (double)large +
                         0x1p-124 * (p.d + norm + p.d * (double)large);  // (and numbers below the normal ones, that may be taken for zero)
      const double low = (double)t - 2.0 * eps, high = (double)t + 2.0 * eps;
      // how many are in for sure, and how many stand between
      uint32_t in = 0, between = 0;
      for (int i = begin + threadIdx.x; i < end; i += kBsThreads) {
        const double x = (double)bs_float(keys[i]);
        if (x > high) ++in;
        else if (x >= low) ++between;
      }
      uint32_t all_in, all_between;
      bs_scan(in, s.scan, all_in);
      bs_scan(between, s.scan, all_between);
      if (all_in + all_between != want) {
        // keys anew: 0 out, all ones in, between the two the score in 64 bits as a fixed-point number of a window that holds it
        double floor_ = (double)t - 3.0 * eps, unit = 4294967290.0 / (6.0 * eps);
        for (int i = begin + threadIdx.x; i < end; i += kBsThreads) {
          const double x = (double)bs_float(keys[i]);
          keys[i] = x > high ? 0xffffffffu : x >= low ? 1u : 0u;
        }
        __syncthreads();
        border = 1u;
        for (;;) {
          bs_rescore(p, s, keys, table, q_at, head, begin, end, border, [&](int i, double x) {
            double u = (x - floor_) * unit;
            u = u > 0.0 ? u < 4294967290.0 ? u : 4294967290.0 : 0.0;
            if (lane == 0) keys[i] = 1u + (uint32_t)u;
          });
          border = bs_nth(keys, begin, end, want, s, above);
          take_equal = want - above;
          uint32_t equal = 0, all_equal;
          for (int i = begin + threadIdx.x; i < end; i += kBsThreads) equal += keys[i] == border;
          bs_scan(equal, s.scan, all_equal);
          if (all_equal == take_equal) break;
          // more of one key than there is room for: equal scores, or a window that is too wide for them
          double least = INFINITY, largest = -INFINITY;
          bs_rescore(p, s, keys, table, q_at, head, begin, end, border, [&](int, double x) {
            least = x < least ? x : least;
            largest = x > largest ? x : largest;
          });
          if (lane == 0) s.low[warp] = least, s.high[warp] = largest;
          __syncthreads();
          for (int w = 0; w < kBsWarps; ++w) {
            least = s.low[w] < least ? s.low[w] : least;
            largest = s.high[w] > largest ? s.high[w] : largest;
          }
          if (least == largest) break;
          floor_ = least;
          unit = 4294967290.0 / (largest - least);
          for (int i = begin + threadIdx.x; i < end; i += kBsThreads) {
            const uint32_t k = keys[i];
            keys[i] = k > border ? 0xffffffffu : k == border ? 1u : 0u;
          }
          border = 1u;
          __syncthreads();
        }
      } else {
        uint32_t least = 0xffffffffu;  // everything down to the smallest key between the two
        for (int i = begin + threadIdx.x; i < end; i += kBsThreads)
          if ((double)bs_float(keys[i]) >= low) least = min(least, keys[i]);
        least = __reduce_min_sync(kFullMask, least);
        if (lane == 0) s.scan[warp] = least;
        __syncthreads();
        for (int w = 0; w < kBsWarps; ++w) least = min(least, s.scan[w]);
        __syncthreads();
        border = least;
        take_equal = 0xffffffffu;
      }
    }
  }

  // the columns in ascending order: each thread a run of neighbours
  const int each = (n + kBsThreads - 1) / kBsThreads, lo = min(n, (int)threadIdx.x * each), hi = min(n, lo + each);
  uint32_t equal = 0, total;
  if (want > 0)
    for (int i = max(lo, begin); i < min(hi, end); ++i) equal += keys[i] == border;
  const uint32_t equal_front = bs_scan(equal, s.scan, total);
  auto chosen = [&](int i, uint32_t& e) {
    if (i < begin || i >= end) return true;
    if (want == 0) return false;
    if (keys[i] == border) return e++ < take_equal;
    return keys[i] > border;
  };
  uint32_t mine = 0, e = equal_front;
  for (int i = lo; i < hi; ++i) mine += chosen(i, e);
  uint32_t at = bs_scan(mine, s.scan, total);
  e = equal_front;
  for (int i = lo; i < hi; ++i)
    if (chosen(i, e)) {
      if (at < (uint32_t)p.budget) out[at] = i;
      ++at;
    }
}

// CTAs per cluster: enough for two on every SM, no more than one per 16 blocks and warp of the widest row.
static int block_select_ctas(long long units, long long columns, int sms) {
  long long c = (2LL * sms + units - 1) / units;
  const long long useful = (columns + 16 * kBsWarps - 1) / (16 * kBsWarps);
  c = c < useful ? c : useful;
  return (int)(c < 1 ? 1 : (c > 8 ? 8 : c));
}

template <typename C, int kD, int kTiles, int kTerms>
static int launch_block_select(const SelectParams& p, cudaStream_t stream) {
  auto* kernel = block_select_kernel<C, kD, kTiles, kTerms>;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBsMostColumns * 4) == cudaSuccess;
      }))
    return NVJ_ERR_LAUNCH;
  const long long tokens = (long long)p.rows * p.width;
  const int ctas = block_select_ctas(tokens * p.hkv, p.table_width, 148);
  if (tokens * ctas > 0x7fffffffLL) return NVJ_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tokens * ctas), p.hkv, 1);
  cfg.blockDim = dim3(kBsThreads, 1, 1);
  cfg.dynamicSmemBytes = p.table_width > p.budget ? (size_t)p.table_width * 4 : 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, ctas) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
}
template <typename C, int kD, int kTerms>
static int launch_block_select_heads(const SelectParams& p, cudaStream_t stream) {
  return p.groups <= 8 ? launch_block_select<C, kD, 1, kTerms>(p, stream) : launch_block_select<C, kD, 2, kTerms>(p, stream);
}
template <typename C, int kTerms>
static int launch_block_select_dims(const SelectParams& p, cudaStream_t stream) {
  if (p.d == 256) return launch_block_select_heads<C, 256, kTerms>(p, stream);
  if (p.d == 128) return launch_block_select_heads<C, 128, kTerms>(p, stream);
  return launch_block_select_heads<C, 64, kTerms>(p, stream);
}
// Tensor-core tiles where bounds and queries are exact in terms of the cache's type: all queries over bf16 bounds (f16's and f32's as two
// terms), f16 ones over f16.
static int launch_block_select_any(const SelectParams& p, cudaStream_t stream) {
  if ((p.d == 64 || p.d == 128 || p.d == 256) && p.groups <= 16) {
    if (p.cache_dtype == NVJ_BF16)
      return p.q_dtype == NVJ_BF16 ? launch_block_select_dims<__nv_bfloat16, 1>(p, stream) : launch_block_select_dims<__nv_bfloat16, 2>(p, stream);
    if (p.cache_dtype == NVJ_F16 && p.q_dtype == NVJ_F16) return launch_block_select_dims<__half, 1>(p, stream);
  }
  return launch_block_select<float, 0, 1, 1>(p, stream);
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
  return launch_block_select_any(p, static_cast<cudaStream_t>(stream));
}
