// Selection of the blocks of a row that its attention is to read.
//
//   score(b) = max over the heads g of the kv head's group of  sum_d max(q_gd, 0) high_bd + min(q_gd, 0) low_bd
// which no key of block b exceeds: low and high are the bounds of its keys (rope_append.cu).  Chosen are the `first` first and the
// `last` last blocks that the token sees and, of the others, those of the highest scores; ties go to the lowest column.  A score
// that is NaN ranks as infinity; blocks outside the pool rank behind all others.
//
// Columns are whole numbers, so the border between chosen and left has to lie where it lies in exact arithmetic.  The scores are
// sums in fp32 whose error is bounded by eps = c * (the largest sum of the products' magnitudes of all blocks), c from the number of
// roundings; with t the border's score, blocks above t + 2 eps are in and those below t - 2 eps are out whatever was rounded, and the
// few between the two are scored again in 64 bits.  Usually that is the block at the border alone, and nothing is left to decide.  Scores that fp32 sums
// did not hold are scored in 64 bits first, and if numbers are among them eps is infinite.  (With |q|_1 * (largest |bound|)
// in place of that sum and the tensor cores' sums over all dims in one, 2 - 8 blocks stood between in nearly every selection: 5 us for
// four rows, 12 - 19 for long ones.)
//
// One thread-block cluster per query token and kv head: its warps score 16 blocks at a time and leave the scores, as ordered
// integers, in the first CTA's shared memory, which finds the border by bins over the scores' range and writes the columns in ascending order.
// No workspace, no second launch.  Bound by the bytes of the bounds, 2 head_dim numbers per block and kv head: 1/block_size of the cache: 64 rows of 1024 - 4096 blocks, 2 heads
// of 256, 336 MB in 79 us (51 at the copy rate), 256 of 128 - 512 41 (26), 4 rows of 59 - 223 8.2.  On the CUDA cores, f32 bounds, 234 registers and two CTAs to an
// SM: 256 rows of 128 - 512 blocks 131 us (52).  The tables' width counts, not the rows' alone: their scores' places are shared memory, and the plan knows no other length.
// 256 rows of 128 - 512 blocks in tables of 4096 columns 48 us, of 16384 68.

#pragma once

#include <cfloat>

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

constexpr int kBsMostWarps = 8;
constexpr int kBsBins = 2048;
constexpr int kBsMostColumns = 45056;  // of a row: their scores fit one SM's shared memory, beside the queries
constexpr int kBsMostCtas = 8;
constexpr int kBsFew = 32;                    // keys that a warp ranks at once
constexpr uint32_t kBsInfinity = 0xff800000u;  // bs_key(+infinity)
constexpr uint32_t kBsLowest = 0x007fffffu;    // bs_key(-infinity)
constexpr uint32_t kBsMissing = 0u;            // a block outside the pool: below every score (kBsLowest at first)

// Floats as integers of the same order; NaN as infinity.
__device__ __forceinline__ uint32_t bs_key(float x) {
  if (x != x) return kBsInfinity;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bs_float(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// What a warp of the cluster leaves with the scores: the largest sum of magnitudes that it has met in a block of a finite score, and the ends of its keys.
struct BsEnds {
  float most;
  uint32_t least, largest;
};
struct BsShared {
  uint32_t hist[kBsBins];  // zero between uses; or a list of columns
  uint32_t scan[2][kBsMostWarps];
  uint32_t pick, above, inside, count;  // of a step of the selection: the bin, the keys above it and in it; entries of a list
  uint32_t few[kBsFew];
  double few_scores[kBsFew];
  BsEnds ends[kBsMostCtas * kBsMostWarps];
  double low[kBsMostWarps], high[kBsMostWarps];
  float reach[kBsMostWarps];
};

// Sum over the CTA of one number per thread: the sum of the threads in front and the whole.  `which` of two places is used in turn, so that one barrier does.
__device__ __forceinline__ uint32_t bs_scan(uint32_t x, BsShared& s, int& which, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_up_sync(kFullMask, y, o);
    if (lane >= o) y += z;
  }
  uint32_t* scan = s.scan[which];
  which ^= 1;
  if (lane == 31) scan[warp] = y;
  __syncthreads();
  uint32_t front = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kBsMostWarps; ++w)
    if (w < warps) {
      const uint32_t v = scan[w];
      if (w < warp) front += v;
      total += v;
    }
  return front + y - x;
}

// Sum over the CTA of one number per thread.
__device__ __forceinline__ uint32_t bs_total(uint32_t x, BsShared& s, int& which) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  x = __reduce_add_sync(kFullMask, x);
  uint32_t* scan = s.scan[which];
  which ^= 1;
  if ((threadIdx.x & 31) == 0) scan[warp] = x;
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kBsMostWarps; ++w)
    if (w < warps) total += scan[w];
  return total;
}

// The `want`-th largest (from 1) of keys[begin .. end), which lie in [least, largest]; `above`: how many are larger.  Each step deals the keys of the
// interval to bins of equal width and goes on in the one that holds it: scores of one size spread over the bins at once, where digits
// of the numbers themselves would put them all into a few.  (Four bins a thread for short rows.)
__device__ __forceinline__ uint32_t bs_nth(const uint32_t* keys, int begin, int end, uint32_t want, uint32_t least, uint32_t largest, BsShared& s,
                                           int& which, uint32_t& above) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = blockDim.x;
  const int each = end - begin > 1024 ? kBsBins / threads : 4, bits = 31 - __clz(each * threads);
  above = 0;
  for (;;) {
    const uint32_t range = largest - least;
    const int width = range == 0 ? 0 : 32 - __clz(range), shift = width > bits ? width - bits : 0;
    for (int i = begin + threadIdx.x; i < end; i += threads) {
      const uint32_t k = keys[i];
      if (k >= least && k <= largest) atomicAdd(&s.hist[(k - least) >> shift], 1u);
    }
    __syncthreads();
    // from the top: thread t holds the t-th `each` bins, and leaves them at zero
    const int top = each * (threads - (int)threadIdx.x);
    uint32_t mine = 0, total;
    for (int i = 4; i <= each; i += 4) {
      const uint4 h = *reinterpret_cast<const uint4*>(&s.hist[top - i]);
      mine += h.x + h.y + h.z + h.w;
    }
    const uint32_t front = above + bs_scan(mine, s, which, total);
    if (front < want && want <= front + mine) {
      uint32_t run = front;
      for (int i = 1; i <= each; ++i) {
        const uint32_t h = s.hist[top - i];
        if (want <= run + h) {
          s.pick = top - i;
          s.above = run;
          s.inside = h;
          s.count = 0;
          break;
        }
        run += h;
      }
    }
    for (int i = 4; i <= each; i += 4) *reinterpret_cast<uint4*>(&s.hist[top - i]) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    above = s.above;
    const uint32_t inside = s.inside, from = least + (s.pick << shift), to = from + min(largest - from, (1u << shift) - 1u);
    if (shift == 0) {
      __syncthreads();  // (s.pick is written again by the next selection)
      return from;
    }
    least = from;
    largest = to;
    if (inside > kBsFew) {
      __syncthreads();
      continue;
    }
    // the few that are left, ranked by one warp
    for (int i = begin + threadIdx.x; i < end; i += threads) {
      const uint32_t k = keys[i];
      if (k >= least && k <= largest) s.few[atomicAdd(&s.count, 1u)] = k;
    }
    __syncthreads();
    if (warp == 0) {
      const uint32_t mine_ = lane < (int)inside ? s.few[lane] : 0u;
      uint32_t larger = 0, same = 0;
      for (int j = 0; j < (int)inside; ++j) {
        const uint32_t k = __shfl_sync(kFullMask, mine_, j);
        larger += k > mine_;
        same += k == mine_;
      }
      // (equal keys agree on what they write)
      if (lane < (int)inside && above + larger < want && want <= above + larger + same) {
        s.pick = mine_;
        s.above = above + larger;
      }
    }
    __syncthreads();
    const uint32_t key = s.pick;
    above = s.above;
    __syncthreads();
    return key;
  }
}

__device__ __forceinline__ float4 bs_load4(const void* p, long long i, int dtype) {
  if (dtype == NVJ_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  const float2 a = dtype == NVJ_F16 ? q_float2(v.x) : bf16x2_to_float2(v.x), b = dtype == NVJ_F16 ? q_float2(v.y) : bf16x2_to_float2(v.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

// Score of one block in 64 bits, by a warp; the same in every lane.  kStrict: bounds and queries may be no numbers, and what they make is kept (a query of any sign
// against a bound that is not finite on either side: NaN or infinity, as the formula has it).
template <bool kStrict = false>
static __device__ double bs_exact(const SelectParams& p, long long q_at, long long bounds_at, int lane) {
  double best = -INFINITY;
  for (int g0 = 0; g0 < p.groups; g0 += 4) {  // four heads' loads in flight
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 128 * i + 4 * lane;
      if (d >= p.d) continue;
      const float4 low = bs_load4(p.bounds, bounds_at + d, p.cache_dtype), high = bs_load4(p.bounds, bounds_at + p.d + d, p.cache_dtype);
      float4 q[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) q[g] = g0 + g < p.groups ? bs_load4(p.q, q_at + (long long)(g0 + g) * p.d + d, p.q_dtype) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        sum[g] += (double)q[g].x * (double)(q[g].x > 0.f ? high.x : low.x);
        sum[g] += (double)q[g].y * (double)(q[g].y > 0.f ? high.y : low.y);
        sum[g] += (double)q[g].z * (double)(q[g].z > 0.f ? high.z : low.z);
        sum[g] += (double)q[g].w * (double)(q[g].w > 0.f ? high.w : low.w);
        if constexpr (kStrict) {  // zero times the other bounds
          sum[g] += 0.0 * (double)(q[g].x > 0.f ? low.x : high.x);
          sum[g] += 0.0 * (double)(q[g].y > 0.f ? low.y : high.y);
          sum[g] += 0.0 * (double)(q[g].z > 0.f ? low.z : high.z);
          sum[g] += 0.0 * (double)(q[g].w > 0.f ? low.w : high.w);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum[g] += __shfl_xor_sync(kFullMask, sum[g], o);
      if (g0 + g < p.groups) best = sum[g] > best || (kStrict && sum[g] != sum[g]) ? sum[g] : best;
    }
  }
  return best;
}

// `f(column, score in 64 bits)` by the warps of the CTA, for the columns whose key is `key`; in batches of what the list holds, which is left at zero.  kStrict: for the columns whose keys are
// no number's (from kBsInfinity on and round to kBsLowest), of blocks that may be outside the pool; those get kBsMissing.
template <bool kStrict = false, class F>
__device__ __forceinline__ void bs_rescore(const SelectParams& p, BsShared& s, uint32_t* keys, const int32_t* table, long long q_at, int head,
                                           int begin, int end, uint32_t key, F&& f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = blockDim.x;
  for (int base = begin; base < end; base += kBsBins) {
    const int stop = min(end, base + kBsBins);
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int i = base + threadIdx.x; i < stop; i += threads)
      if (kStrict ? keys[i] - key <= kBsLowest - kBsInfinity : keys[i] == key) s.hist[atomicAdd(&s.count, 1u)] = i;
    __syncthreads();
    const int m = (int)s.count;
    for (int j = warp; j < m; j += threads >> 5) {
      const int i = (int)s.hist[j], id = table[i];
      if (kStrict && (id < 0 || id >= p.num_blocks)) {
        if (lane == 0) keys[i] = kBsMissing;
        continue;
      }
      f(i, bs_exact<kStrict>(p, q_at, ((long long)id * p.hkv + head) * 2 * p.d, lane));
    }
    __syncthreads();
    for (int j = threadIdx.x; j < m; j += threads) s.hist[j] = 0;
  }
  __syncthreads();
}

// The larger and the smaller of two, NaN if either is.
__device__ __forceinline__ float bs_larger(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float bs_smaller(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A block's score into the first CTA's keys.
__device__ __forceinline__ void bs_leave(uint32_t keys_at, int c, float score, float magnitude, BsEnds& ends, bool mine) {
  const uint32_t key = bs_key(score);
  if (score - score == 0.f) ends.most = fmaxf(ends.most, magnitude);
  ends.least = min(ends.least, key);
  ends.largest = max(ends.largest, key);
  if (mine) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(keys_at + 4 * c), "r"(key) : "memory");
}

// Scores on the CUDA cores, for any type and number of heads: a warp takes eight blocks at a time, a lane four neighbouring dims of each (eight of head_dim > 128); the 32
// sums of eight blocks and four heads go through a butterfly of 31 exchanges that leaves one with each lane.
template <typename C, int kQuads>
struct BsLanes {
  static constexpr int kBlocks = 8;

  static __device__ __forceinline__ float4 load4(const C* at) {
    if constexpr (sizeof(C) == 4) {
      const uint4 v = ld_stream_u4(at);
      return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    } else {
      uint2 v;
      asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(at));
      float2 a, b;
      if constexpr (std::is_same<C, __half>::value) a = q_float2(v.x), b = q_float2(v.y);
      else a = bf16x2_to_float2(v.x), b = bf16x2_to_float2(v.y);
      return make_float4(a.x, a.y, b.x, b.y);
    }
  }
  // sums[i], i < 2 n, over the lanes that differ in bits below 2 n: lane l keeps that of i = l mod 2 n
  template <int n>
  static __device__ __forceinline__ void gather(float (&sums)[2 * n], int lane) {
#pragma unroll
    for (int o = n; o > 0; o >>= 1) {
      const bool upper = lane & o;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float keep = upper ? sums[i + o] : sums[i], send = upper ? sums[i] : sums[i + o];
        sums[i] = keep + __shfl_xor_sync(kFullMask, send, o);
      }
    }
  }

  static __device__ void run(const SelectParams& p, long long q_at, const int32_t* table, int head, int c0, int stride, int n, uint32_t keys_at, BsEnds& ends, int lane) {
    for (; c0 < n; c0 += stride) {
      int id = lane < kBlocks && c0 + lane < n ? table[c0 + lane] : -1;
      if (lane < kBlocks && c0 + lane < n && (id < 0 || id >= p.num_blocks)) {
        atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
        id = -1;
      }
      float4 low[kBlocks][kQuads], high[kBlocks][kQuads];
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const int mine = __shfl_sync(kFullMask, id, k);
        const C* at = static_cast<const C*>(p.bounds) + ((long long)mine * p.hkv + head) * 2 * p.d + 4 * lane;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          low[k][i] = high[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (mine >= 0 && 128 * i + 4 * lane < p.d) {
            low[k][i] = load4(at + 128 * i);
            high[k][i] = load4(at + p.d + 128 * i);
          }
        }
      }
      float best = -INFINITY;
      float4 size[kQuads];  // the largest |q| of the heads
#pragma unroll
      for (int i = 0; i < kQuads; ++i) size[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int g0 = 0; g0 < p.groups; g0 += 4) {
        float sums[32];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          float q[kQuads][4];
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (g0 + h < p.groups && 128 * i + 4 * lane < p.d) x = bs_load4(p.q, q_at + (long long)(g0 + h) * p.d + 128 * i + 4 * lane, p.q_dtype);
            q[i][0] = x.x, q[i][1] = x.y, q[i][2] = x.z, q[i][3] = x.w;
          }
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
            float4& z = size[i];
            z = make_float4(fmaxf(z.x, fabsf(q[i][0])), fmaxf(z.y, fabsf(q[i][1])), fmaxf(z.z, fabsf(q[i][2])), fmaxf(z.w, fabsf(q[i][3])));
          }
#pragma unroll
          for (int k = 0; k < kBlocks; ++k) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kQuads; ++i) {
              const float lo[4] = {low[k][i].x, low[k][i].y, low[k][i].z, low[k][i].w}, hi[4] = {high[k][i].x, high[k][i].y, high[k][i].z, high[k][i].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) sum = fmaf(bs_larger(q[i][j], 0.f), hi[j], fmaf(bs_smaller(q[i][j], 0.f), lo[j], sum));
            }
            sums[4 * k + h] = sum;
          }
        }
        gather<16>(sums, lane);  // lane 4 k + h: block k, head g0 + h
        if (g0 + (lane & 3) < p.groups) best = bs_larger(best, sums[0]);
      }
      float most[kBlocks];
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        most[k] = 0.f;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const float4 a = low[k][i], b = high[k][i], z = size[i];
          most[k] = fmaf(z.x, fmaxf(fabsf(a.x), fabsf(b.x)), most[k]);
          most[k] = fmaf(z.y, fmaxf(fabsf(a.y), fabsf(b.y)), most[k]);
          most[k] = fmaf(z.z, fmaxf(fabsf(a.z), fabsf(b.z)), most[k]);
          most[k] = fmaf(z.w, fmaxf(fabsf(a.w), fabsf(b.w)), most[k]);
        }
      }
      gather<4>(most, lane);  // lane l: block l mod 8, of the lanes that equal it above that
#pragma unroll
      for (int o = 8; o < 32; o <<= 1) most[0] += __shfl_xor_sync(kFullMask, most[0], o);
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) best = bs_larger(best, __shfl_xor_sync(kFullMask, best, o));
      const int k = lane >> 2, c = c0 + k;
      const float m = __shfl_sync(kFullMask, most[0], k);
      if (__shfl_sync(kFullMask, id, k) < 0) best = -INFINITY;
      if (c < n) bs_leave(keys_at, c, best, m, ends, (lane & 3) == 0);
    }
    ends.most = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(ends.most)));
    ends.least = __reduce_min_sync(kFullMask, ends.least);
    ends.largest = __reduce_max_sync(kFullMask, ends.largest);
  }
};

// The same on tensor-core tiles, for bf16 and f16 bounds and up to 16 query heads of a kv head: the blocks are the rows of an mma.sync tile, the heads its
// columns, and the contraction runs over the 2 D bounds, the positive parts of the queries standing against the high ones, the negative parts against the low.
// A lane's 16 bytes of a block's bounds are its operands as they come (selected_decode.cuh); 128 dims of 16 blocks are under way in
// registers and asked for again when all have been used.  (Each piece as soon as it has been used: 64 rows of 1024 - 4096 blocks 90 us instead of 83.  Through shared
// memory, by 16-byte asynchronous copies into two stages per warp, 89; by bulk copies of 256 bytes 134, the copy engine's limit.)
// kRagged: a head_dim below kD, its missing dims zero.
template <typename C, int kD, int kTiles, int kTerms, bool kRagged>
struct BsTiles {
  static constexpr int kPitch = kD + 32;  // elements; the eight columns' pieces of 16 bytes fall into different banks
  static constexpr int kHalves = kD > 128 ? kD / 128 : 1, kPieces = kD / 32 / kHalves;
  static constexpr int kQBytes = kTerms * 2 * 8 * kTiles * kPitch * 2;  // [term][sign][column][pitch]

  // The queries' parts into shared memory, a warp a column at a time, lane l the dims 8 l ..  Returns the largest |q| that this warp has met,
  // infinity if a bf16 one is so small that its products may be taken for zero.
  static __device__ float stage(const SelectParams& p, long long q_at, C* qs, int lane) {
    uint32_t reach = 0u;
    for (int col = threadIdx.x >> 5; col < 8 * kTiles; col += blockDim.x >> 5) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      if (col < p.groups && 8 * lane < (kRagged ? p.d : kD)) {
        const long long at = q_at + (long long)col * p.d + 8 * lane;
        if (p.q_dtype == NVJ_BF16) q_floats(q_load8(static_cast<const __nv_bfloat16*>(p.q) + at), x);
        else if (p.q_dtype == NVJ_F16) q_floats(q_load8(static_cast<const __half*>(p.q) + at), x);
        else q_floats(q_load8(static_cast<const float*>(p.q) + at), x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x[i]);
        reach = max(reach, !std::is_same<C, __half>::value && a > 0.f && a < 0x1p-100f ? 0x7f800000u : __float_as_uint(a));
      }
      if (lane >= kD / 8) continue;
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
        uint32_t up[4], down[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w;
          float2 f;
          if constexpr (kTerms > 1) {  // cut, not rounded: the largest f32 numbers stay finite (kTerms > 1 is bf16)
            w = __byte_perm(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), 0x7632);
            f = bf16x2_to_float2(w);
          } else {
            w = cm_pack<C>(x[2 * i], x[2 * i + 1], false);
          }
          // (NaN goes with the positive ones; what a cut leaves has the number's own sign)
          const uint32_t minus = (x[2 * i] < 0.f ? 0x0000ffffu : 0u) | (x[2 * i + 1] < 0.f ? 0xffff0000u : 0u);
          up[i] = w & ~minus;
          down[i] = w & minus;
          if constexpr (kTerms > 1) {
            x[2 * i] -= f.x;
            x[2 * i + 1] -= f.y;
          }
        }
        C* at = qs + (term * 2 * 8 * kTiles + col) * kPitch + 8 * lane;
        *reinterpret_cast<uint4*>(at) = make_uint4(up[0], up[1], up[2], up[3]);
        *reinterpret_cast<uint4*>(at + 8 * kTiles * kPitch) = make_uint4(down[0], down[1], down[2], down[3]);
      }
    }
    return __uint_as_float(__reduce_max_sync(kFullMask, reach));
  }
  uint4 held[kPieces][2][2];  // [piece][low, high][row g, row g + 8]
  const C* at[2];             // bounds of rows g and g + 8, this lane's dims (of block 0 where there is no block)
  bool there[2];
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
      there[r] = mine >= 0;
      at[r] = static_cast<const C*>(p.bounds) + ((long long)max(mine, 0) * p.hkv + head) * 2 * (kRagged ? p.d : kD) + 8 * (lane & 3);
    }
  }
  __device__ void ask(const SelectParams& p, int piece, int half, int lane) {
    const int dim = 32 * (half * kPieces + piece);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (!kRagged || dim + 8 * (lane & 3) < p.d) held[piece][b][r] = ld_stream_u4(at[r] + b * (kRagged ? p.d : kD) + dim);
        else held[piece][b][r] = make_uint4(0, 0, 0, 0);
  }
  // The larger magnitudes of two words' bounds: low <= high, so that it is that of high or of -low.
  static __device__ __forceinline__ uint32_t size(uint32_t low, uint32_t high) {
    uint32_t y;
    if constexpr (std::is_same<C, __half>::value) {
      const __half2 x = __hmax2(*reinterpret_cast<const __half2*>(&high), __hneg2(*reinterpret_cast<const __half2*>(&low)));
      y = *reinterpret_cast<const uint32_t*>(&x);
    } else {
      const __nv_bfloat162 x = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&high), __hneg2(*reinterpret_cast<const __nv_bfloat162*>(&low)));
      y = *reinterpret_cast<const uint32_t*>(&x);
    }
    return y;
  }
  static __device__ __forceinline__ uint32_t either(uint32_t up, uint32_t down) { return up | (down & 0x7fff7fffu); }

  // All tiles from c0 on, `stride` columns apart.
  __device__ void run(const SelectParams& p, const C* qs, const int32_t* table, int head, int c0, int stride, int n, uint32_t keys_at, BsEnds& ends, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float acc[kTiles][4], most[kTiles][4];  // scores; sums of |q| * (the larger |bound|)
    while (c0 < n) {
      const int next = c0 + stride;
      const bool here[2] = {there[0], there[1]};
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = most[j][i] = 0.f;
#pragma unroll
      for (int half = 0; half < kHalves; ++half) {
        if (half == kHalves - 1) {  // what is asked for from here on is the next tile's
          take(p, head, next, n, lane);
          fetch_id(table, next + stride, n, lane);
        }
#pragma unroll
        for (int piece = 0; piece < kPieces; ++piece) {
          const uint4 low0 = held[piece][0][0], low1 = held[piece][0][1], high0 = held[piece][1][0], high1 = held[piece][1][1];
          const uint32_t m0[4] = {size(low0.x, high0.x), size(low0.y, high0.y), size(low0.z, high0.z), size(low0.w, high0.w)};
          const uint32_t m1[4] = {size(low1.x, high1.x), size(low1.y, high1.y), size(low1.z, high1.z), size(low1.w, high1.w)};
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            float sum[4] = {0.f, 0.f, 0.f, 0.f};  // of these 32 dims alone: the tensor cores cut what they add to a larger sum
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
              const C* q = qs + ((term * 2 * kTiles + j) * 8 + g) * kPitch + 32 * (half * kPieces + piece) + 8 * t;
              const uint4 up = *reinterpret_cast<const uint4*>(q), down = *reinterpret_cast<const uint4*>(q + 8 * kTiles * kPitch);
              cm_mma<C>(sum, {high0.x, high1.x, high0.y, high1.y}, up.x, up.y);
              cm_mma<C>(sum, {high0.z, high1.z, high0.w, high1.w}, up.z, up.w);
              cm_mma<C>(sum, {low0.x, low1.x, low0.y, low1.y}, down.x, down.y);
              cm_mma<C>(sum, {low0.z, low1.z, low0.w, low1.w}, down.z, down.w);
              cm_mma<C>(most[j], {m0[0], m1[0], m0[1], m1[1]}, either(up.x, down.x), either(up.y, down.y));
              cm_mma<C>(most[j], {m0[2], m1[2], m0[3], m1[3]}, either(up.z, down.z), either(up.w, down.w));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] += sum[i];
          }
        }
#pragma unroll
        for (int piece = 0; piece < kPieces; ++piece) ask(p, piece, half == kHalves - 1 ? 0 : half + 1, lane);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float best = -INFINITY, m = 0.f;
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (8 * j + 2 * t + i < p.groups) {
              best = bs_larger(best, acc[j][2 * r + i]);
              m = fmaxf(m, most[j][2 * r + i]);
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          best = bs_larger(best, __shfl_xor_sync(kFullMask, best, o));
          m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        }
        if (!here[r]) best = -INFINITY;
        const int c = c0 + g + 8 * r;
        if (c < n) bs_leave(keys_at, c, best, m, ends, t == 0);
      }
      c0 = next;
    }
    ends.most = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(ends.most)));
    ends.least = __reduce_min_sync(kFullMask, ends.least);
    ends.largest = __reduce_max_sync(kFullMask, ends.largest);
  }
};

// kD 0: on the CUDA cores, kTiles quads of dims per lane.
template <typename C, int kD, int kTiles, int kTerms, bool kRagged>
__global__ void __launch_bounds__(32 * kBsMostWarps, kD == 0 && kTiles > 1 ? 1 : 2) block_select_kernel(SelectParams p, int ctas) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) BsShared s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = blockDim.x, warps = threads >> 5;
  const int rank = ctas > 1 ? (int)cl_rank() : 0;
  // (the heads of a token side by side: their bounds lie next to each other)
  const int unit = blockIdx.x / ctas, token = unit / p.hkv, row = token / p.width, head = unit - token * p.hkv;
  if (ctas > 1) cl_arrive();  // (no CTA is written to before it is there)
  if (rank == 0)
    for (int i = threadIdx.x; i < kBsBins; i += threads) s.hist[i] = 0;
  pdl_wait();
  pdl_release();
  int len = max(p.seq_lens[row], 0);
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
      for (unsigned i = threadIdx.x; i < (unsigned)p.budget; i += threads) out[i] = i < (unsigned)n ? (int)i : -1;  // (the step behind the largest budget passes 2^31)
    return;
  }
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  const long long q_at = ((long long)token * hq + (long long)head * p.groups) * p.d;
  const uint32_t keys_at = ctas > 1 ? cl_map(keys, 0) : smem_u32(keys);

  BsEnds ends{0.f, 0xffffffffu, 0u};
  float reach = 0.f;
  constexpr int kAtOnce = kD > 0 ? 16 : 8;  // blocks that a warp takes
  const int c0 = (rank * warps + warp) * kAtOnce, stride = ctas * warps * kAtOnce;
  if constexpr (kD > 0) {
    using Tiles = BsTiles<C, kD, kTiles, kTerms, kRagged>;
    __shared__ __align__(16) C qs[Tiles::kQBytes / 2];
    Tiles tiles;
    tiles.fetch_id(table, c0, n, lane);
    tiles.take(p, head, c0, n, lane);
#pragma unroll
    for (int piece = 0; piece < Tiles::kPieces; ++piece) tiles.ask(p, piece, 0, lane);
    tiles.fetch_id(table, c0 + stride, n, lane);

    reach = Tiles::stage(p, q_at, qs, lane);
    __syncthreads();
    tiles.run(p, qs, table, head, c0, stride, n, keys_at, ends, lane);
  } else {
    BsLanes<C, kTiles>::run(p, q_at, table, head, c0, stride, n, keys_at, ends, lane);
  }
  if (lane == 0) {
    s.reach[warp] = reach;
    const uint32_t at = (ctas > 1 ? cl_map(&s.ends[rank * warps + warp], 0) : smem_u32(&s.ends[rank * warps + warp]));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(ends.most) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + 4), "r"(ends.least) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + 8), "r"(ends.largest) : "memory");
  }
  if (ctas > 1) {
    cl_sync();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // the border among the columns that are not chosen anyway: chosen are keys above it, and the first `take_equal` of those that equal it
  const int begin = p.first, end = n - p.last;
  const uint32_t want = p.budget - p.first - p.last;
  uint32_t border = 0xffffffffu, take_equal = 0;
  bool all_equal_in = true;  // every key that equals the border is chosen
  int which = 0;
  if (want > 0) {
    uint32_t above, least = 0xffffffffu, largest = 0u, most = 0u;
    for (int i = lane; i < ctas * warps; i += 32) {
      const BsEnds e = s.ends[i];
      most = max(most, __float_as_uint(e.most));
      least = min(least, e.least);
      largest = max(largest, e.largest);
    }
    most = __reduce_max_sync(kFullMask, most);
    least = __reduce_min_sync(kFullMask, least);
    largest = __reduce_max_sync(kFullMask, largest);
    for (int w = 0; w < warps; ++w) reach = fmaxf(reach, s.reach[w]);
    if (largest >= kBsInfinity || least <= kBsLowest) {
      // Scores that an fp32 sum did not hold: of operands that are no numbers, or sums of numbers that left fp32, be it on the way to one that it holds.  In 64 bits
      // no sum of numbers does; such a block's place is found below, among all others that are numbers (eps is infinite).
      bool numbers = false;
      bs_rescore<true>(p, s, keys, table, q_at, head, begin, end, kBsInfinity, [&](int i, double x) {
        const bool number = fabs(x) < INFINITY;
        numbers |= number;
        if (lane == 0) keys[i] = number ? bs_key(fminf(fmaxf((float)x, -FLT_MAX), FLT_MAX)) : x < 0.0 ? kBsLowest : kBsInfinity;
      });
      if (__syncthreads_or(numbers)) most = 0x7f800000u;
      least = kBsMissing;
      largest = kBsInfinity;
    }
    border = bs_nth(keys, begin, end, want, least, largest, s, which, above);
    take_equal = want - above;
    all_equal_in = false;
    const float t = bs_float(border);
    if (t - t == 0.f) {
      // Products are exact on the tensor cores (in a chain of fused multiply-adds, too).  A sum of 32 dims is four steps for each term of the
      // queries, each cuts up to 17 numbers at 2^-23 of the largest: 68 * 2^-23 of the magnitudes for a term; D / 32 of them are added up in fp32.  Two
      // terms of eight bits, both cut, leave 2^-15 of a query at most (with the second one rounded 2^-16, and the compiler spills: 256 rows 51 us instead of
      // 45).  The magnitudes' own sum is off by a thousandth at most.
      constexpr double kCut = kD > 0 ? 68.0 * kTerms : 16.0, kSlip = kTerms > 1 ? 0x1p-15 : 0.0;
      const double eps = ((kCut + p.d / 16) * 0x1p-23 + kSlip) * 1.01 * (double)__uint_as_float(most) +
                         0x1p-124 * p.d * (1.0 + (double)reach);  // (and products and bounds below the normal numbers, that may be taken for zero)
      // (blocks that are not there, and scores that are no numbers, stay what they are)
      const uint32_t low = max(bs_key(__double2float_ru((double)t - 2.0 * eps)), kBsLowest + 1u),
                     high = min(bs_key(__double2float_rd((double)t + 2.0 * eps)), kBsInfinity - 1u);
      // how many are in for sure (in the upper half of the sum), and how many stand between
      uint32_t mine = 0;
      for (int i = begin + threadIdx.x; i < end; i += threads) {
        const uint32_t k = keys[i];
        mine += k > high ? 0x10000u : k >= low ? 1u : 0u;
      }
      const uint32_t all = bs_total(mine, s, which);
      const uint32_t in = all >> 16, between = all & 0xffffu;
      if (in + between == want) {
        border = low;
        all_equal_in = true;
      } else if (between <= kBsFew) {
        // a warp a score, then one warp ranks them; what is chosen gets the largest key, the others the smallest
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        for (int i = begin + threadIdx.x; i < end; i += threads) {
          const uint32_t k = keys[i];
          if (k >= low && k <= high) s.few[atomicAdd(&s.count, 1u)] = i;
        }
        __syncthreads();
        for (int j = warp; j < (int)between; j += warps) {
          const double x = bs_exact(p, q_at, ((long long)table[s.few[j]] * p.hkv + head) * 2 * p.d, lane);
          if (lane == 0) s.few_scores[j] = x;
        }
        __syncthreads();
        if (warp == 0 && lane < (int)between) {
          const double x = s.few_scores[lane];
          const uint32_t i = s.few[lane];
          uint32_t in_front = 0;
          for (int j = 0; j < (int)between; ++j) in_front += s.few_scores[j] > x || (s.few_scores[j] == x && s.few[j] < i);
          keys[i] = in + in_front < want ? 0xffffffffu : 0u;
        }
        __syncthreads();
        border = high;
        all_equal_in = true;
      } else {
        // keys anew: 0 out, all ones in, between the two the score in 64 bits as a fixed-point number of a window that holds it
        double floor_ = (double)t - 3.0 * eps, unit = 4294967290.0 / (6.0 * eps);
        for (int i = begin + threadIdx.x; i < end; i += threads) {
          const uint32_t k = keys[i];
          keys[i] = k > high ? 0xffffffffu : k >= low ? 1u : 0u;
        }
        border = 1u;
        for (;;) {
          bs_rescore(p, s, keys, table, q_at, head, begin, end, border, [&](int i, double x) {
            double u = (x - floor_) * unit;
            u = u > 0.0 ? u < 4294967290.0 ? u : 4294967290.0 : 0.0;
            if (lane == 0) keys[i] = 1u + (uint32_t)u;
          });
          border = bs_nth(keys, begin, end, want, 0u, 0xffffffffu, s, which, above);
          take_equal = want - above;
          uint32_t equal = 0;
          for (int i = begin + threadIdx.x; i < end; i += threads) equal += keys[i] == border;
          if (bs_total(equal, s, which) == take_equal) break;
          // more of one key than there is room for: equal scores, or a window that is too wide for them
          double lowest = INFINITY, highest = -INFINITY;
          bs_rescore(p, s, keys, table, q_at, head, begin, end, border, [&](int, double x) {
            lowest = x < lowest ? x : lowest;
            highest = x > highest ? x : highest;
          });
          if (lane == 0) s.low[warp] = lowest, s.high[warp] = highest;
          __syncthreads();
          for (int w = 0; w < warps; ++w) {
            lowest = s.low[w] < lowest ? s.low[w] : lowest;
            highest = s.high[w] > highest ? s.high[w] : highest;
          }
          if (lowest == highest) break;
          floor_ = lowest;
          unit = 4294967290.0 / (highest - lowest);
          for (int i = begin + threadIdx.x; i < end; i += threads) {
            const uint32_t k = keys[i];
            keys[i] = k > border ? 0xffffffffu : k == border ? 1u : 0u;
          }
          border = 1u;
          __syncthreads();
        }
      }
    }
  }

  // the columns in ascending order: each thread a run of neighbours
  const int each = (n + threads - 1) / threads, lo = min(n, (int)threadIdx.x * each), hi = min(n, lo + each);
  uint32_t total, e = 0;
  if (!all_equal_in) {
    uint32_t equal = 0;
    for (int i = max(lo, begin); i < min(hi, end); ++i) equal += keys[i] == border;
    e = bs_scan(equal, s, which, total);
  } else {
    take_equal = 0xffffffffu;
  }
  auto chosen = [&](int i, uint32_t& seen) {
    if (i < begin || i >= end) return true;
    if (want == 0) return false;
    const uint32_t k = keys[i];
    if (k == border) return seen++ < take_equal;
    return k > border;
  };
  uint32_t mine = 0, seen = e;
  for (int i = lo; i < hi; ++i) mine += chosen(i, seen);
  uint32_t at = bs_scan(mine, s, which, total);
  seen = e;
  for (int i = lo; i < hi; ++i)
    if (chosen(i, seen)) {
      if (at < (uint32_t)p.budget) out[at] = i;
      ++at;
    }
}

// How a call is cut: CTAs per cluster and their warps.  A CTA has ~8 us beside its stream (ids, queries, border, output), which others hide.
//   * Many rows, or short ones: four warps each, four CTAs to an SM (256 rows of 128 - 512 blocks, 2 heads of 256: 42 us, two CTAs each 46, four 52; 250
//     rows of 190: 21, with eight warps 26).
//   * Few long rows: eight warps, as many CTAs as are resident at once (64 rows of 1000: two 27, four 32; 32: four 19, eight 25), and twice as many where each would still
//     have more than 1024 blocks, so that the longest rows are not left alone at the end (64 rows of 1024 - 4096: two 81, four 78).
//   * At most a CTA per tile of its warps, or per two of them where the CTAs do not all have an SM of their own (16 rows of 1000: four 15.2, eight
//     16.2; 8 rows: four 13.4, eight 12.5).
struct BsPlan {
  int ctas, warps;
};
static BsPlan block_select_plan(long long units, long long columns, int sms) {
  const int warps = units > 2LL * sms || columns <= 512 ? 4 : 8;
  long long c = units > 2LL * sms ? 1 : (16LL / warps) * sms / units;
  if (columns > 1024 * c) c *= 2;
  const long long tiles = (columns + 16 * warps - 1) / (16 * warps);
  if (c > tiles) c = tiles;
  if (c > kBsMostCtas) c = kBsMostCtas;
  if (units * c > sms && c > (tiles + 1) / 2) c = (tiles + 1) / 2;
  return {(int)(c < 1 ? 1 : c), warps};
}

template <typename C, int kD, int kTiles, int kTerms, bool kRagged = false>
static int launch_block_select(const SelectParams& p, cudaStream_t stream) {
  auto* kernel = block_select_kernel<C, kD, kTiles, kTerms, kRagged>;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBsMostColumns * 4) == cudaSuccess;
      }))
    return NVJ_ERR_LAUNCH;
  const long long tokens = (long long)p.rows * p.width;
  const BsPlan plan = block_select_plan(tokens * p.hkv, p.table_width, 148);
  if (tokens * p.hkv * plan.ctas > 0x7fffffffLL) return NVJ_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tokens * p.hkv * plan.ctas), 1, 1);
  cfg.blockDim = dim3(32 * plan.warps, 1, 1);
  cfg.dynamicSmemBytes = p.table_width > p.budget ? (size_t)p.table_width * 4 : 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = plan.ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = plan.ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, plan.ctas) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
}
template <typename C, int kD, int kTerms>
static int launch_block_select_heads(const SelectParams& p, cudaStream_t stream) {
  if (p.d != kD) return p.groups <= 8 ? launch_block_select<C, kD, 1, kTerms, true>(p, stream) : launch_block_select<C, kD, 2, kTerms, true>(p, stream);
  return p.groups <= 8 ? launch_block_select<C, kD, 1, kTerms>(p, stream) : launch_block_select<C, kD, 2, kTerms>(p, stream);
}
// Up to 16 query heads of a kv head.
template <typename C, int kTerms>
static int launch_block_select_dims(const SelectParams& p, cudaStream_t stream) {
  if (p.d > 128) return launch_block_select_heads<C, 256, kTerms>(p, stream);
  if (p.d > 64) return launch_block_select_heads<C, 128, kTerms>(p, stream);
  return launch_block_select_heads<C, 64, kTerms>(p, stream);
}
// block_select_bf16.cu, block_select_f16.cu
int launch_block_select_bf16(const SelectParams& p, cudaStream_t stream);
int launch_block_select_f16(const SelectParams& p, cudaStream_t stream);

}  // namespace nvj
