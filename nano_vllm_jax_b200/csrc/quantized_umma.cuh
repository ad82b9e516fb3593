// Attention over the 8-bit paged cache on the 5th-generation tensor cores (tcgen05, kind::f8f6f4): the kernel of large batches of
// rows of few query tokens.  Included by one file per type of query (quantized_umma_*.cu).
//
// e4m3 is an operand type of the tensor cores, so K and V need no conversion and go from memory to shared memory and no further; what
// has to become e4m3 is the other side, and a number becomes a sum of e4m3 terms: t0 = rne(x), t1 = rne(u (x - t0)), ..., each with
// four bits of it; u = 32 for queries, 16 for weights.  bf16 queries are three terms, or two where a CTA has more than eight columns, f16 three, f32
// five (2^-20); the weights of the softmax five (2^-20, and never closer than 2^-26, the last place of the fifth term: the largest weight is kept between
// 2^3 and 2^8, so that a key 2^8 below it still has 2^-21).  The last term's last place bounds a query's small numbers, too: they are right to 2^-23, 2^-28
// or 2^-38 of the row's largest number, with two, three or five terms (exact, in bf16, from 2^-15 of it on with two, in f16 from 2^-17 on).  One of 256 dims
// 2^12 times the others, which decide: 1.2e-6 of the result in bf16 and one token (with two terms and u = 16 it was 3.4e-4), 2.2e-6 in f16, 4e-7 in f32.
// The terms are columns of their own, added with their powers of u when a result is read:
//   S^T = K Q^T    [128 keys x kQTerms * kC]            32 dims per MMA, K and Q from shared memory, K-major;
//   O^T = V^T P^T  [kDim / 128 x 128 dims x 5 * kC]     32 keys per MMA, V and the weights from shared memory, MN-major.
// A tile of 128 keys of one kv head is 64 KiB (head_dim 256), 1.4 us of an SM's share of the memory; its products take a fraction of
// that, and its softmax (thread = key) ~ 150 instructions per warp for four columns, where the mma.sync form, which converts every
// number in registers, spends 5500 on the same bytes.
//
// Work split: CTA = (range, kv head and column tile).  The units of 16 to 64 keys of all rows form one sequence that is cut into equal ranges
// (decode_parts.cuh); rows cut over ranges leave partials, folded by a second small launch.
//   softmax    thread = key, in groups of four warps.  Up to eight columns two groups take the tiles in turn, each with
//              references, sums and accumulators of its own (a tile's chain of waits, from its scores to its weights, is longer than
//              its bytes: one group alone took 1.85 us per tile of 64 KiB); of 16 or 24 two or three groups take eight each (two of twelve
//              columns 2.8 us slower on 64 rows of 5 tokens).
//              Scores from tensor memory, times the K scale of the key's block, plus the log2 of its V scale; weights exp2(that -
//              reference) as e4m3 terms into shared memory; their sum with the V scale divided out again, relative to the largest so far.
//              Thread = dim when a row's segment ends.
//   2 warps    MMA issue: the scores (up to two tiles ahead), the weighted sums.
//   1 warp     TMA producer: boxes of a unit's keys [8-key group][128-byte chunk][8 keys][128 B], 128-byte swizzle, into rings of tiles of K
//              and of V (160 KiB), and with K the scales of its blocks.
//   1 warp     the queries, up to two segments ahead: scaled to 2^7 - 2^8 by a power of two per column, split into terms.
// Measured on several GPUs, 8 bf16 heads of 256 over 2: 256 rows of 1024 - 4096 keys 107 - 113 us (92 - 96% of the copy rate), 64 of 8192 - 32768 200 - 208
// us (99 - 103%), 64 of 1024 - 4096 with 5 tokens each 48 - 50 us (53 - 55%: bound by a tile's way from scores to weights, 1.75 us where its bytes take
// 1.4); 48 f16 rows of 200 - 3000 keys, 32 heads of 128 over 8, 38.1 us (64%: 5 us until the first scores, 5 for the fold).
// Every wait is bounded; after a timeout (NVJ_DEV_TIMEOUT) the kernel stops issuing, lets copies land and frees its tensor
// memory.  A block id outside the pool is flagged, fetched from beyond the tensor (zeros) and its keys are left out.
#pragma once

#include <cuda.h>

#include "decode_parts.cuh"
#include "quantized_kv.cuh"
#include "quantized_umma_params.cuh"
#include "umma.cuh"

namespace nvj {

constexpr int kQuTile = 128;    // keys per tile
constexpr int kQuUnits = 8;     // boxes per tile, at most: a box is a unit of 16, 32 or 64 keys of one block (QuParams::unit)
constexpr int kQuPTerms = 5;
// Named barriers (0 is __syncthreads'): a softmax group's, from this one on; all groups'; everybody's but the producer's.  None has two meanings: after a
// wait that ran out a group may meet the others where another one still votes, with another number of threads.
constexpr int kQuBarGroup = 1, kQuBarAll = 4, kQuBarQueries = 5;
// The reference of a column's weights is set 2^3 below its largest weight and moved when one would pass 2^8 (e4m3 ends at 448).
constexpr float kQuNone = -3e38f, kQuSlack = 8.f, kQuLift = 3.f;
// V scales reach from 2^-117 (the append's for a block of zeros) to 2^119.  A sum of weights is of exp2(score - (reference - v_top)), v_top the
// log2 of the group's largest V scale so far, but for kQuFar; the weight of a key whose block is 2^kQuFar quieter may be zero and says nothing of that
// any more, so that such keys take an exponential of their own (for all keys: 64 rows of 5 tokens 48.6 -> 53 us).  Next to a loud block
// their share may be as large as 2^(score's lead): it ends at 2^kQuMost, where a row's loud keys weigh 2^-kQuMost and less.  So what a
// row's output owes to values 2^-90 of the largest of its blocks and smaller may be off, by 2^-90 of that largest one at most.
constexpr float kQuFar = 40.f, kQuMost = 106.f, kQuMostSum = 0x1p108f;  // (10^6 keys of 2^kQuMost are an f32 number)

template <typename T, int kSharing>
constexpr int quq_terms() {  // (a third one of bf16 is free up to eight columns; with 20 it takes 64 rows 2.8 us of 49)
  return sizeof(T) == 4 ? 5 : std::is_same<T, __half>::value || kSharing == 1 ? 3 : 2;
}

// kCg: columns of a softmax thread; kSharing: groups that share a tile, a region of the columns each.  One: two groups take the tiles in turn.
template <typename T, int kDim, int kCg, int kSharing>
struct QuLayout {
  static constexpr bool kByTiles = kSharing == 1;
  static constexpr int kGroups = kByTiles ? 2 : kSharing, kSoftmaxThreads = 128 * kGroups, kThreads = kSoftmaxThreads + 128;
  static constexpr int kC = kCg * kSharing;  // columns of the CTA
  static constexpr int kRegions = kSharing;  // of a row of query terms or weights
  static constexpr int kQTerms = quq_terms<T, kSharing>();
  static constexpr int kChunks = kDim / 128;
  static constexpr int kSRegion = kQTerms * kCg;                        // columns of S: [region][term][kCg]
  static constexpr int kORegion = kQuPTerms * kCg;                      // columns of O: [region][term][kCg]
  static constexpr int kNS = (kRegions * kSRegion + 15) / 16 * 16;      // (N of an MMA: multiples of 16)
  static constexpr int kNO = (kRegions * kORegion + 15) / 16 * 16;
  static constexpr int kSets0 = (512 - 2 * kNS) / (kNO * kChunks);      // accumulators that take the tiles in turn: shorter sums
  static constexpr int kSets = kByTiles ? (kSets0 < 4 ? 2 : 4) : (kSets0 < 2 ? 1 : 2);
  static constexpr int kColO = 2 * kNS;                                 // S twice, then the sets
  static constexpr int kTileBytes = kQuTile * kDim;                     // of K (or V)
  static constexpr int kQChunk = kNS * 128;                             // bytes of a chunk of the query terms
  static constexpr int kQBytes = kChunks * kQChunk, kWBytes = kQuTile * 128;
  static constexpr int kFit = (232448 - 1024 - 6144 - 2 * kQBytes - 2 * kWBytes) / kTileBytes;
  static constexpr int kSlots = kFit < 160 * 1024 / kTileBytes ? kFit : 160 * 1024 / kTileBytes;
  static constexpr int kKSlots = kSlots / 2, kVSlots = kSlots - kKSlots;  // a ring of tiles of K, one of V (which waits for its weights)
  static_assert(kQuBarGroup + kGroups <= kQuBarAll && kQuBarAll != kQuBarQueries, "a barrier of its own for every meeting");
  static_assert(kNO <= 128 && kNS <= 256, "a row of weights is 128 bytes");
  static_assert(kColO + kSets * kChunks * kNO <= 512, "tensor memory");
  static_assert(kKSlots >= 1 && kVSlots >= 2, "the rings");
};

template <class L>
struct QuSmem {
  alignas(1024) char k[L::kKSlots][L::kTileBytes];
  alignas(1024) char v[L::kVSlots][L::kTileBytes];
  alignas(1024) char q[2][L::kChunks][L::kQChunk];  // by segment parity: [chunk][region, term, column][128 B]
  alignas(1024) char w[2][L::kWBytes];              // by tile parity: weights' terms [key][128 B]
  alignas(8) unsigned long long k_full[L::kKSlots], k_empty[L::kKSlots], v_full[L::kVSlots], v_empty[L::kVSlots], q_full[2], q_free[2], s_full[2], p_full[2], pv_done[2], o_full, o_free;
  alignas(16) float k_unit[8][kQuUnits], v_unit[8][kQuUnits];  // by tile: the scales of its units' blocks; V's -1: no such block
  alignas(16) float factor[4][L::kC];  // by segment: what a column's products are multiplied by, and the keys it may see
  alignas(16) int limit[4][L::kC];
  int seen[4];  // by segment: the largest limit, hence the keys that any column sees
  alignas(16) float red[L::kGroups][4][8];  // per group and warp
  float red_v[L::kGroups][4];
  float m[L::kGroups][8], mv[L::kGroups][8];  // at the end: references of the sum of the weights, and of the weighted sums
  int col_row[L::kC], col_token[L::kC];  // of a column: its row of the row's queries (and of its output), its token
  int lens[L::kThreads];  // of rows lens_from ..
  alignas(16) float out_f[2][L::kC];  // what a group's sums are multiplied by at the end
  int scan[16];
  int start_b, start_j, lens_from, abort_flag;
  uint32_t tmem_base;
};

__device__ __forceinline__ void qu_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// Instruction descriptor, kind::f8f6f4: fp32 accumulate, e4m3 A and B, M = 128.
__device__ __forceinline__ constexpr uint32_t qu_idesc(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void qu_load(uint32_t dst, const CUtensorMap* map, int group, int head, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %2, %2, %3, %4}], [%5], %6;"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(group), "r"(head), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void qu_tmem_st8(uint32_t taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
                 "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
               : "memory");
}
__device__ __forceinline__ void qu_sts4(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void qu_sts2(uint32_t at, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void qu_sts1(uint32_t at, uint32_t x) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }
// N (a multiple of 4) numbers from a 16-byte boundary in shared memory on.
template <int N>
__device__ __forceinline__ void qu_lds(float (&v)[N], const float* from) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(from + i);
    v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
  }
}
template <int N>
__device__ __forceinline__ void qu_lds(int (&v)[N], const int* from) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const int4 x = *reinterpret_cast<const int4*>(from + i);
    v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
  }
}
// Whether `mine` holds in any of the `threads` threads that meet at barrier `id`.
template <int kThreads>
__device__ __forceinline__ bool qu_meet_any(int id, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any) : "r"((uint32_t)mine), "r"(id), "n"(kThreads) : "memory");
  return any != 0;
}
// The warp's largest x (order-preserving integers; a NaN with a clear sign counts as the largest).
__device__ __forceinline__ float qu_warp_max(float x) {
  const int i = __float_as_int(x), k = __reduce_max_sync(kFullMask, i ^ ((i >> 31) & 0x7fffffff));
  return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}
// Inclusive scan of one int per thread over the CTA.
template <int kThreads>
__device__ __forceinline__ int qu_inclusive_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(kFullMask, v, o);
    if (lane >= o) v += n;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int x = warp_sums[w];
    if (w < warp) before += x;
    all += x;
  }
  total = all;
  return v + before;
}

// A place in a ring.  (K and V have rings of their own: the barriers of a ring have to be waited on in the order of its uses, and the two
// products are issued by a warp each.)
template <int kSlots>
struct QuRing {
  int at = 0;
  uint32_t phase = 0;
  bool reuse = false;  // the place has been used before
  __device__ __forceinline__ void step() {
    if (++at == kSlots) { at = 0; phase ^= 1u; reuse = true; }
  }
};
// The CTA's segments: units [j0, j0 + n) of row b, which has nb of them and len keys.  A tile is `per` units.
struct QuSeg {
  int b, j0, n, nb, len;
  __device__ __forceinline__ int tiles(int per) const { return (n + per - 1) / per; }
  __device__ __forceinline__ int tile_units(int t, int per) const { return min(n - t * per, per); }
  __device__ __forceinline__ bool whole() const { return n == nb; }
};
__device__ __forceinline__ int qu_row_units(const QuParams& a, int len) { return (len + a.unit - 1) >> a.unit_log2; }
struct QuWalk {  // (next_seg of decode_parts.cuh, over units)
  int b, j;
  long long g, g1;
  const int* lens;  // in shared memory: an access to global memory takes up to 2 us here while the copies are under way
  int lens_from, lens_count;
  __device__ __forceinline__ bool next(const QuParams& a, const DecodeParams& p, QuSeg& s) {
    while (g < g1 && b < p.batch) {
      const int len = b - lens_from < lens_count ? lens[b - lens_from] : decode_row_len(p, b), nb = qu_row_units(a, len), all = blocks_in_sequence(p, nb);
      if (j >= all) { ++b; j = 0; continue; }
      const int take = (long long)(all - j) < g1 - g ? all - j : (int)(g1 - g);
      const int j0 = j, j1 = min(j + take, nb), row = b;
      g += take; ++b; j = 0;  // either the row is finished or the range is
      if (j1 <= j0) continue;  // only the row's end lies here
      s = QuSeg{row, j0, j1 - j0, nb, len};
      return true;
    }
    return false;
  }
};
// What the range that begins at position j of row b, and at g0 of the sequence, tells the fold (umma_cut of decode_parts.cuh).
__device__ __forceinline__ UmmaCut qu_cut(const QuParams& a, const DecodeParams& p, const Partition& pt, int range, int b, int j, long long g0) {
  const int nb = qu_row_units(a, decode_row_len(p, b));
  const int first = pt.cta_of(g0 - j);
  if (j == 0 || j >= nb || first != range - 1) return kNoCut;
  return UmmaCut{b, first, pt.cta_of(g0 - j + nb - 1), 0};
}

// ---- TMA loads ------------------------------------------------------------------------------------------------------------
template <class L>
__device__ __forceinline__ void qu_producer(const CUtensorMap* k_map, const CUtensorMap* v_map, const QuParams& a, const DecodeParams& p, QuSmem<L>& sm,
                                            int head, QuWalk walk, int lane) {
  const int per = kQuTile / a.unit, per_block = p.block_size / a.unit;
  const uint32_t unit_bytes = (uint32_t)a.unit * L::kChunks * 128;
  const int oob = (int)(p.num_blocks * (p.block_size / 8));  // a box that starts here is filled with zeros
  uint64_t policy;  // every block is read once
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  auto ids_at = [&](const QuSeg& s, int i) {
    return i + lane < s.n ? p.block_tables[(long long)s.b * p.table_width + (s.j0 + i + lane) / per_block] : 0;
  };
  QuRing<L::kKSlots> k_at;
  QuRing<L::kVSlots> v_at;
  uint32_t tile = 0;
  QuSeg s, nxt;
  bool have = walk.next(a, p, s);
  int ids = have ? ids_at(s, 0) : 0;
  while (have) {
    bool more = false;
    int next_first = 0;
    for (int i0 = 0; i0 < s.n; i0 += 32) {  // 32 units = 4 tiles or more at a time
      const int ahead = ids_at(s, i0 + 32);
      const int n = min(s.n - i0, 32);
      const bool bad = lane < n && (ids < 0 || ids >= p.num_blocks);
      if (bad) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      const int group = bad || lane >= n ? oob : ids * (p.block_size / 8) + (s.j0 + i0 + lane) % per_block * (a.unit / 8);
      for (int i = 0; i < n; i += per) {
        const int cnt = min(n - i, per), mine = __shfl_sync(kFullMask, group, (i + lane) & 31);  // a lane per unit
        const int id = __shfl_sync(kFullMask, bad ? -1 : ids, (i + lane) & 31);
        {
          if (k_at.reuse && !um_wait(&sm.k_empty[k_at.at], k_at.phase ^ 1u, &sm.abort_flag, p.status)) return;
          const uint32_t full = smem_u32(&sm.k_full[k_at.at]);
          // The scales with K, counted on its barrier: eight tiles' places, so that the ones of tile n have been read before those
          // of tile n + 8 come.  (Fetched by the softmax threads a tile ahead, each waited ~1100 cycles per tile for them: with the
          // memory busy an access takes longer than two tiles.)
          if (lane < cnt) {
            float *ku = &sm.k_unit[tile & 7u][lane], *vu = &sm.v_unit[tile & 7u][lane];
            if (id >= 0) {
              const long long entry = (long long)id * a.num_kv_heads + head;
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(ku)), "l"(a.k_scale + entry) : "memory");
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(vu)), "l"(a.v_scale + entry) : "memory");
              asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(full) : "memory");
            } else {
              *ku = 0.f;
              *vu = -1.f;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)cnt * unit_bytes);
          __syncwarp();
          if (lane < cnt) qu_load(smem_u32(sm.k[k_at.at]) + lane * unit_bytes, k_map, mine, head, full, policy);
          __syncwarp();
          k_at.step();
        }
        {
          if (v_at.reuse && !um_wait(&sm.v_empty[v_at.at], v_at.phase ^ 1u, &sm.abort_flag, p.status)) return;
          const uint32_t full = smem_u32(&sm.v_full[v_at.at]);
          if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)cnt * unit_bytes);
          __syncwarp();
          if (lane < cnt) qu_load(smem_u32(sm.v[v_at.at]) + lane * unit_bytes, v_map, mine, head, full, policy);
          __syncwarp();
          v_at.step();
        }
        ++tile;
      }
      ids = ahead;
      if (i0 == 0) {  // the row behind this one, once the first copies are on their way
        more = walk.next(a, p, nxt);
        if (more) next_first = ids_at(nxt, 0);
      }
    }
    s = nxt;
    ids = next_first;
    have = more;
  }
}

// ---- MMA issue -------------------------------------------------------------------------------------------------
// A warp for either product: a tile's ~ 500 cycles of waits, descriptors and commits on each side would otherwise add up to more than its
// bytes take (head_dim 128).  S(n) takes the place of S(n - 2), which has been read when that tile's weights are there.
template <class L>
__device__ __forceinline__ void qu_scores_warp(QuSmem<L>& sm, const QuParams& a, const DecodeParams& p, uint32_t tmem, QuWalk walk) {
  constexpr uint32_t idesc = qu_idesc(L::kNS, false, false);
  const uint64_t k_desc0 = umma_desc(smem_u32(sm.k[0]), 16, L::kChunks * 1024);  // keys are rows: groups of 8
  const uint64_t q_desc0 = umma_desc(smem_u32(sm.q[0][0]), 16, 1024);
  QuRing<L::kKSlots> at;
  QuSeg s;
  const int per = kQuTile / a.unit;
  uint32_t n = 0;
  for (uint32_t seg = 0; walk.next(a, p, s); ++seg) {
    const uint32_t qb = seg & 1u;
    const int nt = s.tiles(per);
    for (int t = 0; t < nt; ++t, ++n) {
      if (t == 0 && !um_wait(&sm.q_full[qb], (seg >> 1) & 1u, &sm.abort_flag, p.status)) return;
      if (!um_wait(&sm.k_full[at.at], at.phase, &sm.abort_flag, p.status)) return;
      if (n >= 2 && !um_wait(&sm.p_full[n & 1u], ((n >> 1) - 1) & 1u, &sm.abort_flag, p.status)) return;
      tc_fence_after_sync();
      if (um_elect_one()) {
        // (rows of keys that the tile does not have are computed from whatever lies there, and masked)
        const uint64_t k_desc = k_desc0 + (uint64_t)((at.at * L::kTileBytes) >> 4), q_desc = q_desc0 + (uint64_t)((qb * L::kQBytes) >> 4);
#pragma unroll
        for (int ks = 0; ks < L::kChunks * 4; ++ks)
          qu_mma(tmem + (n & 1u) * L::kNS, k_desc + (uint64_t)(((ks >> 2) * 1024 + (ks & 3) * 32) >> 4),
                 q_desc + (uint64_t)(((ks >> 2) * L::kQChunk + (ks & 3) * 32) >> 4), idesc, ks > 0 ? 1u : 0u);
        umma_commit(smem_u32(&sm.s_full[n & 1u]));
        umma_commit(smem_u32(&sm.k_empty[at.at]));
        if (t == nt - 1) umma_commit(smem_u32(&sm.q_free[qb]));
      }
      __syncwarp();
      at.step();
    }
  }
}
template <class L>
__device__ __forceinline__ void qu_sums_warp(QuSmem<L>& sm, const QuParams& a, const DecodeParams& p, uint32_t tmem, QuWalk walk) {
  constexpr uint32_t idesc = qu_idesc(L::kNO, true, true);
  const uint64_t v_desc0 = umma_desc(smem_u32(sm.v[0]), 1024, L::kChunks * 1024);  // dims are rows, a chunk at a time; keys in groups of 8
  const uint64_t w_desc0 = umma_desc(smem_u32(sm.w[0]), 1024, 1024);
  QuRing<L::kVSlots> at;
  QuSeg s;
  const int per = kQuTile / a.unit;
  uint32_t n = 0;
  for (uint32_t seg = 0; walk.next(a, p, s); ++seg) {
    const int nt = s.tiles(per);
    const uint32_t n0 = n;
    for (int t = 0; t < nt; ++t, ++n) {
      if (!um_wait(&sm.v_full[at.at], at.phase, &sm.abort_flag, p.status)) return;
      if (!um_wait(&sm.p_full[n & 1u], (n >> 1) & 1u, &sm.abort_flag, p.status)) return;
      // the first weighted sums of a segment overwrite O: the segment before must have been read out
      if (t == 0 && seg > 0 && !um_wait(&sm.o_free, (seg - 1) & 1u, &sm.abort_flag, p.status)) return;
      tc_fence_after_sync();
      if (um_elect_one()) {
        const int steps = (s.tile_units(t, per) * a.unit + 31) / 32;
        const uint32_t o = tmem + L::kColO + ((n0 & 1u) + t) % L::kSets * (L::kChunks * L::kNO);
        const uint64_t v_desc = v_desc0 + (uint64_t)((at.at * L::kTileBytes) >> 4), w_desc = w_desc0 + (uint64_t)(((n & 1u) * L::kWBytes) >> 4);
        for (int i = 0; i < steps; ++i) {  // 32 keys, four groups of 8
          const uint32_t accumulate = (t >= L::kSets || i > 0) ? 1u : 0u;
          const uint64_t wd = w_desc + (uint64_t)((i * 32 * 128) >> 4), vd = v_desc + (uint64_t)((i * 32 * L::kChunks * 128) >> 4);
#pragma unroll
          for (int h = 0; h < L::kChunks; ++h) qu_mma(o + h * L::kNO, vd + (uint64_t)((h * 1024) >> 4), wd, idesc, accumulate);
        }
        umma_commit(smem_u32(&sm.pv_done[n & 1u]));
        umma_commit(smem_u32(&sm.v_empty[at.at]));
        if (t == nt - 1) umma_commit(smem_u32(&sm.o_full));
      }
      __syncwarp();
      at.step();
    }
  }
}

// ---- softmax and output.  Thread = key of the tile, then dim of the output ---------------------------------------
// (A wait that runs out does so for one warp and perhaps not for the next: a group's warps leave together, behind a meeting.)
template <class L, int kCg>
__device__ __forceinline__ void qu_softmax_warps(QuSmem<L>& sm, const QuParams& a, const DecodeParams& p, uint32_t tmem, int head, int hct, int ct,
                                                 QuWalk walk, int range, int group, int warp, int lane) {
  constexpr int kSRead = (L::kSRegion + 7) / 8, kORead = (kQuPTerms * kCg + 7) / 8;  // pieces of 8 columns
  constexpr bool kByTiles = L::kByTiles;
  constexpr int kDim = L::kChunks * 128, kWords = L::kORegion / 4;
  const int key = warp * 32 + lane, region = kByTiles ? 0 : group, first_col = kByTiles ? 0 : group * kCg, bar = kQuBarGroup + group;
  tmem += (uint32_t)(warp * 32) << 16;
  // a group that leaves early meets the other one, which waits at a segment's end or leaves as well
  auto give_up = [] { qu_meet_any<L::kSoftmaxThreads>(kQuBarAll, true); };
  QuRing<L::kVSlots> at;  // V's slot of the tile at hand
  QuSeg s;
  const int per = kQuTile / a.unit, my_unit = key >> a.unit_log2;
  uint32_t n = 0;
  for (uint32_t seg = 0; walk.next(a, p, s); ++seg) {
    const float* factor = sm.factor[seg & 3u] + first_col;
    const int* limit = sm.limit[seg & 3u] + first_col;
    const uint32_t n0 = n;
    bool begun = false;  // the group has had a tile of this segment
    float l[kCg], m[kCg], v_top = kQuNone;
#pragma unroll
    for (int c = 0; c < kCg; ++c) {
      l[c] = 0.f;
      m[c] = kQuNone;
    }
    const int nt = s.tiles(per);
    for (int t = 0; t < nt; ++t, ++n) {
      if (kByTiles && (int)(n & 1u) != group) {
        at.step();
        continue;
      }
      const int cnt = s.tile_units(t, per);
      const uint32_t buf = n & 1u, phase = (n >> 1) & 1u;
      // this thread's key; one that the tile does not have is behind everybody's last one
      const int at_key = my_unit < cnt ? (s.j0 + t * per) * a.unit + key : 0x7fffffff;
      const bool ok = um_wait(&sm.s_full[buf], phase, &sm.abort_flag, p.status);
      tc_fence_after_sync();
      const float k_unit = sm.k_unit[n & 7u][my_unit], v_unit = my_unit < cnt ? sm.v_unit[n & 7u][my_unit] : -1.f;
      const float v_log = v_unit >= 0.f ? __log2f(fmaxf(v_unit, 0x1p-126f)) : v_top;
      float sc[kCg];
      {
        float x[kSRead][8];
        const bool there = v_unit >= 0.f;
#pragma unroll
        for (int i = 0; i < kSRead; ++i) tmem_ld8(tmem + buf * L::kNS + region * L::kSRegion + 8 * i, x[i]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kSRead; ++i) tmem_loaded(x[i]);
        float by[kCg];
        int seen[kCg];
        qu_lds(by, factor);
        qu_lds(seen, limit);
#pragma unroll
        for (int c = 0; c < kCg; ++c) {
          float y = x[((L::kQTerms - 1) * kCg + c) / 8][((L::kQTerms - 1) * kCg + c) % 8];
#pragma unroll
          for (int j = L::kQTerms - 2; j >= 0; --j) y = fmaf(y, 0.03125f, x[(j * kCg + c) / 8][(j * kCg + c) % 8]);
          sc[c] = there && at_key < seen[c] ? fmaf(y, by[c] * k_unit, v_log) : -INFINITY;
        }
      }
      bool above = v_log > v_top + kQuFar || !begun;
#pragma unroll
      for (int c = 0; c < kCg; ++c) above |= sc[c] > m[c] + kQuSlack;
      if (qu_meet_any<128>(bar, !ok || above)) {
        // the first tile, or rarely a later one: the tile's maxima; what has been summed so far is brought to the new references, which every
        // thread finds for itself
#pragma unroll
        for (int c = 0; c < kCg; ++c) {
          const float x = qu_warp_max(sc[c]);
          if (lane == 0) sm.red[group][warp][c] = x;
        }
        {
          const float x = qu_warp_max(v_unit >= 0.f ? v_log : kQuNone);
          if (lane == 0) sm.red_v[group][warp] = x;
        }
        // (the group's weighted sums so far have to be complete)
        const uint32_t done = kByTiles ? n - 2 : n - 1;
        const bool complete = !begun || um_wait(&sm.pv_done[done & 1u], (done >> 1) & 1u, &sm.abort_flag, p.status);
        if (qu_meet_any<128>(bar, !ok || !complete)) return give_up();
        float f[kCg];
        const float v_most = fmaxf(fmaxf(sm.red_v[group][0], sm.red_v[group][1]), fmaxf(sm.red_v[group][2], sm.red_v[group][3]));
        const float v_now = v_most > v_top + kQuFar ? v_most : v_top, raised = v_now - v_top;
        v_top = v_now;
#pragma unroll
        for (int c = 0; c < kCg; c += 4) {
          float x[4], y[4];
          qu_lds(x, &sm.red[group][0][c]);
#pragma unroll
          for (int w = 1; w < 4; ++w) {
            qu_lds(y, &sm.red[group][w][c]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaxf(x[e], y[e]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float now = x[e] > m[c + e] + kQuSlack ? x[e] - kQuLift : m[c + e];  // (one whose scores stay under it keeps its reference)
            f[c + e] = ex2_approx(m[c + e] - now);
            l[c + e] *= ex2_approx(fminf((m[c + e] - now) + raised, 126.f));
            l[c + e] = l[c + e] > kQuMostSum ? kQuMostSum : l[c + e];
            m[c + e] = now;
          }
        }
        if (begun) {
          tc_fence_after_sync();
#pragma unroll 1
          for (int k = 0; k < L::kSets; ++k) {
            const int since = (k - (int)(n0 & 1u) + L::kSets) % L::kSets;  // the set's first tile in this segment
            if (since >= t || (kByTiles && (k & 1) != group)) continue;
#pragma unroll 1
            for (int h = 0; h < L::kChunks; ++h) {
              float o[kORead][8];
              const uint32_t from = tmem + L::kColO + (k * L::kChunks + h) * L::kNO + region * L::kORegion;
#pragma unroll
              for (int i = 0; i < kORead; ++i) tmem_ld8(from + 8 * i, o[i]);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < kORead; ++i) {
                tmem_loaded(o[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (8 * i + e < kQuPTerms * kCg) o[i][e] *= f[(8 * i + e) % kCg];
                qu_tmem_st8(from + 8 * i, o[i]);
              }
            }
          }
          tmem_st_wait();
        }
        begun = true;
      }
      // weights as e4m3 terms: byte term * kCg + column of the group's region of the key's row
      {
        float r[kCg];
        const float back = v_top - v_log;
        const bool far = back > kQuFar;
        const float inverse = far ? 0.f : ex2_approx(back);
#pragma unroll
        for (int c = 0; c < kCg; ++c) {
          r[c] = ex2_approx(sc[c] - m[c]);
          l[c] = fmaf(r[c], inverse, l[c]);
        }
        if (__builtin_expect(far, 0)) {
#pragma unroll
          for (int c = 0; c < kCg; ++c) l[c] += ex2_approx(fminf((sc[c] - m[c]) + back, kQuMost));
        }
        uint32_t bytes[kWords];
#pragma unroll
        for (int j = 0; j < kQuPTerms; ++j)
#pragma unroll
          for (int c = 0; c < kCg; c += 4) {
            const uint32_t x = q_pack2(r[c], r[c + 1]), y = q_pack2(r[c + 2], r[c + 3]);
            bytes[(j * kCg + c) / 4] = x | y << 16;
            if (j + 1 < kQuPTerms) {
              const float2 b0 = q_float2(q_half2(x)), b1 = q_float2(q_half2(y));
              r[c] = (r[c] - b0.x) * 16.f;
              r[c + 1] = (r[c + 1] - b0.y) * 16.f;
              r[c + 2] = (r[c + 2] - b1.x) * 16.f;
              r[c + 3] = (r[c + 3] - b1.y) * 16.f;
            }
          }
        // (the weights of tile n - 2, in the same place, have been used: almost always long ago; a wait that runs out shows at the next meeting)
        if (n >= 2) um_wait(&sm.pv_done[buf], ((n >> 1) - 1) & 1u, &sm.abort_flag, p.status);
        const uint32_t w_row = smem_u32(sm.w[buf]) + key * 128;
        // (bytes of the row behind the last region hold anything: they only reach columns of O that nothing reads)
        const int piece = region * (kWords / 2);  // of 8 bytes: a region is 2.5 or 5 of the swizzle's 16
        if constexpr (kWords % 4 == 1) {
#pragma unroll
          for (int i = 0; i < kWords / 4; ++i)
            qu_sts4(w_row + ((i ^ (key & 7)) << 4), bytes[4 * i], bytes[4 * i + 1], bytes[4 * i + 2], bytes[4 * i + 3]);
          qu_sts1(w_row + (((kWords / 4) ^ (key & 7)) << 4), bytes[kWords - 1]);
        } else {
#pragma unroll
          for (int i = 0; i < kWords / 2; ++i)
            qu_sts2(w_row + ((((piece + i) >> 1) ^ (key & 7)) << 4) + ((piece + i) & 1) * 8, bytes[2 * i], bytes[2 * i + 1]);
        }
      }
      // V rows of keys that are not there, or that no column sees, weigh nothing, but may hold anything: 0 x NaN is not 0
      const int seen = sm.seen[seg & 3u];
      if ((kByTiles || group == 0) && ((cnt * a.unit & 31) || (s.j0 + t * per + cnt) * a.unit > seen)) {
        if (qu_meet_any<128>(bar, !um_wait(&sm.v_full[at.at], at.phase, &sm.abort_flag, p.status))) return give_up();
        if (key < (cnt * a.unit + 31) / 32 * 32 && at_key >= seen) {
          const uint32_t v_row = smem_u32(sm.v[at.at]) + (key >> 3) * (8 * kDim) + (key & 7) * 128;
#pragma unroll
          for (int i = 0; i < kDim / 16; ++i) qu_sts4(v_row + (i >> 3) * 1024 + (i & 7) * 16, 0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      mbar_arrive(smem_u32(&sm.p_full[buf]));
      at.step();
    }
    // ---- end of the segment: sums over the keys, then the output or the partial
#pragma unroll
    for (int c = 0; c < kCg; ++c) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l[c] += __shfl_xor_sync(kFullMask, l[c], o);
      if (lane == 0) sm.red[group][warp][c] = l[c];
    }
    if (key == 0) {
#pragma unroll
      for (int c = 0; c < kCg; ++c) {
        sm.mv[group][c] = m[c];
        sm.m[group][c] = m[c] > kQuNone ? m[c] - v_top : kQuNone;
      }
    }
    if (qu_meet_any<L::kSoftmaxThreads>(kQuBarAll, !um_wait(&sm.o_full, seg & 1u, &sm.abort_flag, p.status))) return;
    const bool final_row = s.whole();
    const long long slot = (long long)partial_slot(range, s.j0 == 0) * a.hcts + hct;
    const int tid = group * 128 + key;
    if (tid < L::kC) {
      auto sum_of = [&](int g, int c) { return (sm.red[g][0][c] + sm.red[g][1][c]) + (sm.red[g][2][c] + sm.red[g][3][c]); };
      if constexpr (kByTiles) {
        const float s0 = sum_of(0, tid), s1 = sum_of(1, tid), top = fmaxf(sm.m[0][tid], sm.m[1][tid]);
        const float sum = s0 * ex2_approx(sm.m[0][tid] - top) + s1 * ex2_approx(sm.m[1][tid] - top);
        const float f = sum == 0.f ? 0.f : final_row ? 1.f / sum : 1.f;
        sm.out_f[0][tid] = s0 == 0.f ? 0.f : f * ex2_approx(sm.mv[0][tid] - top);
        sm.out_f[1][tid] = s1 == 0.f ? 0.f : f * ex2_approx(sm.mv[1][tid] - top);
        if (!final_row) *reinterpret_cast<float2*>(a.part_ml + (slot * L::kC + tid) * 2) = make_float2(top, sum);
      } else {
        const int g = tid / kCg, c = tid % kCg;
        const float sum = sum_of(g, c);
        sm.out_f[0][tid] = sum == 0.f ? 0.f : ex2_approx(sm.mv[g][c] - sm.m[g][c]) * (final_row ? 1.f / sum : 1.f);
        if (!final_row) *reinterpret_cast<float2*>(a.part_ml + (slot * L::kC + tid) * 2) = make_float2(sm.m[g][c], sum);
      }
    }
    qu_meet_any<L::kSoftmaxThreads>(kQuBarAll, false);
    tc_fence_after_sync();
    const int columns = min(a.columns - ct * L::kC, L::kC);
    const long long token = a.query_start_loc ? (long long)a.query_start_loc[s.b] : (long long)s.b * a.width;
    // a piece of the output is a chunk of the dims of a region; the single one of head_dim 128 and up to 8 columns is shared
    constexpr bool kShared = L::kChunks * L::kRegions == 1;
#pragma unroll 1
    for (int piece = kShared ? 0 : group; piece < L::kChunks * L::kRegions; piece += L::kGroups) {
      const int h = piece % L::kChunks, r = piece / L::kChunks;
      float y[kCg];
#pragma unroll
      for (int c = 0; c < kCg; ++c) y[c] = 0.f;
#pragma unroll 1
      for (int k = 0; k < L::kSets; ++k) {
        if ((k - (int)(n0 & 1u) + L::kSets) % L::kSets >= nt) continue;  // no tile of this segment
        float o[kORead][8], part[kCg];  // high terms last: small numbers are added first
        const uint32_t from = tmem + L::kColO + (k * L::kChunks + h) * L::kNO + r * L::kORegion;
#pragma unroll
        for (int i = 0; i < kORead; ++i) tmem_ld8(from + 8 * i, o[i]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kORead; ++i) tmem_loaded(o[i]);
#pragma unroll
        for (int c = 0; c < kCg; ++c) {
          part[c] = o[((kQuPTerms - 1) * kCg + c) / 8][((kQuPTerms - 1) * kCg + c) % 8];
#pragma unroll
          for (int j = kQuPTerms - 2; j >= 0; --j) part[c] = fmaf(part[c], 0.0625f, o[(j * kCg + c) / 8][(j * kCg + c) % 8]);
          const float f = sm.out_f[kByTiles ? k & 1 : 0][r * kCg + c];
          if (!(f == 0.f)) y[c] = fmaf(part[c], f, y[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < kCg; ++c) {
        const int col = r * kCg + c;
        if (col >= columns || (kShared && c / (kCg / 2) != group)) continue;
        float* to = final_row ? a.out + (token * a.num_q_heads + sm.col_row[col]) * kDim : a.part_acc + (slot * L::kC + col) * kDim;
        to[h * 128 + key] = y[c];
      }
    }
    tc_fence_before_sync();  // the next segment's first weighted sums overwrite what was just read
    mbar_arrive(smem_u32(&sm.o_free));
  }
}

// ---- queries as e4m3 terms: a column (head_dim 128: two) per warp at a time ---------------------------------------------------------------------------
// (Loops that are rolled up: twelve columns unrolled were 20 KB of code that a CTA runs through once or twice, and waits for: 13 us in front
// of the first scores of rows of five tokens.)
template <class L, typename T>
struct QuColumn {  // from column c on: column c + l / kLanes, dims 8 (l % kLanes) .. in lane l
  static constexpr int kLanes = L::kChunks * 16, kCount = 32 / kLanes;
  QRaw<T> raw;
  int limit;
  __device__ __forceinline__ void load(const QuSmem<L>& sm, const QuParams& a, const QuSeg& s, long long token, int ct, int c, int lane) {
    raw = QRaw<T>{};
    limit = 0;
    c += lane / kLanes;
    if (ct * L::kC + c < a.columns) {
      raw = q_load8(static_cast<const T*>(a.q) + (token * a.num_q_heads + sm.col_row[c]) * (L::kChunks * 128) + 8 * (lane % kLanes));
      const int last = a.positions ? a.positions[token + sm.col_token[c]] : 0x7ffffffe;
      limit = last < s.len ? last + 1 : s.len;
    }
  }
  template <int kCg>
  __device__ __forceinline__ void store(QuSmem<L>& sm, const QuParams& a, uint32_t seg, int c, int lane) const {
    const int d = 8 * (lane % kLanes);
    c += lane / kLanes;
    float x[8];
    q_floats(raw, x);
    int bits = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) bits = max(bits, __float_as_int(x[k]) & 0x7fffffff);
    if constexpr (kCount == 1) {
      bits = __reduce_max_sync(kFullMask, bits);
    } else {
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(kFullMask, bits, o));
    }
    const bool odd = bits >= 0x7f800000;  // an infinity or NaN: the column's scores are NaN
    int e = (bits >> 23) - 127 - 7;       // largest = 2^(e + 7) * [1, 2)
    e = bits == 0 || odd ? 0 : (e < -126 ? -126 : e);
    const float down = q_pow2(-e);
    if (lane % kLanes == 0) {
      sm.factor[seg & 3u][c] = odd ? __int_as_float(0x7fffffff) : q_pow2(e) * a.scale_log2;
      sm.limit[seg & 3u][c] = limit;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] *= down;
    const int row0 = c / kCg * L::kSRegion + c % kCg;
#pragma unroll
    for (int j = 0; j < L::kQTerms; ++j) {
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        b[k] = q_pack2(x[2 * k], x[2 * k + 1]);
        if (j + 1 < L::kQTerms) {
          const float2 y = q_float2(q_half2(b[k]));
          x[2 * k] = (x[2 * k] - y.x) * 32.f;  // (a term is at most 2^8, what its rounding leaves 2^3)
          x[2 * k + 1] = (x[2 * k + 1] - y.y) * 32.f;
        }
      }
      const int row = row0 + j * kCg;
      *reinterpret_cast<uint2*>(sm.q[seg & 1u][d / 128] + row * 128 + (((d % 128 / 16) ^ (row & 7)) << 4) + (d & 8)) =
          make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
    }
  }
};
__device__ __forceinline__ long long qu_first_token(const QuParams& a, int b) {
  return a.query_start_loc ? (long long)a.query_start_loc[b] : (long long)b * a.width;
}
// The query warp: the segments behind the first, whose queries all warps have brought in before.
template <class L, typename T, int kCg>
__device__ __forceinline__ void qu_query_warp(QuSmem<L>& sm, const QuParams& a, const DecodeParams& p, int ct, QuWalk walk, int lane) {
  QuSeg s;
  for (uint32_t seg = 0; walk.next(a, p, s); ++seg) {
    if (seg > 0) {
      const long long token = qu_first_token(a, s.b);
      // a few columns are on their way at a time
      using Column = QuColumn<L, T>;
      constexpr int kAhead = L::kC < 4 * Column::kCount ? L::kC / Column::kCount : 4, kAll = kAhead * Column::kCount;
      static_assert(L::kC % kAll == 0);
      Column column[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) column[i].load(sm, a, s, token, ct, i * Column::kCount, lane);
      int seen = 0;
      // the scores of the segment two before have been computed
      if (seg > 1 && !um_wait(&sm.q_free[seg & 1u], ((seg >> 1) - 1) & 1u, &sm.abort_flag, p.status)) return;
#pragma unroll 1
      for (int c = 0; c < L::kC; c += kAll) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          column[i].template store<kCg>(sm, a, seg, c + i * Column::kCount, lane);
          seen = max(seen, column[i].limit);
          if (c + kAll < L::kC) column[i].load(sm, a, s, token, ct, c + kAll + i * Column::kCount, lane);
        }
      }
      seen = __reduce_max_sync(kFullMask, seen);
      if (lane == 0) sm.seen[seg & 3u] = seen;
      fence_proxy_async_smem();
    }
    mbar_arrive(smem_u32(&sm.q_full[seg & 1u]));
  }
}

template <typename T, int kDim, int kCg, int kSharing>
__global__ void __launch_bounds__(QuLayout<T, kDim, kCg, kSharing>::kThreads, 1)
quantized_umma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const QuParams a, const DecodeParams p) {
  using L = QuLayout<T, kDim, kCg, kSharing>;
  constexpr int kThreads = L::kThreads, kScoresWarp = 4 * L::kGroups, kSumsWarp = kScoresWarp + 1, kTmaWarp = kScoresWarp + 2;
  extern __shared__ unsigned char qu_smem_raw[];
  QuSmem<L>& sm = *reinterpret_cast<QuSmem<L>*>((reinterpret_cast<uintptr_t>(qu_smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hct = blockIdx.x % a.hcts, range = blockIdx.x / a.hcts, ranges = gridDim.x / a.hcts;
  const int head = hct / a.column_tiles, ct = hct % a.column_tiles;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&k_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
    sm.start_b = p.batch; sm.start_j = 0; sm.lens_from = 0; sm.abort_flag = 0; sm.seen[0] = 0;
    for (int i = 0; i < L::kKSlots; ++i) {
      mbar_init(smem_u32(&sm.k_full[i]), 1);
      mbar_init(smem_u32(&sm.k_empty[i]), 1);
    }
    for (int i = 0; i < L::kVSlots; ++i) {
      mbar_init(smem_u32(&sm.v_full[i]), 1);
      mbar_init(smem_u32(&sm.v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.q_full[i]), 32);
      mbar_init(smem_u32(&sm.q_free[i]), 1);
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.p_full[i]), 128 * kSharing);
      mbar_init(smem_u32(&sm.pv_done[i]), 1);
    }
    mbar_init(smem_u32(&sm.o_full), 1);
    mbar_init(smem_u32(&sm.o_free), L::kSoftmaxThreads);
    mbar_fence_init();
  }
  if (threadIdx.x < L::kC) {
    const int at = ct * L::kC + threadIdx.x;
    sm.col_token[threadIdx.x] = at / a.groups;
    sm.col_row[threadIdx.x] = at / a.groups * a.num_q_heads + head * a.groups + at % a.groups;
  }
  // (rows of the query terms that no column fills: finite, and never read)
  for (int i = threadIdx.x; i < (int)sizeof(sm.q) / 16; i += kThreads) reinterpret_cast<uint4*>(sm.q)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  pdl_wait();
  {  // this CTA's share of the block tables into the L2, while the lengths are on their way
    const long long lines = ((long long)p.batch * p.table_width * (long long)sizeof(int32_t) + 127) / 128;
    const long long line = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (line < lines) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.block_tables) + line * 128));
  }
  // ---- pass 1: total number of units; zero the output of rows without keys
  int mine = 0, first_n = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + threadIdx.x;
    int len = 0;
    if (b < p.batch) len = decode_row_len(p, b);
    const int n = blocks_in_sequence(p, qu_row_units(a, len));
    if (base == 0) {
      first_n = n;
      sm.lens[threadIdx.x] = len;
    }
    mine += n;
    const bool ours = b < p.batch && len <= 0 && b % ranges == range &&
                      (!p.packed_rows || packed_row_served(p, b));
    for (unsigned todo = __ballot_sync(kFullMask, ours); todo; todo &= todo - 1) {
      const int bb = base + (warp << 5) + (__ffs(todo) - 1);
      const long long token = a.query_start_loc ? (long long)a.query_start_loc[bb] : (long long)bb * a.width;
      const int columns = min(a.columns - ct * L::kC, L::kC);
      for (int i = lane; i < columns * (kDim / 4); i += 32) {
        const int at = ct * L::kC + i / (kDim / 4);
        reinterpret_cast<float4*>(a.out + ((token + at / a.groups) * a.num_q_heads + head * a.groups + at % a.groups) * kDim)[i % (kDim / 4)] =
            make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  int total = 0;
  const int incl = qu_inclusive_scan<kThreads>(mine, sm.scan, total);
  const Partition pt = make_partition(total > 0 ? total : 1, ranges);
  const long long g0 = pt.start(range), g1 = pt.start(range + 1);
  if (total == 0 || range >= pt.n || g0 == g1) {  // nothing for this CTA
    if (hct == 0 && threadIdx.x == 0) a.cuts[range] = kNoCut;
    return;
  }
  // ---- pass 2: locate (row, unit) of g0
  long long carry = 0;
  if (p.batch <= kThreads) {  // one row per thread: the scan of pass 1 has the answer already
    const long long excl = incl - first_n;
    if (first_n > 0 && excl <= g0 && g0 < excl + first_n) { sm.start_b = threadIdx.x; sm.start_j = (int)(g0 - excl); }
    carry = g0 + 1;  // skips the loop below
  }
  for (int base = 0; base < p.batch && carry <= g0; base += kThreads) {
    const int b = base + threadIdx.x;
    int n = 0;
    if (b < p.batch) n = blocks_in_sequence(p, qu_row_units(a, decode_row_len(p, b)));
    int chunk_total = 0;
    const long long excl = carry + qu_inclusive_scan<kThreads>(n, sm.scan, chunk_total) - n;
    if (n > 0 && excl <= g0 && g0 < excl + n) { sm.start_b = b; sm.start_j = (int)(g0 - excl); }
    carry += chunk_total;
  }
  __syncthreads();
  if (p.batch > kThreads) {  // (else pass 1 has left all lengths)
    const int b = sm.start_b + threadIdx.x;
    sm.lens[threadIdx.x] = b < p.batch ? decode_row_len(p, b) : 0;
    if (threadIdx.x == 0) sm.lens_from = sm.start_b;
    __syncthreads();
  }
  const QuWalk walk{sm.start_b, sm.start_j, g0, g1, sm.lens, sm.lens_from, kThreads};
  if (warp == kTmaWarp) {  // needs neither queries nor tensor memory
    qu_producer<L>(&k_map, &v_map, a, p, sm, head, walk, lane);
  } else {
    if (warp == kScoresWarp) {  // tensor memory between the wait and the release (umma.cuh)
      tmem_alloc(smem_u32(&sm.tmem_base), 512);
      if (lane == 0) pdl_release();
    }
    {  // the first segment's queries
      QuSeg s;
      QuWalk first = walk;
      const bool have = first.next(a, p, s);
      const long long token = have ? qu_first_token(a, s.b) : 0;
#pragma unroll 1
      for (int c = (warp - (warp > kTmaWarp)) * QuColumn<L, T>::kCount; have && c < L::kC; c += (kThreads / 32 - 1) * QuColumn<L, T>::kCount) {
        QuColumn<L, T> column;
        column.load(sm, a, s, token, ct, c, lane);
        column.template store<kCg>(sm, a, 0u, c, lane);
        const int seen = __reduce_max_sync(kFullMask, column.limit);
        if (lane == 0) atomicMax(&sm.seen[0], seen);
      }
      fence_proxy_async_smem();
    }
    tc_fence_before_sync();
    named_bar_sync(kQuBarQueries, kThreads - 32);
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem_base;

    if (warp < kScoresWarp) qu_softmax_warps<L, kCg>(sm, a, p, tmem, head, hct, ct, walk, range, warp >> 2, warp & 3, lane);
    else if (warp == kScoresWarp) qu_scores_warp<L>(sm, a, p, tmem, walk);
    else if (warp == kSumsWarp) {
      if (hct == 0 && lane == 0) a.cuts[range] = qu_cut(a, p, pt, range, walk.b, walk.j, walk.g);
      __syncwarp();
      qu_sums_warp<L>(sm, a, p, tmem, walk);
    }
    else qu_query_warp<L, T, kCg>(sm, a, p, ct, walk, lane);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (sm.abort_flag) {  // give copies and MMAs in flight time to land before the CTA's memory is released
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == kScoresWarp) tmem_dealloc(sm.tmem_base, 512);
}

template <typename T, int kDim, int kCg, int kSharing>
static int launch_quantized_umma(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int ranges,
                                 cudaStream_t stream) {
  using L = QuLayout<T, kDim, kCg, kSharing>;
  constexpr int bytes = (int)sizeof(QuSmem<L>) + 1024;
  static_assert(bytes <= 232448, "the ring exceeds the shared memory of one CTA");
  auto* kernel = quantized_umma_kernel<T, kDim, kCg, kSharing>;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess; }))
    return NVJ_ERR_LAUNCH;
  return launch_after(kernel, dim3((unsigned)(ranges * a.hcts)), dim3(L::kThreads), bytes, stream, k_map, v_map, a, p) == cudaSuccess ? NVJ_OK
                                                                                                                             : NVJ_ERR_LAUNCH;
}
template <typename T>
static int launch_quantized_umma_shape(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int head_dim,
                                       int ranges, cudaStream_t stream) {
  auto columns = [&](auto dim) {
    constexpr int kDim = decltype(dim)::value;
    switch (a.tile_columns) {
      case 4: return launch_quantized_umma<T, kDim, 4, 1>(k_map, v_map, a, p, ranges, stream);
      case 8: return launch_quantized_umma<T, kDim, 8, 1>(k_map, v_map, a, p, ranges, stream);
      case 16: return launch_quantized_umma<T, kDim, 8, 2>(k_map, v_map, a, p, ranges, stream);
      default: return launch_quantized_umma<T, kDim, 8, 3>(k_map, v_map, a, p, ranges, stream);
    }
  };
  return head_dim == 256 ? columns(std::integral_constant<int, 256>{}) : columns(std::integral_constant<int, 128>{});
}

}  // namespace nvj
