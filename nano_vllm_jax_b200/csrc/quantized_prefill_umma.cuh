// Ragged packed prefill over the 8-bit paged cache on the 5th-generation tensor cores (tcgen05, kind::f16).  Included by one file per type of
// query (quantized_prefill_*.cu).
//
// Every number of the cache is an f16 number (e4m3 has fewer bits and a smaller range), so K and V become f16 on their way into shared
// memory and nothing is rounded; a block's scale is a power of two and joins the scores (K) or the weights (V) in f32.
//   S = Q K^T    [128 query rows x 64 keys]   16 dims per MMA; bf16 and f16 queries are f16 times a power of two per row (exact, but for bf16
//                numbers below 2^-31 of their row's largest), f32 ones two f16 terms (2^-22);
//   O = P V      [128 query rows x head_dim]  16 keys per MMA; P from tensor memory, as two f16 terms (2^-22 of a weight).
// A tile of 64 keys takes 4 * 128 * 64 * head_dim flops for S and twice that for O's two terms: 2200 cycles of an SM at head_dim 256.  A softmax
// thread's way from a tile's scores to its weights takes as long: scores out of tensor memory 400, the pair's meeting 500, exponentials and terms
// 700, back 250.  head_dim 64 takes just that, 128 2500, 256 3400, where queries, keys and values move 220 KB through shared memory per tile.
// Against the tiles of mma.sync that stood here before: 1984 f16 tokens behind 727, 32 heads of 128 over 8, 452 -> 187 us; 1018 tokens of
// four rows behind 1232 each 165 -> 74; 55 f32 tokens of two rows behind 1214 (8 heads of 256 over 2) 160 -> 27; 54 tokens behind 1398 (16
// heads of 64 over 2) 62 -> 16; the smallest calls as long as they took (20 tokens, heads of 256: 17.7 -> 17).  A small call at head_dim
// 256 is start and end: row and lengths 2.4 us, queries 3, a tile 2, rows staged 3, folded over DSMEM 5.
//
// CTA: 128 query rows (token major, a kv head's `groups` heads minor) of one table row and kv head.  While that gives fewer tiles than the GPU
// has room for, a tile's keys are split over a cluster of up to eight CTAs, which fold their rows through each other's shared memory.
//   warps 0 - 7    softmax, thread = (query row, half of the tile's keys); a row's two halves are a pair of warps
//   warps 8 - 11   keys: 16-byte pieces of the blocks to registers, one tile ahead, and from there as f16 to their tiles
//   warps 12 - 15  values, in the same way; the first issues the weighted sums' MMAs, the second the scores', a tile ahead
// The weights of a row are exp2(score - reference) times the V scale; the reference is set so that the largest weight is 2^7,
// and moved when a later one would pass 2^15 (f16 ends at 2^16), which is rare.  Their sum is taken in f32, relative to the largest score's: the
// weights of 16 keys of one block with the block's V scale divided out again, or, where a block is so quiet that its weights may be
// zero although its keys count in that sum (the append gives a block of zeros 2^-117), exponentials of their own.
// The tensor cores cut the last place of what they add to: 1.2e-5 of a sum over 16384 keys.  After kQtFlush tiles the sums are
// emptied into the output row (clusters: into scratch) and begun again.
// Every wait is bounded; after a timeout (NVJ_DEV_TIMEOUT) the kernel stops issuing, lets MMAs land and frees its tensor memory.
#pragma once

#include "cluster.cuh"
#include "quantized_kv.cuh"
#include "quantized_prefill_params.cuh"
#include "umma.cuh"

namespace nvj {

constexpr int kQtRows = 128, kQtKeys = 64, kQtThreads = 512, kQtSoftmax = 256, kQtLoaders = 128;
constexpr int kQtColS = 256, kQtColP = 384;  // of tensor memory: O from 0, S twice, P twice (two terms of 32 columns)
constexpr float kQtNone = -3e38f, kQtSlack = 8.f, kQtLift = 7.f;
constexpr float kQtFar = 40.f;  // log2 of what weights are multiplied by, at most, on their way into their sum

template <typename T, int kD>
struct QtSmem {
  static constexpr int kQTerms = std::is_same<T, float>::value ? 2 : 1;
  static constexpr int kChunks = kD / 64;                 // of 64 dims: 128 bytes of f16
  static constexpr int kTileBytes = kQtKeys * kD * 2;
  static constexpr int kFit = (232448 - 1024 - 4096 - kQTerms * kChunks * 16384) / kTileBytes;
  static constexpr int kKSlots = kFit >= 3 ? 2 : 1, kVSlots = kFit >= 4 ? 2 : 1;
  alignas(1024) char q[kQTerms][kChunks][kQtRows * 128];  // [chunk][row][128 B]
  alignas(1024) char k[kKSlots][kTileBytes];              // [8-key group][chunk][8 keys][128 B]
  alignas(1024) char v[kVSlots][kTileBytes];
  alignas(8) unsigned long long k_full[kKSlots], k_empty[kKSlots], v_full[kVSlots], v_empty[kVSlots], s_full[2], p_full[2], pv_done[2];
  // by tile and 16 keys: the block's scales; V's -1: no such block.  Those of tile n + 1 are asked for when S(n - 2) is complete, hence when the weights
  // of n - 4 are there: eight places, so that n - 7's have been read.
  alignas(16) float k_unit[8][4], v_unit[8][4];
  float factor[kQtRows];
  int limit[kQtRows];
  float2 red[kQtRows];  // between the two threads of a row
  int found[3], most, abort_flag;
  uint32_t tmem_base;
};

__device__ __forceinline__ bool qt_pair_any(int id, bool mine) {  // of the 64 threads of two warps
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any) : "r"((uint32_t)mine), "r"(id) : "memory");
  return any != 0;
}
// Instruction descriptor, kind::f16: fp32 accumulate, f16 A and B, M = 128.
__device__ __forceinline__ constexpr uint32_t qt_idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// Where 16-byte piece `piece` of row r of the staged output lies: rows of 4 kD bytes, pieces swapped so that 32 rows fall into different banks.
template <int kD>
__device__ __forceinline__ int qt_piece(int r, int piece) { return r * kD + ((piece ^ (r & 15)) << 2); }

// ---- MMA issue ------------------------------------------------------------------------------------------------------------------------
// S of tile n takes the place of S of n - 2, which has been read when that tile's weights are there.
template <typename T, int kD>
__device__ __forceinline__ bool qt_issue_scores(QtSmem<T, kD>& sm, const QtParams& p, uint32_t tmem, int n) {
  using L = QtSmem<T, kD>;
  constexpr uint32_t idesc = qt_idesc(kQtKeys, false);
  const int slot = n % L::kKSlots;
  if (!um_wait(&sm.k_full[slot], (n / L::kKSlots) & 1u, &sm.abort_flag, p.status)) return false;
  if (n >= 2 && !um_wait(&sm.p_full[n & 1], ((n >> 1) - 1) & 1u, &sm.abort_flag, p.status)) return false;
  tc_fence_after_sync();
  if (um_elect_one()) {
    const uint64_t q_desc = umma_desc(smem_u32(sm.q[0][0]), 16, 1024), k_desc = umma_desc(smem_u32(sm.k[slot]), 16, L::kChunks * 1024);
#pragma unroll
    for (int term = L::kQTerms - 1; term >= 0; --term)
#pragma unroll
      for (int ks = 0; ks < kD / 16; ++ks)
        umma_bf16_ss(tmem + kQtColS + (n & 1) * kQtKeys,
                     q_desc + (uint64_t)((((term * L::kChunks + (ks >> 2)) * kQtRows * 128) + (ks & 3) * 32) >> 4),
                     k_desc + (uint64_t)(((ks >> 2) * 1024 + (ks & 3) * 32) >> 4), idesc, ks > 0 || term < L::kQTerms - 1 ? 1u : 0u);
    umma_commit(smem_u32(&sm.s_full[n & 1]));
    umma_commit(smem_u32(&sm.k_empty[slot]));
  }
  __syncwarp();
  return true;
}
template <typename T, int kD>
__device__ __forceinline__ bool qt_issue_sums(QtSmem<T, kD>& sm, const QtParams& p, uint32_t tmem, int n, bool flush) {
  using L = QtSmem<T, kD>;
  constexpr uint32_t idesc = qt_idesc(kD, true);
  const int slot = n % L::kVSlots;
  if (!um_wait(&sm.v_full[slot], (n / L::kVSlots) & 1u, &sm.abort_flag, p.status)) return false;
  if (!um_wait(&sm.p_full[n & 1], (n >> 1) & 1u, &sm.abort_flag, p.status)) return false;
  tc_fence_after_sync();
  if (um_elect_one()) {
    const uint64_t v_desc = umma_desc(smem_u32(sm.v[slot]), 1024, L::kChunks * 1024);  // chunks of 64 dims, groups of 8 keys
    const bool anew = flush ? n % kQtFlush == 0 : n == 0;
#pragma unroll
    for (int ks = 0; ks < kQtKeys / 16; ++ks)
#pragma unroll
      for (int term = 1; term >= 0; --term)
        umma_bf16_ts(tmem, tmem + kQtColP + (n & 1) * 64 + term * 32 + ks * 8, v_desc + (uint64_t)((ks * 2 * L::kChunks * 1024) >> 4), idesc,
                     anew && ks == 0 && term == 1 ? 0u : 1u);
    umma_commit(smem_u32(&sm.pv_done[n & 1]));
    umma_commit(smem_u32(&sm.v_empty[slot]));
  }
  __syncwarp();
  return true;
}

// ---- warps 8 - 15 -------------------------------------------------------------------------------------------------------------
template <bool kV, typename T, int kD>
__device__ __forceinline__ void qt_loaders(QtSmem<T, kD>& sm, const QtParams& p, uint32_t tmem, bool flush, int row, int head, int len, int tile0,
                                           int tiles, int tid) {
  using L = QtSmem<T, kD>;
  constexpr int kPieces = kD / 32, kStep = kQtLoaders / (kD / 16);  // pieces per thread; keys between them (8, 16 or 32)
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  // Of the tile's first kStep keys: the thread's key, 64 dims and 16 bytes of them.  (Eight lanes of a store: four pieces each of an even and an
  // odd key, which the swizzle puts into different banks.)
  const int key_of = (tid >> 2 & 1) + tid / (8 * L::kChunks) * 2, chunk = tid / 8 % L::kChunks, piece = chunk * 4 + (tid & 3);
  // Blocks are walked 16 keys at a time, four to a tile, by every thread for itself: ids of the tile ahead, and where in the cache the
  // thread's pieces of the one at hand lie.
  const int per_block = p.block_size / 16, hop = 4 / per_block, over = 4 % per_block;
  const int row_bytes = p.num_kv_heads * kD, block_bytes = row_bytes * p.block_size;
  const unsigned ids_end = p.num_blocks < 0x80000000ll ? (unsigned)p.num_blocks : 0x80000000u;
  int block[4], rest[4], id[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    block[j] = (tile0 * 4 + j) / per_block;
    rest[j] = (tile0 * 4 + j) % per_block;
  }
  auto ids_of = [&](int tile) {  // tiles in turn
#pragma unroll
    for (int j = 0; j < 4; ++j) id[j] = tile * kQtKeys + j * 16 < len ? table[block[j]] : -1;
  };
  long long at[4];     // of 16 keys: bytes from the cache's beginning to the thread's key and piece; -1: no such block, or behind the last key
  bool whole = false;  // all of the tile's keys are there
  const int mine = (key_of & 15) * row_bytes + head * kD + piece * 16;
  auto locate = [&](int tile) {
    whole = (tile + 1) * kQtKeys <= len;
    if (!kV && tid < 4) {  // the scales, counted with K
      const int i = tid == 0 ? id[0] : tid == 1 ? id[1] : tid == 2 ? id[2] : id[3], slot = (tile - tile0) & 7;
      if ((unsigned)i < ids_end) {
        const long long entry = (long long)i * p.num_kv_heads + head;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&sm.k_unit[slot][tid])), "l"(p.k_scale + entry) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&sm.v_unit[slot][tid])), "l"(p.v_scale + entry) : "memory");
      } else {
        sm.k_unit[slot][tid] = 0.f;
        sm.v_unit[slot][tid] = -1.f;
        if (tile * kQtKeys + tid * 16 < len) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool ok = (unsigned)id[j] < ids_end;
      at[j] = ok ? (long long)id[j] * block_bytes + (rest[j] * 16 * row_bytes + mine) : -1ll;
      whole = whole && ok;
      block[j] += hop;
      rest[j] += over;
      if (rest[j] >= per_block) {
        rest[j] -= per_block;
        ++block[j];
      }
    }
  };
  // (Four warps for K and V, and two that only issued MMAs: up to 20% slower with f32 queries, 5% with heads of 128, 5 - 7% faster on 4096 tokens of
  // heads of 64, or of 256 in f16.  The pieces by way of shared memory instead of registers: 0 - 5% slower.)
  const uint8_t* cache = kV ? p.v_cache : p.k_cache;
  uint4 held[kPieces];
  auto fetch = [&](int tile) {
    const int step_bytes = kStep * row_bytes;
    if (whole) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        if constexpr (kStep == 32) held[i] = ld_stream_u4(cache + (key_of >= 16 ? at[2 * i + 1] : at[2 * i]));
        else held[i] = ld_stream_u4(cache + (at[i * kStep / 16] + i * kStep % 16 / kStep * step_bytes));
      }
    } else {  // keys behind the row's last one become zeros, which as values weigh nothing
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int key = key_of + i * kStep;
        long long from;
        if constexpr (kStep == 32) from = key_of >= 16 ? at[2 * i + 1] : at[2 * i];
        else from = at[i * kStep / 16];
        held[i] = make_uint4(0, 0, 0, 0);
        if (from >= 0 && tile * kQtKeys + key < len) held[i] = ld_stream_u4(cache + from + (kStep < 16 ? i * kStep % 16 / kStep * step_bytes : 0));
      }
    }
  };
  const uint32_t dst = (key_of >> 3) * (L::kChunks * 1024) + chunk * 1024 + (key_of & 7) * 128 + ((((tid & 3) * 2) ^ (key_of & 7)) << 4);
  auto store = [&](char* tile) {
    if (!kV && tid < 4) asm volatile("cp.async.wait_all;" ::: "memory");
    const uint32_t to = smem_u32(tile) + dst;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t w[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                     ::"r"((h ? to ^ 16u : to) + i * (kStep / 8 * L::kChunks * 1024)), "r"(q_half2(w[2 * h])), "r"(q_half2_high(w[2 * h])),
                       "r"(q_half2(w[2 * h + 1])), "r"(q_half2_high(w[2 * h + 1])) : "memory");
    }
  };
  constexpr int kSlots = kV ? L::kVSlots : L::kKSlots;
  ids_of(tile0);
  locate(tile0);
  fetch(tile0);
  ids_of(tile0 + 1);
  // The values' first two warps issue the MMAs: one the weighted sums, one the scores, a tile ahead.  (By the first warps of the keys and of the values,
  // each issuing what its own tiles are for, 3700 cycles per tile of 64 keys of 256: the keys' warp had the scales to bring as well.)
  const bool sums = kV && tid < 32, scores = kV && tid >= 32 && tid < 64;
  bool alive = true;
  if (scores) {
    named_bar_sync(5, kQtSoftmax + 32);  // the queries are there
    alive = qt_issue_scores(sm, p, tmem, 0);
  }
#pragma unroll 1
  for (int n = 0; alive && n < tiles; ++n) {
    const int slot = n % kSlots;
    if (scores && n + 1 < tiles && !(alive = qt_issue_scores(sm, p, tmem, n + 1))) break;
    if (sums && n > 0 && !(alive = qt_issue_sums(sm, p, tmem, n - 1, flush))) break;
    if (n >= kSlots && !(alive = um_wait(kV ? &sm.v_empty[slot] : &sm.k_empty[slot], (n / kSlots - 1) & 1u, &sm.abort_flag, p.status))) break;
    store(kV ? sm.v[slot] : sm.k[slot]);
    fence_proxy_async_smem();
    mbar_arrive(smem_u32(kV ? &sm.v_full[slot] : &sm.k_full[slot]));
    if (n + 1 < tiles) {
      locate(tile0 + n + 1);
      fetch(tile0 + n + 1);
      ids_of(tile0 + n + 2);
    }
  }
  if (sums && alive) qt_issue_sums(sm, p, tmem, tiles - 1, flush);
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- queries: 8 dims a lane, so many rows of a warp at a time -----------------------------------------------------------------------------
template <typename T, int kD>
struct QtQueries {
  static constexpr int kWarps = 8, kLanes = kD / 8, kAtOnce = 32 / kLanes;
  static constexpr int kAll = (kQtRows + kWarps * kAtOnce - 1) / (kWarps * kAtOnce);  // passes of a warp
  static constexpr int kMost = sizeof(T) == 4 ? 4 : 8, kRounds = kAll < kMost ? kAll : kMost;  // of them on their way at a time
  static __device__ __forceinline__ int row_of(int round, int warp, int lane) { return (round * kWarps + warp) * kAtOnce + lane / kLanes; }
  // Times a power of two per row that makes the largest 2^14 - 2^15.
  static __device__ __forceinline__ void store(QtSmem<T, kD>& sm, const QRaw<T>& raw, int r, int lane, float scale_log2) {
    float x[8];
    q_floats(raw, x);
    int bits = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) bits = max(bits, __float_as_int(x[k]) & 0x7fffffff);
    if constexpr (kLanes == 32) {
      bits = __reduce_max_sync(kFullMask, bits);
    } else {
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(kFullMask, bits, o));
    }
    const bool odd = bits >= 0x7f800000;  // an infinity or NaN: the row's scores are NaN
    int e = (bits >> 23) - 127 - 14;
    e = bits == 0 || odd ? 0 : (e < -126 ? -126 : e);
    const float down = q_pow2(-e);
    if (r >= kQtRows) return;
    if (lane % kLanes == 0) sm.factor[r] = odd ? __int_as_float(0x7fffffff) : q_pow2(e) * scale_log2;
    uint32_t w[4], low[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = x[2 * k] * down, b = x[2 * k + 1] * down;
      w[k] = q_pair(a, b);
      low[k] = q_pair_rest(a, b, w[k]);
    }
    const int d = 8 * (lane % kLanes), at = r * 128 + (((d % 64 / 8) ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(sm.q[0][d / 64] + at) = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (QtSmem<T, kD>::kQTerms == 2) *reinterpret_cast<uint4*>(sm.q[1][d / 64] + at) = make_uint4(low[0], low[1], low[2], low[3]);
  }
};

// ---- warps 0 - 7 ----------------------------------------------------------------------------------------------------------------
// (A scale of zero is as good as the smallest there is.)
__device__ __forceinline__ float qt_log(float v_unit) { return v_unit < 0.f ? -INFINITY : __log2f(fmaxf(v_unit, 0x1p-126f)); }
struct QtRow {  // what a softmax thread knows of its row at the end: references of the weighted sums and of the sum l of the weights
  float m, top, l, m_flushed;
};
template <typename T, int kD>
__device__ __forceinline__ bool qt_softmax(QtSmem<T, kD>& sm, const QtParams& p, uint32_t tmem, int tile0, int tiles, int r, int half, int pair, float* flush_row,
                                           bool flush, QtRow& o) {
  constexpr int kHalf = kD / 2;  // columns of O that the thread handles
  const float factor = sm.factor[r];
  const int limit = sm.limit[r];
  const int fewest = __reduce_min_sync(kFullMask, limit);
  o.m = o.top = kQtNone;
  o.l = 0.f;
  o.m_flushed = 0.f;
  bool begun = false;
  for (int n = 0; n < tiles; ++n) {
    const int buf = n & 1;
    const bool ok = um_wait(&sm.s_full[buf], (n >> 1) & 1u, &sm.abort_flag, p.status);
    tc_fence_after_sync();
    float x[32];
    tmem_ld32(tmem + kQtColS + buf * kQtKeys + half * 32, x);
    const float2 unit = *reinterpret_cast<const float2*>(&sm.k_unit[n & 7][2 * half]), v_unit = *reinterpret_cast<const float2*>(&sm.v_unit[n & 7][2 * half]);
    const int key0 = (tile0 + n) * kQtKeys + half * 32;
    const float by[2] = {factor * unit.x, factor * unit.y}, plus[2] = {qt_log(v_unit.x), qt_log(v_unit.y)};
    // scores are x * mul; the exponents of the weights that and add - reference
    float top, most, mul[2], add[2] = {plus[0], plus[1]};  // the largest score with its V scale, and the largest without
    if (key0 + 32 > fewest || plus[0] == -INFINITY || plus[1] == -INFINITY || !(p.scale_log2 > 0.f)) {
      float big[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        x[j] = key0 + j < limit && plus[j >> 4] != -INFINITY ? x[j] * by[j >> 4] : -INFINITY;
        big[j >> 4] = fmaxf(big[j >> 4], x[j]);
      }
      most = fmaxf(big[0], big[1]);
      top = fmaxf(big[0] + plus[0], big[1] + plus[1]);
      mul[0] = mul[1] = 1.f;
    } else {  // the largest score of 16 keys of one block is the largest product's
      float big[2] = {x[0], x[16]};
#pragma unroll
      for (int j = 0; j < 32; ++j) big[j >> 4] = fmaxf(big[j >> 4], x[j]);
      most = fmaxf(big[0] * by[0], big[1] * by[1]);
      top = fmaxf(fmaf(big[0], by[0], plus[0]), fmaf(big[1], by[1], plus[1]));
      mul[0] = by[0];
      mul[1] = by[1];
    }
    if (qt_pair_any(1 + pair, !ok || !begun || top > o.m + kQtSlack || most > o.top + kQtSlack)) {
      if (half == 0) sm.red[r] = make_float2(top, most);
      const bool complete = !begun || um_wait(&sm.pv_done[buf ^ 1], ((n - 1) >> 1) & 1u, &sm.abort_flag, p.status);
      if (qt_pair_any(1 + pair, !ok || !complete)) return false;
      tc_fence_after_sync();
      float2 both = make_float2(top, most);
      if (half == 1) sm.red[r] = both = make_float2(fmaxf(top, sm.red[r].x), fmaxf(most, sm.red[r].y));
      qt_pair_any(1 + pair, false);
      if (half == 0) both = sm.red[r];
      const float now = both.x > o.m + kQtSlack ? both.x - kQtLift : o.m;  // (a row whose scores stay under it keeps its reference)
      const float now_top = both.y > o.top + kQtSlack ? both.y : o.top;
      const float f = ex2_approx(o.m - now);
      o.l *= ex2_approx(o.top - now_top);
      o.m = now;
      o.top = now_top;
      if (begun) {
#pragma unroll 1
        for (int c = half * kHalf; c < (half + 1) * kHalf; c += 32) {
          float y[32];
          tmem_ld32(tmem + c, y);
#pragma unroll
          for (int j = 0; j < 32; ++j) y[j] *= f;
          tmem_st32(tmem + c, y);
        }
      }
      begun = true;
    }
    if (flush && n > 0 && n % kQtFlush == 0) {  // the sums so far to memory; the next weighted sums overwrite them
      if (qt_pair_any(1 + pair, !um_wait(&sm.pv_done[buf ^ 1], ((n - 1) >> 1) & 1u, &sm.abort_flag, p.status))) return false;
      tc_fence_after_sync();
      const float back = n > kQtFlush ? ex2_approx(o.m_flushed - o.m) : 0.f;
      o.m_flushed = o.m;
#pragma unroll 1
      for (int c = half * kHalf; c < (half + 1) * kHalf; c += 32) {
        float y[32];
        __syncwarp();
        tmem_ld32(tmem + c, y);
        if (!flush_row) continue;
        float4* to = reinterpret_cast<float4*>(flush_row + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float4 was = back == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : to[j];
          to[j] = make_float4(fmaf(was.x, back, y[4 * j]), fmaf(was.y, back, y[4 * j + 1]), fmaf(was.z, back, y[4 * j + 2]), fmaf(was.w, back, y[4 * j + 3]));
        }
      }
    }
    float sum[2] = {0.f, 0.f};
    add[0] -= o.m;
    add[1] -= o.m;
    uint32_t high[16], low[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = ex2_approx(fmaf(x[2 * j], mul[j >> 3], add[j >> 3])), b = ex2_approx(fmaf(x[2 * j + 1], mul[j >> 3], add[j >> 3]));
      sum[j >> 3] += a + b;
      high[j] = q_pair(a, b);
      low[j] = q_pair_rest(a, b, high[j]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float back = (o.m - o.top) - plus[h];
      if (back > kQtFar) {
#pragma unroll
        for (int j = 0; j < 16; ++j) o.l += ex2_approx(fmaf(x[16 * h + j], mul[h], -o.top));
      } else {
        o.l = fmaf(sum[h], ex2_approx(back), o.l);
      }
    }
    // (the weights of tile n - 2, in the same place, have been used: almost always long ago; a wait that runs out shows at the next meeting)
    if (n >= 2) um_wait(&sm.pv_done[buf], ((n >> 1) - 1) & 1u, &sm.abort_flag, p.status);
    tc_fence_after_sync();
    tmem_st16(tmem + kQtColP + buf * 64 + half * 16, high);
    tmem_st16(tmem + kQtColP + buf * 64 + 32 + half * 16, low);
    tmem_st_wait();
    tc_fence_before_sync();
    mbar_arrive(smem_u32(&sm.p_full[buf]));
  }
  // all sums are there
  if (tiles > 0 && qt_pair_any(1 + pair, !um_wait(&sm.pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1u, &sm.abort_flag, p.status))) return false;
  tc_fence_after_sync();
  if (half == 1) sm.red[r].x = o.l;
  qt_pair_any(1 + pair, false);
  if (half == 0) sm.red[r].x = o.l = o.l + sm.red[r].x;
  qt_pair_any(1 + pair, false);
  o.l = sm.red[r].x;
  return true;
}

template <typename T, int kD>
__global__ void __launch_bounds__(kQtThreads, 1) quantized_prefill_umma_kernel(const QtParams p) {
  using L = QtSmem<T, kD>;
  extern __shared__ unsigned char qt_raw[];
  L& sm = *reinterpret_cast<L*>((reinterpret_cast<uintptr_t>(qt_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, head = blockIdx.y, hq = p.num_kv_heads * p.groups;
  const int splits = p.splits, rank = splits > 1 ? (int)cl_rank() : 0;
  // clusters, at the end: the rows from the beginning of the queries on, behind them a row's reference and sum, the sum's reference
  float* stage = reinterpret_cast<float*>(sm.q);
  float2* ml = reinterpret_cast<float2*>(stage + kQtRows * kD);
  float* mv_of = reinterpret_cast<float*>(ml + kQtRows);
  if (tid == 0) {
    for (int i = 0; i < L::kKSlots; ++i) {
      mbar_init(smem_u32(&sm.k_full[i]), kQtLoaders);
      mbar_init(smem_u32(&sm.k_empty[i]), 1);
    }
    for (int i = 0; i < L::kVSlots; ++i) {
      mbar_init(smem_u32(&sm.v_full[i]), kQtLoaders);
      mbar_init(smem_u32(&sm.v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.p_full[i]), kQtSoftmax);
      mbar_init(smem_u32(&sm.pv_done[i]), 1);
    }
    mbar_fence_init();
    sm.found[0] = -1;
    sm.most = 0;
    sm.abort_flag = 0;
  }
  __syncthreads();
  pdl_wait();

  // which table row and tile this CTA has: tiles are counted row by row; the last ones (most keys) go first
  const int tile_at = (int)blockIdx.x / splits;
  if (warp == 0) {
    auto tiles_of = [&](int r) {
      const int from = p.query_start_loc[r], to = p.query_start_loc[r + 1];
      if (from < 0 || (p.skip_single && to - from == 1)) return 0;
      const int n = min(to, p.token_bucket) - from;
      return n <= 0 ? 0 : (int)(((long long)n * p.groups + kQtRows - 1) / kQtRows);
    };
    const int first_tiles = lane < p.rows ? tiles_of(lane) : 0;
    int total = first_tiles;
    for (int r = 32 + lane; r < p.rows; r += 32) total += tiles_of(r);
    total = __reduce_add_sync(kFullMask, total);
    const int want = total - 1 - tile_at;
    int before = 0;
    for (int r0 = 0; r0 < p.rows && want >= 0; r0 += 32) {
      const int mine = r0 == 0 ? first_tiles : r0 + lane < p.rows ? tiles_of(r0 + lane) : 0;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(kFullMask, upto, o);
        if (lane >= o) upto += a;
      }
      const int first = before + upto - mine;
      if (want >= first && want < first + mine) {
        sm.found[0] = r0 + lane;
        sm.found[1] = want - first;
      }
      before += __shfl_sync(kFullMask, upto, 31);
      if (want < before) break;
    }
  } else if (warp == 8) {
    tmem_alloc(smem_u32(&sm.tmem_base), 512);  // (between the wait and the release: umma.cuh)
    if (lane == 0) pdl_release();
    tc_fence_before_sync();
  } else if (warp >= 12) {  // padding behind the last row's tokens
    const int end = p.query_start_loc[p.rows], from = end > 0 ? end : 0;
    const long long per_token = (long long)p.groups * (kD / 4), pad = from < p.token_bucket ? (long long)(p.token_bucket - from) * per_token : 0;
    for (long long i = (long long)blockIdx.x * kQtLoaders + tid - 384; i < pad; i += (long long)gridDim.x * kQtLoaders) {
      const long long token = from + i / per_token;
      reinterpret_cast<float4*>(p.out + (token * hq + head * p.groups) * kD)[i % per_token] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  const int row = sm.found[0], first_row = row >= 0 ? sm.found[1] * kQtRows : 0;  // of the row's query rows
  const int token0 = row >= 0 ? p.query_start_loc[row] : -1;
  int query_rows = 0;
  if (row >= 0 && token0 >= 0 && token0 < p.token_bucket) query_rows = min(p.query_start_loc[row + 1] - token0, p.token_bucket - token0) * p.groups;
  if (row < 0 || (long long)sm.found[1] * kQtRows >= query_rows) {  // nothing, for all CTAs of a cluster
    if (warp == 8) tmem_dealloc(tmem, 512);
    return;
  }
  int len = p.kv_lens[row];
  if (len > (long long)p.table_width * p.block_size) {
    if (tid == 0) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    len = p.table_width * p.block_size;
  }
  // queries on their way before anything else is asked for
  using Q = QtQueries<T, kD>;
  auto query = [&](int r) {
    const int at = first_row + r;
    QRaw<T> raw{};
    if (r < kQtRows && at < query_rows)
      raw = q_load8(static_cast<const T*>(p.q) + ((long long)(token0 + at / p.groups) * hq + head * p.groups + at % p.groups) * kD + 8 * (lane % Q::kLanes));
    return raw;
  };
  QRaw<T> queries[Q::kRounds];
  if (warp < 8) {
#pragma unroll
    for (int u = 0; u < Q::kRounds; ++u) queries[u] = query(Q::row_of(u, warp, lane));
  }
  if (tid < kQtRows) {  // how many keys the tile's rows see
    const int at = first_row + tid;
    int limit = 0;
    if (at < query_rows) {
      const int last = p.positions[token0 + at / p.groups];
      limit = last < len ? last + 1 : len;
    }
    sm.limit[tid] = limit;
    const int most = __reduce_max_sync(kFullMask, limit);
    if (lane == 0) atomicMax(&sm.most, most);
  }
  __syncthreads();
  len = sm.most;  // (keys that none of the rows sees may hold anything, as those behind the table row's last one)
  const int all_tiles = (len + kQtKeys - 1) / kQtKeys;
  const int parts = splits == 1 ? 1 : min(splits, max(1, all_tiles / kQtSplitTiles));
  const int tile0 = rank < parts ? (int)((long long)all_tiles * rank / parts) : 0;
  const int tiles = rank < parts ? (int)((long long)all_tiles * (rank + 1) / parts) - tile0 : 0;
  // (a cluster's CTAs empty their sums into scratch, if there is some)
  float* scratch = splits == 1 ? nullptr : p.flush;
  const bool flush = tiles > kQtFlush && (splits == 1 || scratch);

  if (warp >= 8) {
    if (tiles > 0 && warp >= 12) qt_loaders<true>(sm, p, tmem, flush, row, head, len, tile0, tiles, tid - 384);
    else if (tiles > 0) qt_loaders<false>(sm, p, tmem, flush, row, head, len, tile0, tiles, tid - 256);
  } else {
    for (int i0 = 0; tiles > 0; ) {
#pragma unroll
      for (int u = 0; u < Q::kRounds; ++u) Q::store(sm, queries[u], Q::row_of(i0 + u, warp, lane), lane, p.scale_log2);
      i0 += Q::kRounds;
      if (i0 >= Q::kAll) break;
#pragma unroll
      for (int u = 0; u < Q::kRounds; ++u) queries[u] = query(Q::row_of(i0 + u, warp, lane));
    }
    fence_proxy_async_smem();
    if (tiles > 0) named_bar_sync(5, kQtSoftmax + 32);
    {
      const int r = (warp & 3) * 32 + lane, half = warp >> 2, at = first_row + r;
      const uint32_t my_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      float* out_row = at < query_rows ? p.out + ((long long)(token0 + at / p.groups) * hq + head * p.groups + at % p.groups) * kD : nullptr;
      float* flush_row = splits == 1 ? out_row : scratch ? scratch + (((long long)blockIdx.y * gridDim.x + blockIdx.x) * kQtRows + r) * kD : nullptr;
      QtRow o;
      const bool alive = qt_softmax(sm, p, my_tmem, tile0, tiles, r, half, warp & 3, flush_row, flush, o);
      // (the staged rows take the place of the queries, keys and values of all rows: every product has to be over)
      named_bar_sync(6, kQtSoftmax);
      if (alive) {
        const float f = splits > 1 ? 1.f : o.l == 0.f ? 0.f : ex2_approx(o.m - o.top) / o.l;
        const float back = flush ? ex2_approx(o.m_flushed - o.m) : 0.f;
        if (splits > 1 && half == 0) {
          ml[r] = make_float2(o.top, o.l);
          mv_of[r] = o.m;
        }
#pragma unroll 1
        for (int c = half * (kD / 2); c < (half + 1) * (kD / 2); c += 32) {
          float y[32];
          __syncwarp();
          if (tiles > 0) tmem_ld32(my_tmem + c, y);
          if (!out_row || (splits > 1 && o.l == 0.f)) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!(o.l == 0.f)) {
              z = make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
              if (flush) {
                const float4 was = *reinterpret_cast<const float4*>(flush_row + c + 4 * j);
                z = make_float4(fmaf(was.x, back, z.x), fmaf(was.y, back, z.y), fmaf(was.z, back, z.z), fmaf(was.w, back, z.w));
              }
              z = make_float4(z.x * f, z.y * f, z.z * f, z.w * f);
            }
            *reinterpret_cast<float4*>(stage + qt_piece<kD>(r, c / 4 + j)) = z;
          }
        }
      } else if (splits > 1) {  // (the others fold without it; the status says so)
        if (half == 0) {
          ml[r] = make_float2(kQtNone, 0.f);
          mv_of[r] = kQtNone;
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  bool odd = false;
  constexpr int kLanes = kD / 4 < 32 ? kD / 4 : 32, kHalves = kD / 4 / kLanes;  // of a warp, a piece of the row each; head_dim 256: two
  constexpr int kWarps = kQtThreads / 32;
  auto out_of = [&](int r) {
    const int at = first_row + r;
    return reinterpret_cast<float4*>(p.out + ((long long)(token0 + at / p.groups) * hq + head * p.groups + at % p.groups) * kD);
  };
  const int last_row = min(query_rows - first_row, kQtRows);
  if (splits == 1) {
    if (lane < kLanes && !sm.abort_flag) {
#pragma unroll 4
      for (int i = warp; i < last_row * kHalves; i += kWarps) {
        const int piece = i % kHalves * kLanes + lane;
        out_of(i / kHalves)[piece] = *reinterpret_cast<const float4*>(stage + qt_piece<kD>(i / kHalves, piece));
      }
    }
  } else {
    cl_sync();  // every CTA's rows are staged
    const int row0 = rank * kQtRows / splits, row1 = min((rank + 1) * kQtRows / splits, last_row);
    // four rows of a warp at a time: lane 8 i + s has CTA s's reference, sum and, in the end, weight in row i of them
    for (int first = row0 + 4 * warp; first < row1; first += 4 * kWarps) {
      const int mine = first + lane / kQtMostSplits, s = lane % kQtMostSplits;
      float2 e = make_float2(kQtNone, 0.f);
      float mv = kQtNone;
      if (s < parts && mine < row1) {
        e = cl_ld2(cl_map(&ml[mine], s));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(mv) : "r"(cl_map(&mv_of[mine], s)) : "memory");
      }
      const bool none = e.y == 0.f;
      float top = none ? kQtNone : e.x;
#pragma unroll
      for (int o = 1; o < kQtMostSplits; o <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
      float sum = none ? 0.f : e.y * ex2_approx(e.x - top);
#pragma unroll
      for (int o = 1; o < kQtMostSplits; o <<= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
      const float f = none ? 0.f : ex2_approx(mv - top) / sum;
      const unsigned real = __ballot_sync(kFullMask, !none);
      odd |= !(f <= 1.f) || !(mv <= 3e38f);
      const int items = min(4, row1 - first) * kHalves;
#pragma unroll 1
      for (int i = 0; i < items; i += 2) {  // two pieces' loads at a time
        float4 x[2][kQtMostSplits];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int k = (i + u) / kHalves, piece = (i + u) % kHalves * kLanes + lane;
#pragma unroll
          for (int c = 0; c < kQtMostSplits; ++c) {
            x[u][c] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i + u < items && (real >> (k * kQtMostSplits + c) & 1) && lane < kLanes) x[u][c] = cl_ld4(cl_map(stage + qt_piece<kD>(first + k, piece), c));
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int k = min((i + u) / kHalves, 3);
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int c = 0; c < kQtMostSplits; ++c) {
            const float g = __shfl_sync(kFullMask, f, k * kQtMostSplits + c);
            if (real >> (k * kQtMostSplits + c) & 1) y = make_float4(fmaf(x[u][c].x, g, y.x), fmaf(x[u][c].y, g, y.y), fmaf(x[u][c].z, g, y.z), fmaf(x[u][c].w, g, y.w));
          }
          odd |= cl_not_finite(y);
          if (i + u < items && lane < kLanes) out_of(first + k)[(i + u) % kHalves * kLanes + lane] = y;
        }
      }
    }
  }
  if (sm.abort_flag) {  // give MMAs in flight time to land before the CTA's memory is released
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (splits > 1) cl_sync_read(odd);
  else __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

template <typename T, int kD>
static int launch_quantized_prefill_umma(QtParams p, int tiles, int most_tiles, cudaStream_t stream) {
  using L = QtSmem<T, kD>;
  constexpr int need = (int)sizeof(L) + 1024, bytes = need < 120 * 1024 ? 120 * 1024 : need;  // (one CTA per SM: all of its tensor memory)
  static_assert(need <= 232448, "shared memory of one CTA");
  static_assert((int)sizeof(L) - (int)offsetof(L, k_full) <= 4096 && offsetof(L, k_full) >= kQtRows * (kD * 4 + 12), "tiles, and staged rows in their place");
  auto* kernel = quantized_prefill_umma_kernel<T, kD>;
  static PerDeviceFlags ready, clusters[kQtMostSplits + 1];
  if (!once_per_device(ready, [&](int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess; }))
    return NVJ_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kQtThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  const int dev = current_device();
  p.splits = 1;
  // As many CTAs per tile as leave all tiles room at once (what the GPU's clusters have room for is asked once per device), and no more than
  // the longest row has tiles for.
  const long long room = ((long long)p.table_width * p.block_size + kQtKeys - 1) / kQtKeys / kQtSplitTiles;
  for (int s = 2; dev >= 0 && s <= kQtMostSplits && s <= room && (long long)tiles * p.num_kv_heads * s <= 148; ++s) {
    int n = clusters[s].v[dev].load(std::memory_order_acquire);  // the number + 1
    if (n == 0) {
      attr[0].val.clusterDim.x = s;
      cfg.gridDim = dim3(148 / s * s);
      cfg.numAttrs = 1;
      int count = 0;
      if (cudaOccupancyMaxActiveClusters(&count, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        count = 0;
      }
      n = count + 1;
      clusters[s].v[dev].store(n, std::memory_order_release);
    }
    if ((long long)tiles * p.num_kv_heads <= n - 1) p.splits = s;
  }
  if ((long long)most_tiles * p.splits > 0x7fffffffLL) return NVJ_ERR_TOO_LARGE;
  // (scratch for the CTAs of clusters only as far as it goes)
  if (p.splits == 1 || (long long)most_tiles * p.splits * p.num_kv_heads * kQtRows * kD * 4 > p.flush_bytes) p.flush = nullptr;
  attr[0].val.clusterDim.x = p.splits;
  cfg.gridDim = dim3((unsigned)(most_tiles * p.splits), p.num_kv_heads);
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
}
template <typename T>
static int launch_quantized_prefill_type(const QtParams& p, int head_dim, int tiles, int most_tiles, cudaStream_t stream) {
  if (head_dim == 256) return launch_quantized_prefill_umma<T, 256>(p, tiles, most_tiles, stream);
  if (head_dim == 128) return launch_quantized_prefill_umma<T, 128>(p, tiles, most_tiles, stream);
  return launch_quantized_prefill_umma<T, 64>(p, tiles, most_tiles, stream);
}

}  // namespace nvj
