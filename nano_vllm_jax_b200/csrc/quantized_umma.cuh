// Attention over the 8-bit paged cache on the 5th-generation tensor cores (tcgen05, kind::f8f6f4): the kernel of large batches of
// rows of few query tokens.  Included by one file per type of query (quantized_umma_*.cu).
//
// e4m3 is an operand type of the tensor cores, so K and V need no conversion and go from memory to shared memory and no further; what
// has to become e4m3 is the other side, and a number becomes a sum of e4m3 terms: t0 = rne(x), t1 = rne(16 (x - t0)), ..., each with
// four bits of it.  bf16 queries (8 bits) are two terms exactly, f16 three, f32 five (2^-20); the weights of the softmax five (2^-20).  The
// terms are columns of their own, added with their powers of 16 when a result is read:
//   S^T = K Q^T    [128 keys x kQTerms * kC]            32 dims per MMA, K and Q from shared memory, K-major;
//   O^T = V^T P^T  [kDim / 128 x 128 dims x 5 * kC]     32 keys per MMA, V and the weights from shared memory, MN-major.
// A tile of 128 keys of one kv head is 64 KiB (head_dim 256), 1.4 us of an SM's share of the memory; its products take a fraction of
// that, and its softmax (thread = key) ~ 150 instructions per warp for four columns, where the mma.sync form, which converts every
// number in registers, spends 5500 on the same bytes.
//
// Work split: CTA = (range, kv head and column tile).  The 16-key units of all rows form one sequence that is cut into equal ranges
// (decode_parts.cuh); rows cut over ranges leave partials, folded by a second small launch.
//   warps 0 - 3  softmax, thread = key: scores from tensor memory, times the K scale of the key's block; weights
//                exp2(s + log2 V scale - reference) as e4m3 terms into shared memory; their sum without the V scale under a
//                reference of its own.  References move only when a score passes one by 2^8 (weights up to 2^8 <= 448).  Thread = dim when
//                a row's segment ends.
//   warp 4       MMA issue.
//   warp 5       TMA producer: 16-key boxes [8-key group][128-byte chunk][8 keys][128 B], 128-byte swizzle, into a ring of tiles of K
//                and V in turn (160 KiB).
//   warps 6, 7   the next segment's queries: scaled to 2^7 - 2^8 by a power of two per column, split into terms.
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
constexpr int kQuUnit = 16;     // keys per box
constexpr int kQuUnits = kQuTile / kQuUnit;
constexpr int kQuPTerms = 5;
constexpr float kQuNone = -3e38f, kQuSlack = 8.f;

template <typename T>
constexpr int quq_terms() {
  return sizeof(T) == 4 ? 5 : std::is_same<T, __half>::value ? 3 : 2;
}

template <typename T, int kDim, int kC>
struct QuLayout {
  static constexpr int kQTerms = quq_terms<T>();
  static constexpr int kChunks = kDim / 128;
  static constexpr int kNS = (kQTerms * kC + 15) / 16 * 16;   // columns of S (N of an MMA: multiples of 16)
  static constexpr int kNO = (kQuPTerms * kC + 15) / 16 * 16;  // columns of O
  static constexpr int kSets0 = (512 - kNS) / (kNO * kChunks);
  static constexpr int kSets = kSets0 < 1 ? 1 : (kSets0 > 3 ? 3 : kSets0);  // accumulators that take the tiles in turn: shorter sums
  static constexpr int kColO = kNS;
  static constexpr int kTileBytes = kQuTile * kDim;           // of K (or V)
  static constexpr int kUnitBytes = kQuUnit * kDim;
  static constexpr int kSlots = 160 * 1024 / kTileBytes;
  static constexpr int kQChunk = kNS * 128;                   // bytes of a chunk of the query terms
  static_assert(kNO <= 128 && kNS <= 256, "a row of weights is 128 bytes");
  static_assert(kNS + kSets * kChunks * kNO <= 512, "tensor memory");
};

template <typename T, int kDim, int kC>
struct QuSmem {
  using L = QuLayout<T, kDim, kC>;
  alignas(1024) char slot[L::kSlots][L::kTileBytes];
  alignas(1024) char q[L::kChunks][L::kQChunk];  // [chunk][term * kC + column][128 B]
  alignas(1024) char w[kQuTile * 128];           // weights' terms [key][128 B]
  alignas(8) unsigned long long full[L::kSlots], empty[L::kSlots], q_full, q_free, s_full, p_full, o_full, o_free;
  alignas(16) float factor[2][kC];  // by segment parity: what a column's products are multiplied by, and the keys it may see
  alignas(16) int limit[2][kC];
  alignas(16) float red[4][kC], red_v[4][kC];
  alignas(16) float m[kC], mv[kC], f[kC], fv[kC];
  int scan[16];
  int start_b, start_j, abort_flag;
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
// Whether `mine` holds in any thread of the softmax warps, which meet here.
__device__ __forceinline__ bool qu_meet_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any) : "r"((uint32_t)mine) : "memory");
  return any != 0;
}
// The warp's largest x (order-preserving integers; a NaN with a clear sign counts as the largest).
__device__ __forceinline__ float qu_warp_max(float x) {
  const int i = __float_as_int(x), k = __reduce_max_sync(kFullMask, i ^ ((i >> 31) & 0x7fffffff));
  return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}

// A place in the ring: K and V of a tile follow one another.
template <int kSlots>
struct QuRing {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step() {
    if (++at == kSlots) { at = 0; phase ^= 1u; }
  }
};
// The CTA's segments: 16-key units [j0, j0 + n) of row b, which has nb of them and len keys.
struct QuSeg {
  int b, j0, n, nb, len;
  __device__ __forceinline__ int tiles() const { return (n + kQuUnits - 1) / kQuUnits; }
  __device__ __forceinline__ int tile_units(int t) const { return min(n - t * kQuUnits, kQuUnits); }
  __device__ __forceinline__ bool whole() const { return n == nb; }
};
struct QuWalk {
  int b, j;
  long long g, g1;
  __device__ __forceinline__ bool next(const DecodeParams& p, QuSeg& s) {
    Seg r;
    if (!next_seg(p, b, j, g, g1, r)) return false;
    s = QuSeg{r.b, r.j0, r.j1 - r.j0, r.nb, r.len};
    return true;
  }
};

// ---- warp 5: TMA loads ------------------------------------------------------------------------------------------------------------
template <typename T, int kDim, int kC>
__device__ __forceinline__ void qu_producer(const CUtensorMap* k_map, const CUtensorMap* v_map, const QuParams& a, const DecodeParams& p,
                                            QuSmem<T, kDim, kC>& sm, int head, QuWalk walk, int lane) {
  using L = QuLayout<T, kDim, kC>;
  const int per_block = p.block_size / kQuUnit;
  const int oob = (int)(p.num_blocks * (p.block_size / 8));  // a box that starts here is filled with zeros
  uint64_t policy;  // every block is read once
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  auto ids_at = [&](const QuSeg& s, int i) {
    return i + lane < s.n ? p.block_tables[(long long)s.b * p.table_width + (s.j0 + i + lane) / per_block] : 0;
  };
  QuRing<L::kSlots> at;
  bool reuse = false;  // the slot has been used before
  QuSeg s, nxt;
  bool have = walk.next(p, s);
  int ids = have ? ids_at(s, 0) : 0;
  while (have) {
    bool more = false;
    int next_first = 0;
    for (int i0 = 0; i0 < s.n; i0 += 32) {  // 32 units = 4 tiles at a time
      const int ahead = ids_at(s, i0 + 32);
      const int n = min(s.n - i0, 32);
      const bool bad = lane < n && (ids < 0 || ids >= p.num_blocks);
      if (bad) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      const int group = bad || lane >= n ? oob : ids * (p.block_size / 8) + (s.j0 + i0 + lane) % per_block * 2;
      for (int i = 0; i < n; i += kQuUnits) {
        const int cnt = min(n - i, kQuUnits), mine = __shfl_sync(kFullMask, group, (i + lane) & 31);  // a lane per unit
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (reuse && !um_wait(&sm.empty[at.at], at.phase ^ 1u, &sm.abort_flag, p.status)) return;
          const uint32_t full = smem_u32(&sm.full[at.at]), dst = smem_u32(sm.slot[at.at]) + lane * L::kUnitBytes;
          if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)cnt * L::kUnitBytes);
          __syncwarp();
          if (lane < cnt) qu_load(dst, kv == 0 ? k_map : v_map, mine, head, full, policy);
          __syncwarp();
          at.step();
          if (at.at == 0) reuse = true;
        }
      }
      ids = ahead;
      if (i0 == 0) {  // the row behind this one, once the first copies are on their way
        more = walk.next(p, nxt);
        if (more) next_first = ids_at(nxt, 0);
      }
    }
    s = nxt;
    ids = next_first;
    have = more;
  }
}

// ---- warp 4: MMA issue ------------------------------------------------------------------------------------------------------------
template <typename T, int kDim, int kC>
__device__ __forceinline__ void qu_mma_warp(QuSmem<T, kDim, kC>& sm, const DecodeParams& p, uint32_t tmem, QuWalk walk) {
  using L = QuLayout<T, kDim, kC>;
  constexpr uint32_t idesc_s = qu_idesc(L::kNS, false, false), idesc_o = qu_idesc(L::kNO, true, true);
  const uint64_t k_desc0 = umma_desc(smem_u32(sm.slot[0]), 16, L::kChunks * 1024);  // keys are rows: groups of 8
  const uint64_t v_desc0 = umma_desc(smem_u32(sm.slot[0]), 1024, L::kChunks * 1024);  // dims are rows, a chunk at a time; keys in groups of 8
  const uint64_t q_desc = umma_desc(smem_u32(sm.q[0]), 16, 1024);
  const uint64_t w_desc = umma_desc(smem_u32(sm.w), 1024, 1024);
  QuRing<L::kSlots> at;
  QuSeg s;
  uint32_t tile = 0;
  for (uint32_t seg = 0; walk.next(p, s); ++seg) {
    const int nt = s.tiles();
    for (int t = 0; t < nt; ++t, ++tile) {
      // (rows of keys that the tile does not have are computed from whatever lies there, and masked)
      if (t == 0 && !um_wait(&sm.q_full, seg & 1u, &sm.abort_flag, p.status)) return;
      if (!um_wait(&sm.full[at.at], at.phase, &sm.abort_flag, p.status)) return;
      tc_fence_after_sync();
      if (um_elect_one()) {
        const uint64_t k_desc = k_desc0 + (uint64_t)((at.at * L::kTileBytes) >> 4);
#pragma unroll
        for (int ks = 0; ks < kDim / 32; ++ks)
          qu_mma(tmem, k_desc + (uint64_t)(((ks >> 2) * 1024 + (ks & 3) * 32) >> 4), q_desc + (uint64_t)(((ks >> 2) * L::kQChunk + (ks & 3) * 32) >> 4),
                 idesc_s, ks > 0 ? 1u : 0u);
        umma_commit(smem_u32(&sm.s_full));
        umma_commit(smem_u32(&sm.empty[at.at]));
        if (t == nt - 1) umma_commit(smem_u32(&sm.q_free));
      }
      __syncwarp();
      at.step();
      if (!um_wait(&sm.full[at.at], at.phase, &sm.abort_flag, p.status)) return;
      if (!um_wait(&sm.p_full, tile & 1u, &sm.abort_flag, p.status)) return;
      // the first weighted sum of a segment overwrites O: the segment before must have been read out
      if (t == 0 && seg > 0 && !um_wait(&sm.o_free, (seg - 1) & 1u, &sm.abort_flag, p.status)) return;
      tc_fence_after_sync();
      if (um_elect_one()) {
        const int steps = (s.tile_units(t) + 1) / 2;
        const uint32_t o = tmem + L::kColO + (t % L::kSets) * (L::kChunks * L::kNO);
        const uint64_t v_desc = v_desc0 + (uint64_t)((at.at * L::kTileBytes) >> 4);
        for (int i = 0; i < steps; ++i) {  // 32 keys, four groups of 8
          const uint32_t more = (t >= L::kSets || i > 0) ? 1u : 0u;
          const uint64_t wd = w_desc + (uint64_t)((i * 32 * 128) >> 4), vd = v_desc + (uint64_t)((i * 2 * L::kUnitBytes) >> 4);
#pragma unroll
          for (int h = 0; h < L::kChunks; ++h) qu_mma(o + h * L::kNO, vd + (uint64_t)((h * 1024) >> 4), wd, idesc_o, more);
        }
        umma_commit(smem_u32(&sm.empty[at.at]));
        if (t == nt - 1) umma_commit(smem_u32(&sm.o_full));
      }
      __syncwarp();
      at.step();
    }
  }
}

// Scales of the CTA's tiles, one tile ahead: thread = key.  `id` belongs to the tile behind `k_unit` and `v_unit`.
struct QuScales {
  QuWalk walk;
  QuSeg s;
  int t;
  bool have;
  int id;

  __device__ __forceinline__ void fetch_id(const DecodeParams& p, int key) {
    id = -1;
    const int u = t * kQuUnits + key / kQuUnit;
    if (have && u < s.n) id = p.block_tables[(long long)s.b * p.table_width + (s.j0 + u) / (p.block_size / kQuUnit)];
  }
  __device__ __forceinline__ void begin(const DecodeParams& p, const QuWalk& w, int key) {
    walk = w;
    t = 0;
    have = walk.next(p, s);
    fetch_id(p, key);
  }
  // the scales of the tile whose id is here (of -1: no key), and the id of the one behind it
  __device__ __forceinline__ void step(const QuParams& a, const DecodeParams& p, int key, int head, float& k_unit, float& v_unit) {
    k_unit = 0.f;
    v_unit = -1.f;
    if (id >= 0 && id < p.num_blocks) {
      k_unit = a.k_scale[(long long)id * a.num_kv_heads + head];
      v_unit = a.v_scale[(long long)id * a.num_kv_heads + head];
    }
    if (have && ++t == s.tiles()) {
      t = 0;
      have = walk.next(p, s);
    }
    fetch_id(p, key);
  }
};

// ---- warps 0 - 3: softmax and output.  Thread = key of the tile, then dim of the output ---------------------------------------
// (A wait that runs out does so for one warp and perhaps not for the next: they leave together, behind a meeting.)
template <typename T, int kDim, int kC>
__device__ __forceinline__ void qu_softmax_warps(QuSmem<T, kDim, kC>& sm, const QuParams& a, const DecodeParams& p, uint32_t tmem, int head, int hct,
                                                 int ct, QuWalk walk, int range, int warp, int lane) {
  using L = QuLayout<T, kDim, kC>;
  constexpr int kSRead = (L::kQTerms * kC + 7) / 8, kORead = (kQuPTerms * kC + 7) / 8;  // pieces of 8 columns
  const int key = warp * 32 + lane;
  const uint32_t w_row = smem_u32(sm.w) + key * 128;
  tmem += (uint32_t)(warp * 32) << 16;
  QuScales scales;
  scales.begin(p, walk, key);
  float next_k, next_v;
  scales.step(a, p, key, head, next_k, next_v);
  QuRing<L::kSlots> at;
  QuSeg s;
  uint32_t tile = 0;
  for (uint32_t seg = 0; walk.next(p, s); ++seg) {
    const float* factor = sm.factor[seg & 1u];
    const int* limit = sm.limit[seg & 1u];
    float l[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) l[c] = 0.f;
    const int nt = s.tiles();
    for (int t = 0; t < nt; ++t, ++tile) {
      at.step();  // V's slot
      const int cnt = s.tile_units(t);
      // this thread's key; one that the tile does not have is behind everybody's last one
      const int at_key = (key >> 4) < cnt ? (s.j0 + t * kQuUnits) * kQuUnit + key : 0x7fffffff;
      const float k_unit = next_k, v_unit = next_v;
      scales.step(a, p, key, head, next_k, next_v);
      const bool there = v_unit >= 0.f;
      const float v_log = there ? __log2f(v_unit) : 0.f;
      const bool ok = um_wait(&sm.s_full, tile & 1u, &sm.abort_flag, p.status);
      tc_fence_after_sync();
      float sc[kC];
      {
        float x[kSRead][8];
#pragma unroll
        for (int i = 0; i < kSRead; ++i) tmem_ld8(tmem + 8 * i, x[i]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kSRead; ++i) tmem_loaded(x[i]);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          float y = x[((L::kQTerms - 1) * kC + c) / 8][((L::kQTerms - 1) * kC + c) % 8];
#pragma unroll
          for (int j = L::kQTerms - 2; j >= 0; --j) y = fmaf(y, 0.0625f, x[(j * kC + c) / 8][(j * kC + c) % 8]);
          sc[c] = there && at_key < limit[c] ? y * (factor[c] * k_unit) : -INFINITY;
        }
      }
      bool above = false;
      if (t > 0) {
#pragma unroll
        for (int c = 0; c < kC; ++c) above |= sc[c] > sm.m[c] + kQuSlack || sc[c] + v_log > sm.mv[c] + kQuSlack;
      }
      if (qu_meet_any(!ok || t == 0 || above)) {
        // the first tile, or rarely a later one: the tile's maxima; what has been summed so far is brought to the new references
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const float x = qu_warp_max(sc[c]), y = qu_warp_max(sc[c] + v_log);
          if (lane == 0) {
            sm.red[warp][c] = x;
            sm.red_v[warp][c] = y;
          }
        }
        if (qu_meet_any(!ok)) return;
        if (key < kC) {
          const float x = fmaxf(fmaxf(sm.red[0][key], sm.red[1][key]), fmaxf(sm.red[2][key], sm.red[3][key]));
          const float y = fmaxf(fmaxf(sm.red_v[0][key], sm.red_v[1][key]), fmaxf(sm.red_v[2][key], sm.red_v[3][key]));
          const float old = t == 0 ? kQuNone : sm.m[key], old_v = t == 0 ? kQuNone : sm.mv[key];
          const float now = fmaxf(old, x), now_v = fmaxf(old_v, y);
          sm.f[key] = ex2_approx(old - now);
          sm.fv[key] = ex2_approx(old_v - now_v);
          sm.m[key] = now;
          sm.mv[key] = now_v;
        }
        qu_meet_any(false);
        if (t > 0) {  // (the weighted sums so far are complete: S of this tile was issued behind them)
#pragma unroll
          for (int c = 0; c < kC; ++c) l[c] *= sm.f[c];
          const int sets = t < L::kSets ? t : L::kSets;
#pragma unroll 1
          for (int i = 0; i < sets * L::kChunks; ++i) {
#pragma unroll
            for (int c8 = 0; c8 < kORead; ++c8) {
              float o[8];
              tmem_ld8(tmem + L::kColO + i * L::kNO + 8 * c8, o);
              tmem_ld_wait();
              tmem_loaded(o);
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] *= sm.fv[(8 * c8 + k) % kC];
              qu_tmem_st8(tmem + L::kColO + i * L::kNO + 8 * c8, o);
            }
          }
          tmem_st_wait();
        }
      }
      // weights as e4m3 terms: byte term * kC + column of the key's row
      {
        float r[kC];
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          l[c] += ex2_approx(sc[c] - sm.m[c]);
          r[c] = ex2_approx(sc[c] + v_log - sm.mv[c]);
        }
        uint32_t bytes[(kQuPTerms * kC / 4 + 3) / 4 * 4];
#pragma unroll
        for (int i = 0; i < (kQuPTerms * kC / 4 + 3) / 4 * 4; ++i) bytes[i] = 0u;
#pragma unroll
        for (int j = 0; j < kQuPTerms; ++j)
#pragma unroll
          for (int c = 0; c < kC; c += 4) {
            const uint32_t x = q_pack2(r[c], r[c + 1]), y = q_pack2(r[c + 2], r[c + 3]);
            bytes[(j * kC + c) / 4] = x | y << 16;
            if (j + 1 < kQuPTerms) {
              const float2 b0 = q_float2(q_half2(x)), b1 = q_float2(q_half2(y));
              r[c] = (r[c] - b0.x) * 16.f;
              r[c + 1] = (r[c + 1] - b0.y) * 16.f;
              r[c + 2] = (r[c + 2] - b1.x) * 16.f;
              r[c + 3] = (r[c + 3] - b1.y) * 16.f;
            }
          }
#pragma unroll
        for (int i = 0; i < (kQuPTerms * kC / 4 + 3) / 4; ++i)
          qu_sts4(w_row + ((i ^ (key & 7)) << 4), bytes[4 * i], bytes[4 * i + 1], bytes[4 * i + 2], bytes[4 * i + 3]);
      }
      // V rows of keys that are not there weigh nothing, but may hold anything: 0 x NaN is not 0
      if (t == nt - 1 && ((cnt & 1) || (s.j0 + s.n == s.nb && (s.len & (kQuUnit - 1))))) {
        if (qu_meet_any(!um_wait(&sm.full[at.at], at.phase, &sm.abort_flag, p.status))) return;
        if (key < ((cnt + 1) / 2) * 32 && (at_key == 0x7fffffff || at_key >= s.len)) {
          const uint32_t v_row = smem_u32(sm.slot[at.at]) + (key >> 3) * (8 * kDim) + (key & 7) * 128;
#pragma unroll
          for (int i = 0; i < kDim / 16; ++i) qu_sts4(v_row + (i >> 3) * 1024 + (i & 7) * 16, 0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      mbar_arrive(smem_u32(&sm.p_full));
      at.step();
    }
    // ---- end of the segment: sums over the keys, then the output or the partial
#pragma unroll
    for (int c = 0; c < kC; ++c) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l[c] += __shfl_xor_sync(kFullMask, l[c], o);
      if (lane == 0) sm.red[warp][c] = l[c];
    }
    if (qu_meet_any(!um_wait(&sm.o_full, seg & 1u, &sm.abort_flag, p.status))) return;
    const bool final_row = s.whole();
    const long long slot = (long long)partial_slot(range, s.j0 == 0) * a.hcts + hct;
    if (key < kC) {
      const float sum = (sm.red[0][key] + sm.red[1][key]) + (sm.red[2][key] + sm.red[3][key]);
      const float up = ex2_approx(sm.mv[key] - sm.m[key]);
      sm.f[key] = sum == 0.f ? 0.f : final_row ? up / sum : up;
      if (!final_row) *reinterpret_cast<float2*>(a.part_ml + (slot * kC + key) * 2) = make_float2(sm.m[key], sum);
    }
    qu_meet_any(false);
    tc_fence_after_sync();
    const int sets = nt < L::kSets ? nt : L::kSets;
    const int columns = min(a.columns - ct * kC, kC);
    const long long token = a.query_start_loc ? (long long)a.query_start_loc[s.b] : (long long)s.b * a.width;
#pragma unroll 1
    for (int h = 0; h < L::kChunks; ++h) {
      float y[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) y[c] = 0.f;
#pragma unroll 1
      for (int k = 0; k < sets; ++k) {
        float part[kC];  // high terms last: small numbers are added first
#pragma unroll
        for (int c = 0; c < kC; ++c) part[c] = 0.f;
#pragma unroll
        for (int i = kORead - 1; i >= 0; --i) {
          float o[8];
          tmem_ld8(tmem + L::kColO + (k * L::kChunks + h) * L::kNO + 8 * i, o);
          tmem_ld_wait();
          tmem_loaded(o);
#pragma unroll
          for (int e = 7; e >= 0; --e) {
            const int n = 8 * i + e;
            if (n < kQuPTerms * kC) part[n % kC] = fmaf(part[n % kC], 0.0625f, o[e]);
          }
        }
#pragma unroll
        for (int c = 0; c < kC; ++c) y[c] += part[c];
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        if (c < columns) {
          const int at_col = ct * kC + c;
          float* to = final_row ? a.out + ((token + at_col / a.groups) * a.num_q_heads + head * a.groups + at_col % a.groups) * kDim
                                : a.part_acc + (slot * kC + c) * kDim;
          const float f = sm.f[c];
          to[h * 128 + key] = f == 0.f ? 0.f : y[c] * f;
        }
      }
    }
    tc_fence_before_sync();  // the next segment's first weighted sums overwrite what was just read
    mbar_arrive(smem_u32(&sm.o_free));
  }
}

// ---- warps 6 and 7: a segment's queries as e4m3 terms -------------------------------------------------------------------------
template <typename T, int kDim, int kC>
__device__ __forceinline__ void qu_query_warps(QuSmem<T, kDim, kC>& sm, const QuParams& a, const DecodeParams& p, int head, int ct, QuWalk walk, int tid) {
  using L = QuLayout<T, kDim, kC>;
  constexpr int kFly = kC / 2 < 4 ? kC / 2 : 4;  // columns of a warp in flight
  const int half = tid >> 5, lane = tid & 31;
  const int d = 8 * lane;  // (head_dim 128: half of the lanes)
  QuSeg s;
  for (uint32_t seg = 0; walk.next(p, s); ++seg) {
    const long long token = a.query_start_loc ? (long long)a.query_start_loc[s.b] : (long long)s.b * a.width;
#pragma unroll 1
    for (int c0 = 0; c0 < kC; c0 += 2 * kFly) {
      float x[kFly][8];
      int limit[kFly];
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int at = ct * kC + c0 + 2 * i + half;
        limit[i] = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = 0.f;
        if (at < a.columns) {
          const long long row = token + at / a.groups;
          if (d < kDim) q_floats(q_load8(static_cast<const T*>(a.q) + (row * a.num_q_heads + head * a.groups + at % a.groups) * kDim + d), x[i]);
          const int last = a.positions ? a.positions[row] : 0x7ffffffe;
          limit[i] = last < s.len ? last + 1 : s.len;
        }
      }
      if (c0 == 0 && seg > 0 && !um_wait(&sm.q_free, (seg - 1) & 1u, &sm.abort_flag, p.status)) return;
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int c = c0 + 2 * i + half;
        const int bits = __reduce_max_sync(kFullMask, __float_as_int(q_largest(0.f, x[i])));
        int e = (bits >> 23) - 127 - 7;  // largest = 2^(e + 7) * [1, 2)
        e = bits == 0 ? 0 : (e < -126 ? -126 : e);
        const float down = q_pow2(-e);
        bool odd = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          odd |= !(x[i][k] - x[i][k] == 0.f);  // an infinity or NaN: the column's scores are NaN
          x[i][k] *= down;
        }
        odd = __any_sync(kFullMask, odd);
        if (lane == 0) {
          sm.factor[seg & 1u][c] = odd ? __int_as_float(0x7fffffff) : q_pow2(e) * a.scale_log2;
          sm.limit[seg & 1u][c] = limit[i];
        }
#pragma unroll
        for (int j = 0; j < L::kQTerms; ++j) {
          uint32_t b[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            b[k] = q_pack2(x[i][2 * k], x[i][2 * k + 1]);
            const float2 y = q_float2(q_half2(b[k]));
            x[i][2 * k] = (x[i][2 * k] - y.x) * 16.f;
            x[i][2 * k + 1] = (x[i][2 * k + 1] - y.y) * 16.f;
          }
          const int row = j * kC + c;
          if (d < kDim)
            *reinterpret_cast<uint2*>(sm.q[d / 128] + row * 128 + (((d % 128 / 16) ^ (row & 7)) << 4) + (d & 8)) =
                make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        }
      }
    }
    fence_proxy_async_smem();
    mbar_arrive(smem_u32(&sm.q_full));
  }
}

template <typename T, int kDim, int kC>
__global__ void __launch_bounds__(kDecodeThreads, 1)
quantized_umma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const QuParams a, const DecodeParams p) {
  using L = QuLayout<T, kDim, kC>;
  extern __shared__ unsigned char qu_smem_raw[];
  QuSmem<T, kDim, kC>& sm = *reinterpret_cast<QuSmem<T, kDim, kC>*>((reinterpret_cast<uintptr_t>(qu_smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hct = blockIdx.x % a.hcts, range = blockIdx.x / a.hcts, ranges = gridDim.x / a.hcts;
  const int head = hct / a.column_tiles, ct = hct % a.column_tiles;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&k_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
    sm.start_b = p.batch; sm.start_j = 0; sm.abort_flag = 0;
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(smem_u32(&sm.full[i]), 1);
      mbar_init(smem_u32(&sm.empty[i]), 1);
    }
    mbar_init(smem_u32(&sm.q_full), 64);
    mbar_init(smem_u32(&sm.q_free), 1);
    mbar_init(smem_u32(&sm.s_full), 1);
    mbar_init(smem_u32(&sm.p_full), 128);
    mbar_init(smem_u32(&sm.o_full), 1);
    mbar_init(smem_u32(&sm.o_free), 128);
    mbar_fence_init();
  }
  pdl_wait();
  {  // this CTA's share of the block tables into the L2, while the lengths are on their way
    const long long lines = ((long long)p.batch * p.table_width * (long long)sizeof(int32_t) + 127) / 128;
    const long long line = (long long)blockIdx.x * kDecodeThreads + threadIdx.x;
    if (line < lines) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.block_tables) + line * 128));
  }
  // ---- pass 1: total number of units; zero the output of rows without keys
  int mine = 0, first_n = 0;
  for (int base = 0; base < p.batch; base += kDecodeThreads) {
    const int b = base + threadIdx.x;
    int len = 0;
    if (b < p.batch) len = decode_row_len(p, b);
    const int n = blocks_in_sequence(p, (len + kBlk - 1) / kBlk);
    if (base == 0) first_n = n;
    mine += n;
    const bool ours = b < p.batch && len <= 0 && b % ranges == range &&
                      (!p.query_start_loc || p.query_start_loc[b + 1] - p.query_start_loc[b] == 1);
    for (unsigned todo = __ballot_sync(kFullMask, ours); todo; todo &= todo - 1) {
      const int bb = base + (warp << 5) + (__ffs(todo) - 1);
      const long long token = a.query_start_loc ? (long long)a.query_start_loc[bb] : (long long)bb * a.width;
      const int columns = min(a.columns - ct * kC, kC);
      for (int i = lane; i < columns * (kDim / 4); i += 32) {
        const int at = ct * kC + i / (kDim / 4);
        reinterpret_cast<float4*>(a.out + ((token + at / a.groups) * a.num_q_heads + head * a.groups + at % a.groups) * kDim)[i % (kDim / 4)] =
            make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  int total = 0;
  const int incl = cta_inclusive_scan(mine, sm.scan, total);
  const Partition pt = make_partition(total > 0 ? total : 1, ranges);
  const long long g0 = pt.start(range), g1 = pt.start(range + 1);
  if (total == 0 || range >= pt.n || g0 == g1) {  // nothing for this CTA
    if (hct == 0 && threadIdx.x == 0) a.cuts[range] = kNoCut;
    return;
  }
  // ---- pass 2: locate (row, unit) of g0
  long long carry = 0;
  if (p.batch <= kDecodeThreads) {  // one row per thread: the scan of pass 1 has the answer already
    const long long excl = incl - first_n;
    if (first_n > 0 && excl <= g0 && g0 < excl + first_n) { sm.start_b = threadIdx.x; sm.start_j = (int)(g0 - excl); }
    carry = g0 + 1;  // skips the loop below
  }
  for (int base = 0; base < p.batch && carry <= g0; base += kDecodeThreads) {
    const int b = base + threadIdx.x;
    int n = 0;
    if (b < p.batch) n = blocks_in_sequence(p, (decode_row_len(p, b) + kBlk - 1) / kBlk);
    int chunk_total = 0;
    const long long excl = carry + cta_inclusive_scan(n, sm.scan, chunk_total) - n;
    if (n > 0 && excl <= g0 && g0 < excl + n) { sm.start_b = b; sm.start_j = (int)(g0 - excl); }
    carry += chunk_total;
  }
  // (rows of the query terms that no column fills: finite, and never read)
  for (int i = threadIdx.x; i < (int)sizeof(sm.q) / 16; i += kDecodeThreads) reinterpret_cast<uint4*>(sm.q)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  const QuWalk walk{sm.start_b, sm.start_j, g0, g1};
  if (warp == 4) {  // tensor memory between the wait and the release (umma.cuh)
    tmem_alloc(smem_u32(&sm.tmem_base), 512);
    if (lane == 0) pdl_release();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sm.tmem_base;

  if (warp < 4) qu_softmax_warps<T, kDim, kC>(sm, a, p, tmem, head, hct, ct, walk, range, warp, lane);
  else if (warp == 4) {
    if (hct == 0 && lane == 0) a.cuts[range] = umma_cut(p, pt, range, walk.b, walk.j, walk.g);
    __syncwarp();
    qu_mma_warp<T, kDim, kC>(sm, p, tmem, walk);
  }
  else if (warp == 5) qu_producer<T, kDim, kC>(&k_map, &v_map, a, p, sm, head, walk, lane);
  else qu_query_warps<T, kDim, kC>(sm, a, p, head, ct, walk, threadIdx.x - 192);

  tc_fence_before_sync();
  __syncthreads();
  if (sm.abort_flag) {  // give copies and MMAs in flight time to land before the CTA's memory is released
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 4) tmem_dealloc(tmem, 512);
}

template <typename T, int kDim, int kC>
static int launch_quantized_umma(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int ranges,
                                 cudaStream_t stream) {
  constexpr int bytes = (int)sizeof(QuSmem<T, kDim, kC>) + 1024;
  static_assert(bytes <= 232448, "the ring exceeds the shared memory of one CTA");
  auto* kernel = quantized_umma_kernel<T, kDim, kC>;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess; }))
    return NVJ_ERR_LAUNCH;
  return launch_after(kernel, dim3((unsigned)(ranges * a.hcts)), dim3(kDecodeThreads), bytes, stream, k_map, v_map, a, p) == cudaSuccess ? NVJ_OK
                                                                                                                                 : NVJ_ERR_LAUNCH;
}
template <typename T>
static int launch_quantized_umma_shape(const CUtensorMap& k_map, const CUtensorMap& v_map, const QuParams& a, const DecodeParams& p, int head_dim,
                                       int ranges, cudaStream_t stream) {
  auto columns = [&](auto dim) {
    constexpr int kDim = decltype(dim)::value;
    switch (a.tile_columns) {
      case 4: return launch_quantized_umma<T, kDim, 4>(k_map, v_map, a, p, ranges, stream);
      case 8: return launch_quantized_umma<T, kDim, 8>(k_map, v_map, a, p, ranges, stream);
      case 16: return launch_quantized_umma<T, kDim, 16>(k_map, v_map, a, p, ranges, stream);
      default: return launch_quantized_umma<T, kDim, 24>(k_map, v_map, a, p, ranges, stream);
    }
  };
  return head_dim == 256 ? columns(std::integral_constant<int, 256>{}) : columns(std::integral_constant<int, 128>{});
}

}  // namespace nvj
