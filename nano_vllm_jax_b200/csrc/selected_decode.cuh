// Decode attention over selected blocks of a row: what its kernels share, and the one on tensor-core tiles.
//
//   out[t, h] = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale * q[t, h] . k_p),  p in the blocks that selected[t, kv head] lists, p < len, p <= position[t]
//
// A list holds columns of the row's block table, -1 where it has ended; every entry counts, also one that is there twice.
//
// Bound by the bytes of K and V of the listed blocks, which lie scattered over the pool, block_size * head_dim numbers at a stretch if a block had
// one kv head only.  selected_decode_kernel, for bf16 and f16 caches with blocks of whole 16-key tiles:
//   * one thread-block cluster per (query token, kv head, tile of query columns); the list's 16-key tiles are dealt to the cluster's warps in
//     turn, and warps and CTAs merge through shared and distributed shared memory: no workspace, no second launch;
//   * K and V go from global memory to registers in 16-byte pieces and nowhere else: both products are taken transposed
//     (S^T = K Q^T, O^T = V^T P^T), and since the order of a contraction is free, the 16 bytes that a lane holds of a row ARE its
//     operands, permuted the same way on the other side; V takes one byte permute per word besides, which pairs its keys;
//   * queries of another type than the cache's are sums of three terms of its type, 24 bits; weights of three bf16 or two f16 terms, 24 and 22 bits (two of
//     bf16, 2^-17: 64 selected blocks of 256 rows 2.1e-6 from 64 bits, relative to the size of the result, instead of 4.5e-7).  With up to four columns
//     two terms of the weights are the two halves of the eight columns of one mma.sync.  A tile's products are summed by themselves and added in fp32 (left in the
//     tensor cores' sums, which cut their last place, 8192 keys 3e-6 - 9e-6 from 64 bits instead of 1e-7 - 5e-7; 2% of the time);
//   * a warp walks only the tiles that are there: it holds the places of its next 32 in its lanes and takes the set bits of their vote.
// 256 rows, 64 blocks of 16 keys, 8 heads over 2 of 256: 540 MB in 90.5 us, 91% of the copy rate (f16 89; f32 queries 103); 48 rows, 32 heads over 8 of 128 49.7, 92%.  Other
// head_dims take the form of three query terms and eight columns: 256 rows of 6 heads over 3 of 96 74.5 us, 62%.
// Maxima are lazy: one vote per tile says whether a score has left them behind, and only then the sums are rescaled.
#pragma once

#include "cluster.cuh"
#include "decode_cluster.cuh"
#include "quantized_kv.cuh"

namespace nvj {

struct SelectedParams {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  const int32_t* positions;  // nullable [rows, width]
  const int32_t* selected;   // [rows, width, hkv, entries]
  float* out;
  int32_t* status;
  long long num_blocks;
  int q_dtype, rows, width, table_width, block_size, hkv, groups, d, entries;
  int column_tiles;  // tiles of query columns of a token and kv head
  float scale_log2;  // scale * log2(e)
};

// Keys that a token of row `row` sees.
__device__ __forceinline__ int sd_visible(const SelectedParams& p, int row, int token) {
  int len = max(p.seq_lens[row], 0);
  if (len > (long long)p.table_width * p.block_size) {
    if (threadIdx.x == 0) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    len = p.table_width * p.block_size;
  }
  return p.positions ? min(len - 1, p.positions[token]) + 1 : len;
}

constexpr float kSdNone = -3e38f;  // a maximum that no score has touched
constexpr int kSdWarps = 4, kSdThreads = 32 * kSdWarps;

// Shared memory: the queries while the tiles are walked, then each warp's sums.  kTiles: mma column tiles of 8.  kPack: at most four columns, the low
// term of the weights in columns 4 - 7.  kTerms: of the queries.
template <int kD, int kTiles, bool kPack, int kTerms>
struct SdShape {
  static constexpr int kCols = kPack ? 4 : 8 * kTiles;  // query columns
  static constexpr int kQCols = 8 * kTiles;             // columns of the operand
  static constexpr int kQPitch = kD + 32;               // elements; the eight columns' pieces of 16 bytes fall into different banks
  static constexpr int kQBytes = kTerms * kQCols * kQPitch * 2;
  static constexpr int kAccPitch = kD + 4;  // floats
  static constexpr int kAccBytes = kSdWarps * kCols * kAccPitch * 4;
  static constexpr int kBytes = kQBytes > kAccBytes ? kQBytes : kAccBytes;
};

template <typename C>
__device__ __forceinline__ uint32_t sd_pair(float x, float y) { return cm_pack<C>(x, y, false); }
template <typename C>
__device__ __forceinline__ float2 sd_floats(uint32_t w) {
  if constexpr (std::is_same<C, __half>::value) return q_float2(w);
  else return bf16x2_to_float2(w);
}
// Eight elements of a query in its own type.
__device__ __forceinline__ void sd_query8(const SelectedParams& p, long long at, float (&x)[8]) {
  if (p.q_dtype == NVJ_F32) q_floats(q_load8(static_cast<const float*>(p.q) + at), x);
  else if (p.q_dtype == NVJ_F16) q_floats(q_load8(static_cast<const __half*>(p.q) + at), x);
  else q_floats(q_load8(static_cast<const __nv_bfloat16*>(p.q) + at), x);
}

// The end of a kernel: the sums of the CTA's warps, kCols columns of `dims` numbers each relative to its reference, and those of the cluster's CTAs into one: the output
// of the heads first_head .. of this kv head's group.
template <int kCols, int kAccPitch>
__device__ __forceinline__ void sd_merge(const SelectedParams& p, float* all, const float2 (&sd_ml)[kSdWarps][kCols], float2 (&sd_ML)[kCols], int token, int head,
                                         int first_head, int dims, int ctas, int rank) {
  const int quads = dims >> 2;
  auto place = [&](int col, int d) {
    return p.out + (((long long)token * p.hkv + head) * p.groups + first_head + col) * dims + d;
  };
  const int used = min(kCols, p.groups - first_head);
  for (int i = threadIdx.x; i < used * quads; i += kSdThreads) {
    const int col = i / quads, d = i % quads * 4;
    float top = kSdNone, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kSdWarps; ++w) top = fmaxf(top, sd_ml[w][col].x);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSdWarps; ++w) {
      const float2 ml = sd_ml[w][col];
      const float f = ex2_approx(ml.x - top);
      sum = fmaf(ml.y, f, sum);
      const float4 x = *reinterpret_cast<const float4*>(all + (w * kCols + col) * kAccPitch + d);
      y.x = fmaf(x.x, f, y.x);
      y.y = fmaf(x.y, f, y.y);
      y.z = fmaf(x.z, f, y.z);
      y.w = fmaf(x.w, f, y.w);
    }
    if (ctas == 1) {
      const float inverse = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<float4*>(place(col, d)) = make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
    } else {
      *reinterpret_cast<float4*>(all + col * kAccPitch + d) = y;  // (read above by this thread alone)
      if (d == 0) sd_ML[col] = make_float2(top, sum);
    }
  }
  if (ctas == 1) return;
  cl_sync();
  bool odd = false;
  const int pieces = used * quads, per = (pieces + ctas - 1) / ctas;
  for (int i = threadIdx.x; i < per; i += kSdThreads) {
    const int piece = rank * per + i;
    if (piece >= pieces) break;
    const int col = piece / quads, d = piece % quads * 4;
    float top = kSdNone, sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int first = 0; first < ctas; first += 4) {  // four CTAs' shares in flight
      float2 e[4];
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int from = first + k < ctas ? first + k : first;
        e[k] = cl_ld2(cl_map(&sd_ML[col], from));
        x[k] = cl_ld4(cl_map(all + col * kAccPitch + d, from));
        if (first + k >= ctas) e[k] = make_float2(kSdNone, 0.f), x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float now = top;
#pragma unroll
      for (int k = 0; k < 4; ++k) now = fmaxf(now, e[k].x);
      const float f = ex2_approx(top - now);
      sum *= f;
      y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
      top = now;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float w = ex2_approx(e[k].x - top);
        sum = fmaf(e[k].y, w, sum);
        y.x = fmaf(x[k].x, w, y.x);
        y.y = fmaf(x[k].y, w, y.y);
        y.z = fmaf(x[k].z, w, y.z);
        y.w = fmaf(x[k].w, w, y.w);
      }
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    y = make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
    odd |= cl_not_finite(y) || !(sum - sum == 0.f);
    *reinterpret_cast<float4*>(place(col, d)) = y;
  }
  cl_sync_read(odd);  // no CTA goes while another reads its sums
}

// kRagged: a head_dim below kD, its missing dims zero.
template <typename C, int kD, int kTiles, bool kPack, int kTerms, bool kRagged>
__global__ void __launch_bounds__(kSdThreads) selected_decode_kernel(SelectedParams p, int ctas) {
  using S = SdShape<kD, kTiles, kPack, kTerms>;
  constexpr bool kF16 = std::is_same<C, __half>::value;
  constexpr int kCols = S::kCols, kParts = kD / 32;  // K: parts of 32 dims, 16 bytes per lane and key row
  constexpr int kVParts = kD / 64;                   // V: parts of 64 dims
  constexpr int kAhead = kD == 64 ? 2 : 1;           // tiles that a warp has under way
  constexpr int kMTiles = kD / 16;
  constexpr int kWTerms = kF16 ? 2 : 3;              // of the weights
  // The reference of the sums moves when a score passes it by more than kLift + 2^8.  f16 weights: they end at 65504 above and lose bits below 2^-14, so that the
  // reference is set 2^7 below the largest score.
  constexpr float kLift = kF16 ? 7.f : 0.f, kSlack = 8.f;
  extern __shared__ __align__(16) char sd_smem[];
  __shared__ __align__(8) float sd_factor[S::kQCols];  // what the products of a column are to be multiplied by
  __shared__ float2 sd_ml[kSdWarps][kCols];     // a warp's reference and sum
  __shared__ float2 sd_ML[kCols];               // the CTA's
  C* qs = reinterpret_cast<C*>(sd_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = ctas > 1 ? (int)cl_rank() : 0;
  const int token = blockIdx.x / ctas, row = token / p.width;
  const int head = blockIdx.y / p.column_tiles, ct = blockIdx.y % p.column_tiles;
  const int hq = p.hkv * p.groups, dims = kRagged ? p.d : kD;
  pdl_wait();
  pdl_release();
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  const int32_t* list = p.selected + ((long long)token * p.hkv + head) * p.entries;
  const int per_block = p.block_size >> 4, tiles = p.entries * per_block, step = ctas * kSdWarps;
  // the next 32 tiles of this warp, one per lane: block id (-1: not there), position of the tile's first key, its place in the block
  int chunk = rank * kSdWarps + warp, id = -1, base = 0, off = 0;
  unsigned there = 0;
  auto entry_of = [&](int first) {
    const long long at = first + (long long)lane * step;
    return at < tiles ? list[(int)at / per_block] : -1;
  };
  int c = entry_of(chunk);
  const int visible = sd_visible(p, row, token);
  auto look = [&]() {
    off = ((int)(chunk + (long long)lane * step) % per_block) * 16;
    id = -1;
    if (c >= 0 && c < p.table_width && (long long)c * p.block_size + off < visible) {
      id = table[c];
      if (id < 0 || id >= p.num_blocks) {
        atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
        id = -1;
      }
    }
    base = id >= 0 ? c * p.block_size + off : 0;
    there = __ballot_sync(kFullMask, id >= 0);
  };
  look();
  const long long key_stride = (long long)p.hkv * dims;
  uint4 k_held[kAhead][kParts][2];   // keys g and g + 8: dims 32 part + 8 t ..
  uint4 v_held[kAhead][kVParts][4];  // keys 2t, 2t + 1, 2t + 8, 2t + 9: dims 64 part + 8 g ..
  int left[kAhead];                  // keys of the tile that are to be seen; 0: no tile
  const C* next_v[kAhead];
  // the next tile's K rows on their way; its V rows' place
  auto ask_k = [&](int u) {
    left[u] = 0;
    while (there == 0) {
      chunk += 32 * step;
      if (chunk >= tiles) return;
      c = entry_of(chunk);
      look();
    }
    const int slot = __ffs(there) - 1;
    there &= there - 1;
    const long long key = (long long)__shfl_sync(kFullMask, id, slot) * p.block_size + __shfl_sync(kFullMask, off, slot);
    left[u] = visible - __shfl_sync(kFullMask, base, slot);
    const long long at = (key * p.hkv + head) * dims;
    const C* kp = static_cast<const C*>(p.k_cache) + at + g * key_stride + 8 * t;
    next_v[u] = static_cast<const C*>(p.v_cache) + at;
#pragma unroll
    for (int s = 0; s < kParts; ++s) {
      if (!kRagged || 32 * s + 8 * t < dims) {
        k_held[u][s][0] = ld_stream_u4(kp + 32 * s);
        k_held[u][s][1] = ld_stream_u4(kp + 8 * key_stride + 32 * s);
      } else {
        k_held[u][s][0] = k_held[u][s][1] = make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto ask_v = [&](int u) {
    if (left[u] <= 0) return;
    const C* vp = next_v[u] + 2 * t * key_stride + 8 * g;
    if (!kRagged && left[u] >= 16) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int h = 0; h < kVParts; ++h) v_held[u][h][k] = ld_stream_u4(vp + ((k & 1) + 8 * (k >> 1)) * key_stride + 64 * h);
      return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // keys behind the last one hold anything: they must not reach a product
      const int key = (k & 1) + 8 * (k >> 1);
#pragma unroll
      for (int h = 0; h < kVParts; ++h) {
        v_held[u][h][k] = make_uint4(0, 0, 0, 0);
        if (2 * t + key < left[u] && (!kRagged || 64 * h + 8 * g < dims)) v_held[u][h][k] = ld_stream_u4(vp + key * key_stride + 64 * h);
      }
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    ask_k(u);
    ask_v(u);
  }

  // queries into shared memory: a warp a column at a time, lane l the dims 8 l ..  (f16 terms of another type: after a power of two that brings the
  // largest magnitude next to 2^14)
  for (int col = warp; col < S::kQCols; col += kSdWarps) {
    const int at = ct * kCols + (kPack ? (col & 3) : col);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (at < p.groups && lane < dims / 8) sd_query8(p, ((long long)token * hq + head * p.groups + at) * dims + 8 * lane, x);
    float factor = p.scale_log2;
    if constexpr (kF16 && kTerms > 1) {
      const int bits = __reduce_max_sync(kFullMask, __float_as_int(q_largest(0.f, x)));
      int e = (bits >> 23) - 127 - 14;
      e = bits == 0 ? 0 : (e < -126 ? -126 : e);
      const float down = q_pow2(-e > 126 ? 126 : -e);
      factor *= q_pow2(e);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= down;
    }
    if (lane == 0) sd_factor[col] = factor;
    if (lane < kD / 8) {
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kTerms > 1 && !kF16) w[i] = __byte_perm(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), 0x7632);  // (cut: three times 8 bits)
          else w[i] = sd_pair<C>(x[2 * i], x[2 * i + 1]);
          const float2 f = sd_floats<C>(w[i]);
          x[2 * i] -= f.x;
          x[2 * i + 1] -= f.y;
        }
        *reinterpret_cast<uint4*>(qs + (term * S::kQCols + col) * S::kQPitch + 8 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  __syncthreads();

  // this lane's columns 2t, 2t + 1 of each column tile
  float m[kTiles][2], l[kTiles][2], acc[kTiles][kMTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[j][i] = kSdNone;
      l[j][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kMTiles; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[j][i][k] = 0.f;
  }

  auto work_on = [&](int u) {
    // S^T = K Q^T: rows keys, columns queries; two sums, so that a product does not wait for the one before
    float s[kTiles][4], s2[kTiles][4];
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[j][k] = s2[j][k] = 0.f;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const uint4 lo = k_held[u][part][0], hi = k_held[u][part][1];
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
          const uint4 b = *reinterpret_cast<const uint4*>(qs + ((term * kTiles + j) * 8 + g) * S::kQPitch + 32 * part + 8 * t);
          cm_mma<C>(s[j], {lo.x, hi.x, lo.y, hi.y}, b.x, b.y);
          cm_mma<C>(s2[j], {lo.z, hi.z, lo.w, hi.w}, b.z, b.w);
        }
    }
    const int seen = left[u];
    ask_k(u);  // the K rows of the tile that is to take these registers

    // scores in log2 units; whether one passes its reference by more than the slack
    bool over = false;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const float2 factor = *reinterpret_cast<const float2*>(&sd_factor[8 * j + 2 * t]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = k & 1;
        s[j][k] = g + 8 * (k >> 1) < seen ? (s[j][k] + s2[j][k]) * (i ? factor.y : factor.x) : -INFINITY;
        over |= s[j][k] > m[j][i] + (kSlack + kLift);
      }
    }
    if (__any_sync(kFullMask, over)) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(s[j][i], s[j][i + 2]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
          const float now = fmaxf(m[j][i], top - kLift), f = ex2_approx(m[j][i] - now);
          m[j][i] = now;
          l[j][i] *= f;
#pragma unroll
          for (int a = 0; a < kMTiles; ++a) {
            acc[j][a][i] *= f;
            acc[j][a][i + 2] *= f;
          }
        }
    }
    // weights: their sum, and P^T as terms
    uint32_t part[kTiles][2][3];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] = ex2_approx(s[j][k] - m[j][k & 1]);
        l[j][k & 1] += w[k];
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t term[kWTerms];
#pragma unroll
        for (int i = 0; i < kWTerms; ++i) {
          term[i] = sd_pair<C>(w[2 * r], w[2 * r + 1]);
          const float2 f = sd_floats<C>(term[i]);
          w[2 * r] -= f.x;
          w[2 * r + 1] -= f.y;
        }
        if constexpr (kPack) {
          part[j][r][0] = cm_transpose(t < 2 ? term[0] : term[1]);
          if constexpr (kWTerms > 2) part[j][r][1] = cm_transpose(t < 2 ? term[2] : 0u);
        } else {
#pragma unroll
          for (int i = 0; i < kWTerms; ++i) part[j][r][i] = cm_transpose(term[i]);
        }
      }
    }
    // O^T += V^T P^T: rows dims 64 part + 8 g + 2 w and + 1
#pragma unroll
    for (int h = 0; h < kVParts; ++h) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        auto word = [&](int k) { return w == 0 ? v_held[u][h][k].x : w == 1 ? v_held[u][h][k].y : w == 2 ? v_held[u][h][k].z : v_held[u][h][k].w; };
        const uint32_t a[4] = {__byte_perm(word(0), word(1), 0x5410), __byte_perm(word(0), word(1), 0x7632),
                               __byte_perm(word(2), word(3), 0x5410), __byte_perm(word(2), word(3), 0x7632)};
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};  // of this tile alone: the tensor cores cut the last place of what they add to a longer sum
#pragma unroll
          for (int i = 0; i < (kPack ? kWTerms - 1 : kWTerms); ++i) cm_mma<C>(sum, a, part[j][0][i], part[j][1][i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][h * 4 + w][i] += sum[i];
        }
      }
    }
    ask_v(u);
  };
  bool more = true;
  while (more) {
    more = false;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (left[u] > 0) {
        work_on(u);
        more = true;
      }
  }

  // the warps' sums into shared memory (the queries are no longer needed)
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[j][i] += __shfl_xor_sync(kFullMask, l[j][i], o);
    }
  __syncthreads();
  float* sums = reinterpret_cast<float*>(sd_smem) + warp * kCols * S::kAccPitch;
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    const int col = 8 * j + 2 * t;
#pragma unroll
    for (int a = 0; a < kMTiles; ++a) {
      if constexpr (kPack) {  // the low terms' share of a column is two lanes away
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[j][a][k] += __shfl_xor_sync(kFullMask, acc[j][a][k], 2);
      }
      const int d = (a / 4) * 64 + 8 * g + 2 * (a % 4);
      if (!kPack || t < 2) {
        *reinterpret_cast<float2*>(sums + col * S::kAccPitch + d) = make_float2(acc[j][a][0], acc[j][a][2]);
        *reinterpret_cast<float2*>(sums + (col + 1) * S::kAccPitch + d) = make_float2(acc[j][a][1], acc[j][a][3]);
      }
    }
    if (g == 0 && (!kPack || t < 2)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) sd_ml[warp][col + i] = make_float2(m[j][i], l[j][i]);
    }
  }
  __syncthreads();
  sd_merge<kCols, S::kAccPitch>(p, reinterpret_cast<float*>(sd_smem), sd_ml, sd_ML, token, head, ct * kCols, dims, ctas, rank);
}

// CTAs per cluster: as many as are resident at once, two to an SM less what clusters leave unused, up to 8 (16, which are placed one by one, for up to four lists), and no
// more than one per four tiles.  Lists are of one length, so that more CTAs than that gain nothing at the end and cost their start.  64 16-key tiles of 256 dims:
// 2 lists 16 CTAs 7.5 us, 8 8.8; 16 lists 8 11.6, 16 17.6; 64 lists 4 19.3, 6 29.4; 128 lists 2 29.2, 1 36.1; 512 lists 1 92, 2 108.
static int selected_decode_ctas(long long units, long long tiles, int sms) {
  long long c = 7LL * sms / (4 * units);
  if (c < 1 && 2 * units < 5LL * sms) c = 2;  // (a round and a bit: halves; 320 lists of 64: one CTA 84, two 78; 384 of 96 tiles of 128 dims: 52, 58)
  const long long useful = (tiles + kSdWarps - 1) / kSdWarps, most = units > 4 ? 8 : 16;
  c = c < useful ? c : useful;
  return (int)(c < 1 ? 1 : (c > most ? most : c));
}

// A launch of `kernel`, whose CTAs take `columns` heads of a group and `keys` keys of a list at a time.
inline int launch_selected_clusters(void (*kernel)(SelectedParams, int), PerDeviceFlags& ready, SelectedParams p, int columns, int keys, int smem,
                                    cudaStream_t stream) {
  if (!once_per_device(ready, [&](int) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
               cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
      }))
    return NVJ_ERR_LAUNCH;
  p.column_tiles = (p.groups + columns - 1) / columns;
  const long long tokens = (long long)p.rows * p.width, per_block = (p.block_size + keys - 1) / keys;
  if ((long long)p.hkv * p.column_tiles > 65535) return NVJ_ERR_TOO_LARGE;
  const int ctas = selected_decode_ctas(tokens * p.hkv * p.column_tiles, p.entries * per_block, 148);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * tokens), p.hkv * p.column_tiles, 1);
  cfg.blockDim = dim3(kSdThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
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

template <typename C, int kD, int kTiles, bool kPack, int kTerms, bool kRagged = false>
static int launch_selected(const SelectedParams& p, cudaStream_t stream) {
  using S = SdShape<kD, kTiles, kPack, kTerms>;
  static PerDeviceFlags ready;
  return launch_selected_clusters(selected_decode_kernel<C, kD, kTiles, kPack, kTerms, kRagged>, ready, p, S::kCols, 16, S::kBytes, stream);
}

template <typename C, int kD>
static int launch_selected_columns(const SelectedParams& p, bool same, cudaStream_t stream) {
  if (p.d != kD) return launch_selected<C, kD, 1, false, 3, true>(p, stream);
  // (16 columns of 256 dims do not fit a thread's registers: two clusters read the blocks, the second mostly from the L2)
  if constexpr (kD < 256)
    if (p.groups > 8) return same ? launch_selected<C, kD, 2, false, 1>(p, stream) : launch_selected<C, kD, 2, false, 3>(p, stream);
  if (!same) return launch_selected<C, kD, 1, false, 3>(p, stream);
  if (p.groups <= 4) return launch_selected<C, kD, 1, true, 1>(p, stream);
  return launch_selected<C, kD, 1, false, 1>(p, stream);
}
// A cache of type C and blocks of whole 16-key tiles; `same`: the queries are of the cache's type.
template <typename C>
static int launch_selected_dims(const SelectedParams& p, bool same, cudaStream_t stream) {
  if (p.d > 128) return launch_selected_columns<C, 256>(p, same, stream);
  if (p.d > 64) return launch_selected_columns<C, 128>(p, same, stream);
  return launch_selected_columns<C, 64>(p, same, stream);
}
// selected_decode_bf16.cu, selected_decode_f16.cu
int launch_selected_bf16(const SelectedParams& p, cudaStream_t stream);
int launch_selected_f16(const SelectedParams& p, cudaStream_t stream);

}  // namespace nvj
