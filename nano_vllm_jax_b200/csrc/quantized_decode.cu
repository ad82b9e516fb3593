// Paged attention over the 8-bit cache (quantized_kv.cuh) for rows of few query tokens: decode and verification of speculated tokens.
//
//   out[t, h] = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale * q[t, h] . k_p),  p < len and p <= position[t]
//
// Bound by the bytes of K and V: 2 * kv_heads * head_dim per key, half of the bf16 cache's.  At the same byte rate an SM meets twice
// as many numbers per second as over bf16, so what a number costs in instructions decides:
//   * one thread-block cluster per (row, kv head, tile of query columns), a warp per 16-key tile, tiles dealt to the
//     cluster's warps in turn: no scan of the lengths, no workspace, no counter; warps merge through shared memory, CTAs through
//     distributed shared memory;
//   * K and V go from global memory to registers in 16-byte pieces and nowhere else: both products are taken transposed
//     (S^T = K Q^T, O^T = V^T P^T), and since the order of a contraction is free, the 16 bytes that a lane holds of a
//     row ARE its operands, permuted the same way on the other side.  No shared memory, no ldmatrix on the way;
//   * e4m3 becomes f16 exactly, two numbers per instruction; V takes one byte permute per two numbers besides, which pairs its keys;
//   * f16 queries times a power of two per column (exact for bf16 and f16; f32 queries go as a high and a low term), weights as
//     a high and a low f16 term: products as good as in f32.  With up to four columns the two terms of the weights are the
//     two halves of the eight columns of one mma.sync, with more they are two of them;
//   * the K scale of a block multiplies its scores, the V scale goes into the exponent of the weights: a running maximum of
//     its own for the weighted sum keeps blocks of any scale apart from the sum of the weights.
// Maxima are lazy: one vote per tile says whether a score has left them behind, and only then the sums are rescaled.
// Measured: four rows of 64 - 512 keys, 8 heads of 256 over 2, 6.9 - 7.5 us, which is launch, trips and merge; 126 rows of 4850 - 9700 keys, 4 heads of 64, 157
// us (46% of the copy rate), 16 over 2 94 us (38%): instructions.

#include "cluster.cuh"
#include "decode_parts.cuh"
#include "quantized_kv.cuh"
#include "quantized_umma_params.cuh"
#include "umma.cuh"

namespace nvj {

struct QDecodeParams {
  const void* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  const int32_t* positions;        // nullable: [rows, width], packed: per token
  const int32_t* query_start_loc;  // packed: the rows of one query token, one of `tokens`, are served, the others left alone
  float* out;
  int32_t* status;
  long long num_blocks;
  int rows, width, tokens, table_width, block_size, num_kv_heads, groups;
  int column_tiles;  // tiles of query columns of a row and kv head
  float scale_log2;  // scale * log2(e)
};

constexpr int kQdWarps = 4, kQdThreads = 32 * kQdWarps;
constexpr float kQdNone = -3e38f;  // a maximum that no score has touched
// The reference of the sum of weights moves when a score passes it by 2^8; that of the weighted sum is set 2^7 below the largest weight and moves
// when one would pass 2^15: f16 ends at 65504 above and at 2^-24 below, and a key 2^10 below the largest still has 22 bits in two terms.
constexpr float kQdSlack = 8.f, kQdLift = 7.f;

// Shared memory: the queries as f16 while the tiles are walked, then each warp's sums.
// kTiles: mma column tiles of 8.  kPack: at most four columns, the low term of the weights in columns 4 - 7.  kF32: f32 queries.
template <int kD, int kTiles, bool kPack, bool kF32>
struct QdShape {
  static constexpr int kCols = kPack ? 4 : 8 * kTiles;  // query columns
  static constexpr int kQCols = 8 * kTiles;             // columns of the operand
  static constexpr int kQPitch = kD + 8;                // f16 elements; two columns' pieces fall into different banks
  static constexpr int kQTerms = kF32 && !kPack ? 2 : 1;
  static constexpr int kQBytes = kQTerms * kQCols * kQPitch * 2;
  static constexpr int kAccPitch = kD + 4;  // floats
  static constexpr int kAccBytes = kQdWarps * kCols * kAccPitch * 4;
  static constexpr int kBytes = kQBytes > kAccBytes ? kQBytes : kAccBytes;
};

// CTAs that an SM is to hold at least.  head_dim 64: a warp has half or a quarter of the bytes of the other forms under way, so more warps have to be
// there (126 rows of 4850 - 9700 keys, 4 heads of 64: 180 us with as few as there were, 160 with five; six, at 80 registers, 152
// and small calls 7% slower; 64 rows of 4 tokens, 16 heads over 2, 43 -> 34 with four).
constexpr int qd_resident(int dim, int tiles, bool pack) { return dim == 64 ? (tiles > 1 ? 4 : pack ? 5 : 1) : pack && dim == 256 ? 3 : 1; }
template <typename T, int kD, int kTiles, bool kPack>
__global__ void __launch_bounds__(kQdThreads, qd_resident(kD, kTiles, kPack)) quantized_decode_kernel(QDecodeParams p, int ctas) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  using S = QdShape<kD, kTiles, kPack, kF32>;
  constexpr int kCols = S::kCols, kParts = kD / 64;  // parts of 64 dims: one 16-byte piece per lane and key row
  // Tiles that a warp has under way; one of 64 dims is 2 KiB (with one of them 126 rows of 4850 - 9700 keys, 4 heads, 160 us instead of 154, 16 heads
  // over 2 104 instead of 94).
  constexpr int kAhead = kD == 64 && kTiles == 1 ? 2 : 1;
  constexpr int kVHalves = kD >= 128 ? kD / 128 : 1;  // parts of 128 dims of V (64: 8-byte pieces)
  constexpr int kVWords = kD >= 128 ? 4 : 2;          // words of a V piece
  constexpr int kMTiles = kD / 16;
  extern __shared__ __align__(16) char qd_smem[];
  __shared__ float qd_factor[S::kQCols];                  // what the products of a column are to be multiplied by
  __shared__ float2 qd_ml[kQdWarps][kCols];               // a warp's maximum and sum
  __shared__ float qd_mv[kQdWarps][kCols];                // ... and the reference of its weighted sums
  __shared__ float2 qd_ML[kCols];                         // the CTA's
  __half* qs = reinterpret_cast<__half*>(qd_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = ctas > 1 ? (int)cl_rank() : 0;
  const int row = blockIdx.x / ctas;
  const int head = blockIdx.y / p.column_tiles, ct = blockIdx.y % p.column_tiles;
  const int hq = p.num_kv_heads * p.groups;
  pdl_wait();
  pdl_release();

  // the row's first query token and how many it has; a packed batch's rows of several tokens are not ours
  int token = row * p.width, width = p.width, live = 1;
  if (p.query_start_loc) {
    token = p.query_start_loc[row];
    width = 1;
    live = p.query_start_loc[row + 1] - token == 1 && token >= 0 && token < p.tokens;
  }
  const int columns = width * p.groups;  // of the row and kv head: column c = (token c / groups, head c % groups)
  int len = p.seq_lens[row];
  const int step = ctas * kQdWarps;
  int tile = rank * kQdWarps + warp;  // this warp's tiles: tile, tile + step, ..
  const int per_block = p.block_size >> 4;
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  // ids of this warp's next 32 tiles, one per lane (a table entry exists whatever the length is)
  auto fetch_id = [&](int first) {
    const int b = (first + lane * step) / per_block;
    return b < p.table_width ? table[b] : -1;
  };
  int id = fetch_id(tile);
  // (the 32 tiles behind them, if registers run two tiles ahead: one outside the pool is flagged with its scales)
  int next_ids = -1;
  auto fetch_next_ids = [&](int first) {
    if constexpr (kAhead > 1) {
      next_ids = fetch_id(first + 32 * step);
      if (next_ids >= p.num_blocks) next_ids = -1;
    }
  };
  fetch_next_ids(tile);
  int last = 0x7fffffff;  // position of the last key that a token of the row sees
  if (p.positions && live) {
    last = lane < width ? p.positions[token + lane] : -1;
    for (int i = lane + 32; i < width; i += 32) last = max(last, p.positions[token + i]);
    last = __reduce_max_sync(kFullMask, last);
  }
  if (!live) len = 0;
  if (len > p.table_width * (long long)p.block_size) {
    if (threadIdx.x == 0 && rank == 0) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    len = p.table_width * p.block_size;
  }
  len = min(len - 1, last) + 1;  // (keys that none of them sees may hold anything, as those behind the row's last one)
  const int tiles = (len + 15) >> 4;
  float ks = 0.f, lv = 0.f;  // scales of this lane's tile: of K, and log2 of V's
  auto fetch_scales = [&](int first) {
    const bool used = first + lane * step < tiles;
    if (used && (id < 0 || id >= p.num_blocks)) {
      atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      id = -1;
    }
    if (used && id >= 0) {
      ks = p.k_scale[(long long)id * p.num_kv_heads + head];
      lv = p.v_scale[(long long)id * p.num_kv_heads + head];
    }
  };
  const long long key_stride = (long long)p.num_kv_heads * kD;
  uint4 k_held[kAhead][kParts][2];    // keys g and g + 8: dims 64 part + 16 t ..
  uint4 v_held[kAhead][kVHalves][4];  // keys 2t, 2t + 1, 2t + 8, 2t + 9: dims 128 half + 16 g .. (64 dims: 8 g ..)
  auto load_k = [&](uint4 (&kr)[kParts][2], int tile_id, int which) {
    if (tile_id < 0) {
#pragma unroll
      for (int s = 0; s < kParts; ++s) kr[s][0] = kr[s][1] = make_uint4(0, 0, 0, 0);
      return;
    }
    const uint8_t* at = p.k_cache + (((long long)tile_id * p.block_size + (which % per_block) * 16 + g) * p.num_kv_heads + head) * kD + 16 * t;
#pragma unroll
    for (int s = 0; s < kParts; ++s) {
      kr[s][0] = ld_stream_u4(at + 64 * s);
      kr[s][1] = ld_stream_u4(at + 8 * key_stride + 64 * s);
    }
  };
  auto load_v = [&](uint4 (&vr)[kVHalves][4], int tile_id, int which) {
    const int first = which * 16 + 2 * t;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = (k & 1) + 8 * (k >> 1);  // behind 2t
      // keys behind the row's last one hold anything: they must not reach a product
      const bool ok = tile_id >= 0 && first + key < len;
      const uint8_t* at = p.v_cache + (((long long)tile_id * p.block_size + (which % per_block) * 16 + 2 * t + key) * p.num_kv_heads + head) * kD;
#pragma unroll
      for (int h = 0; h < kVHalves; ++h) {
        vr[h][k] = make_uint4(0, 0, 0, 0);
        if (ok) {
          if constexpr (kD >= 128) {
            vr[h][k] = ld_stream_u4(at + 128 * h + 16 * g);
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(at + 8 * g);
            vr[h][k].x = w.x;
            vr[h][k].y = w.y;
          }
        }
      }
    }
  };

  int slot = 0;  // lane that holds the current tile's id and scales
  if (tile < tiles) {
    fetch_scales(tile);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int first_id = __shfl_sync(kFullMask, id, u);
      if (tile + u * step < tiles) {
        load_k(k_held[u], first_id, tile + u * step);
        load_v(v_held[u], first_id, tile + u * step);
      }
    }
  }

  // queries into shared memory: a warp a column at a time, lane l the dims 8 l .. (f16 after a power of two that brings the largest
  // magnitude next to 2^14, so that numbers down to 2^-28 of it keep 11 bits)
  for (int c = warp; c < S::kQCols; c += kQdWarps) {
    const int col = kPack ? (c & 3) : c;
    const int at = ct * kCols + col;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (live && at < columns && lane < kD / 8)
      q_floats(q_load8(static_cast<const T*>(p.q) + ((long long)(token + at / p.groups) * hq + head * p.groups + at % p.groups) * kD + 8 * lane), x);
    float largest = 0.f;
    largest = q_largest(largest, x);
    const int bits = __reduce_max_sync(kFullMask, __float_as_int(largest));
    int e = (bits >> 23) - 127 - 14;  // largest = 2^(e + 14) * [1, 2)
    e = bits == 0 ? 0 : (e < -126 ? -126 : e);
    const float down = q_pow2(-e > 126 ? 126 : -e);
    if (lane == 0) qd_factor[c] = q_pow2(e) * p.scale_log2;
    if (lane < kD / 8) {
      uint32_t w[4], low[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = x[2 * i] * down, b = x[2 * i + 1] * down;
        w[i] = q_pair(a, b);
        low[i] = q_pair_rest(a, b, w[i]);
      }
      const bool second = kF32 && kPack && c >= 4;  // packed f32 queries: columns 4 - 7 hold the low terms
      uint4* at4 = reinterpret_cast<uint4*>(qs + c * S::kQPitch + 8 * lane);
      *at4 = second ? make_uint4(low[0], low[1], low[2], low[3]) : make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (S::kQTerms == 2)
        *reinterpret_cast<uint4*>(qs + (S::kQCols + c) * S::kQPitch + 8 * lane) = make_uint4(low[0], low[1], low[2], low[3]);
    }
  }
  __syncthreads();

  // this lane's columns 2t, 2t + 1 of each column tile
  float factor[kTiles][2], m[kTiles][2], mv[kTiles][2], l[kTiles][2];
  int limit[kTiles][2];
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = 8 * j + 2 * t + i, at = ct * kCols + (kPack ? (c & 3) : c);
      factor[j][i] = qd_factor[c];
      m[j][i] = mv[j][i] = kQdNone;
      l[j][i] = 0.f;
      limit[j][i] = len;
      if (p.positions && at < columns && live) {  // (a row that is not ours may begin behind the last token)
        const int last = p.positions[token + at / p.groups];
        limit[j][i] = last < len ? last + 1 : len;
      }
    }
  float acc[kTiles][kMTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < kMTiles; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[j][i][k] = 0.f;

  auto work_on = [&](uint4 (&kr)[kParts][2], uint4 (&vr)[kVHalves][4]) {
    const float k_unit = __shfl_sync(kFullMask, ks, slot), v_log = __log2f(__shfl_sync(kFullMask, lv, slot));
    const bool usable = __shfl_sync(kFullMask, id, slot) >= 0;
    // S^T = K Q^T: rows keys, columns queries
    float s[kTiles][4];
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[j][k] = 0.f;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const uint32_t lo[4] = {kr[part][0].x, kr[part][0].y, kr[part][0].z, kr[part][0].w};
      const uint32_t hi[4] = {kr[part][1].x, kr[part][1].y, kr[part][1].z, kr[part][1].w};
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int term = 0; term < S::kQTerms; ++term) {
          const uint4* b4 = reinterpret_cast<const uint4*>(qs + ((term * kTiles + j) * 8 + g) * S::kQPitch + 64 * part + 16 * t);
          const uint4 b0 = b4[0], b1 = b4[1];
          const uint32_t b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            q_mma(s[j], q_half2(lo[k]), q_half2(hi[k]), q_half2_high(lo[k]), q_half2_high(hi[k]), b[2 * k], b[2 * k + 1]);
        }
    }
    // the K rows of the tile that is to take these registers
    const int this_tile = tile;
    tile += step;
    const int next = tile + (kAhead - 1) * step;
    if (++slot == 32) {
      slot = 0;
      if (tile < tiles) {
        id = kAhead > 1 ? next_ids : fetch_id(tile);
        fetch_scales(tile);
        fetch_next_ids(tile);
      }
    }
    int next_id = __shfl_sync(kFullMask, id, (slot + kAhead - 1) & 31);
    if constexpr (kAhead > 1) {
      const int behind = __shfl_sync(kFullMask, next_ids, (slot + kAhead - 1) & 31);
      if (slot + kAhead - 1 >= 32) next_id = behind;
    }
    if (next < tiles) load_k(kr, next_id, next);

    // scores in log2 units; whether one passes its maximum by more than the slack
    bool over = false;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (kF32 && kPack) s[j][k] += __shfl_xor_sync(kFullMask, s[j][k], 2);  // the low terms' columns are two lanes away
        const int i = k & 1, key = this_tile * 16 + g + 8 * (k >> 1);
        s[j][k] = key < limit[j][i] && usable ? s[j][k] * (factor[j][i] * k_unit) : -INFINITY;
        over |= s[j][k] > m[j][i] + kQdSlack || s[j][k] + v_log > mv[j][i] + (kQdSlack + kQdLift);
      }
    if (__any_sync(kFullMask, over)) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(s[j][i], s[j][i + 2]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
          const float now = fmaxf(m[j][i], top), now_v = fmaxf(mv[j][i], top + v_log - kQdLift);
          l[j][i] *= ex2_approx(m[j][i] - now);
          const float f = ex2_approx(mv[j][i] - now_v);
          m[j][i] = now;
          mv[j][i] = now_v;
#pragma unroll
          for (int a = 0; a < kMTiles; ++a) {
            acc[j][a][i] *= f;
            acc[j][a][i + 2] *= f;
          }
        }
    }
    // weights: their sum, and P^T as high and low f16 terms
    uint32_t high[kTiles][2], low[kTiles][2];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = k & 1;
        l[j][i] += ex2_approx(s[j][k] - m[j][i]);
        w[k] = ex2_approx(s[j][k] + v_log - mv[j][i]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t h = q_pair(w[2 * r], w[2 * r + 1]);
        const uint32_t rest = q_pair_rest(w[2 * r], w[2 * r + 1], h);
        if constexpr (kPack) {
          high[j][r] = q_transpose(t < 2 ? h : rest);
        } else {
          high[j][r] = q_transpose(h);
          low[j][r] = q_transpose(rest);
        }
      }
    }
    // O^T += V^T P^T: rows dims 16 g + 2 i and 16 g + 2 i + 1 of a part of 128 (64: 8 g + ..)
#pragma unroll
    for (int h = 0; h < kVHalves; ++h) {
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        auto word = [&](int k) { return w == 0 ? vr[h][k].x : w == 1 ? vr[h][k].y : w == 2 ? vr[h][k].z : vr[h][k].w; };
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // bytes 2b, 2b + 1 of the word
          const uint32_t near = __byte_perm(word(0), word(1), b ? 0x7362 : 0x5140);  // keys 2t, 2t + 1
          const uint32_t far = __byte_perm(word(2), word(3), b ? 0x7362 : 0x5140);   // keys 2t + 8, 2t + 9
          const uint32_t a0 = q_half2(near), a1 = q_half2_high(near), a2 = q_half2(far), a3 = q_half2_high(far);
          const int at = (h * kVWords + w) * 2 + b;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            q_mma(acc[j][at], a0, a1, a2, a3, high[j][0], high[j][1]);
            if constexpr (!kPack) q_mma(acc[j][at], a0, a1, a2, a3, low[j][0], low[j][1]);
          }
        }
      }
    }
    if (next < tiles) load_v(vr, next_id, next);
  };
  while (tile < tiles) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (tile < tiles) work_on(k_held[u], v_held[u]);
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
  float* sums = reinterpret_cast<float*>(qd_smem) + warp * kCols * S::kAccPitch;
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    const int c = 8 * j + 2 * t;
#pragma unroll
    for (int a = 0; a < kMTiles; ++a) {
      if constexpr (kPack) {  // the low terms' share of a column is two lanes away
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[j][a][k] += __shfl_xor_sync(kFullMask, acc[j][a][k], 2);
      }
      const int d = kD >= 128 ? (a / 8) * 128 + 16 * g + 2 * (a % 8) : 8 * g + 2 * a;
      if (!kPack || t < 2) {
        *reinterpret_cast<float2*>(sums + c * S::kAccPitch + d) = make_float2(acc[j][a][0], acc[j][a][2]);
        *reinterpret_cast<float2*>(sums + (c + 1) * S::kAccPitch + d) = make_float2(acc[j][a][1], acc[j][a][3]);
      }
    }
    if (g == 0 && (!kPack || t < 2)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qd_ml[warp][c + i] = make_float2(m[j][i], l[j][i]);
        qd_mv[warp][c + i] = mv[j][i];
      }
    }
  }
  __syncthreads();
  // ... and into one, in the first warp's place: relative to the largest maximum of the scores
  float* all = reinterpret_cast<float*>(qd_smem);
  for (int i = threadIdx.x; i < kCols * (kD / 4); i += kQdThreads) {
    const int c = i / (kD / 4), d = i % (kD / 4) * 4;
    float top = kQdNone, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kQdWarps; ++w) top = fmaxf(top, qd_ml[w][c].x);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kQdWarps; ++w) {
      const float2 ml = qd_ml[w][c];
      sum = fmaf(ml.y, ex2_approx(ml.x - top), sum);
      const float f = ml.y == 0.f ? 0.f : ex2_approx(qd_mv[w][c] - top);
      const float4 x = *reinterpret_cast<const float4*>(all + (w * kCols + c) * S::kAccPitch + d);
      y.x = fmaf(x.x, f, y.x);
      y.y = fmaf(x.y, f, y.y);
      y.z = fmaf(x.z, f, y.z);
      y.w = fmaf(x.w, f, y.w);
    }
    *reinterpret_cast<float4*>(all + c * S::kAccPitch + d) = y;  // (read above by this thread alone)
    if (d == 0) qd_ML[c] = make_float2(top, sum);
  }
  auto place = [&](int c, int d) {  // of column c's dims d .. d + 3 in the output
    const int at = ct * kCols + c;
    return p.out + ((long long)(token + at / p.groups) * hq + head * p.groups + at % p.groups) * kD + d;
  };
  const int used = live ? min(kCols, columns - ct * kCols) : 0;
  if (ctas == 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < used * (kD / 4); i += kQdThreads) {
      const int c = i / (kD / 4), d = i % (kD / 4) * 4;
      const float sum = qd_ML[c].y, inverse = sum == 0.f ? 0.f : 1.f / sum;
      const float4 y = *reinterpret_cast<const float4*>(all + c * S::kAccPitch + d);
      *reinterpret_cast<float4*>(place(c, d)) = make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
    }
    return;
  }
  cl_sync();
  bool odd = false;
  const int pieces = used * (kD / 4), per = (pieces + ctas - 1) / ctas;
  for (int i = threadIdx.x; i < per; i += kQdThreads) {
    const int piece = rank * per + i;
    if (piece >= pieces) break;
    const int c = piece / (kD / 4), d = piece % (kD / 4) * 4;
    float top = kQdNone, sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int first = 0; first < ctas; first += 4) {  // four CTAs' shares in flight
      float2 e[4];
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int from = first + k < ctas ? first + k : first;
        e[k] = cl_ld2(cl_map(&qd_ML[c], from));
        x[k] = cl_ld4(cl_map(all + c * S::kAccPitch + d, from));
        if (first + k >= ctas) e[k] = make_float2(kQdNone, 0.f), x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
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
        const float f = ex2_approx(e[k].x - top);
        sum = fmaf(e[k].y, f, sum);
        y.x = fmaf(x[k].x, f, y.x);
        y.y = fmaf(x[k].y, f, y.y);
        y.z = fmaf(x[k].z, f, y.z);
        y.w = fmaf(x[k].w, f, y.w);
      }
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    y = make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
    odd |= cl_not_finite(y) || !(sum - sum == 0.f);
    *reinterpret_cast<float4*>(place(c, d)) = y;
  }
  cl_sync_read(odd);  // no CTA goes while another reads its sums
}

// CTAs per cluster: as many as give every SM its three resident CTAs, up to 16, and no more than one per four tiles of the widest
// row; at least four in batches of long rows, so that the last CTAs to finish are short ones.
static int quantized_decode_ctas(long long units, long long tiles, int sms) {
  long long c = (3LL * sms + units / 2) / units;
  if (c < 4 && tiles > 128) c = 4;
  const long long useful = (tiles + kQdWarps - 1) / kQdWarps;
  c = c < useful ? c : useful;
  return (int)(c < 1 ? 1 : (c > 16 ? 16 : c));
}

template <typename T, int kD, int kTiles, bool kPack>
static int launch_quantized_decode(QDecodeParams p, cudaStream_t stream) {
  using S = QdShape<kD, kTiles, kPack, std::is_same<T, float>::value>;
  auto* kernel = quantized_decode_kernel<T, kD, kTiles, kPack>;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) == cudaSuccess &&
               cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
      }))
    return NVJ_ERR_LAUNCH;
  p.column_tiles = (p.width * p.groups + S::kCols - 1) / S::kCols;
  const long long units = (long long)p.rows * p.num_kv_heads * p.column_tiles;
  const int ctas = quantized_decode_ctas(units, (long long)p.table_width * p.block_size / 16, 148);
  if ((long long)ctas * p.rows > 0x7fffffffLL || (long long)p.num_kv_heads * p.column_tiles > 65535) return NVJ_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas * (unsigned)p.rows, p.num_kv_heads * p.column_tiles, 1);
  cfg.blockDim = dim3(kQdThreads, 1, 1);
  cfg.dynamicSmemBytes = S::kBytes;
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

template <typename T, int kD>
static int launch_quantized_decode_columns(const QDecodeParams& p, cudaStream_t stream) {
  const long long columns = (long long)p.width * p.groups;
  if (columns <= 4) return launch_quantized_decode<T, kD, 1, true>(p, stream);
  if (columns <= 8) return launch_quantized_decode<T, kD, 1, false>(p, stream);
  return launch_quantized_decode<T, kD, 2, false>(p, stream);
}
template <typename T>
static int launch_quantized_decode_dims(const QDecodeParams& p, int head_dim, cudaStream_t stream) {
  if (head_dim == 256) return launch_quantized_decode_columns<T, 256>(p, stream);
  if (head_dim == 128) return launch_quantized_decode_columns<T, 128>(p, stream);
  return launch_quantized_decode_columns<T, 64>(p, stream);
}

// ---- the tcgen05 form (quantized_umma.cuh): its tensor maps, workspace, launch and fold ------------------------------------------
typedef CUresult (*QuEncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                    const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static QuEncodeTiledFn qu_encode_fn() {
  static QuEncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<QuEncodeTiledFn>(ptr);
  }();
  return fn;
}
// A layer [token, kv head, head_dim] of bytes seen as {128 dims, token of a group of 8, 128-dim chunk, group, kv head}: a box is 16, 32 or 64 keys
// of one kv head and lands as [group][chunk][8 keys][128 B] with the 128-byte swizzle.  (An SM takes in ~20 B per cycle through boxes of
// 2 KiB, 16 keys of head_dim 128, and needs 23.)  `extent` = (tokens << 14) | log2(keys / 16) << 12 | kv heads << 1 | head_dim 256.
static bool qu_make_map(CUtensorMap* map, const void* base, uint64_t extent) {
  const cuuint32_t unit = 16u << ((extent >> 12) & 3);
  const cuuint64_t tokens = extent >> 14, heads = (extent >> 1) & 0x7ff, dim = extent & 1 ? 256 : 128;
  const cuuint64_t dims[5] = {128, 8, dim / 128, tokens / 8, heads};
  const cuuint64_t strides[4] = {heads * dim, 128, 8 * heads * dim, dim};
  const cuuint32_t box[5] = {128, 8, (cuuint32_t)(dim / 128), unit / 8, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return qu_encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
constexpr int kQuMapKind = 6;  // (tensor_map_cached)

// How a call is cut: column tiles, ranges, and where its partials lie in the workspace.
struct QuPlan {
  int column_tiles, tile_columns, hcts, ranges;
  size_t acc_bytes, ml_bytes, cut_bytes;
  size_t bytes() const { return acc_bytes + ml_bytes + cut_bytes; }
};
static QuPlan qu_plan(int columns, int num_kv_heads, int head_dim, int sms) {
  QuPlan w{};
  w.column_tiles = (columns + 23) / 24;
  const int each = (columns + w.column_tiles - 1) / w.column_tiles;
  w.tile_columns = each <= 4 ? 4 : each <= 8 ? 8 : each <= 16 ? 16 : 24;
  w.hcts = num_kv_heads * w.column_tiles;
  w.ranges = sms / w.hcts > 1 ? sms / w.hcts : 1;
  const size_t slots = w.ranges > 1 ? (size_t)2 * w.ranges * w.hcts * w.tile_columns : 0;
  w.acc_bytes = ws_round(slots * head_dim * sizeof(float));
  w.ml_bytes = ws_round(slots * 2 * sizeof(float));
  w.cut_bytes = ws_round((size_t)w.ranges * sizeof(UmmaCut));
  return w;
}

// The first boundary that cuts a row folds the row's columns from the ranges' partials.  Grid: boundary, kv head and column tile, 256 pieces of
// (column, 4 dims); a thread a piece.  Behind boundary c lies a row that begins in range c and goes on in c + 1, if any does: those two
// parts are asked for together with what was cut.  (A CTA for all columns, that asked first and loaded then: 11 us behind rows of five tokens.)
__global__ void __launch_bounds__(256) quantized_umma_fold_kernel(QuParams a, int head_dim) {
  const int hct = blockIdx.y, head = hct / a.column_tiles, ct = hct % a.column_tiles, pieces = head_dim / 4;
  const int item = blockIdx.z * 256 + threadIdx.x, c = item / pieces, d = item % pieces * 4, at = ct * a.tile_columns + c;
  const int out_row = at / a.groups * a.num_q_heads + head * a.groups + at % a.groups;
  const bool mine = c < min(a.columns - ct * a.tile_columns, a.tile_columns);
  const int first = blockIdx.x;
  pdl_wait();
  pdl_release();
  if (!mine) return;
  auto slot_of = [&](int part) { return ((long long)partial_slot(part, part == first) * a.hcts + hct) * a.tile_columns + c; };
  auto load = [&](int part, float2& e, float4& x) {
    e = __ldcg(reinterpret_cast<const float2*>(a.part_ml + slot_of(part) * 2));
    x = __ldcg(reinterpret_cast<const float4*>(a.part_acc + slot_of(part) * head_dim + d));
  };
  float2 e[8];
  float4 x[8];
  load(first, e[0], x[0]);
  load(first + 1, e[1], x[1]);
  const int4 cut = __ldcg(reinterpret_cast<const int4*>(a.cuts + first + 1));  // row, its first and last range
  if (cut.x < 0) return;
  float top = -3e38f, sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int from = first;;) {
    const int n = from == first ? 2 : min(cut.z + 1 - from, 8);
    float now = top;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) now = fmaxf(now, e[k].x);
    const float f = ex2_approx(top - now);
    sum *= f;
    y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
    top = now;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) {
        const float w = ex2_approx(e[k].x - top);
        sum = fmaf(e[k].y, w, sum);
        y.x = fmaf(x[k].x, w, y.x);
        y.y = fmaf(x[k].y, w, y.y);
        y.z = fmaf(x[k].z, w, y.z);
        y.w = fmaf(x[k].w, w, y.w);
      }
    from += n;
    if (from > cut.z) break;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (from + k <= cut.z) load(from + k, e[k], x[k]);
  }
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
  const long long token = a.query_start_loc ? (long long)a.query_start_loc[cut.x] : (long long)cut.x * a.width;
  *reinterpret_cast<float4*>(a.out + (token * a.num_q_heads + out_row) * head_dim + d) =
      make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
}

// What a row's end costs a CTA, in keys (decode_parts.cuh), up to eight columns and beyond.  256 rows of 1024 - 4096 keys 107.4 us with 64, 107.2 with
// 128, 106.5 with 192, 106.8 with 256, 107.1 with 384; 48 rows of 8 heads 39.2, 38.5, 38.4, 38.1, 38.5; 64 rows of 5 tokens 58.4, 56.7, 55.8, 55.2, 53.6.
constexpr int kQuRowEndCost = 256, kQuWideRowEndCost = 384;

static int run_quantized_umma(const QDecodeParams& q, int q_dtype, int head_dim, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const int sms = decode_wide_num_ctas();
  if (sms <= 0) return NVJ_ERR_LAUNCH;
  if (head_dim < 128 || !qu_encode_fn()) return NVJ_ERR_UNSUPPORTED;
  if (q.num_blocks < 1 || q.num_blocks * (q.block_size / 8) >= 0x7fffffffLL) return NVJ_ERR_UNSUPPORTED;
  const int columns = q.width * q.groups;
  const QuPlan w = qu_plan(columns, q.num_kv_heads, head_dim, sms);
  if (!workspace || !aligned16(workspace) || workspace_bytes < w.bytes()) return NVJ_ERR_WORKSPACE;
  CUtensorMap k_map, v_map;
  const int unit_log2 = q.block_size % 64 == 0 ? 6 : q.block_size % 32 == 0 ? 5 : 4;
  const uint64_t extent = (uint64_t)q.num_blocks * q.block_size << 14 | (uint64_t)(unit_log2 - 4) << 12 | (uint64_t)q.num_kv_heads << 1 | (head_dim == 256 ? 1u : 0u);
  if (!tensor_map_cached(&k_map, kQuMapKind, q.k_cache, extent, qu_make_map) || !tensor_map_cached(&v_map, kQuMapKind, q.v_cache, extent, qu_make_map))
    return NVJ_ERR_UNSUPPORTED;
  char* at = static_cast<char*>(workspace);
  QuParams a{};
  a.q = q.q;
  a.k_scale = q.k_scale;
  a.v_scale = q.v_scale;
  a.positions = q.positions;
  a.query_start_loc = q.query_start_loc;
  a.out = q.out;
  a.part_acc = reinterpret_cast<float*>(at);
  a.part_ml = reinterpret_cast<float*>(at + w.acc_bytes);
  a.cuts = reinterpret_cast<UmmaCut*>(at + w.acc_bytes + w.ml_bytes);
  a.width = q.width;
  a.columns = columns;
  a.groups = q.groups;
  a.num_q_heads = q.groups * q.num_kv_heads;
  a.num_kv_heads = q.num_kv_heads;
  a.unit = 1 << unit_log2;
  a.unit_log2 = unit_log2;
  a.column_tiles = w.column_tiles;
  a.tile_columns = w.tile_columns;
  a.hcts = w.hcts;
  a.scale_log2 = q.scale_log2;
  DecodeParams p{};
  p.block_tables = q.block_tables;
  p.seq_lens = q.seq_lens;
  p.query_start_loc = q.query_start_loc;
  p.query_positions = q.positions;
  p.packed_rows = q.query_start_loc ? q.tokens : 0;
  p.status = q.status;
  p.num_blocks = q.num_blocks;
  p.batch = q.rows;
  p.table_width = q.table_width;
  p.block_size = q.block_size;
  p.row_end_cost = (w.tile_columns <= 8 ? kQuRowEndCost : kQuWideRowEndCost) >> unit_log2;
  const auto launch = q_dtype == NVJ_BF16 ? launch_quantized_umma_bf16 : q_dtype == NVJ_F16 ? launch_quantized_umma_f16 : launch_quantized_umma_f32;
  const int rc = launch(k_map, v_map, a, p, head_dim, w.ranges, stream);
  if (rc != NVJ_OK || w.ranges < 2) return rc;
  return launch_after(quantized_umma_fold_kernel, dim3(w.ranges - 1, w.hcts, (w.tile_columns * head_dim / 4 + 255) / 256), dim3(256), 0, stream, a, head_dim) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
}

// Whether a call goes to the tcgen05 form: by the room of its tables, since the lengths are on the GPU.  That form starts and folds 5 us later, and
// takes 3 - 8 us for a row and head even if they have few keys, but 0.4 - 1.2 us per 128 keys behind them where this file's takes up to 2.8 (head_dim
// 256).  Over 272 batches of 1 - 512 rows, 64 - 65536 keys, 4 - 80 columns and four head layouts (drawn once, their times are not kept) the rule cost
// 1.5% against the better of both, 30% at most (always this file's form: 23%, always the other: 19%).  Either side of it, us: 64 rows of 64 - 128 keys, 2 heads of 256 and 4
// columns 10.2 against 14.9, 64 of 1024 - 2048 keys 45 against 27; one row of 4096 keys 11.7 against 15.1, one of 32768 45.9 against 22.6.
static bool quantized_umma_pays(int rows, int width, int table_width, int block_size, int num_kv_heads, int head_dim, int groups) {
  const long long room = (long long)table_width * block_size, columns = ((long long)width * groups + 3) / 4;
  return head_dim >= 128 && room >= 320 && (double)rows * room * num_kv_heads * head_dim * columns >= 6 * 1048576.;
}

}  // namespace nvj

extern "C" size_t nvj_paged_decode_quantized_workspace_bytes(int rows, int width, int table_width, int block_size, int num_kv_heads,
                                                              int head_dim, int num_q_heads, int form) {
  using namespace nvj;
  if (rows <= 0 || width <= 0 || table_width <= 0 || !quantized_cache_shape_ok(block_size, num_kv_heads, head_dim) || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads != 0 || head_dim < 128 || form < 0 || form == 1)
    return 0;
  const int groups = num_q_heads / num_kv_heads, sms = decode_wide_num_ctas();
  if (sms <= 0 || (long long)width * groups > 0xffff) return 0;
  if (form == 0 && !quantized_umma_pays(rows, width, table_width, block_size, num_kv_heads, head_dim, groups)) return 0;
  return qu_plan(width * groups, num_kv_heads, head_dim, sms).bytes();
}

namespace nvj {
// `tokens`: how many a packed batch's q, positions and out hold; rows whose token lies elsewhere are not served.
int paged_decode_quantized(const void* q, int q_dtype, const void* k_cache_layer, const void* v_cache_layer, const float* k_scale, const float* v_scale,
                           int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int num_q_heads, const int32_t* block_tables,
                           int table_width, const int32_t* seq_lens, const int32_t* positions, const int32_t* query_start_loc, int rows, int width,
                           int tokens, float scale, float* out, int32_t* status, void* workspace, size_t workspace_bytes, int form,
                           nvj_stream_t stream) {
  if (form < 0 || form > 2) return NVJ_ERR_INVALID_ARGUMENT;
  if (rows < 0 || width < 0 || table_width < 0 || num_blocks < 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (q_dtype < NVJ_BF16 || q_dtype > NVJ_F32 || !quantized_cache_shape_ok(block_size, num_kv_heads, head_dim)) return NVJ_ERR_UNSUPPORTED;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (rows == 0 || width == 0) return NVJ_OK;
  if (query_start_loc && (width != 1 || !positions)) return NVJ_ERR_INVALID_ARGUMENT;
  if (!q || !k_cache_layer || !v_cache_layer || !k_scale || !v_scale || !seq_lens || !out || !status) return NVJ_ERR_INVALID_ARGUMENT;
  if (table_width > 0 && !block_tables) return NVJ_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache_layer) || !aligned16(v_cache_layer)) return NVJ_ERR_INVALID_ARGUMENT;
  if ((long long)table_width * block_size > 0x7fffffffLL - 65536) return NVJ_ERR_TOO_LARGE;
  if ((long long)width * (num_q_heads / num_kv_heads) > 0xffff || (long long)rows * width > 0x7fffffffLL) return NVJ_ERR_TOO_LARGE;
  QDecodeParams p{};
  p.q = q;
  p.k_cache = static_cast<const uint8_t*>(k_cache_layer);
  p.v_cache = static_cast<const uint8_t*>(v_cache_layer);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.positions = positions;
  p.query_start_loc = query_start_loc;
  p.out = out;
  p.status = status;
  p.num_blocks = num_blocks;
  p.rows = rows;
  p.width = width;
  p.tokens = tokens;
  p.table_width = table_width;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.groups = num_q_heads / num_kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (form == 2 || (form == 0 && workspace && quantized_umma_pays(rows, width, table_width, block_size, num_kv_heads, head_dim, p.groups))) {
    const int rc = run_quantized_umma(p, q_dtype, head_dim, workspace, workspace_bytes, s);
    if (form == 2 || (rc != NVJ_ERR_UNSUPPORTED && rc != NVJ_ERR_WORKSPACE)) return rc;
  }
  if (q_dtype == NVJ_BF16) return launch_quantized_decode_dims<__nv_bfloat16>(p, head_dim, s);
  if (q_dtype == NVJ_F16) return launch_quantized_decode_dims<__half>(p, head_dim, s);
  return launch_quantized_decode_dims<float>(p, head_dim, s);
}
}  // namespace nvj

extern "C" int nvj_paged_decode_quantized(const void* q, int q_dtype, const void* k_cache_layer, const void* v_cache_layer,
                                          const float* k_scale, const float* v_scale, int64_t num_blocks, int block_size,
                                          int num_kv_heads, int head_dim, int num_q_heads, const int32_t* block_tables, int table_width,
                                          const int32_t* seq_lens, const int32_t* positions, const int32_t* query_start_loc, int rows,
                                          int width, float scale, float* out, int32_t* status, void* workspace,
                                          size_t workspace_bytes, int form, nvj_stream_t stream) {
  return nvj::paged_decode_quantized(q, q_dtype, k_cache_layer, v_cache_layer, k_scale, v_scale, num_blocks, block_size, num_kv_heads, head_dim,
                                     num_q_heads, block_tables, table_width, seq_lens, positions, query_start_loc, rows, width, 0x7fffffff, scale, out,
                                     status, workspace, workspace_bytes, form, stream);
}
