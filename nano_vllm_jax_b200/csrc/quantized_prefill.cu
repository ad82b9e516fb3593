// Ragged packed prefill attention over the 8-bit paged cache (quantized_kv.cuh).  Two routes:
//
//   * the model's shape with bf16 queries: the rows' blocks are written out once as bf16 (exact: a scale is a power of two) into
//     pages of a scratch cache, and the tcgen05 tiles of the bf16 cache run over it (paged_prefill_umma2.cu).  Writing
//     out moves 5 bytes per number, once per call; the products take 4 * query heads * head_dim flops per key and
//     query token, so that a prompt's pages are ~1% of its time;
//   * every other head layout, block size and query type: quantized_prefill_kernel below, flash attention on mma.sync tiles with the
//     numbers converted to f16 on their way into shared memory.
// Rows of a single query token go to the decode kernel, which reads the 8-bit blocks and spreads a row over SMs.

#include "quantized_kv.cuh"

namespace nvj {

int prefill_over_pages(const void* q, const void* k_pages, const void* v_pages, long long pages, const int32_t* page_tables, int table_width,
                       const int32_t* kv_lens, const int32_t* positions, const int32_t* query_start_loc, int rows, int token_bucket, float scale,
                       float* out, int32_t* status, void* workspace, size_t workspace_bytes, int part, int tile_pairs, cudaStream_t stream);

// ---- pages of a scratch bf16 cache ----------------------------------------------------------------------------------------------
struct QUnpackParams {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* kv_lens;
  const int32_t* query_start_loc;
  char* k_pages;  // page row * table_width + b: block b of the row
  char* v_pages;
  int32_t* page_tables;
  int32_t* status;
  long long num_blocks;
  int rows, table_width, skip_single;
};

// Grid (x: blocks of a row in strides, y: rows); the model's shape, 16 tokens of 2 heads of 256: a thread four pieces of 16 numbers, two of K and two
// of V, of one head.  The block's id is asked for together with the row's length: two trips to memory in a row.  A block whose id is outside
// the pool becomes a page of zeros, as the other kernels take it, and so do the rows behind the last key, which hold anything.
__global__ void __launch_bounds__(256) quantized_unpack_kernel(QUnpackParams p) {
  constexpr int kRow = 512, kBlock = 16 * kRow;  // bytes of a token, and of a block
  pdl_wait();
  pdl_release();
  const int row = blockIdx.y;
  const int len = p.kv_lens[row], from = p.query_start_loc[row], to = p.query_start_loc[row + 1];
  const bool skip = to <= from || (p.skip_single && to - from == 1);
  const int head = (threadIdx.x * 16 % kRow) / 256, token = threadIdx.x * 16 / kRow;  // of the first piece; the second is eight tokens on
  for (int b = blockIdx.x; b < p.table_width; b += gridDim.x) {
    const long long page = (long long)row * p.table_width + b;
    const int id = p.block_tables[page];
    if (threadIdx.x == 0) p.page_tables[page] = (int)page;
    const int left = len - b * 16;  // tokens of the row from this block on
    if (skip || left <= 0) continue;
    const bool ok = id >= 0 && id < p.num_blocks;
    if (!ok && threadIdx.x == 0) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
    uint4 w[4];
    float unit[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (ok && token + 8 * (i & 1) < left)
        w[i] = ld_stream_u4((i < 2 ? p.k_cache : p.v_cache) + (long long)id * kBlock + (i & 1) * (kBlock / 2) + threadIdx.x * 16);
    }
    if (ok) {
      unit[0] = p.k_scale[(long long)id * 2 + head];
      unit[1] = p.v_scale[(long long)id * 2 + head];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t in[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      const float u = unit[i >> 1];
      uint32_t out[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = q_float2(q_half2(in[k])), y = q_float2(q_half2_high(in[k]));
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * u, x.y * u), hi = __floats2bfloat162_rn(y.x * u, y.y * u);
        out[2 * k] = *reinterpret_cast<const uint32_t*>(&lo);
        out[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&hi);
      }
      uint4* at = reinterpret_cast<uint4*>((i < 2 ? p.k_pages : p.v_pages) + 2 * (page * kBlock + (i & 1) * (kBlock / 2) + threadIdx.x * 16));
      at[0] = make_uint4(out[0], out[1], out[2], out[3]);
      at[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
}

// ---- mma.sync tiles ---------------------------------------------------------------------------------------------------------------
struct QPrefillParams {
  const void* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* kv_lens;
  const int32_t* positions;
  const int32_t* query_start_loc;
  float* out;
  int32_t* status;
  long long num_blocks;
  int rows, table_width, block_size, num_kv_heads, groups, token_bucket, skip_single;
  float scale_log2;
};

// CTA: 128 query rows (token major, a kv head's `groups` heads minor) of one table row and kv head, 16 per warp; keys in tiles.
// The numbers of a tile are fetched into registers while the tile in front is worked on, and become f16 in shared memory: every
// warp reads them by ldmatrix.  Scores, both references of the maxima and both terms of the weights as in the decode kernel.
constexpr int kQpWarps = 8, kQpThreads = 32 * kQpWarps, kQpRows = 16 * kQpWarps;
constexpr float kQpNone = -3e38f, kQpSlack = 8.f, kQpLift = 7.f;  // (the references are the decode kernel's)

template <typename T, int kD>
struct QpShape {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int kKeys = kD == 256 ? 32 : 64;
  static constexpr int kPitch = kD + 8;  // f16 elements: ldmatrix rows fall into different banks
  static constexpr int kQTerms = kF32 ? 2 : 1;
  static constexpr int kQBytes = kQTerms * kQpRows * kPitch * 2;
  static constexpr int kTileBytes = kKeys * kPitch * 2;
  static constexpr int kBytes = kQBytes + 2 * kTileBytes;
  static constexpr int kPieces = kKeys * kD / 16 / kQpThreads;  // 16-byte pieces of K (and of V) that a thread fetches
};

__device__ __forceinline__ void qp_ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void qp_ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T, int kD>
__global__ void __launch_bounds__(kQpThreads, 1) quantized_prefill_kernel(QPrefillParams p) {
  using S = QpShape<T, kD>;
  constexpr int kKeys = S::kKeys, kPitch = S::kPitch, kNT = kKeys / 8, kSteps = kD / 16, kOT = kD / 8;
  extern __shared__ __align__(16) char qp_smem[];
  __half* qs = reinterpret_cast<__half*>(qp_smem);
  __half* k_tile = reinterpret_cast<__half*>(qp_smem + S::kQBytes);
  __half* v_tile = k_tile + kKeys * kPitch;
  __shared__ float qp_k_unit[2][kKeys], qp_v_log[2][kKeys];
  __shared__ float qp_factor[kQpRows];
  __shared__ int qp_found[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y, hq = p.num_kv_heads * p.groups;
  pdl_wait();
  pdl_release();

  // which table row and tile this CTA has: tiles are counted row by row; the last ones (most keys) go first
  if (tid == 0) qp_found[0] = -1;
  __syncthreads();
  {
    // total first, so that the order can be turned round
    auto tiles_of = [&](int r) {
      const int n = p.query_start_loc[r + 1] - p.query_start_loc[r];
      return n <= 0 || (p.skip_single && n == 1) ? 0 : (n * p.groups + kQpRows - 1) / kQpRows;
    };
    if (warp == 0) {
      int total = 0;
      for (int r = lane; r < p.rows; r += 32) total += tiles_of(r);
      total = __reduce_add_sync(kFullMask, total);
      const int want = total - 1 - (int)blockIdx.x;
      int before = 0;
      for (int r0 = 0; r0 < p.rows && want >= 0; r0 += 32) {
        const int mine = r0 + lane < p.rows ? tiles_of(r0 + lane) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(kFullMask, upto, o);
          if (lane >= o) upto += a;
        }
        const int first = before + upto - mine;
        if (want >= first && want < first + mine) {
          qp_found[0] = r0 + lane;
          qp_found[1] = want - first;
        }
        before += __shfl_sync(kFullMask, upto, 31);
        if (want < before) break;
      }
    }
    // padding behind the last row's tokens
    const int end = p.query_start_loc[p.rows];
    const long long per_token = (long long)p.groups * (kD / 4);
    const long long pad = end < p.token_bucket ? (long long)(p.token_bucket - (end > 0 ? end : 0)) * per_token : 0;
    for (long long i = (long long)blockIdx.x * kQpThreads + tid; i < pad; i += (long long)gridDim.x * kQpThreads) {
      const long long token = (end > 0 ? end : 0) + i / per_token;
      reinterpret_cast<float4*>(p.out + (token * hq + head * p.groups) * kD)[i % per_token] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __syncthreads();
  const int row = qp_found[0];
  if (row < 0) return;
  const int first_row = qp_found[1] * kQpRows;  // of the row's query rows
  const int token0 = p.query_start_loc[row];
  int n = p.query_start_loc[row + 1] - token0;
  if (token0 < 0 || token0 >= p.token_bucket) return;
  n = n < p.token_bucket - token0 ? n : p.token_bucket - token0;
  const int query_rows = n * p.groups;
  int len = p.kv_lens[row];
  if (len > (long long)p.table_width * p.block_size) {
    if (tid == 0) atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    len = p.table_width * p.block_size;
  }
  const int32_t* table = p.block_tables + (long long)row * p.table_width;

  // queries as f16 (a power of two per query row, as in the decode kernel): a warp its own 16 rows
  for (int i = 0; i < 16; ++i) {
    const int r = warp * 16 + i, at = first_row + r;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.f;
    if (at < query_rows && lane < kD / 8)
      q_floats(q_load8(static_cast<const T*>(p.q) + ((long long)(token0 + at / p.groups) * hq + head * p.groups + at % p.groups) * kD + 8 * lane), x);
    const int bits = __reduce_max_sync(kFullMask, __float_as_int(q_largest(0.f, x)));
    int e = (bits >> 23) - 127 - 14;
    e = bits == 0 ? 0 : (e < -126 ? -126 : e);
    const float down = q_pow2(-e);
    if (lane == 0) qp_factor[r] = q_pow2(e) * p.scale_log2;
    if (lane < kD / 8) {
      uint32_t w[4], low[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float a = x[2 * k] * down, b = x[2 * k + 1] * down;
        w[k] = q_pair(a, b);
        low[k] = q_pair_rest(a, b, w[k]);
      }
      *reinterpret_cast<uint4*>(qs + r * kPitch + 8 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (S::kF32) *reinterpret_cast<uint4*>(qs + (kQpRows + r) * kPitch + 8 * lane) = make_uint4(low[0], low[1], low[2], low[3]);
    }
  }
  __syncwarp();
  // this lane's query rows g and g + 8 of the warp's: how many keys they see
  int limit[2], most = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = first_row + warp * 16 + g + 8 * i;
    limit[i] = 0;
    if (at < query_rows) {
      const int last = p.positions[token0 + at / p.groups];
      limit[i] = last < len ? last + 1 : len;
    }
    most = max(most, limit[i]);
  }
  const float factor[2] = {qp_factor[warp * 16 + g], qp_factor[warp * 16 + g + 8]};
  most = __reduce_max_sync(kFullMask, most);
  const int fewest = __reduce_min_sync(kFullMask, min(limit[0], limit[1]));
  if (tid == 0) qp_found[2] = 0;
  __syncthreads();
  if (lane == 0) atomicMax(&qp_found[2], most);
  __syncthreads();
  const int tiles = (max(qp_found[2], 0) + kKeys - 1) / kKeys;

  // a tile's pieces into registers, and from there as f16 into shared memory
  constexpr int kPerKey = kD / 16;
  uint4 kr[S::kPieces], vr[S::kPieces];
  float unit = 0.f, v_unit = 0.f;
  auto fetch = [&](int tile) {
    const int key0 = tile * kKeys;
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int piece = i * kQpThreads + tid, key = key0 + piece / kPerKey, d = piece % kPerKey * 16;
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (key < len) {
        const int id = table[key / p.block_size];
        if (id >= 0 && id < p.num_blocks) {
          const long long at = (((long long)id * p.block_size + key % p.block_size) * p.num_kv_heads + head) * kD + d;
          kr[i] = ld_stream_u4(p.k_cache + at);
          vr[i] = ld_stream_u4(p.v_cache + at);
        }
      }
    }
    if (tid < kKeys) {  // the key's scales; -1 marks a key that is not there
      const int key = key0 + tid;
      unit = 0.f;
      v_unit = -1.f;
      if (key < len) {
        const int id = table[key / p.block_size];
        if (id >= 0 && id < p.num_blocks) {
          unit = p.k_scale[(long long)id * p.num_kv_heads + head];
          v_unit = p.v_scale[(long long)id * p.num_kv_heads + head];
        } else {
          atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
        }
      }
    }
  };
  auto expand = [&](const uint4& w, __half* to) {
    uint4* at = reinterpret_cast<uint4*>(to);
    at[0] = make_uint4(q_half2(w.x), q_half2_high(w.x), q_half2(w.y), q_half2_high(w.y));
    at[1] = make_uint4(q_half2(w.z), q_half2_high(w.z), q_half2(w.w), q_half2_high(w.w));
  };

  float m[2] = {kQpNone, kQpNone}, mv[2] = {kQpNone, kQpNone}, l[2] = {0.f, 0.f};
  float acc[kOT][4];
#pragma unroll
  for (int i = 0; i < kOT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = 0.f;
  const uint32_t q_at = smem_u32(qs + (warp * 16 + (lane & 15)) * kPitch + (lane >> 4) * 8);
  const uint32_t k_at = smem_u32(k_tile + ((lane & 7) + (lane >> 4) * 8) * kPitch + ((lane >> 3) & 1) * 8);
  const uint32_t v_at = smem_u32(v_tile + ((lane & 7) + ((lane >> 3) & 1) * 8) * kPitch + (lane >> 4) * 8);
  if (tiles > 0) fetch(0);
  for (int tile = 0; tile < tiles; ++tile) {
    const int buf = tile & 1;
    __syncthreads();  // the tile in front has been read
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int piece = i * kQpThreads + tid, key = piece / kPerKey, d = piece % kPerKey * 16;
      expand(kr[i], k_tile + key * kPitch + d);
      expand(vr[i], v_tile + key * kPitch + d);
    }
    if (tid < kKeys) {
      qp_k_unit[buf][tid] = unit;
      qp_v_log[buf][tid] = v_unit < 0.f ? -INFINITY : __log2f(v_unit);
    }
    if (tile + 1 < tiles) fetch(tile + 1);
    __syncthreads();
    const int key0 = tile * kKeys;
    if (key0 >= most) continue;  // none of the warp's rows sees the tile
    float s[kNT][4];
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[j][k] = 0.f;
#pragma unroll
    for (int d = 0; d < kSteps; ++d) {
      uint32_t a[4], low[4];
      qp_ldsm4(q_at + d * 32, a);
      if constexpr (S::kF32) qp_ldsm4(q_at + kQpRows * kPitch * 2 + d * 32, low);
#pragma unroll
      for (int j = 0; j < kNT; j += 2) {
        uint32_t b[4];
        qp_ldsm4(k_at + j * 8 * kPitch * 2 + d * 32, b);
        q_mma(s[j], a[0], a[1], a[2], a[3], b[0], b[1]);
        q_mma(s[j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
        if constexpr (S::kF32) {
          q_mma(s[j], low[0], low[1], low[2], low[3], b[0], b[1]);
          q_mma(s[j + 1], low[0], low[1], low[2], low[3], b[2], b[3]);
        }
      }
    }
    const bool masked = key0 + kKeys > fewest;
    float top[2] = {kQpNone, kQpNone}, top_v[2] = {kQpNone, kQpNone};
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      const float2 ku = *reinterpret_cast<const float2*>(&qp_k_unit[buf][8 * j + 2 * t]);
      const float2 vl = *reinterpret_cast<const float2*>(&qp_v_log[buf][8 * j + 2 * t]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = k >> 1, key = key0 + 8 * j + 2 * t + (k & 1);
        float x = s[j][k] * (factor[i] * (k & 1 ? ku.y : ku.x));
        const float v = k & 1 ? vl.y : vl.x;
        if ((masked && key >= limit[i]) || v == -INFINITY) x = -INFINITY;  // hidden, or of no block
        s[j][k] = x;
        top[i] = fmaxf(top[i], x);
        top_v[i] = fmaxf(top_v[i], x + v);
      }
    }
    const bool over = top[0] > m[0] + kQpSlack || top[1] > m[1] + kQpSlack || top_v[0] > mv[0] + (kQpSlack + kQpLift) ||
                      top_v[1] > mv[1] + (kQpSlack + kQpLift);
    if (__any_sync(kFullMask, over)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          top[i] = fmaxf(top[i], __shfl_xor_sync(kFullMask, top[i], o));
          top_v[i] = fmaxf(top_v[i], __shfl_xor_sync(kFullMask, top_v[i], o));
        }
        const float now = fmaxf(m[i], top[i]), now_v = fmaxf(mv[i], top_v[i] - kQpLift);
        l[i] *= ex2_approx(m[i] - now);
        const float f = ex2_approx(mv[i] - now_v);
        m[i] = now;
        mv[i] = now_v;
#pragma unroll
        for (int a = 0; a < kOT; ++a) {
          acc[a][2 * i] *= f;
          acc[a][2 * i + 1] *= f;
        }
      }
    }
    uint32_t high[kNT / 2][4], low[kNT / 2][4];  // the weights' pairs are the operand of the second product
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      const float2 vl = *reinterpret_cast<const float2*>(&qp_v_log[buf][8 * j + 2 * t]);
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = k >> 1;
        l[i] += ex2_approx(s[j][k] - m[i]);
        w[k] = ex2_approx(s[j][k] + (k & 1 ? vl.y : vl.x) - mv[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t& h = high[j / 2][2 * (j & 1) + i];
        h = q_pair(w[2 * i], w[2 * i + 1]);
        low[j / 2][2 * (j & 1) + i] = q_pair_rest(w[2 * i], w[2 * i + 1], h);
      }
    }
    // A tile's weighted sum is taken from zero and added in f32: the tensor cores cut the last place of what they add to, and 1000 steps on one sum
    // cost 3e-5 of it (8000 keys).
#pragma unroll
    for (int d = 0; d < kOT; d += 2) {
      float part[2][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) part[0][k] = part[1][k] = 0.f;
#pragma unroll
      for (int j = 0; j < kNT / 2; ++j) {
        uint32_t b[4];
        qp_ldsm4_t(v_at + (j * 16 * kPitch + d * 8) * 2, b);
        q_mma(part[0], low[j][0], low[j][1], low[j][2], low[j][3], b[0], b[1]);
        q_mma(part[1], low[j][0], low[j][1], low[j][2], low[j][3], b[2], b[3]);
        q_mma(part[0], high[j][0], high[j][1], high[j][2], high[j][3], b[0], b[1]);
        q_mma(part[1], high[j][0], high[j][1], high[j][2], high[j][3], b[2], b[3]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        acc[d][k] += part[0][k];
        acc[d + 1][k] += part[1][k];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) l[i] += __shfl_xor_sync(kFullMask, l[i], o);
    const int at = first_row + warp * 16 + g + 8 * i;
    if (at < query_rows) {
      const float f = l[i] == 0.f ? 0.f : ex2_approx(mv[i] - m[i]) / l[i];
      float* to = p.out + ((long long)(token0 + at / p.groups) * hq + head * p.groups + at % p.groups) * kD + 2 * t;
#pragma unroll
      for (int d = 0; d < kOT; ++d) *reinterpret_cast<float2*>(to + 8 * d) = make_float2(acc[d][2 * i] * f, acc[d][2 * i + 1] * f);
    }
  }
}

template <typename T, int kD>
static int launch_quantized_prefill(const QPrefillParams& p, cudaStream_t stream) {
  using S = QpShape<T, kD>;
  auto* kernel = quantized_prefill_kernel<T, kD>;
  static PerDeviceFlags ready;
  if (!once_per_device(ready, [&](int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) == cudaSuccess; }))
    return NVJ_ERR_LAUNCH;
  // as many CTAs per kv head as the bucket's tokens can make tiles: full ones, and one that is not per row
  const long long most = (long long)p.token_bucket * p.groups / kQpRows + (p.rows < p.token_bucket ? p.rows : p.token_bucket) + 1;
  return launch_after(kernel, dim3((unsigned)most, p.num_kv_heads), dim3(kQpThreads), S::kBytes, stream, p) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
}
template <typename T>
static int launch_quantized_prefill_dims(const QPrefillParams& p, int head_dim, cudaStream_t stream) {
  if (head_dim == 256) return launch_quantized_prefill<T, 256>(p, stream);
  if (head_dim == 128) return launch_quantized_prefill<T, 128>(p, stream);
  return launch_quantized_prefill<T, 64>(p, stream);
}

// Whether a call's rows are written out as bf16 pages for the tcgen05 tiles.
static bool quantized_unpacks(int q_dtype, int block_size, int num_kv_heads, int head_dim, int num_q_heads, float scale) {
  return q_dtype == NVJ_BF16 && block_size == 16 && num_kv_heads == 2 && head_dim == 256 && num_q_heads == 8 && scale > 0.f;
}
// Pages of at most 1 GiB; a batch with more table room than that goes to the mma.sync tiles.
constexpr long long kQMostPages = 32768;  // (rows among them: the grid's y)

}  // namespace nvj

namespace nvj {
// Bytes of a batch's pages, 0 where there are none.
static size_t quantized_page_bytes(int q_dtype, int rows, int table_width, int block_size, int num_kv_heads, int head_dim, int num_q_heads, float scale) {
  const long long pages = (long long)rows * table_width;
  if (pages <= 0 || pages > kQMostPages || !quantized_unpacks(q_dtype, block_size, num_kv_heads, head_dim, num_q_heads, scale)) return 0;
  return (size_t)(pages * 2 * block_size * num_kv_heads * head_dim * 2 + (pages * 4 + 255) / 256 * 256);
}
}  // namespace nvj

// The scratch serves the decode kernel's partials and then the pages, one launch behind the other.
extern "C" size_t nvj_paged_prefill_quantized_workspace_bytes(int q_dtype, int rows, int table_width, int block_size, int num_kv_heads,
                                                              int head_dim, int num_q_heads, float scale, int single_rows) {
  using namespace nvj;
  if (rows <= 0 || table_width <= 0) return 0;
  const size_t pages = quantized_page_bytes(q_dtype, rows, table_width, block_size, num_kv_heads, head_dim, num_q_heads, scale);
  const size_t partials =
      single_rows == 0 ? 0 : nvj_paged_decode_quantized_workspace_bytes(rows, 1, table_width, block_size, num_kv_heads, head_dim, num_q_heads, 0);
  return pages > partials ? pages : partials;
}

extern "C" int nvj_paged_prefill_quantized(const void* q, int q_dtype, const void* k_cache_layer, const void* v_cache_layer,
                                           const float* k_scale, const float* v_scale, int64_t num_blocks, int block_size,
                                           int num_kv_heads, int head_dim, int num_q_heads, const int32_t* block_tables, int table_width,
                                           const int32_t* kv_lens, const int32_t* positions, const int32_t* query_start_loc, int rows,
                                           int token_bucket, float scale, float* out, int32_t* status, void* workspace,
                                           size_t workspace_bytes, int single_rows, int tile_pairs, nvj_stream_t stream) {
  using namespace nvj;
  if (rows < 0 || token_bucket < 0 || table_width < 0 || num_blocks < 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (q_dtype < NVJ_BF16 || q_dtype > NVJ_F32 || !quantized_cache_shape_ok(block_size, num_kv_heads, head_dim)) return NVJ_ERR_UNSUPPORTED;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (token_bucket == 0) return NVJ_OK;
  if (!q || !out || !status || !query_start_loc || !positions || !k_cache_layer || !v_cache_layer || !k_scale || !v_scale)
    return NVJ_ERR_INVALID_ARGUMENT;
  if (rows > 0 && (!kv_lens || (table_width > 0 && !block_tables))) return NVJ_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache_layer) || !aligned16(v_cache_layer)) return NVJ_ERR_INVALID_ARGUMENT;
  if ((long long)table_width * block_size > 0x7fffffffLL - 65536 || (long long)token_bucket * num_q_heads > 0x7fffffffLL - 65536)
    return NVJ_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int skip_single = single_rows != 0;
  if (skip_single && rows > 0) {
    const int rc = nvj_paged_decode_quantized(q, q_dtype, k_cache_layer, v_cache_layer, k_scale, v_scale, num_blocks, block_size, num_kv_heads,
                                              head_dim, num_q_heads, block_tables, table_width, kv_lens, positions, query_start_loc, rows, 1,
                                              scale, out, status, workspace, workspace_bytes, 0, stream);
    if (rc != NVJ_OK) return rc;
  }
  const size_t needed = quantized_page_bytes(q_dtype, rows, table_width, block_size, num_kv_heads, head_dim, num_q_heads, scale);
  if (needed > 0 && workspace && workspace_bytes >= needed && aligned16(workspace)) {
    const long long pages = (long long)rows * table_width, page_bytes = 2LL * block_size * num_kv_heads * head_dim;
    QUnpackParams u{};
    u.k_cache = static_cast<const uint8_t*>(k_cache_layer);
    u.v_cache = static_cast<const uint8_t*>(v_cache_layer);
    u.k_scale = k_scale;
    u.v_scale = v_scale;
    u.block_tables = block_tables;
    u.kv_lens = kv_lens;
    u.query_start_loc = query_start_loc;
    u.k_pages = static_cast<char*>(workspace);
    u.v_pages = u.k_pages + pages * page_bytes;
    u.page_tables = reinterpret_cast<int32_t*>(u.v_pages + pages * page_bytes);
    u.status = status;
    u.num_blocks = num_blocks;
    u.rows = rows;
    u.table_width = table_width;
    u.skip_single = skip_single;
    const int across = (148 * 8 + rows - 1) / rows;
    if (launch_after(quantized_unpack_kernel, dim3(across < table_width ? across : table_width, rows), dim3(256), 0, s, u) != cudaSuccess)
      return NVJ_ERR_LAUNCH;
    // (with no rows of one token the key ranges may be split; part 3 asks for that by a workspace, and writes nothing there)
    const int rc = prefill_over_pages(q, u.k_pages, u.v_pages, pages, u.page_tables, table_width, kv_lens, positions, query_start_loc, rows, token_bucket,
                                      scale, out, status, skip_single ? nullptr : workspace, skip_single ? 0 : workspace_bytes, skip_single ? 2 : 3,
                                      tile_pairs, s);
    if (rc != NVJ_ERR_UNSUPPORTED) return rc;  // (without a tensor-map encoder)
  }
  QPrefillParams p{};
  p.q = q;
  p.k_cache = static_cast<const uint8_t*>(k_cache_layer);
  p.v_cache = static_cast<const uint8_t*>(v_cache_layer);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.kv_lens = kv_lens;
  p.positions = positions;
  p.query_start_loc = query_start_loc;
  p.out = out;
  p.status = status;
  p.num_blocks = num_blocks;
  p.rows = rows;
  p.table_width = table_width;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.groups = num_q_heads / num_kv_heads;
  p.token_bucket = token_bucket;
  p.skip_single = skip_single;
  p.scale_log2 = scale * 1.4426950408889634f;
  if (q_dtype == NVJ_BF16) return launch_quantized_prefill_dims<__nv_bfloat16>(p, head_dim, s);
  if (q_dtype == NVJ_F16) return launch_quantized_prefill_dims<__half>(p, head_dim, s);
  return launch_quantized_prefill_dims<float>(p, head_dim, s);
}
