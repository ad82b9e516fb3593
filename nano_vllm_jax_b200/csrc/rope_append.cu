// Append of new K/V rows to the paged cache with the position rotation on the way, and the bounds of every block's keys beside it.
//
//   (a, b) -> (a c - b s, b c + a s),  c = cos(pos * inv_freq[i]), s = sin(pos * inv_freq[i]),  i < rot / 2
// for the pairs (x[i], x[i + rot/2]) of a query's or key's first `rot` dims, or (x[2i], x[2i + 1]) when they are interleaved.  The angle is a
// product in 64 bits (31 bits of position x 24 of frequency), cosine and sine are good to fp32, the products are formed in fp32 and the
// result is rounded once, to the type of the query or of the cache.
// Bounds: per block and kv head the smallest and the largest stored number of each dim, low in front of high; a block that begins with
// this call's tokens starts anew, another's widen.  NaN stays NaN.
//
// The unit of work for K and V is a run, as in the 8-bit append: tokens of the call that stand together and fall into one block; a warp
// (decode steps) or a CTA's four (prompts) take one run of one kv head, so that the bounds need no atomics.  Queries are dealt by token, so that a warp makes a token's cosines once for
// several heads.  A row is held by 8, 16 or 32 lanes, 8 elements each; its pairs meet by a shuffle of the loaded words.  Cosines and
// sines go through shared memory, and serve all heads that the warp takes.
// Bytes: tokens * head_dim * (2 hq + 2 hkv) * element.  Small calls are launch and the chain positions -> block id -> rows, old bounds -> stores: 256 tokens of 8 heads over 2 of 256,
// one per row, 4.6 us.  Prompts: 16384 bf16 tokens, 64 dims rotated, 45.5 us (203 MB: 31 at the copy rate), 777 f32 tokens of 32 heads over 8 of 128 12.9 (5.9).  Neither bytes (35% of the DRAM's
// peak) nor issue slots (50%) are full: too few warps, 29% of an SM's (96 registers of a thread, f32 127), wait for results of their own, of memory and for code, some 140
// instructions for a row in every form that a call may take.  (Bounds as they are stored, two numbers of 16 bits at a time, spared 2 us.)

#include "quantized_kv.cuh"

namespace nvj {

struct RopeAppendParams {
  const void* q;
  const void* k;
  const void* v;
  long long q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  void* q_out;                                                  // [tokens, hq, D]
  void* k_cache;
  void* v_cache;
  void* bounds;  // nullable [num_blocks, hkv, 2, D]
  const float* inv_freq;
  const int32_t* positions;
  const int32_t* block_tables;
  const int32_t* token_row_ids;    // packed batches
  const int32_t* query_start_loc;  // nullable
  const int32_t* seq_lens;         // nullable: rows with seq_lens[r] <= 0 are left alone
  int32_t* status;
  long long num_blocks;
  int rot, interleaved, hq, hkv, d, qsl_rows, packed, n_tokens, n_cols, table_rows, table_width, block_size;
  int window, kv_ctas, kv_heads, q_ctas, item_heads;  // tokens of a CTA; grid y: CTAs of K and V runs of `kv_heads` heads, then of queries, `item_heads` heads of a token at a time
};

constexpr int kRaWarps = 4, kRaHold = 4;  // rows (steps of rows) that a warp has in flight

__device__ __forceinline__ float ra_min(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float ra_max(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Eight numbers in the type C, rounded to nearest even, and back.
template <typename C>
__device__ __forceinline__ QRaw<C> ra_pack(const float (&x)[8]) {
  QRaw<C> r;
  if constexpr (sizeof(C) == 4) {
    r.v = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    r.w = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<C, __half>::value) {
        w[i] = q_pair(x[2 * i], x[2 * i + 1]);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    r.v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}
// The smaller and the larger of two words of numbers of the type C, NaN where either is.
template <typename C, bool kLarger>
__device__ __forceinline__ uint32_t ra_end(uint32_t a, uint32_t b) {
  if constexpr (sizeof(C) == 4) {
    return __float_as_uint(kLarger ? ra_max(__uint_as_float(a), __uint_as_float(b)) : ra_min(__uint_as_float(a), __uint_as_float(b)));
  } else {
    using Pair = typename std::conditional<std::is_same<C, __half>::value, __half2, __nv_bfloat162>::type;
    const Pair x = *reinterpret_cast<const Pair*>(&a), y = *reinterpret_cast<const Pair*>(&b), z = kLarger ? __hmax2_nan(x, y) : __hmin2_nan(x, y);
    return *reinterpret_cast<const uint32_t*>(&z);
  }
}
template <typename C, bool kLarger>
__device__ __forceinline__ uint4 ra_ends4(const uint4& a, const uint4& b) {
  return make_uint4(ra_end<C, kLarger>(a.x, b.x), ra_end<C, kLarger>(a.y, b.y), ra_end<C, kLarger>(a.z, b.z), ra_end<C, kLarger>(a.w, b.w));
}
// Bounds of eight dims, as they are stored.
template <typename C>
struct RaEnds {
  QRaw<C> low, high;
  __device__ __forceinline__ void clear() {
    constexpr uint32_t up = sizeof(C) == 4 ? 0x7f800000u : std::is_same<C, __half>::value ? 0x7c007c00u : 0x7f807f80u;  // infinities
    constexpr uint32_t down = up | (sizeof(C) == 4 ? 0x80000000u : 0x80008000u);
    low.v = make_uint4(up, up, up, up);
    high.v = make_uint4(down, down, down, down);
    if constexpr (sizeof(C) == 4) low.w = low.v, high.w = high.v;
  }
  __device__ __forceinline__ void take(const QRaw<C>& smaller, const QRaw<C>& larger) {
    low.v = ra_ends4<C, false>(low.v, smaller.v);
    high.v = ra_ends4<C, true>(high.v, larger.v);
    if constexpr (sizeof(C) == 4) {
      low.w = ra_ends4<C, false>(low.w, smaller.w);
      high.w = ra_ends4<C, true>(high.w, larger.w);
    }
  }
};
template <typename C>
__device__ __forceinline__ void ra_store(C* at, const QRaw<C>& r) {
  *reinterpret_cast<uint4*>(at) = r.v;
  if constexpr (sizeof(C) == 4) *reinterpret_cast<uint4*>(at + 4) = r.w;
}

// How a row's pairs lie: `whole` where a lane's eight elements are turned or left together and their partners are another lane's eight, or their own neighbours.
struct RaPairs {
  int rot, half;
  bool pairs, whole, turns;  // turns: this lane's elements are (where whole)
  int from;                  // the lane that has the partners
};
template <int kLanes>
__device__ __forceinline__ RaPairs ra_pairs(const RopeAppendParams& p, int lane) {
  RaPairs r;
  const int col = (lane % kLanes) * 8;
  r.rot = p.rot;
  r.half = p.rot >> 1;
  r.pairs = p.interleaved;
  r.whole = (p.rot & (r.pairs ? 7 : 15)) == 0;
  r.turns = col < p.rot;
  r.from = (lane & ~(kLanes - 1)) + (col < r.half ? (col + r.half) >> 3 : col < r.rot ? (col - r.half) >> 3 : col >> 3);
  return r;
}
// Cosine and sine to a few units of 2^-24 of an angle: in units of half a turn, a rounding in 64 bits away.  (qk_norm_rope_append.cu, which rounds them to bf16, keeps their relative
// accuracy next to the zeros; here they are multiplied and added in fp32.)
__device__ __forceinline__ float2 ra_cos_sin(double angle) {
  const double turns = angle * 0x1.45f306dc9c883p-2;  // 1 / pi
  const long long halves = __double2ll_rn(2.0 * turns);
  float s, c;
  sincospif((float)fma(-0.5, (double)halves, turns), &s, &c);
  const int quarter = (int)halves & 3;
  const float cq = (quarter & 1) ? s : c, sq = (quarter & 1) ? c : s;
  return make_float2(quarter == 1 || quarter == 2 ? -cq : cq, quarter & 2 ? -sq : sq);
}
// Cosines and sines of a position, by the lanes `mine` of `lanes`.
__device__ __forceinline__ void ra_angles(float2* cs, const float* inv_freq, int half, int pos, int mine, int lanes) {
  for (int f = mine; f < half; f += lanes) cs[f] = ra_cos_sin((double)pos * (double)inv_freq[f]);
}
// What this lane's elements and their partners are multiplied by (whole rows).
struct RaFactors {
  float c[8], s[8];
};
__device__ __forceinline__ void ra_factors(RaFactors& f, const float2* cs, const RaPairs& r, int col) {
  if (!r.turns) return;
  if (r.pairs) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = cs[(col >> 1) + j];
      f.c[2 * j] = f.c[2 * j + 1] = t.x;
      f.s[2 * j] = -t.y;
      f.s[2 * j + 1] = t.y;
    }
  } else {
    const float2* at = cs + (col < r.half ? col : col - r.half);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 t = at[j];
      f.c[j] = t.x;
      f.s[j] = col < r.half ? -t.y : t.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ QRaw<T> ra_shuffle(const QRaw<T>& r, int from) {
  QRaw<T> o;
  o.v = make_uint4(__shfl_sync(kFullMask, r.v.x, from), __shfl_sync(kFullMask, r.v.y, from), __shfl_sync(kFullMask, r.v.z, from),
                   __shfl_sync(kFullMask, r.v.w, from));
  if constexpr (sizeof(T) == 4)
    o.w = make_uint4(__shfl_sync(kFullMask, r.w.x, from), __shfl_sync(kFullMask, r.w.y, from), __shfl_sync(kFullMask, r.w.z, from),
                     __shfl_sync(kFullMask, r.w.w, from));
  return o;
}
// One row turned: x from `raw`.  All lanes of the warp are here.
template <typename T>
__device__ __forceinline__ void ra_turn(float (&x)[8], const QRaw<T>& raw, const RaFactors& f, const RaPairs& r) {
  q_floats(raw, x);
  if (r.pairs) {
    if (r.turns) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float a = x[j], b = x[j + 1];
        x[j] = fmaf(a, f.c[j], b * f.s[j]);
        x[j + 1] = fmaf(b, f.c[j + 1], a * f.s[j + 1]);
      }
    }
    return;
  }
  float other[8];
  q_floats(ra_shuffle(raw, r.from), other);
  if (r.turns) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(x[j], f.c[j], other[j] * f.s[j]);
  }
}
// The same where a lane's elements differ: element by element, partners from memory.
template <typename T>
__device__ __forceinline__ void ra_turn_odd(float (&x)[8], const T* src, const float2* cs, const RaPairs& r, int col) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = col + j;
    if (i >= r.rot) continue;
    const bool first = r.pairs ? !(i & 1) : i < r.half;
    const float other = (float)src[r.pairs ? i ^ 1 : first ? i + r.half : i - r.half];
    const float2 t = cs[r.pairs ? i >> 1 : first ? i : i - r.half];
    x[j] = fmaf(x[j], t.x, first ? -(other * t.y) : other * t.y);
  }
}

// Table entry (row * table_width + block of the row) and block of a token, or -1 for a token that is not written.
struct RaToken {
  long long entry;
  int block;
};
__device__ __forceinline__ RaToken ra_token(const RopeAppendParams& p, int i) {
  RaToken t{-1, 0};
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
  const int block = pos / p.block_size;
  if (pos < 0 || block >= p.table_width) {
    atomicOr(p.status, NVJ_DEV_BAD_LENGTH);
    return t;
  }
  t.entry = (long long)row * p.table_width + block;
  t.block = block;
  return t;
}

constexpr int kRaTable = 512;  // cosines and sines that a warp's table holds

// One run: `n` tokens from `first` on, of table entry `entry`, of the kv heads head0 .. head1, by kShare warps that meet at the CTA's barriers.
template <typename T, typename C, int kLanes, int kShare>
__device__ __forceinline__ void ra_run(const RopeAppendParams& p, int first, int n, long long entry, int block, int head0, int head1, bool is_v,
                                       float2 (&tables)[kRaWarps][kRaTable], int warp, int lane) {
  constexpr int kRows = 32 / kLanes;
  const int lane_row = lane / kLanes, sub = (kShare > 1 ? warp * kRows : 0) + lane_row, col = (lane % kLanes) * 8;
  constexpr int kStep = kShare * kRows;  // rows from one step to the next
  float2* table = tables[warp];
  const bool inside = col < p.d;
  const T* src = static_cast<const T*>(is_v ? p.v : p.k);
  const long long token_stride = is_v ? p.v_token : p.k_token, head_stride = is_v ? p.v_head : p.k_head;
  const int id = p.block_tables[entry];
  const bool turned = !is_v && p.rot > 0;
  const RaPairs pairs = ra_pairs<kLanes>(p, lane);
  const long long slot = (long long)p.hkv * p.d;
  const bool bounded = !is_v && p.bounds;
  const int steps = (n + kStep - 1) / kStep;
  const bool kept = steps * kRows * pairs.half <= kRaTable;  // the table holds the angles of all rows of this warp, for all heads
  bool made = false, begins = false;
  for (int head = head0; head < head1; ++head) {
    C* base = static_cast<C*>(is_v ? p.v_cache : p.k_cache) + (((long long)id * p.block_size - (long long)block * p.block_size) * p.hkv + head) * p.d + col;
    RaEnds<C> ends;
    ends.clear();
    for (int at = 0; at < n; at += kRaHold * kStep) {
      QRaw<T> raw[kRaHold];
      int pos[kRaHold];
#pragma unroll
      for (int s = 0; s < kRaHold; ++s) {
        const int r = at + s * kStep + sub;
        pos[s] = 0;
        if (r < n) {
          pos[s] = p.positions[first + r];
          if (inside) raw[s] = q_load8(src + (long long)(first + r) * token_stride + head * head_stride + col);
        }
      }
      if (id < 0 || id >= p.num_blocks) {  // (the rows have been asked for before the id is there)
        if (lane == 0) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
        return;
      }
      if (turned && !made) {
        __syncwarp();
        if (kept) {
          for (int s = 0; s < steps; ++s)
            if (s * kStep + sub < n)
              ra_angles(table + (s * kRows + lane_row) * pairs.half, p.inv_freq, pairs.half, p.positions[first + s * kStep + sub], lane % kLanes, kLanes);
          made = true;
        } else {
#pragma unroll
          for (int s = 0; s < kRaHold; ++s)
            if (at + s * kStep + sub < n) ra_angles(table + (s * kRows + lane_row) * pairs.half, p.inv_freq, pairs.half, pos[s], lane % kLanes, kLanes);
        }
        __syncwarp();
      }
#pragma unroll
      for (int s = 0; s < kRaHold; ++s) {
        if (at + s * kStep + (kShare > 1 ? warp * kRows : 0) >= n) break;
        const int r = at + s * kStep + sub;
        const bool live = r < n && inside;
        const float2* cs = table + ((kept ? at / kStep + s : s) * kRows + lane_row) * pairs.half;
        float x[8];
        if (turned && pairs.whole) {
          RaFactors f;
          ra_factors(f, cs, pairs, col);
          ra_turn(x, raw[s], f, pairs);
        } else {
          q_floats(raw[s], x);
          if (turned && live) ra_turn_odd(x, src + (long long)(first + r) * token_stride + head * head_stride, cs, pairs, col);
        }
        if (live) {
          const QRaw<C> w = ra_pack<C>(x);
          ra_store<C>(base + (long long)pos[s] * slot, w);
          if (bounded) {
            begins |= pos[s] == block * p.block_size;
            ends.take(w, w);
          }
        }
      }
    }
    if (!bounded) continue;
    begins = __any_sync(kFullMask, begins);
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) ends.take(ra_shuffle(ends.low, lane ^ o), ra_shuffle(ends.high, lane ^ o));
    if constexpr (kShare > 1) {
      __shared__ __align__(16) QRaw<C> of_warps[kRaWarps][2][32];
      begins = __syncthreads_or(begins);  // (and the ends of the head before have been read)
      if (lane_row == 0 && inside) of_warps[warp][0][lane] = ends.low, of_warps[warp][1][lane] = ends.high;
      __syncthreads();
      if ((head - head0) % kShare == warp && lane_row == 0 && inside)  // (the heads in turn)
#pragma unroll
        for (int w = 0; w < kShare; ++w) ends.take(of_warps[w][0][lane], of_warps[w][1][lane]);
    }
    if ((kShare == 1 || (head - head0) % kShare == warp) && lane_row == 0 && inside) {
      C* at = static_cast<C*>(p.bounds) + ((long long)id * p.hkv + head) * 2 * p.d + col;
      if (!begins) ends.take(q_load8(at), q_load8(at + p.d));
      ra_store<C>(at, ends.low);
      ra_store<C>(at + p.d, ends.high);
    }
  }
}

// kShare 1: a warp takes the runs of its part (K or V of a kv head); 4: the CTA's warps share them.
template <typename T, typename C, int kLanes, int kShare>
__global__ void __launch_bounds__(32 * kRaWarps, sizeof(T) == 4 ? 4 : 5) rope_append_kernel(RopeAppendParams p) {
  __shared__ __align__(16) float2 tables[kRaWarps][kRaTable];  // rows x rot / 2 frequencies
  constexpr int kRows = 32 / kLanes;
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long base = (long long)blockIdx.x * p.window;  // first token of the window
  if ((int)blockIdx.y < p.kv_ctas) {
    const int part = kShare > 1 ? (int)blockIdx.y : (int)blockIdx.y * kRaWarps + warp, head = (part >> 1) * p.kv_heads;
    if (head >= p.hkv) return;
    if constexpr (kShare > 1) {  // a prompt: the window's rows on their way to the L2 while their places are looked up
      const int heads = min(p.kv_heads, p.hkv - head), lines = (p.d * (int)sizeof(T) + 127) / 128;
      const char* from = static_cast<const char*>(part & 1 ? p.v : p.k);
      const long long token_stride = (part & 1 ? p.v_token : p.k_token) * (long long)sizeof(T), head_stride = (part & 1 ? p.v_head : p.k_head) * (long long)sizeof(T);
      for (int i = threadIdx.x; i < p.window * heads * lines; i += 32 * kRaWarps) {
        const long long token = base + i / (heads * lines);
        const int j = i % (heads * lines);
        if (token < p.n_tokens)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(from + token * token_stride + (head + j / lines) * head_stride + j % lines * 128));
      }
    }
    // lane l looks at token base - 1 + l: the one in front tells whether the window's first token begins a run
    const RaToken t = ra_token(p, (int)base - 1 + lane);
    const long long in_front = __shfl_up_sync(kFullMask, t.entry, 1);
    const bool same = lane > 0 && t.entry >= 0 && t.entry == in_front;
    const unsigned chain = __ballot_sync(kFullMask, same);
    unsigned starts = __ballot_sync(kFullMask, lane > 0 && lane <= p.window && t.entry >= 0 && !same);
    for (; starts; starts &= starts - 1) {
      const int at = __ffs(starts) - 1;  // lane of the run's first token
      const long long entry = __shfl_sync(kFullMask, t.entry, at);
      const int block = __shfl_sync(kFullMask, t.block, at);
      const int first = (int)base - 1 + at;
      const unsigned follow = at == 31 ? 0u : ~(chain >> (at + 1));  // bit j clear: token first + 1 + j is of the run
      int n = 1 + (follow ? __ffs(follow) - 1 : 32);
      if (at + n > 31) {  // the run may go on behind what the lanes have seen
        n = 32 - at;
        for (;;) {
          const unsigned more = __ballot_sync(kFullMask, ra_token(p, first + n + lane).entry == entry);
          const int add = more == kFullMask ? 32 : __ffs(~more) - 1;
          n += add;
          if (add < 32) break;
        }
      }
      ra_run<T, C, kLanes, kShare>(p, first, n, entry, block, head, min(p.hkv, head + p.kv_heads), part & 1, tables, warp, lane);
    }
    return;
  }
  // queries: items of `item_heads` heads of a token
  constexpr int kHold = sizeof(T) == 4 ? 4 : 8;  // a token's rows of eight heads on their way before its angles are made
  float2* table = tables[warp];
  const int sub = lane / kLanes, col = (lane % kLanes) * 8;
  const bool inside = col < p.d;
  const RaPairs pairs = ra_pairs<kLanes>(p, lane);
  const int chunks = (p.hq + p.item_heads - 1) / p.item_heads, items = p.window * chunks;
  for (int item = ((int)blockIdx.y - p.kv_ctas) * kRaWarps + warp; item < items; item += p.q_ctas * kRaWarps) {
    const long long token = base + item / chunks;
    if (token >= p.n_tokens) break;
    const int h0 = item % chunks * p.item_heads, h1 = min(p.hq, h0 + p.item_heads);
    const T* src = static_cast<const T*>(p.q) + token * p.q_token + (h0 + sub) * p.q_head;
    T* dst = static_cast<T*>(p.q_out) + (token * p.hq + h0 + sub) * p.d + col;
    const long long step = kRows * p.q_head;
    RaFactors f;
    bool made = false;
    for (int h = h0; h < h1; h += kHold * kRows) {
      QRaw<T> raw[kHold];
#pragma unroll
      for (int s = 0; s < kHold; ++s) {
        const int mine = h + s * kRows + sub;
        if (mine < h1 && inside) raw[s] = q_load8(src + s * step + col);
      }
      if (!made && pairs.half > 0) {
        __syncwarp();
        ra_angles(table, p.inv_freq, pairs.half, p.positions[token], lane, 32);
        __syncwarp();
        if (pairs.whole) ra_factors(f, table, pairs, col);
        made = true;
      }
#pragma unroll
      for (int s = 0; s < kHold; ++s) {
        if (h + s * kRows >= h1) break;
        const int mine = h + s * kRows + sub;
        const bool live = mine < h1 && inside;
        float x[8];
        if (pairs.half > 0 && pairs.whole) {
          ra_turn(x, raw[s], f, pairs);
        } else {
          q_floats(raw[s], x);
          if (pairs.half > 0 && live) ra_turn_odd(x, src + s * step, table, pairs, col);
        }
        if (live) ra_store<T>(dst + s * kRows * p.d, ra_pack<T>(x));
      }
      src += kHold * step;
      dst += kHold * kRows * p.d;
    }
  }
}

template <typename T, typename C>
static int launch_rope_append(RopeAppendParams p, cudaStream_t stream) {
  // Batches of a few tokens per row: a token per CTA column, its parts and heads dealt to warps.  Prompts: windows of up to 16 tokens, a row's mean, so that one run begins in
  // each, mostly (a window's runs come one behind the other: 8 rows of 5 tokens 18.7 us with windows of 16), shared by a CTA's warps.  The more tokens, the more heads a warp
  // takes, so that cosines are made less often.
  const long long n = p.n_tokens, rows = p.packed ? (p.query_start_loc ? p.qsl_rows : 1) : (n + p.n_cols - 1) / p.n_cols;
  const long long mean = n / (rows > 0 ? rows : 1);
  const bool prompt = mean > 4;
  const int lanes = p.d <= 64 ? 8 : p.d <= 128 ? 16 : 32, at_once = 32 / lanes;
  p.window = prompt ? (int)(mean < 16 ? mean : 16) : 1;
  const long long windows = (n + p.window - 1) / p.window;
  auto within = [](long long x, long long low, long long high) { return (int)(x < low ? low : x > high ? high : x); };
  p.kv_heads = prompt ? (windows * 2 * p.hkv > 20 * 148 ? 2 : 1) : within(n * 2 * p.hkv / (32 * 148), 1, 4);
  const int parts = 2 * ((p.hkv + p.kv_heads - 1) / p.kv_heads);
  p.kv_ctas = prompt ? parts : (parts + kRaWarps - 1) / kRaWarps;
  const int steps = (p.hq + at_once - 1) / at_once, each = within(n * steps / (20 * 148), 1, 16);  // of a token; of a warp
  const int item = within(each, 1, steps < 8 ? (steps > 0 ? steps : 1) : 8);
  p.item_heads = item * at_once;
  const int items = p.hq > 0 ? p.window * ((p.hq + p.item_heads - 1) / p.item_heads) : 0, of_warp = prompt && each > item ? each / item : 1;
  p.q_ctas = (items + kRaWarps * of_warp - 1) / (kRaWarps * of_warp);
  const dim3 grid((unsigned)((p.n_tokens + p.window - 1LL) / p.window), p.kv_ctas + p.q_ctas);
  auto go = [&](auto* kernel) { return launch_after(kernel, grid, dim3(32 * kRaWarps), 0, stream, p) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH; };
  auto shared = [&](auto width) {
    constexpr int kLanes = decltype(width)::value;
    return prompt ? go(rope_append_kernel<T, C, kLanes, kRaWarps>) : go(rope_append_kernel<T, C, kLanes, 1>);
  };
  if (lanes == 8) return shared(std::integral_constant<int, 8>{});
  if (lanes == 16) return shared(std::integral_constant<int, 16>{});
  return shared(std::integral_constant<int, 32>{});
}
template <typename T>
static int launch_rope_append_cache(const RopeAppendParams& p, int cache_dtype, cudaStream_t s) {
  if (cache_dtype == NVJ_BF16) return launch_rope_append<T, __nv_bfloat16>(p, s);
  if (cache_dtype == NVJ_F16) return launch_rope_append<T, __half>(p, s);
  return launch_rope_append<T, float>(p, s);
}

}  // namespace nvj

extern "C" int nvj_rope_kv_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                                  int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, int act_dtype,
                                  const float* inv_freq, int rotary_dim, int interleaved, const int32_t* positions,
                                  const int32_t* block_tables, const int32_t* token_row_ids, int table_rows, int table_width,
                                  const int32_t* query_start_loc, int qsl_rows, const int32_t* seq_lens, int n_rows, int n_cols,
                                  void* k_cache_layer, void* v_cache_layer, void* k_bounds, int cache_dtype, int64_t num_blocks,
                                  int block_size, int num_q_heads, int num_kv_heads, int head_dim, void* q_out, int32_t* status,
                                  nvj_stream_t stream) {
  using namespace nvj;
  if (n_rows < 0 || n_cols < 0 || table_rows < 0 || table_width < 0 || qsl_rows < 0 || num_blocks < 0 || num_q_heads < 0 || num_kv_heads < 1 ||
      block_size < 1 || rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1))
    return NVJ_ERR_INVALID_ARGUMENT;
  if (act_dtype < NVJ_BF16 || act_dtype > NVJ_F32 || cache_dtype < NVJ_BF16 || cache_dtype > NVJ_F32 || head_dim < 8 || head_dim > 256 ||
      head_dim % 8 != 0 || num_kv_heads > 1024 || num_q_heads > 65536)
    return NVJ_ERR_UNSUPPORTED;
  const long long n = (long long)n_rows * n_cols;
  if (n == 0) return NVJ_OK;
  if (n > 0x7fffffffLL - 64) return NVJ_ERR_TOO_LARGE;
  if (!k || !v || !positions || !block_tables || !k_cache_layer || !v_cache_layer || !status || (q && !q_out) || (rotary_dim > 0 && !inv_freq))
    return NVJ_ERR_INVALID_ARGUMENT;
  if (table_rows == 0 || table_width == 0 || num_blocks == 0) return NVJ_ERR_INVALID_ARGUMENT;
  if (token_row_ids && n_rows != 1) return NVJ_ERR_INVALID_ARGUMENT;
  const bool placed = aligned16(q) && aligned16(k) && aligned16(v) && aligned16(k_cache_layer) && aligned16(v_cache_layer) && aligned16(k_bounds) &&
                      aligned16(q_out);
  const int64_t strides = q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride;
  if (!placed || (strides & (act_dtype == NVJ_F32 ? 3 : 7)) != 0) return NVJ_ERR_INVALID_ARGUMENT;
  RopeAppendParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.q_out = q_out;
  p.k_cache = k_cache_layer;
  p.v_cache = v_cache_layer;
  p.bounds = k_bounds;
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.block_tables = block_tables;
  p.token_row_ids = token_row_ids;
  p.query_start_loc = query_start_loc;
  p.seq_lens = seq_lens;
  p.status = status;
  p.num_blocks = num_blocks;
  p.rot = rotary_dim;
  p.interleaved = interleaved;
  p.hq = q ? num_q_heads : 0;
  p.hkv = num_kv_heads;
  p.d = head_dim;
  p.qsl_rows = qsl_rows;
  p.packed = token_row_ids != nullptr;
  p.n_tokens = (int)n;
  p.n_cols = n_cols;
  p.table_rows = table_rows;
  p.table_width = table_width;
  p.block_size = block_size;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (act_dtype == NVJ_BF16) return launch_rope_append_cache<__nv_bfloat16>(p, cache_dtype, s);
  if (act_dtype == NVJ_F16) return launch_rope_append_cache<__half>(p, cache_dtype, s);
  return launch_rope_append_cache<float>(p, cache_dtype, s);
}
