// Decode attention over selected blocks (selected_decode.cuh): the form on the CUDA cores, for f32 caches and for blocks that are not whole 16-key tiles, and the C
// entry.
//
// At four heads per kv head a number of an f32 cache is worth four fused multiply-adds, a fifth of what an SM does while the number arrives, so the CUDA cores
// keep up, in f32 throughout.  A warp takes eight keys at a time, a lane four neighbouring dims of each (eight of head_dim > 128): the 32 scores of
// eight keys and four heads are summed over the lanes by a butterfly of 31 exchanges that leaves one score with each lane, which turns it
// into a weight; for the second product a lane fetches the 32 weights one after the other.  Clusters, lists and the merge are those of the tensor-core form.

#include "selected_decode.cuh"

namespace nvj {

constexpr int kSlKeys = 8;

// Four neighbouring numbers of a cache row.
template <typename C>
__device__ __forceinline__ float4 sl_load4(const C* p) {
  if constexpr (sizeof(C) == 4) {
    const uint4 v = ld_stream_u4(p);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    const float2 a = sd_floats<C>(v.x), b = sd_floats<C>(v.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// kQuads: of a lane, 4 lane .. and 128 + 4 lane ..  kHeads: of the group, at a time.
template <typename C, int kQuads, int kHeads>
__global__ void __launch_bounds__(kSdThreads) selected_decode_lanes_kernel(SelectedParams p, int ctas) {
  constexpr int kPitch = 128 * kQuads + 4;  // floats
  extern __shared__ __align__(16) char sl_smem[];  // the queries [head][pitch]; then each warp's sums
  __shared__ float2 sd_ml[kSdWarps][kHeads];
  __shared__ float2 sd_ML[kHeads];
  float* qs = reinterpret_cast<float*>(sl_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = ctas > 1 ? (int)cl_rank() : 0;
  const int token = blockIdx.x / ctas, row = token / p.width;
  const int head = blockIdx.y / p.column_tiles, first_head = blockIdx.y % p.column_tiles * kHeads;
  const int hq = p.hkv * p.groups;
  pdl_wait();
  pdl_release();
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  const int32_t* list = p.selected + ((long long)token * p.hkv + head) * p.entries;
  const int per_block = (p.block_size + kSlKeys - 1) / kSlKeys, step = ctas * kSdWarps;
  const long long units = (long long)p.entries * per_block;
  // the next 32 units of this warp, one per lane: block id (-1: not there), its first key's place in the block, keys that are to be seen
  long long chunk = rank * kSdWarps + warp;
  int id = -1, off = 0, keys = 0;
  unsigned there = 0;
  auto entry_of = [&]() {
    const long long at = chunk + (long long)lane * step;
    return at < units ? list[at / per_block] : -1;
  };
  int c = entry_of();
  const int visible = sd_visible(p, row, token);
  auto look = [&]() {
    off = (int)((chunk + (long long)lane * step) % per_block) * kSlKeys;
    id = -1;
    if (c >= 0 && c < p.table_width && (long long)c * p.block_size + off < visible) {
      id = table[c];
      if (id < 0 || id >= p.num_blocks) {
        atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
        id = -1;
      }
    }
    keys = id >= 0 ? min(min(kSlKeys, p.block_size - off), visible - (c * p.block_size + off)) : 0;
    there = __ballot_sync(kFullMask, id >= 0);
  };
  look();
  const long long key_stride = (long long)p.hkv * p.d;
  bool inside[kQuads];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) inside[i] = 128 * i + 4 * lane < p.d;
  float4 k_held[kSlKeys][kQuads], v_held[kSlKeys][kQuads];
  int left = 0;  // keys of the unit under way; 0: none
  const C* next_v = nullptr;
  auto ask = [&](float4 (&held)[kSlKeys][kQuads], const C* at) {
#pragma unroll
    for (int k = 0; k < kSlKeys; ++k)
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
        if (k < left && inside[i]) held[k][i] = sl_load4(at + k * key_stride + 128 * i);
        else held[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
  };
  auto ask_k = [&]() {
    left = 0;
    while (there == 0) {
      chunk += 32 * step;
      if (chunk >= units) return;
      c = entry_of();
      look();
    }
    const int slot = __ffs(there) - 1;
    there &= there - 1;
    const long long key = (long long)__shfl_sync(kFullMask, id, slot) * p.block_size + __shfl_sync(kFullMask, off, slot);
    left = __shfl_sync(kFullMask, keys, slot);
    const long long at = (key * p.hkv + head) * p.d + 4 * lane;
    next_v = static_cast<const C*>(p.v_cache) + at;
    ask(k_held, static_cast<const C*>(p.k_cache) + at);
  };
  ask_k();
  if (left > 0) ask(v_held, next_v);

  for (int h = warp; h < kHeads; h += kSdWarps) {
    const int at = first_head + h;
    for (int d = 8 * lane; d < 128 * kQuads; d += 256) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      if (at < p.groups && d < p.d) sd_query8(p, ((long long)token * hq + head * p.groups + at) * p.d + d, x);
#pragma unroll
      for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(qs + h * kPitch + d + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
  }
  __syncthreads();

  // lane 4 k + h has the score, the weight and the sums of key k and head h (of each four heads)
  constexpr int kFours = kHeads / 4;
  float m[kFours], l[kFours];
  float4 acc[kHeads][kQuads];
#pragma unroll
  for (int f = 0; f < kFours; ++f) m[f] = kSdNone, l[f] = 0.f;
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
#pragma unroll
    for (int i = 0; i < kQuads; ++i) acc[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
  while (left > 0) {
    float w[kFours];
    const int seen = left;
#pragma unroll
    for (int f = 0; f < kFours; ++f) {
      float s[32];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float4 q[kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) q[i] = *reinterpret_cast<const float4*>(qs + (4 * f + h) * kPitch + 128 * i + 4 * lane);
#pragma unroll
        for (int k = 0; k < kSlKeys; ++k) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
            sum = fmaf(q[i].x, k_held[k][i].x, sum);
            sum = fmaf(q[i].y, k_held[k][i].y, sum);
            sum = fmaf(q[i].z, k_held[k][i].z, sum);
            sum = fmaf(q[i].w, k_held[k][i].w, sum);
          }
          s[4 * k + h] = sum;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const float keep = upper ? s[i + o] : s[i], send = upper ? s[i] : s[i + o];
          s[i] = keep + __shfl_xor_sync(kFullMask, send, o);
        }
      }
      w[f] = (lane >> 2) < seen ? s[0] * p.scale_log2 : -INFINITY;
    }
    ask_k();  // the K rows of the unit that is to take these registers
#pragma unroll
    for (int f = 0; f < kFours; ++f) {
      if (__any_sync(kFullMask, w[f] > m[f] + 8.f)) {
        float top = w[f];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
        const float now = fmaxf(m[f], top), down = ex2_approx(m[f] - now);
        m[f] = now;
        l[f] *= down;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float x = __shfl_sync(kFullMask, down, h);
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
            float4& a = acc[4 * f + h][i];
            a = make_float4(a.x * x, a.y * x, a.z * x, a.w * x);
          }
        }
      }
      w[f] = ex2_approx(w[f] - m[f]);
      l[f] += w[f];
    }
#pragma unroll
    for (int k = 0; k < kSlKeys; ++k) {  // (rows that are not to be seen are zeros, and so are their weights)
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float x = __shfl_sync(kFullMask, w[h / 4], 4 * k + h % 4);
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          float4& a = acc[h][i];
          a.x = fmaf(x, v_held[k][i].x, a.x);
          a.y = fmaf(x, v_held[k][i].y, a.y);
          a.z = fmaf(x, v_held[k][i].z, a.z);
          a.w = fmaf(x, v_held[k][i].w, a.w);
        }
      }
    }
    if (left > 0) ask(v_held, next_v);
  }
#pragma unroll
  for (int f = 0; f < kFours; ++f) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l[f] += __shfl_xor_sync(kFullMask, l[f], o);
    if (lane < 4) sd_ml[warp][4 * f + lane] = make_float2(m[f], l[f]);
  }
  __syncthreads();
  float* sums = reinterpret_cast<float*>(sl_smem) + warp * kHeads * kPitch;
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
#pragma unroll
    for (int i = 0; i < kQuads; ++i) *reinterpret_cast<float4*>(sums + h * kPitch + 128 * i + 4 * lane) = acc[h][i];
  __syncthreads();
  sd_merge<kHeads, kPitch>(p, reinterpret_cast<float*>(sl_smem), sd_ml, sd_ML, token, head, first_head, p.d, ctas, rank);
}

template <typename C, int kQuads, int kHeads>
static int launch_selected_lanes(const SelectedParams& p, cudaStream_t stream) {
  static PerDeviceFlags ready;
  return launch_selected_clusters(selected_decode_lanes_kernel<C, kQuads, kHeads>, ready, p, kHeads, kSlKeys, kSdWarps * kHeads * (128 * kQuads + 4) * 4,
                                  stream);
}
template <typename C>
static int launch_selected_lanes_heads(const SelectedParams& p, cudaStream_t stream) {
  if (p.d > 128) return launch_selected_lanes<C, 2, 4>(p, stream);  // (eight heads' sums of 256 dims do not fit the registers)
  return p.groups <= 4 ? launch_selected_lanes<C, 1, 4>(p, stream) : launch_selected_lanes<C, 1, 8>(p, stream);
}

}  // namespace nvj

extern "C" int nvj_paged_decode_selected(const void* q, int q_dtype, const void* k_cache_layer, const void* v_cache_layer, int cache_dtype,
                                         int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int num_q_heads,
                                         const int32_t* block_tables, int table_width, const int32_t* seq_lens, const int32_t* positions,
                                         const int32_t* selected, int entries, int rows, int width, float scale, float* out,
                                         int32_t* status, nvj_stream_t stream) {
  using namespace nvj;
  if (rows < 0 || width < 0 || table_width < 0 || num_blocks < 0 || entries < 0 || block_size < 1 || num_kv_heads < 1 || num_q_heads < 1 ||
      num_q_heads % num_kv_heads != 0)
    return NVJ_ERR_INVALID_ARGUMENT;
  if (q_dtype < NVJ_BF16 || q_dtype > NVJ_F32 || cache_dtype < NVJ_BF16 || cache_dtype > NVJ_F32 || head_dim < 8 || head_dim > 256 ||
      head_dim % 8 != 0 || num_kv_heads > 1024 || num_q_heads / num_kv_heads > 65535 || block_size > 65536)
    return NVJ_ERR_UNSUPPORTED;
  if ((long long)rows * width == 0) return NVJ_OK;
  if ((long long)table_width * block_size > 0x7fffffffLL || (long long)entries * block_size > 0x7fffffffLL ||
      (long long)rows * width > 0x7fffffffLL / 16)
    return NVJ_ERR_TOO_LARGE;
  if (!q || !k_cache_layer || !v_cache_layer || !seq_lens || !out || !status || (entries > 0 && !selected) || (table_width > 0 && !block_tables))
    return NVJ_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k_cache_layer) || !aligned16(v_cache_layer) || !aligned16(out)) return NVJ_ERR_INVALID_ARGUMENT;
  SelectedParams p{};
  p.q = q;
  p.k_cache = k_cache_layer;
  p.v_cache = v_cache_layer;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.positions = positions;
  p.selected = selected;
  p.out = out;
  p.status = status;
  p.num_blocks = num_blocks;
  p.q_dtype = q_dtype;
  p.rows = rows;
  p.width = width;
  p.table_width = table_width;
  p.block_size = block_size;
  p.hkv = num_kv_heads;
  p.groups = num_q_heads / num_kv_heads;
  p.d = head_dim;
  p.entries = entries;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (block_size % 16 == 0 && cache_dtype == NVJ_BF16) return launch_selected_bf16(p, s);
  if (block_size % 16 == 0 && cache_dtype == NVJ_F16) return launch_selected_f16(p, s);
  if (cache_dtype == NVJ_BF16) return launch_selected_lanes_heads<__nv_bfloat16>(p, s);
  if (cache_dtype == NVJ_F16) return launch_selected_lanes_heads<__half>(p, s);
  return launch_selected_lanes_heads<float>(p, s);
}
