// Decode attention over selected blocks (selected_decode.cuh): the form for any type and head layout, and the C entry.

#include "selected_decode.cuh"

namespace nvj {

__device__ __forceinline__ float sd_float(const void* p, long long i, int dtype) {
  if (dtype == NVJ_F32) return static_cast<const float*>(p)[i];
  if (dtype == NVJ_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Any type and head layout: on the CUDA cores, a warp per entry and key, the dims over the lanes, four heads at a time.
constexpr int kSgWarps = 4, kSgHeads = 4, kSgEach = 8;
template <typename C>
__global__ void __launch_bounds__(32 * kSgWarps) selected_decode_generic_kernel(SelectedParams p) {
  __shared__ float sums[kSgWarps][kSgHeads][256];
  __shared__ float2 ml[kSgWarps][kSgHeads];
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x, row = token / p.width, head = blockIdx.y, g0 = blockIdx.z * kSgHeads;
  const int heads = min(kSgHeads, p.groups - g0), hq = p.hkv * p.groups;
  const int visible = sd_visible(p, row, token);
  const int32_t* table = p.block_tables + (long long)row * p.table_width;
  const int32_t* list = p.selected + ((long long)token * p.hkv + head) * p.entries;
  const long long q_at = ((long long)token * hq + (long long)head * p.groups + g0) * p.d;
  float q[kSgHeads][kSgEach], acc[kSgHeads][kSgEach], m[kSgHeads], l[kSgHeads];
#pragma unroll
  for (int h = 0; h < kSgHeads; ++h) {
    m[h] = kSdNone;
    l[h] = 0.f;
#pragma unroll
    for (int j = 0; j < kSgEach; ++j) {
      acc[h][j] = 0.f;
      q[h][j] = h < heads && lane + 32 * j < p.d ? sd_float(p.q, q_at + (long long)h * p.d + lane + 32 * j, p.q_dtype) : 0.f;
    }
  }
  for (int e = warp; e < p.entries; e += kSgWarps) {
    const int c = list[e];
    if (c < 0 || c >= p.table_width || (long long)c * p.block_size >= visible) continue;
    const int id = table[c];
    if (id < 0 || id >= p.num_blocks) {
      if (lane == 0) atomicOr(p.status, NVJ_DEV_BAD_BLOCK_ID);
      continue;
    }
    const int keys = min(p.block_size, visible - c * p.block_size);
    for (int o = 0; o < keys; ++o) {
      const long long at = (((long long)id * p.block_size + o) * p.hkv + head) * p.d;
      const C *kp = static_cast<const C*>(p.k_cache) + at, *vp = static_cast<const C*>(p.v_cache) + at;
      float k[kSgEach], v[kSgEach];
#pragma unroll
      for (int j = 0; j < kSgEach; ++j) {
        const int d = lane + 32 * j;
        k[j] = d < p.d ? (float)kp[d] : 0.f;
        v[j] = d < p.d ? (float)vp[d] : 0.f;
      }
#pragma unroll
      for (int h = 0; h < kSgHeads; ++h) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < kSgEach; ++j) s = fmaf(q[h][j], k[j], s);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(kFullMask, s, x);
        s *= p.scale_log2;
        if (s > m[h]) {
          const float f = exp2f(m[h] - s);
          m[h] = s;
          l[h] *= f;
#pragma unroll
          for (int j = 0; j < kSgEach; ++j) acc[h][j] *= f;
        }
        const float w = exp2f(s - m[h]);
        l[h] += w;
#pragma unroll
        for (int j = 0; j < kSgEach; ++j) acc[h][j] = fmaf(w, v[j], acc[h][j]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kSgHeads; ++h) {
    if (lane == 0) ml[warp][h] = make_float2(m[h], l[h]);
#pragma unroll
    for (int j = 0; j < kSgEach; ++j) sums[warp][h][lane + 32 * j] = acc[h][j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * p.d; i += 32 * kSgWarps) {
    const int h = i / p.d, d = i % p.d;
    float top = kSdNone, sum = 0.f, y = 0.f;
    for (int w = 0; w < kSgWarps; ++w) top = fmaxf(top, ml[w][h].x);
    for (int w = 0; w < kSgWarps; ++w) {
      const float f = exp2f(ml[w][h].x - top);
      sum = fmaf(ml[w][h].y, f, sum);
      y = fmaf(sums[w][h][d], f, y);
    }
    p.out[((long long)token * hq + (long long)head * p.groups + g0 + h) * p.d + d] = sum == 0.f ? 0.f : y / sum;
  }
}

template <typename C>
static int launch_selected_generic(const SelectedParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)(p.rows * p.width), p.hkv, (p.groups + kSgHeads - 1) / kSgHeads);
  return launch_after(selected_decode_generic_kernel<C>, grid, dim3(32 * kSgWarps), 0, stream, p) == cudaSuccess ? NVJ_OK : NVJ_ERR_LAUNCH;
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
  const bool tiled = (head_dim == 64 || head_dim == 128 || head_dim == 256) && block_size % 16 == 0;
  if (tiled && cache_dtype == NVJ_BF16) return launch_selected_bf16(p, s);
  if (tiled && cache_dtype == NVJ_F16) return launch_selected_f16(p, s);
  if (cache_dtype == NVJ_BF16) return launch_selected_generic<__nv_bfloat16>(p, s);
  if (cache_dtype == NVJ_F16) return launch_selected_generic<__half>(p, s);
  return launch_selected_generic<float>(p, s);
}
