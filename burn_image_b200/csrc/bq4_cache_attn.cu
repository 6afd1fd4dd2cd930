// bq4_cache_attn.cu -- attention over the paged key/value cache: out =
// softmax(scale q K^T + mask) V for the newest tokens of every sequence, the
// keys being a prefix that the whole batch shares (if any) and the
// sequence's own rows.
//
// One warp takes one (sequence, query, head) row and walks its keys with a
// running maximum m and sum l in f32; each lane holds four values of q, of
// the key and of the output.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "bq4_cache.h"

namespace bq4 {
namespace {

constexpr int kWThreads = 128;

__device__ __forceinline__ void widen4(const CacheView& c, const uint8_t* src, const uint16_t* sc, int kv, int L,
                                       float (&x)[4]) {
  if (c.format == BQ4_CACHE_F16) {
    const uint2 u = reinterpret_cast<const uint2*>(src)[L];
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  } else if (c.format == BQ4_CACHE_Q8) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(src)[L];
    const float s = __uint_as_float((uint32_t)sc[0] << 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)((int)(w >> 8 * j & 255) - 128) * s;
  } else {
    const int blk = L >> 3, g = L & 7;
    const float s = __uint_as_float((uint32_t)sc[blk] << 16);
    if (kv == 0) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(src)[(g >> 1) * c.nb + blk] >> 8 * (L & 1);
      x[0] = (float)((int)(w & 15) - 8) * s;
      x[1] = (float)((int)(w >> 16 & 15) - 8) * s;
      x[2] = (float)((int)(w >> 4 & 15) - 8) * s;
      x[3] = (float)((int)(w >> 20 & 15) - 8) * s;
    } else {
      const uint32_t w = reinterpret_cast<const uint16_t*>(src)[g * c.nb + blk];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (float)((int)(w >> 4 * j & 15) - 8) * s;
    }
  }
}

__global__ void __launch_bounds__(kWThreads) cache_attn_kernel(const CacheAttnCall a, unsigned rows) {
  const unsigned row = (blockIdx.x * kWThreads + threadIdx.x) >> 5;
  if (row >= rows) return;
  const int L = threadIdx.x & 31;
  const unsigned bi = row / (unsigned)a.q_heads;
  const int h = (int)(row - bi * a.q_heads);
  const unsigned b = bi / (unsigned)a.tokens;
  const int i = (int)(bi - b * a.tokens);
  const int kvh = h / (a.q_heads / a.c.kv_heads);
  const bool mine = 4 * L < a.c.head_dim;
  float q[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (mine) {
    const __half* p = reinterpret_cast<const __half*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] +
                      h * a.q_stride[2] + 4 * L;
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = __half2float(p[j]);
  }
  const float c = a.scale * 1.4426950408889634f;  // log2(e)
  float m = -INFINITY, l = 0.0f;
  for (int part = a.prefix_table ? 0 : 1; part < 2; ++part) {
    const int32_t* table = part == 0 ? a.prefix_table : a.s.table + b * a.s.table_stride;
    const int64_t cap = part == 0 ? (int64_t)a.prefix_width * a.c.page_size
                                  : min((int64_t)a.max_length, (int64_t)a.s.table_width * a.c.page_size);
    int n = part == 0 ? a.prefix_length[0] : a.s.lengths[b];
    if (n < 0 || n > cap) {
      atomicCAS(a.err, 0, (int)BQ4_EINVAL_ARG);
      n = n < 0 ? 0 : (int)cap;
    }
    if (part == 1 && a.causal) n = n - a.tokens + i + 1;
    for (int j = 0; j < n; ++j) {
      const int pi = j / a.c.page_size, place = j - pi * a.c.page_size;
      const int page = table[pi];
      if (page < 0 || page >= a.c.pages) {
        atomicCAS(a.err, 0, (int)BQ4_EINVAL_ARG);
        continue;
      }
      const int64_t ph = (int64_t)page * a.c.kv_heads + kvh;
      const uint8_t* kr = a.c.values + ph * 2 * a.c.kv_bytes + (int64_t)place * a.c.row_bytes;
      const uint16_t* sc = a.c.scales + (ph * a.c.page_size + place) * 2 * a.c.nb;
      float k[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (mine) {
        widen4(a.c, kr, sc, 0, L, k);
        widen4(a.c, kr + a.c.kv_bytes, sc + a.c.nb, 1, L, v);
      }
      float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
      for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= c;
      const float mn = fmaxf(m, s), r = exp2f(m - mn), p = exp2f(s - mn);
      m = mn;
      l = l * r + p;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o[e] * r + p * v[e];
    }
  }
  if (mine) {
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    __half* out = reinterpret_cast<__half*>(a.out) + (int64_t)row * a.c.head_dim + 4 * L;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = __float2half_rn(o[j] * inv);
  }
}

}  // namespace

size_t cache_attn_workspace(const CacheAttnCall&, int) { return 0; }

bq4_status run_cache_attn(const CacheAttnCall& a, int, void*, cudaStream_t s) {
  const unsigned rows = (unsigned)((int64_t)a.s.batch * a.tokens * a.q_heads);
  const unsigned per = kWThreads / 32;
  cache_attn_kernel<<<(rows + per - 1) / per, kWThreads, 0, s>>>(a, rows);
  note_launch();
  return check_cuda(cudaGetLastError(), "cache attention launch");
}

}  // namespace bq4
