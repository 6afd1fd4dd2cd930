// bq4_cache.cu -- the paged key/value cache: rows quantised as they are
// written, rows read back, and the host entry points of the cache (the
// attention kernels are in bq4_cache_attn.cu).
//
// Both kernels move each byte once and compute next to nothing, so HBM (and,
// for a decode step's few rows, the launch) bounds them.  A row of HP values
// is taken by HP / 4 lanes, four consecutive values each: 16- or 8-byte
// accesses on the wide side, the block maximum by shuffles over the 8 lanes
// of a q4 block or all lanes of a q8 row, and one store of 4 (q8), 2 (q4) or
// 8 (f16) bytes a lane on the cache side.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "bq4_cache.h"

namespace bq4 {
namespace {

constexpr int kCThreads = 256;

struct CacheRow {
  uint8_t* rows;   // k or v rows of the page and head
  uint16_t* scales;
};

// Rows of (page, head) and the scales of the row at `place`; kv: 0 k, 1 v.
__device__ __forceinline__ CacheRow cache_row(const CacheView& c, int page, int head, int place, int kv) {
  const int64_t ph = (int64_t)page * c.kv_heads + head;
  CacheRow r;
  r.rows = c.values + (ph * 2 + kv) * c.kv_bytes;
  r.scales = c.scales + ((ph * c.page_size + place) * 2 + kv) * c.nb;
  return r;
}

// Rows that sequence b holds; records a length that its pages cannot.
__device__ __forceinline__ int seq_length(const SeqView& s, int page_size, int b, int* err) {
  const int64_t cap = (int64_t)s.table_width * page_size;
  const int n = s.lengths[b];
  if (n < 0 || n > cap) {
    atomicCAS(err, 0, (int)BQ4_EINVAL_ARG);
    return n < 0 ? 0 : (int)cap;
  }
  return n;
}

template <bool kF16>
__device__ __forceinline__ void load4(const void* base, int64_t at, bool vec, float (&x)[4]) {
  if constexpr (kF16) {
    const __half* p = static_cast<const __half*>(base) + at;
    if (vec) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
      x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __half2float(p[j]);
    }
  } else {
    const float* p = static_cast<const float*>(base) + at;
    if (vec) {
      const float4 u = *reinterpret_cast<const float4*>(p);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = p[j];
    }
  }
}

struct AppendArgs {
  CacheView c;
  SeqView s;
  const void* x[2];       // k, v
  int64_t stride[2][3];   // batch, token, head
  int vec;                // every row of x starts on a 4-value boundary
  int tokens;
  unsigned rows;          // batch * tokens * kv_heads
  int* err;
};

// One row a group of HP / 4 lanes; blockIdx.y: k or v.
template <int kFmt, bool kF16>
__global__ void __launch_bounds__(kCThreads) cache_append_kernel(const AppendArgs a) {
  const int kv = blockIdx.y;
  const int lpr = a.c.hp >> 2;                     // lanes of a row: 16 or 32
  const int L = threadIdx.x & (lpr - 1), d0 = 4 * L;
  const unsigned row = blockIdx.x * (unsigned)(kCThreads / lpr) + threadIdx.x / lpr;
  int page = -1, place = 0, h = 0;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < a.rows) {
    const unsigned bi = row / (unsigned)a.c.kv_heads;
    h = (int)(row - bi * a.c.kv_heads);
    const unsigned b = bi / (unsigned)a.tokens, i = bi - b * a.tokens;
    const int pos = seq_length(a.s, a.c.page_size, (int)b, a.err) - a.tokens + (int)i;
    if (pos >= 0) {
      const int pi = pos / a.c.page_size;
      page = a.s.table[b * a.s.table_stride + pi];
      place = pos - pi * a.c.page_size;
      if (page < 0 || page >= a.c.pages) {
        atomicCAS(a.err, 0, (int)BQ4_EINVAL_ARG);
        page = -1;
      }
    }
    if (page >= 0 && d0 < a.c.head_dim)
      load4<kF16>(a.x[kv], b * a.stride[kv][0] + i * a.stride[kv][1] + h * a.stride[kv][2] + d0, a.vec, x);
  }
  const CacheRow r = cache_row(a.c, page < 0 ? 0 : page, h, place, kv);
  auto dst = [&](int at) { return r.rows + cache_swizzle(kv, a.c.row_bytes, place, at); };
  if constexpr (kFmt == BQ4_CACHE_F16) {
    const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&lo);
    u.y = *reinterpret_cast<const uint32_t*>(&hi);
    if (page >= 0) *reinterpret_cast<uint2*>(dst(8 * L)) = u;
    return;
  }
  constexpr float kTop = kFmt == BQ4_CACHE_Q8 ? 127.0f : 7.0f;
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float m = fabsf(x[j]);
    top = m <= 3.402823466e38f ? fmaxf(top, m) : INFINITY;  // NaN too; INFINITY stays the maximum
    if (top == INFINITY) break;
  }
  const int span = kFmt == BQ4_CACHE_Q8 ? lpr : kCacheBlock / 4;
  for (int o = span >> 1; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // f32 quotients, rounded to nearest: the scale and every q follow from the
  // definition bit for bit.
  const __nv_bfloat16 sb =
      top == INFINITY ? __float2bfloat16_rn(__int_as_float(0x7fc00000)) : __float2bfloat16_rn(__fdiv_rn(top, kTop));
  const float s = __bfloat162float(sb);
  int q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    q[j] = s > 0.0f ? (int)fminf(fmaxf(rintf(__fdiv_rn(x[j], s)), -kTop), kTop) : 0;
  if constexpr (kFmt == BQ4_CACHE_Q8) {
    const uint32_t w = (uint32_t)(q[0] + 128) | (uint32_t)(q[1] + 128) << 8 | (uint32_t)(q[2] + 128) << 16 |
                       (uint32_t)(q[3] + 128) << 24;
    if (page >= 0) {
      *reinterpret_cast<uint32_t*>(dst(4 * L)) = w;
      if (L == 0) r.scales[0] = __bfloat16_as_ushort(sb);
    }
  } else {
    const int blk = L >> 3, g = L & 7;
    if (kv == 0) {
      // values o = 4 (L & 1) + j of the word: nibble o / 2 + 4 (o & 1)
      uint32_t w = (uint32_t)(q[0] + 8) | (uint32_t)(q[1] + 8) << 16 | (uint32_t)(q[2] + 8) << 4 |
                   (uint32_t)(q[3] + 8) << 20;
      w <<= 8 * (L & 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      if (page >= 0 && !(L & 1)) *reinterpret_cast<uint32_t*>(dst(4 * ((g >> 1) * a.c.nb + blk))) = w;
    } else {
      const uint16_t w = (uint16_t)((q[0] + 8) | (q[1] + 8) << 4 | (q[2] + 8) << 8 | (q[3] + 8) << 12);
      if (page >= 0) *reinterpret_cast<uint16_t*>(dst(2 * (g * a.c.nb + blk))) = w;
    }
    if (page >= 0 && g == 0) r.scales[blk] = __bfloat16_as_ushort(sb);
  }
}

struct ReadArgs {
  CacheView c;
  SeqView s;
  const int32_t* starts;
  void* out[2];
  int64_t stride[3];      // batch, head, position
  int vec;
  int count;
  unsigned rows;          // batch * kv_heads * count
  int* err;
};

template <int kFmt, bool kF16>
__global__ void __launch_bounds__(kCThreads) cache_read_kernel(const ReadArgs a) {
  const int kv = blockIdx.y;
  const int lpr = a.c.hp >> 2;
  const int L = threadIdx.x & (lpr - 1), d0 = 4 * L;
  const unsigned row = blockIdx.x * (unsigned)(kCThreads / lpr) + threadIdx.x / lpr;
  if (row >= a.rows || d0 >= a.c.head_dim) return;
  const unsigned bh = row / (unsigned)a.count;
  const int i = (int)(row - bh * a.count);
  const unsigned b = bh / (unsigned)a.c.kv_heads;
  const int h = (int)(bh - b * a.c.kv_heads);
  const int64_t pos = (a.starts ? (int64_t)a.starts[b] : 0) + i;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (pos >= 0 && pos < seq_length(a.s, a.c.page_size, (int)b, a.err)) {
    const int pi = (int)pos / a.c.page_size;
    const int page = a.s.table[b * a.s.table_stride + pi];
    if (page < 0 || page >= a.c.pages) {
      atomicCAS(a.err, 0, (int)BQ4_EINVAL_ARG);
    } else {
      const int place = (int)pos - pi * a.c.page_size;
      const CacheRow r = cache_row(a.c, page, h, place, kv);
      auto src = [&](int at) { return r.rows + cache_swizzle(kv, a.c.row_bytes, place, at); };
      if constexpr (kFmt == BQ4_CACHE_F16) {
        load4<true>(src(2 * d0), 0, true, x);
      } else if constexpr (kFmt == BQ4_CACHE_Q8) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(src(4 * L));
        const float s = __uint_as_float((uint32_t)r.scales[0] << 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (float)((int)(w >> 8 * j & 255) - 128) * s;
      } else {
        const int blk = L >> 3, g = L & 7;
        const float s = __uint_as_float((uint32_t)r.scales[blk] << 16);
        if (kv == 0) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(src(4 * ((g >> 1) * a.c.nb + blk))) >> 8 * (L & 1);
          x[0] = (float)((int)(w & 15) - 8) * s;
          x[1] = (float)((int)(w >> 16 & 15) - 8) * s;
          x[2] = (float)((int)(w >> 4 & 15) - 8) * s;
          x[3] = (float)((int)(w >> 20 & 15) - 8) * s;
        } else {
          const uint32_t w = *reinterpret_cast<const uint16_t*>(src(2 * (g * a.c.nb + blk)));
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = (float)((int)(w >> 4 * j & 15) - 8) * s;
        }
      }
    }
  }
  const int64_t at = b * a.stride[0] + h * a.stride[1] + i * a.stride[2] + d0;
  if constexpr (kF16) {
    __half* o = static_cast<__half*>(a.out[kv]) + at;
    const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
    if (a.vec) {
      uint2 u;
      u.x = *reinterpret_cast<const uint32_t*>(&lo);
      u.y = *reinterpret_cast<const uint32_t*>(&hi);
      *reinterpret_cast<uint2*>(o) = u;
    } else {
      o[0] = __low2half(lo), o[1] = __high2half(lo), o[2] = __low2half(hi), o[3] = __high2half(hi);
    }
  } else {
    float* o = static_cast<float*>(a.out[kv]) + at;
    if (a.vec) {
      *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = x[j];
    }
  }
}

// ------------------------------------------------------------------ host side

struct Guard {  // restores the caller's current device
  int prev = -1;
  explicit Guard(int dev) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~Guard() {
    int cur = -1;
    cudaGetDevice(&cur);
    if (prev >= 0 && cur != prev) cudaSetDevice(prev);
  }
};

bool al(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Geometry of a cache, without its pointers and device.
bq4_status check_geometry(const bq4_cache* c) {
  if (!c) return set_error(BQ4_EINVAL_ARG, "cache is NULL");
  if (c->format != BQ4_CACHE_F16 && c->format != BQ4_CACHE_Q8 && c->format != BQ4_CACHE_Q4)
    return set_error(BQ4_EINVAL_ARG, "format %d is not BQ4_CACHE_F16/Q8/Q4", (int)c->format);
  if (c->pages <= 0 || c->pages > 0x7fffffff)
    return set_error(BQ4_EINVAL_SHAPE, "pages=%lld must be in [1, 2^31)", (long long)c->pages);
  if (c->page_size <= 0 || c->page_size % kCachePageUnit || c->page_size > 65536)
    return set_error(BQ4_EINVAL_SHAPE, "page_size=%d must be a multiple of 16 in [16, 65536]", (int)c->page_size);
  if (c->kv_heads <= 0 || c->kv_heads > 65535)
    return set_error(BQ4_EINVAL_SHAPE, "kv_heads=%d must be in [1, 65535]", (int)c->kv_heads);
  if (c->head_dim <= 0 || c->head_dim % 8 || c->head_dim > kCacheMaxHeadDim)
    return set_error(BQ4_EINVAL_SHAPE, "head_dim=%d must be a multiple of 8 in [8, 128]", (int)c->head_dim);
  // pages < 2^31, page_size <= 2^16, kv_heads < 2^16: their product fits 63 bits, its bytes may not
  const int64_t rows = c->pages * c->page_size;
  if (rows > ((int64_t)1 << 53) / c->kv_heads)
    return set_error(BQ4_EINVAL_SHAPE, "pages * page_size * kv_heads above 2^53");
  return BQ4_OK;
}

CacheView view_of(const bq4_cache* c) {
  CacheView v;
  v.values = static_cast<uint8_t*>(c->values);
  v.scales = static_cast<uint16_t*>(c->scales);
  v.pages = (int32_t)c->pages;
  v.page_size = c->page_size;
  v.kv_heads = c->kv_heads;
  v.head_dim = c->head_dim;
  v.hp = cache_hp(c->head_dim);
  v.nb = cache_nb(c->format, v.hp);
  v.row_bytes = cache_row_bytes(c->format, v.hp);
  v.format = c->format;
  v.kv_bytes = (int64_t)c->page_size * v.row_bytes;
  return v;
}

bq4_status check_cache(const bq4_cache* c) {
  bq4_status st = check_geometry(c);
  if (st) return st;
  if (!c->values || (!c->scales && c->format != BQ4_CACHE_F16))
    return set_error(BQ4_EINVAL_ARG, "the cache's values/scales are NULL");
  if (!al(c->values, 256) || !al(c->scales, 256))
    return set_error(BQ4_EALIGN, "the cache's buffers must be 256-byte aligned");
  return BQ4_OK;
}

bq4_status check_seqs(const bq4_cache* c, const bq4_cache_sequences* s, SeqView* v) {
  if (!s) return set_error(BQ4_EINVAL_ARG, "seqs is NULL");
  if (s->batch < 0 || s->table_width < 0 || s->table_stride < 0)
    return set_error(BQ4_EINVAL_SHAPE, "batch=%lld table_width=%lld table_stride=%lld", (long long)s->batch,
                     (long long)s->table_width, (long long)s->table_stride);
  if (s->batch && (!s->lengths || (!s->page_table && s->table_width)))
    return set_error(BQ4_EINVAL_ARG, "page_table/lengths is NULL");
  if (!al(s->page_table, 4) || !al(s->lengths, 4)) return set_error(BQ4_EALIGN, "page_table/lengths misaligned");
  if (s->batch > 0x7fffffff || s->table_width * (int64_t)c->page_size > ((int64_t)1 << 30) ||
      s->table_width > ((int64_t)1 << 30))
    return set_error(BQ4_EINVAL_SHAPE, "batch=%lld or table_width=%lld pages of %d rows: above 2^31 or 2^30 rows",
                     (long long)s->batch, (long long)s->table_width, (int)c->page_size);
  v->table = s->page_table;
  v->lengths = s->lengths;
  v->table_stride = s->table_stride;
  v->table_width = (int32_t)s->table_width;
  v->batch = (int32_t)s->batch;
  return BQ4_OK;
}

// rows = a * b * c when that is below 2^31
bool row_count(int64_t a, int64_t b, int64_t c, int64_t* rows) {
  constexpr int64_t kMost = 0x7fffffff;
  if (a > kMost || b > kMost || c > kMost) return false;
  if (a * b > kMost || a * b * c > kMost) return false;
  *rows = a * b * c;
  return true;
}

bq4_status device_ready(int device) {
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
    cudaGetLastError();
    return set_error(BQ4_EINVAL_ARG, "device %d not present", device);
  }
  if (!device_is_sm100(device))
    return set_error(BQ4_EUNSUPPORTED, "device %d is not sm_100 (B200); libbq4 has no kernels for it", device);
  return BQ4_OK;
}

bool strides_vec(const void* base, const int64_t* st, int esize) {
  return al(base, 4 * esize) && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

template <int kFmt>
void launch_append(const AppendArgs& a, bool f16, dim3 grid, cudaStream_t s) {
  if (f16)
    cache_append_kernel<kFmt, true><<<grid, kCThreads, 0, s>>>(a);
  else
    cache_append_kernel<kFmt, false><<<grid, kCThreads, 0, s>>>(a);
}

template <int kFmt>
void launch_read(const ReadArgs& a, bool f16, dim3 grid, cudaStream_t s) {
  if (f16)
    cache_read_kernel<kFmt, true><<<grid, kCThreads, 0, s>>>(a);
  else
    cache_read_kernel<kFmt, false><<<grid, kCThreads, 0, s>>>(a);
}

// The sizes that both the workspace query and the calls check and plan with.
bq4_status attention_shape(const bq4_cache* cache, int64_t batch, int64_t tokens, int64_t q_heads, int64_t max_length,
                           int64_t max_prefix, CacheAttnCall* call) {
  if (batch < 0 || tokens < 0 || q_heads <= 0 || max_length < 0 || max_prefix < 0)
    return set_error(BQ4_EINVAL_SHAPE, "batch=%lld tokens=%lld q_heads=%lld max_length=%lld max_prefix=%lld",
                     (long long)batch, (long long)tokens, (long long)q_heads, (long long)max_length,
                     (long long)max_prefix);
  if (q_heads % cache->kv_heads)
    return set_error(BQ4_EINVAL_SHAPE, "q_heads=%lld is not a multiple of kv_heads=%d", (long long)q_heads,
                     (int)cache->kv_heads);
  int64_t rows = 0;
  if (!row_count(batch, tokens, q_heads, &rows) || max_length > ((int64_t)1 << 30) ||
      max_prefix > ((int64_t)1 << 30))
    return set_error(BQ4_EINVAL_SHAPE, "batch * tokens * q_heads must be below 2^31, lengths at most 2^30");
  call->c = view_of(cache);
  call->s.batch = (int32_t)batch;
  call->tokens = (int32_t)tokens;
  call->q_heads = (int32_t)q_heads;
  call->max_length = (int32_t)max_length;
  call->prefix_width = (int32_t)((max_prefix + cache->page_size - 1) / cache->page_size);
  return BQ4_OK;
}

bq4_status attention(const bq4_cache* cache, const int32_t* prefix_pages, int64_t prefix_width,
                     const int32_t* prefix_length, bool prefix, const bq4_cache_sequences* seqs, int64_t max_length,
                     const void* q, const int64_t q_strides[3], int64_t tokens, int64_t q_heads, int32_t causal,
                     float scale, void* out, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  bq4_status st = check_cache(cache);
  if (st) return st;
  CacheAttnCall call = {};
  SeqView sv = {};
  st = check_seqs(cache, seqs, &sv);
  if (st) return st;
  if (prefix) {
    if (prefix_width < 0 || prefix_width > ((int64_t)1 << 30) ||
        prefix_width * (int64_t)cache->page_size > ((int64_t)1 << 30))
      return set_error(BQ4_EINVAL_SHAPE, "prefix_width=%lld", (long long)prefix_width);
    if (!prefix_length || (!prefix_pages && prefix_width))
      return set_error(BQ4_EINVAL_ARG, "prefix_pages/prefix_length is NULL");
    if (!al(prefix_pages, 4) || !al(prefix_length, 4))
      return set_error(BQ4_EALIGN, "prefix_pages/prefix_length misaligned");
  }
  const int64_t held = seqs->table_width * cache->page_size;
  st = attention_shape(cache, seqs->batch, tokens, q_heads, max_length > 0 && max_length < held ? max_length : held,
                       prefix ? prefix_width * cache->page_size : 0, &call);
  if (st) return st;
  if (max_length < 0) return set_error(BQ4_EINVAL_SHAPE, "max_length=%lld", (long long)max_length);
  if (seqs->batch == 0 || tokens == 0) return BQ4_OK;
  if (!q || !q_strides || !out) return set_error(BQ4_EINVAL_ARG, "q/q_strides/out is NULL");
  if (!al(q, 2) || !al(out, 16)) return set_error(BQ4_EALIGN, "q misaligned or out not 16-byte aligned");
  if (!(scale == scale)) return set_error(BQ4_EINVAL_ARG, "scale is NaN");
  st = device_ready(cache->device);
  if (st) return st;
  Guard guard(cache->device);
  const int sms = device_sm_count(cache->device);
  size_t need = 0;
  st = cache_attn_workspace(call, sms, &need);
  if (st) return st;
  if (need > workspace_bytes || (need && !workspace))
    return set_error(BQ4_EWORKSPACE, "workspace of %zu bytes; cache attention needs %zu", workspace_bytes, need);
  if (need && !al(workspace, 256)) return set_error(BQ4_EALIGN, "workspace not 256-byte aligned");
  call.s = sv;
  call.prefix_table = prefix ? prefix_pages : nullptr;
  call.prefix_length = prefix ? prefix_length : nullptr;
  call.q = static_cast<const uint16_t*>(q);
  for (int i = 0; i < 3; ++i) call.q_stride[i] = q_strides[i];
  call.out = static_cast<uint16_t*>(out);
  call.causal = causal ? 1 : 0;
  call.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)cache->head_dim);
  call.err = device_error_word();
  if (!call.err) return set_error(BQ4_ECUDA, "device error word unavailable");
  return run_cache_attn(call, sms, workspace, stream);
}

}  // namespace
}  // namespace bq4

using namespace bq4;

extern "C" {

bq4_status bq4_cache_sizes(const bq4_cache* cache, size_t* values_bytes, size_t* scales_bytes) {
  bq4_status st = check_geometry(cache);
  if (st) return st;
  if (!values_bytes || !scales_bytes) return set_error(BQ4_EINVAL_ARG, "values_bytes/scales_bytes is NULL");
  const CacheView v = view_of(cache);
  const size_t rows = (size_t)cache->pages * cache->kv_heads * 2 * cache->page_size;
  *values_bytes = rows * v.row_bytes;
  *scales_bytes = rows * v.nb * 2;
  return BQ4_OK;
}

bq4_status bq4_cache_append(const bq4_cache* cache, const bq4_cache_sequences* seqs, const void* k,
                            const int64_t k_strides[3], const void* v, const int64_t v_strides[3], bq4_dtype dtype,
                            int64_t tokens, bq4_stream_t stream) {
  bq4_status st = check_cache(cache);
  if (st) return st;
  AppendArgs a = {};
  st = check_seqs(cache, seqs, &a.s);
  if (st) return st;
  if (dtype != BQ4_DTYPE_F32 && dtype != BQ4_DTYPE_F16)
    return set_error(BQ4_EINVAL_ARG, "dtype %d is not BQ4_DTYPE_F32/F16", (int)dtype);
  if (tokens < 0) return set_error(BQ4_EINVAL_SHAPE, "tokens=%lld", (long long)tokens);
  int64_t rows = 0;
  if (!row_count(seqs->batch, tokens, cache->kv_heads, &rows))
    return set_error(BQ4_EINVAL_SHAPE, "batch * tokens * kv_heads must be below 2^31");
  if (rows == 0) return BQ4_OK;
  if (!k || !v || !k_strides || !v_strides) return set_error(BQ4_EINVAL_ARG, "k/v or their strides are NULL");
  const int es = dtype == BQ4_DTYPE_F16 ? 2 : 4;
  if (!al(k, es) || !al(v, es)) return set_error(BQ4_EALIGN, "k/v misaligned");
  st = device_ready(cache->device);
  if (st) return st;
  Guard guard(cache->device);
  a.c = view_of(cache);
  a.x[0] = k;
  a.x[1] = v;
  for (int i = 0; i < 3; ++i) {
    a.stride[0][i] = k_strides[i];
    a.stride[1][i] = v_strides[i];
  }
  a.vec = strides_vec(k, k_strides, es) && strides_vec(v, v_strides, es);
  a.tokens = (int)tokens;
  a.rows = (unsigned)rows;
  a.err = device_error_word();
  if (!a.err) return set_error(BQ4_ECUDA, "device error word unavailable");
  const int per = kCThreads / (a.c.hp / 4);
  const dim3 grid((unsigned)((rows + per - 1) / per), 2);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (cache->format == BQ4_CACHE_F16)
    launch_append<BQ4_CACHE_F16>(a, es == 2, grid, s);
  else if (cache->format == BQ4_CACHE_Q8)
    launch_append<BQ4_CACHE_Q8>(a, es == 2, grid, s);
  else
    launch_append<BQ4_CACHE_Q4>(a, es == 2, grid, s);
  note_launch();
  return check_cuda(cudaGetLastError(), "cache append launch");
}

bq4_status bq4_cache_read(const bq4_cache* cache, const bq4_cache_sequences* seqs, const int32_t* starts,
                          int64_t count, void* k_out, void* v_out, const int64_t strides[3], bq4_dtype dtype,
                          bq4_stream_t stream) {
  bq4_status st = check_cache(cache);
  if (st) return st;
  ReadArgs a = {};
  st = check_seqs(cache, seqs, &a.s);
  if (st) return st;
  if (dtype != BQ4_DTYPE_F32 && dtype != BQ4_DTYPE_F16)
    return set_error(BQ4_EINVAL_ARG, "dtype %d is not BQ4_DTYPE_F32/F16", (int)dtype);
  if (count < 0) return set_error(BQ4_EINVAL_SHAPE, "count=%lld", (long long)count);
  int64_t rows = 0;
  if (!row_count(seqs->batch, count, cache->kv_heads, &rows))
    return set_error(BQ4_EINVAL_SHAPE, "batch * count * kv_heads must be below 2^31");
  if (rows == 0) return BQ4_OK;
  if (!k_out || !v_out || !strides) return set_error(BQ4_EINVAL_ARG, "k_out/v_out/strides is NULL");
  const int es = dtype == BQ4_DTYPE_F16 ? 2 : 4;
  if (!al(k_out, es) || !al(v_out, es) || !al(starts, 4))
    return set_error(BQ4_EALIGN, "k_out/v_out/starts misaligned");
  st = device_ready(cache->device);
  if (st) return st;
  Guard guard(cache->device);
  a.c = view_of(cache);
  a.starts = starts;
  a.out[0] = k_out;
  a.out[1] = v_out;
  for (int i = 0; i < 3; ++i) a.stride[i] = strides[i];
  a.vec = strides_vec(k_out, strides, es) && strides_vec(v_out, strides, es);
  a.count = (int)count;
  a.rows = (unsigned)rows;
  a.err = device_error_word();
  if (!a.err) return set_error(BQ4_ECUDA, "device error word unavailable");
  const int per = kCThreads / (a.c.hp / 4);
  const dim3 grid((unsigned)((rows + per - 1) / per), 2);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (cache->format == BQ4_CACHE_F16)
    launch_read<BQ4_CACHE_F16>(a, es == 2, grid, s);
  else if (cache->format == BQ4_CACHE_Q8)
    launch_read<BQ4_CACHE_Q8>(a, es == 2, grid, s);
  else
    launch_read<BQ4_CACHE_Q4>(a, es == 2, grid, s);
  note_launch();
  return check_cuda(cudaGetLastError(), "cache read launch");
}

bq4_status bq4_cache_attention_workspace_size(const bq4_cache* cache, int64_t batch, int64_t tokens, int64_t q_heads,
                                              int64_t max_length, int64_t max_prefix, size_t* bytes) {
  bq4_status st = check_geometry(cache);
  if (st) return st;
  if (!bytes) return set_error(BQ4_EINVAL_ARG, "bytes is NULL");
  *bytes = 0;
  CacheAttnCall call = {};
  st = attention_shape(cache, batch, tokens, q_heads, max_length, max_prefix, &call);
  if (st) return st;
  if (batch == 0 || tokens == 0) return BQ4_OK;
  st = device_ready(cache->device);
  if (st) return st;
  return cache_attn_workspace(call, device_sm_count(cache->device), bytes);
}

bq4_status bq4_cache_attention(const bq4_cache* cache, const bq4_cache_sequences* seqs, int64_t max_length,
                               const void* q, const int64_t q_strides[3], int64_t tokens, int64_t q_heads,
                               int32_t causal, float scale, void* out, void* workspace, size_t workspace_bytes,
                               bq4_stream_t stream) {
  return attention(cache, nullptr, 0, nullptr, false, seqs, max_length, q, q_strides, tokens, q_heads, causal, scale,
                   out, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

bq4_status bq4_cache_prefix_attention(const bq4_cache* cache, const int32_t* prefix_pages, int64_t prefix_width,
                                      const int32_t* prefix_length, const bq4_cache_sequences* seqs,
                                      int64_t max_length, const void* q, const int64_t q_strides[3], int64_t tokens,
                                      int64_t q_heads, int32_t causal, float scale, void* out, void* workspace,
                                      size_t workspace_bytes, bq4_stream_t stream) {
  return attention(cache, prefix_pages, prefix_width, prefix_length, true, seqs, max_length, q, q_strides, tokens,
                   q_heads, causal, scale, out, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
