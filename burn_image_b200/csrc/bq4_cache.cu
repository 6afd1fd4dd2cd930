// bq4_cache.cu -- the paged key/value cache: rows quantised as they are
// written, rows read back, and the host entry points of the cache (the
// attention kernels are in bq4_cache_attn.cu).
//
// Both kernels move each byte once and compute next to nothing, so HBM (and,
// for a decode step's few rows, the launch) bounds them: 8 x 4352 rows of 8 kv
// heads, 8 bits to f16, are read in 43.5 us (211 MB, 4.9 TB/s, 0.74 of the copy
// rate); 4352 f32 rows are written in 4 bits in 14.1 us (41 MB; some 110
// instructions a row for two roundings and the packing); a decode step of 32
// sequences takes 3.0 us to write and 2.3 to read back, an empty launch 1.4.
// A warp takes 2 to 16 neighbouring positions of one page, for one head's k or
// v, as many as it loads before it uses the first: page, row and sequence are
// worked out once for them.  A row of HP values is taken by HP / W lanes, W
// consecutive values each: 8 when they are written (what a block's maximum and
// scale cost is shared by fewer lanes then; f32 rows 18.7 -> 15.9 us against 4),
// 16 bytes when they are read.  Block maxima come from shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>

#include "bq4_cache.h"

namespace bq4 {
namespace {

constexpr int kCThreads = 256;

struct CacheRow {
  uint8_t* rows;     // k or v rows of the step
  uint16_t* scales;  // of its row at `place`
};

// Rows of the step of (page, head) that holds `place`; kv: 0 k, 1 v.  The next row's
// scales lie 2 nb on.
__device__ __forceinline__ CacheRow cache_row(const CacheView& c, int page, int head, int place, int kv) {
  uint8_t* step = cache_step(c, page, head, place);
  CacheRow r;
  r.rows = step + kv * 16 * c.row_bytes;
  r.scales = reinterpret_cast<uint16_t*>(step + 32 * c.row_bytes) + ((place & 15) * 2 + kv) * c.nb;
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

// kW consecutive values at element `at`, in f32; vec: they lie on 16 bytes.
template <bool kF16, int kW>
__device__ __forceinline__ void load_values(const void* base, int64_t at, bool vec, float (&x)[kW]) {
  if constexpr (kF16) {
    const __half* p = static_cast<const __half*>(base) + at;
    if (vec) {
      uint32_t u[kW / 2];
      if constexpr (kW == 8)
        *reinterpret_cast<uint4*>(u) = __ldg(reinterpret_cast<const uint4*>(p));
      else
        *reinterpret_cast<uint2*>(u) = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
      for (int j = 0; j < kW / 2; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
        x[2 * j] = f.x, x[2 * j + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kW; ++j) x[j] = __half2float(p[j]);
    }
  } else {
    const float* p = static_cast<const float*>(base) + at;
    if (vec) {
#pragma unroll
      for (int j = 0; j < kW; j += 4) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(p + j));
        x[j] = u.x, x[j + 1] = u.y, x[j + 2] = u.z, x[j + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kW; ++j) x[j] = p[j];
    }
  }
}

// n bytes (2, 4, 8 or 16) of packed words.
template <int kBytes>
__device__ __forceinline__ void store_words(uint8_t* dst, const uint32_t* w) {
  if constexpr (kBytes == 2)
    *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w[0];
  else if constexpr (kBytes == 4)
    *reinterpret_cast<uint32_t*>(dst) = w[0];
  else if constexpr (kBytes == 8)
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <int kBytes>
__device__ __forceinline__ void load_words(const uint8_t* src, uint32_t* w) {
  if constexpr (kBytes == 2)
    w[0] = *reinterpret_cast<const uint16_t*>(src);
  else if constexpr (kBytes == 4)
    w[0] = *reinterpret_cast<const uint32_t*>(src);
  else if constexpr (kBytes == 8)
    *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(src);
  else
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(src);
}

// How a warp of the append and of the read kernel (kF16: of f16 rows) takes
// rows: kW values a lane, kLanes lanes a row, kPer rows at a time, kTake in all.
template <int kHP, bool kMany>
struct TakeAppend {
  static constexpr int kW = 8, kLanes = kHP / kW, kPer = 32 / kLanes, kRounds = !kMany ? 1 : kPer < 4 ? 4 : 2;
  static constexpr int kTake = kPer * kRounds;
};
template <bool kF16, int kHP, bool kMany>
struct TakeRead {
  static constexpr int kW = kF16 ? 8 : 4, kLanes = kHP / kW, kPer = 32 / kLanes;
  static constexpr int kRounds = !kMany ? 2 : kPer < 4 ? 8 : 4;
  static constexpr int kTake = kPer * kRounds;
};
// Calls of more rows than this (k and v, of all heads) take kMany: 8 rounds a warp
// read 557056 rows of 8 bits in 43.5 us (4: 45.2, 2: 51.9), 2 rounds the 512 of a
// decode step in 2.3 (4: 2.8, 8: 3.2); 1 round a warp writes 2590 in 3.0 us (4: 4.3).
// Around the switch, few / many in us, f16 rows of 128: 8 bits written 4096 rows
// 3.3 / 5.4, 8192 3.9 / 5.5, 16384 5.9 / 6.2, 32768 8.9 / 8.2, read 2.5 / 3.4, 2.7 / 3.5,
// 3.6 / 3.5, 4.8 / 4.4; 4 bits written 3.2 / 5.7, 4.0 / 5.8, 6.0 / 6.4, 9.3 / 10.6, read
// 2.8 / 4.9, 3.0 / 4.8, 3.9 / 5.0, 6.0 / 6.0; f16 written 2.4 / 3.2, 2.9 / 3.3, 3.8 / 3.7,
// 5.9 / 4.6, read 2.4 / 3.2, 2.6 / 3.2, 3.1 / 3.3, 4.2 / 4.0.
constexpr int64_t kManyRows = 16384;

struct AppendArgs {
  CacheView c;
  SeqView s;
  const void* x[2];       // k, v
  int64_t stride[2][3];   // batch, token, head
  int vec;                // every row of x lies on 16 bytes
  int tokens, steps;      // steps: the most warps that a sequence's new rows of a head take
  unsigned items;         // batch * steps * kv_heads * 2
  int* err;
};

__device__ __forceinline__ int page_of(const CacheView& c, const SeqView& s, int b, int base, int* place, int* err) {
  const int pi = base / c.page_size;
  const int page = s.table[b * s.table_stride + pi];
  *place = base - pi * c.page_size;
  if (page >= 0 && page < c.pages) return page;
  atomicCAS(err, 0, (int)BQ4_EINVAL_ARG);
  return -1;
}

template <int kFmt, bool kF16, int kHP, bool kMany>
__global__ void __launch_bounds__(kCThreads) cache_append_kernel(const __grid_constant__ AppendArgs a) {
  using T = TakeAppend<kHP, kMany>;
  constexpr int kW = T::kW, kLanes = T::kLanes, kPer = T::kPer, kAhead = T::kRounds, kTake = T::kTake;
  constexpr int kRow = kFmt == BQ4_CACHE_F16 ? 2 * kHP : kFmt == BQ4_CACHE_Q8 ? kHP : kHP / 2;
  constexpr int kNb = kFmt == BQ4_CACHE_Q8 ? 1 : kHP / kCacheBlock;
  const int lane = threadIdx.x & 31, L = lane % kLanes, sub = lane / kLanes, d0 = kW * L;
  unsigned item = blockIdx.x * (kCThreads / 32) + (threadIdx.x >> 5);
  if (item >= a.items) return;
  // kv, then head, fastest: neighbouring warps read neighbouring rows
  const int kv = item & 1;
  item >>= 1;
  const int head = (int)(item % (unsigned)a.c.kv_heads);
  item /= (unsigned)a.c.kv_heads;
  const int b = (int)(item / (unsigned)a.steps), step = (int)(item - (unsigned)b * a.steps);
  const int end = seq_length(a.s, a.c.page_size, b, a.err), from = end - a.tokens, first = max(from, 0);
  const int aligned = first & ~(kTake - 1);
  if (step >= (end - aligned + kTake - 1) / kTake) return;  // (the last of 2^31 tokens' steps pass an int)
  const int base = aligned + kTake * step;
  int place0;
  const int page = page_of(a.c, a.s, b, base, &place0, a.err);
  if (page < 0) return;
  const CacheRow r = cache_row(a.c, page, head, place0, kv);
  const int64_t src = b * a.stride[kv][0] + head * a.stride[kv][2] + d0;

  {
    float xs[kAhead][kW];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int pos = base + j * kPer + sub;
#pragma unroll
      for (int e = 0; e < kW; ++e) xs[j][e] = 0.0f;
      if (pos >= first && pos < end && d0 < a.c.head_dim)
        load_values<kF16, kW>(a.x[kv], src + (int64_t)(pos - from) * a.stride[kv][1], a.vec, xs[j]);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int row = j * kPer + sub;
      const bool live = base + row >= first && base + row < end;
      if (!__any_sync(0xffffffffu, live)) continue;
      float(&x)[kW] = xs[j];
      auto dst = [&](int at) { return r.rows + cache_swizzle(kv, kRow, (place0 & 15) + row, at); };
      uint16_t* sc = r.scales + row * 2 * kNb;
      if constexpr (kFmt == BQ4_CACHE_F16) {
        uint32_t w[kW / 2];
#pragma unroll
        for (int e = 0; e < kW / 2; ++e) {
          const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
          w[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if (live) store_words<2 * kW>(dst(2 * d0), w);
      } else {
        constexpr float kTop = kFmt == BQ4_CACHE_Q8 ? 127.0f : 7.0f;
        // magnitudes as their bits, which order like them, infinities and NaN on top
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < kW; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
        for (int o = (kFmt == BQ4_CACHE_Q8 ? kLanes : kCacheBlock / kW) >> 1; o; o >>= 1)
          most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        // f32 quotients, rounded to nearest: the scale and every q follow from the
        // definition bit for bit.
        const float top = __uint_as_float(most);
        const __nv_bfloat16 sb =
            __float2bfloat16_rn(most >= 0x7f800000u ? __int_as_float(0x7fc00000) : __fdiv_rn(top, kTop));
        const float s = __bfloat162float(sb);
        // x (1 / s) is the quotient but for 2^-23 of the inverse and two roundings, 2^-22 in all of
        // at most kTop (1 + 2^-9): where it lies 2^-14 or more from a half, both round to the same
        // whole number, which needs no clamping.  The divisions are left for a lane that holds
        // another one, and for scales whose inverse is not normal.  y + 1.5 2^23 rounds y to a
        // whole number in the low bits of the sum.
        constexpr float kRound = 12582912.0f;
        constexpr uint32_t kZero = kFmt == BQ4_CACHE_Q8 ? 128 : 8;
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        if (!(s > 0.0f)) inv = 0.0f;
        uint32_t q[kW];  // u = q + 128 or q + 8
        float far = s > 0.0f && !(s >= 0x1p-120f && s <= 0x1p120f) ? 1.0f : 0.0f;
#pragma unroll
        for (int e = 0; e < kW; ++e) {
          const float y = x[e] * inv, t = y + kRound;
          q[e] = __float_as_uint(t) - (__float_as_uint(kRound) - kZero);
          far = fmaxf(far, fabsf(y - (t - kRound)));
        }
        if (far > 0.5f - 0x1p-14f) {
#pragma unroll
          for (int e = 0; e < kW; ++e)
            q[e] = (uint32_t)((int)fminf(fmaxf(rintf(__fdiv_rn(x[e], s)), -kTop), kTop) + (int)kZero);
        }
        if (!(s > 0.0f)) {  // a scale of 0, or NaN
#pragma unroll
          for (int e = 0; e < kW; ++e) q[e] = kZero;
        }
        if constexpr (kFmt == BQ4_CACHE_Q8) {
          uint32_t w[kW / 4];
#pragma unroll
          for (int e = 0; e < kW / 4; ++e)
            w[e] = q[4 * e] | q[4 * e + 1] << 8 | q[4 * e + 2] << 16 | q[4 * e + 3] << 24;
          if (live) {
            store_words<kW>(dst(d0), w);
            if (L == 0) sc[0] = __bfloat16_as_ushort(sb);
          }
        } else {
          const int blk = d0 >> 5;
          if (kv == 0) {
            // value o of the 8 of a word: nibble o / 2 + 4 (o & 1)
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < kW; ++e) w |= q[e] << (4 * (e >> 1) + 16 * (e & 1));
            if (live) store_words<4>(dst(4 * (((d0 >> 3) & 3) * kNb + blk)), &w);
          } else {
#pragma unroll
            for (int e = 0; e < kW; e += 4) {
              const uint32_t w = q[e] | q[e + 1] << 4 | q[e + 2] << 8 | q[e + 3] << 12;
              if (live) store_words<2>(dst(2 * ((((d0 + e) >> 2) & 7) * kNb + blk)), &w);
            }
          }
          if (live && (d0 & 31) == 0) sc[blk] = __bfloat16_as_ushort(sb);
        }
      }
    }
  }
}

struct ReadArgs {
  CacheView c;
  SeqView s;
  const int32_t* starts;
  void* out[2];
  int64_t stride[3];      // batch, head, position
  int vec;                // every row of out lies on 16 bytes
  int count, steps;       // steps: the most warps that `count` positions of a head take
  unsigned items;         // batch * kv_heads * 2 * steps
  int* err;
};

template <int kFmt, bool kF16, int kHP, bool kMany>
__global__ void __launch_bounds__(kCThreads) cache_read_kernel(const __grid_constant__ ReadArgs a) {
  using T = TakeRead<kF16, kHP, kMany>;
  constexpr int kW = T::kW, kLanes = T::kLanes, kPer = T::kPer, kAhead = T::kRounds, kTake = T::kTake;
  constexpr int kRow = kFmt == BQ4_CACHE_F16 ? 2 * kHP : kFmt == BQ4_CACHE_Q8 ? kHP : kHP / 2;
  constexpr int kNb = kFmt == BQ4_CACHE_Q8 ? 1 : kHP / kCacheBlock;
  constexpr int kHeld = kFmt == BQ4_CACHE_F16 ? 2 * kW : kFmt == BQ4_CACHE_Q8 ? kW : kW / 2;  // bytes of kW values
  constexpr int kWords = kHeld < 4 ? 1 : kHeld / 4;
  const int lane = threadIdx.x & 31, L = lane % kLanes, sub = lane / kLanes, d0 = kW * L;
  unsigned item = blockIdx.x * (kCThreads / 32) + (threadIdx.x >> 5);
  if (item >= a.items) return;
  const int step = (int)(item % (unsigned)a.steps);
  item /= (unsigned)a.steps;
  const int kv = item & 1;
  item >>= 1;
  const int b = (int)(item / (unsigned)a.c.kv_heads), head = (int)(item - (unsigned)b * a.c.kv_heads);
  const int64_t start = a.starts ? (int64_t)a.starts[b] : 0;
  const int64_t base = (start & ~(int64_t)(kTake - 1)) + (int64_t)kTake * step, to = start + a.count;
  if (base >= to) return;
  const int end = seq_length(a.s, a.c.page_size, b, a.err);
  int place0 = 0, page = -1;
  if (base >= 0 && base < end) page = page_of(a.c, a.s, b, (int)base, &place0, a.err);
  const CacheRow r = cache_row(a.c, max(page, 0), head, place0, kv);
  const int64_t dst = b * a.stride[0] + head * a.stride[1] + (base - start) * a.stride[2] + d0;

  {
    uint32_t held[kAhead][kWords];
    uint32_t scale[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int row = j * kPer + sub;
      const bool live = page >= 0 && base + row < end;
#pragma unroll
      for (int e = 0; e < kWords; ++e) held[j][e] = 0;
      scale[j] = 0;
      if (live) {
        auto src = [&](int at) { return r.rows + cache_swizzle(kv, kRow, (place0 & 15) + row, at); };
        const uint16_t* sc = r.scales + row * 2 * kNb;
        if constexpr (kFmt == BQ4_CACHE_F16) {
          load_words<kHeld>(src(2 * d0), held[j]);
        } else if constexpr (kFmt == BQ4_CACHE_Q8) {
          load_words<kHeld>(src(d0), held[j]);
          scale[j] = sc[0];
        } else {
          const int blk = d0 >> 5;
          scale[j] = sc[blk];
          if (kv == 0) {
            load_words<4>(src(4 * (((d0 >> 3) & 3) * kNb + blk)), held[j]);
          } else {
#pragma unroll
            for (int e = 0; e < kW; e += 4) {
              uint32_t w;
              load_words<2>(src(2 * ((((d0 + e) >> 2) & 7) * kNb + blk)), &w);
              held[j][0] |= w << 4 * e;
            }
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int row = j * kPer + sub;
      const float s = __uint_as_float(scale[j] << 16);
      float x[kW];
#pragma unroll
      for (int e = 0; e < kW; ++e) {
        if constexpr (kFmt == BQ4_CACHE_F16) {
          x[e] = __half2float(__ushort_as_half((unsigned short)(held[j][e >> 1] >> 16 * (e & 1))));
        } else if constexpr (kFmt == BQ4_CACHE_Q8) {
          // byte u under the exponent of 2^23: 2^23 + u, exactly
          x[e] = (__uint_as_float(__byte_perm(held[j][e >> 2], 0x4b000000u, 0x7540 + (e & 3))) - 8388736.0f) * s;
        } else {
          const int o = kW == 4 ? 4 * (L & 1) + e : e;
          const int nibble = kv == 0 ? 4 * (o >> 1) + 16 * (o & 1) : 4 * e;
          x[e] = (__uint_as_float((held[j][0] >> nibble & 15) | 0x4b000000u) - 8388616.0f) * s;
        }
      }
      const bool live = page >= 0 && base + row < end;
      if (kFmt != BQ4_CACHE_F16 && !live) {  // the zero words stand for -128 (-8) and a scale of 0: make it +0
#pragma unroll
        for (int e = 0; e < kW; ++e) x[e] = 0.0f;
      }
      if (base + row < start || base + row >= to || d0 >= a.c.head_dim) continue;
      const int64_t at = dst + (int64_t)row * a.stride[2];
      if constexpr (kF16) {
        uint32_t w[kW / 2];
#pragma unroll
        for (int e = 0; e < kW / 2; ++e) {
          const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
          w[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        __half* o = static_cast<__half*>(a.out[kv]) + at;
        if (a.vec) {
          store_words<16>(reinterpret_cast<uint8_t*>(o), w);
        } else {
#pragma unroll
          for (int e = 0; e < kW; ++e) o[e] = __ushort_as_half((unsigned short)(w[e >> 1] >> 16 * (e & 1)));
        }
      } else {
        float* o = static_cast<float*>(a.out[kv]) + at;
        if (a.vec) {
          *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
          for (int e = 0; e < kW; ++e) o[e] = x[e];
        }
      }
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
  v.data = static_cast<uint8_t*>(c->data);
  v.pages = (int32_t)c->pages;
  v.page_size = c->page_size;
  v.kv_heads = c->kv_heads;
  v.head_dim = c->head_dim;
  v.hp = cache_hp(c->head_dim);
  v.nb = cache_nb(c->format, v.hp);
  v.row_bytes = cache_row_bytes(c->format, v.hp);
  v.format = c->format;
  v.step_bytes = cache_step_bytes(v.row_bytes, v.nb);
  return v;
}

bq4_status check_cache(const bq4_cache* c) {
  bq4_status st = check_geometry(c);
  if (st) return st;
  if (!c->data) return set_error(BQ4_EINVAL_ARG, "the cache's data is NULL");
  if (!al(c->data, 256)) return set_error(BQ4_EALIGN, "the cache's data must be 256-byte aligned");
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
  static std::atomic<uint64_t> ready{0};  // a bit for each device found fit before
  if (device >= 0 && device < 64 && ready.load(std::memory_order_relaxed) >> device & 1) return BQ4_OK;
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
    cudaGetLastError();
    return set_error(BQ4_EINVAL_ARG, "device %d not present", device);
  }
  if (!device_is_sm100(device))
    return set_error(BQ4_EUNSUPPORTED, "device %d is not sm_100 (B200); libbq4 has no kernels for it", device);
  if (device < 64) ready.fetch_or(1ull << device, std::memory_order_relaxed);
  return BQ4_OK;
}

bool strides_vec(const void* base, const int64_t* st, int esize) {
  const int64_t n = 16 / esize;
  return al(base, 16) && st[0] % n == 0 && st[1] % n == 0 && st[2] % n == 0;
}

// Launches; false: too many warps for one.
template <int kFmt, bool kF16, int kHP, bool kMany>
bool launch_append(AppendArgs& a, int64_t batch, cudaStream_t s) {
  constexpr int kTake = TakeAppend<kHP, kMany>::kTake;
  a.steps = (int)(((int64_t)a.tokens + 2 * kTake - 2) / kTake);
  int64_t items = 0;
  if (!row_count(2 * batch, a.steps, a.c.kv_heads, &items)) return false;
  a.items = (unsigned)items;
  const unsigned grid = (unsigned)((items + kCThreads / 32 - 1) / (kCThreads / 32));
  cache_append_kernel<kFmt, kF16, kHP, kMany><<<grid, kCThreads, 0, s>>>(a);
  return true;
}
template <int kFmt, bool kF16, int kHP>
bool launch_append(AppendArgs& a, int64_t batch, cudaStream_t s) {
  return 2 * batch * a.tokens * a.c.kv_heads > kManyRows ? launch_append<kFmt, kF16, kHP, true>(a, batch, s)
                                                         : launch_append<kFmt, kF16, kHP, false>(a, batch, s);
}
template <int kFmt>
bool launch_append(AppendArgs& a, bool f16, int64_t batch, cudaStream_t s) {
  if (a.c.hp == 64)
    return f16 ? launch_append<kFmt, true, 64>(a, batch, s) : launch_append<kFmt, false, 64>(a, batch, s);
  return f16 ? launch_append<kFmt, true, 128>(a, batch, s) : launch_append<kFmt, false, 128>(a, batch, s);
}

template <int kFmt, bool kF16, int kHP, bool kMany>
bool launch_read(ReadArgs& a, int64_t batch, int64_t count, cudaStream_t s) {
  constexpr int kTake = TakeRead<kF16, kHP, kMany>::kTake;
  a.steps = (int)((count + 2 * kTake - 2) / kTake);
  int64_t items = 0;
  if (!row_count(2 * batch, a.steps, a.c.kv_heads, &items)) return false;
  a.items = (unsigned)items;
  const unsigned grid = (unsigned)((items + kCThreads / 32 - 1) / (kCThreads / 32));
  cache_read_kernel<kFmt, kF16, kHP, kMany><<<grid, kCThreads, 0, s>>>(a);
  return true;
}
template <int kFmt, bool kF16, int kHP>
bool launch_read(ReadArgs& a, int64_t batch, int64_t count, cudaStream_t s) {
  return 2 * batch * count * a.c.kv_heads > kManyRows ? launch_read<kFmt, kF16, kHP, true>(a, batch, count, s)
                                                      : launch_read<kFmt, kF16, kHP, false>(a, batch, count, s);
}
template <int kFmt>
bool launch_read(ReadArgs& a, bool f16, int64_t batch, int64_t count, cudaStream_t s) {
  if (a.c.hp == 64)
    return f16 ? launch_read<kFmt, true, 64>(a, batch, count, s) : launch_read<kFmt, false, 64>(a, batch, count, s);
  return f16 ? launch_read<kFmt, true, 128>(a, batch, count, s) : launch_read<kFmt, false, 128>(a, batch, count, s);
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
  if (!(scale <= 3.402823466e38f)) return set_error(BQ4_EINVAL_ARG, "scale is NaN or infinite");
  st = device_ready(cache->device);
  if (st) return st;
  Guard guard(cache->device);
  const int sms = device_sm_count(cache->device);
  call.s = sv;
  call.bounded = max_length > 0;
  call.prefix_table = prefix ? prefix_pages : nullptr;
  call.prefix_length = prefix ? prefix_length : nullptr;
  call.q = static_cast<const uint16_t*>(q);
  for (int i = 0; i < 3; ++i) call.q_stride[i] = q_strides[i];
  call.out = static_cast<uint16_t*>(out);
  call.causal = causal ? 1 : 0;
  call.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)cache->head_dim);
  call.err = device_error_word();
  if (!call.err) return set_error(BQ4_ECUDA, "device error word unavailable");
  return run_cache_attn(call, sms, workspace, workspace_bytes, stream);
}

}  // namespace
}  // namespace bq4

using namespace bq4;

extern "C" {

bq4_status bq4_cache_size(const bq4_cache* cache, size_t* bytes) {
  bq4_status st = check_geometry(cache);
  if (st) return st;
  if (!bytes) return set_error(BQ4_EINVAL_ARG, "bytes is NULL");
  *bytes = (size_t)cache->pages * cache->kv_heads * (cache->page_size / kCachePageUnit) * view_of(cache).step_bytes;
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
  a.err = device_error_word();
  if (!a.err) return set_error(BQ4_ECUDA, "device error word unavailable");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool ok = cache->format == BQ4_CACHE_F16  ? launch_append<BQ4_CACHE_F16>(a, es == 2, seqs->batch, s)
                  : cache->format == BQ4_CACHE_Q8 ? launch_append<BQ4_CACHE_Q8>(a, es == 2, seqs->batch, s)
                                                  : launch_append<BQ4_CACHE_Q4>(a, es == 2, seqs->batch, s);
  if (!ok) return set_error(BQ4_EINVAL_SHAPE, "batch * tokens * kv_heads too large for one launch");
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
  a.err = device_error_word();
  if (!a.err) return set_error(BQ4_ECUDA, "device error word unavailable");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool ok = cache->format == BQ4_CACHE_F16  ? launch_read<BQ4_CACHE_F16>(a, es == 2, seqs->batch, count, s)
                  : cache->format == BQ4_CACHE_Q8 ? launch_read<BQ4_CACHE_Q8>(a, es == 2, seqs->batch, count, s)
                                                  : launch_read<BQ4_CACHE_Q4>(a, es == 2, seqs->batch, count, s);
  if (!ok) return set_error(BQ4_EINVAL_SHAPE, "batch * count * kv_heads too large for one launch");
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
  const bool bounded = max_length >= 0;
  if (max_length < -((int64_t)1 << 30)) return set_error(BQ4_EINVAL_SHAPE, "max_length=%lld", (long long)max_length);
  st = attention_shape(cache, batch, tokens, q_heads, bounded ? max_length : -max_length, max_prefix, &call);
  if (st) return st;
  call.bounded = bounded;
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
