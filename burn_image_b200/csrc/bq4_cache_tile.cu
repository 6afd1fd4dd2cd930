// bq4_cache_tile.cu -- attention over the key/value cache for many query rows
// a kv head (a chunk of a prompt, or a large batch behind a shared prefix).
//
// With hundreds of rows on the same keys the products dominate, and every
// CTA of rows would widen the same cache rows again.  So the rows of the cache
// are widened once (cache_widen_kernel), into records of 128 keys laid out as
// the tensor core reads them, and cache_tile_kernel runs the two products of
// 256 query rows a CTA on tcgen05 with scores, P and O in TMEM.
//
// A record of one (key set, kv head, 128 keys):
//   k tile  [hp / 64][128 keys][64] f16, 128-byte swizzle: whole numbers q
//           (8 bits), q s_b / s (4 bits: s the power of two above the row's
//           scales, the product has 11 bits and is exact), or the rows (f16);
//   v tile  [2][hp][64 keys] f16 (transposed), 128-byte swizzle: q s_v 2^-e,
//           rounded once (2^-11 of it; exact for 4 bits and f16), with the key's own
//           e, 0 unless its v pass 2^15 (one of a whole record would take the others'
//           bits, of rows that do not see that key too);
//   consts  per key the factor ck that turns its raw score into log2 units (s_k,
//           s or 1, times scale log2(e)), lv = e, or -inf for a row that does
//           not exist, and w = 2^-e; whether some lv is not 0 and some e is not.
//           (k rounded to f16 instead, without a factor a score, gained 7 %: not
//           worth its error.)
// A v value that is not finite would carry 0 * NaN into the rows that do not see
// it.  It is stored as 0 and its key marked: the rows that see the key take it from
// the cache at their end.  (A row of 8 bits has one scale: its key gets ck = NaN,
// as one of a k that is not finite does.)
//
// cache_tile_kernel, one CTA for 256 rows and a range of records:
//   warp 0        bulk copies of the records (2 stages), q tiles once
//   warp 1        S_t = q_t k^T and O_t += P_t v for the two 128-row tiles in
//                 turn, so that one tile's softmax runs beside the other's products
//   warps 4..11   a thread a row: y = S ck (+ lv), p = 2^(y - m) as f16 into
//                 TMEM, l += p (w); O is rescaled only when some p would
//                 pass 2^14
// Every wait is bounded (BQ4_ETIMEOUT), as in bq4_attn_fused.cu.
//
// What bounds it: the softmax threads' chain from S to P.  A 512-token chunk of 32
// / 8 heads on 8704 rows of 8 bits takes 113 us (widening 13, products 92, join
// 8 with its start hidden): 71 GFLOP, 0.37 of the bf16 peak; a record of 256 rows
// takes 2.6 us, 1.5 at the peak.  Not tried: widening in this kernel, from raw rows
// beside the operand stages (32,448 bytes are free; a record's 128 raw tokens take
// 18,432 in 4 bits and 33,280 in 8, which the consts' addends and weights would have
// to make room for).  Tried: two threads a row
// (their exchange and the registers that it costs: 152 us), a row's 128 scores
// in registers (spilled), equal shares of all records for every CTA instead of
// halves of a range on 128 of 148 SMs (113 to 118 us; 103 against 99 us behind
// a shared prefix, for the second piece's start).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "attn_tile.cuh"
#include "bq4_cache.h"
#include "sm100_ptx.cuh"

namespace bq4 {
namespace {

constexpr int kKeys = 128;                   // keys of a record
constexpr int kTThreads = 384;
constexpr int kRing = 2;                     // stages of k and of v
constexpr uint32_t kConsts = kKeys * 12 + 32;  // bytes of a record's consts
constexpr float kTNone = -1e30f;             // the maximum of no score
// log2 units: m is set 2^6 below the maximum and moves when p would pass 2^14, so
// that f16 holds p to its 2^-11 down to 2^-20 of the row's largest (a small p
// may meet a large v)
constexpr float kTHead = 6.0f, kTJump = 14.0f;

struct Consts {
  float ck[kKeys], lv[kKeys], w[kKeys];
  unsigned odd[4];  // a bit for each key with a v value that is not finite
  int flags;        // 1: some lv is not 0; 2: some e is not; 4: some bit of odd is set
  int pad[3];
};
static_assert(sizeof(Consts) == kConsts, "a record's consts are copied in 16-byte units");

struct TileArgs {
  CacheAttnCall a;
  float c;            // scale * log2(e)
  int group;
  int prefix;         // the key set is the prefix and the rows are the whole batch's
  int sets;           // key sets: 1 or the batch
  int tiles;          // 256-row tiles of a set
  int blocks;         // records of a set and kv head, at most
  int span, chunks;   // records of a chunk; chunks of a tile, at most
  int q_vec;          // q rows lie on 16 bytes
  int finish;         // one chunk and no other source: rows are finished here
  uint64_t page_magic;  // floor(u / (page_size / 16)) = u * page_magic >> 38
  uint8_t* k;         // [sets][kv_heads][blocks] tiles
  uint8_t* v;
  Consts* consts;
  uint8_t* q;         // [sets][kv_heads][2 tiles][128 rows] tiles
  float* part;        // [sets][tiles][kv_heads][chunks][256][hp]
  float2* ml;         // m, l likewise
};

__device__ __forceinline__ int set_length(const TileArgs& s, int set, int* err) {
  const int64_t cap = s.prefix ? (int64_t)s.a.prefix_width * s.a.c.page_size
                               : min((int64_t)s.a.max_length, (int64_t)s.a.s.table_width * s.a.c.page_size);
  const int n = s.prefix ? s.a.prefix_length[0] : s.a.s.lengths[set];
  if (n >= 0 && n <= cap) return n;
  atomicCAS(err, 0, (int)BQ4_EINVAL_ARG);
  return n < 0 ? 0 : (int)cap;
}

// ---------------------------------------------------------------- widening

template <int kFmt, int kHP>
__global__ void __launch_bounds__(256) cache_widen_kernel(const __grid_constant__ TileArgs s) {
  constexpr int kRow = kFmt == BQ4_CACHE_F16 ? 2 * kHP : kFmt == BQ4_CACHE_Q8 ? kHP : kHP / 2;
  constexpr int kNb = kFmt == BQ4_CACHE_Q4 ? kHP / kCacheBlock : 1;
  constexpr int kCh = kHP / 8;                 // 16-byte pieces of a row
  constexpr int kTile = kKeys * kHP * 2;       // bytes of a k or v tile
  constexpr int kPitch = kHP + 2;              // halves; an odd number of words
  const CacheView& c = s.a.c;
  const int tid = threadIdx.x;
  const int64_t records = (int64_t)s.sets * c.kv_heads * s.blocks;
  ptx::griddep_launch_dependents();

  if (blockIdx.x >= records) {
    // ---- a q tile: 128 rows, swizzled
    const int64_t i = blockIdx.x - records;
    const int tile = (int)(i % (2 * s.tiles));
    const int64_t sh = i / (2 * s.tiles);
    const int kvh = (int)(sh % c.kv_heads), set = (int)(sh / c.kv_heads);
    const int rows = (s.prefix ? s.a.s.batch : 1) * s.a.tokens * s.group;
    uint8_t* dst = s.q + i * (128 * kHP * 2);
    for (int p = tid; p < 128 * kCh; p += 256) {
      const int r = p / kCh, ch = p % kCh;
      int row = tile * 128 + r, b = set;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (row < rows && 8 * ch < c.head_dim) {
        if (s.prefix) {
          b = row / (s.a.tokens * s.group);
          row -= b * s.a.tokens * s.group;
        }
        const int tok = row / s.group, h = kvh * s.group + row - tok * s.group;
        const uint16_t* src = s.a.q + b * s.a.q_stride[0] + tok * s.a.q_stride[1] + h * s.a.q_stride[2] + 8 * ch;
        if (s.q_vec)
          u = *reinterpret_cast<const uint4*>(src);
        else
          u = make_uint4(src[0] | (uint32_t)src[1] << 16, src[2] | (uint32_t)src[3] << 16,
                         src[4] | (uint32_t)src[5] << 16, src[6] | (uint32_t)src[7] << 16);
      }
      *reinterpret_cast<uint4*>(dst + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = u;
    }
    // this grid does not end before the one that it was launched beside
    if (blockIdx.x == gridDim.x - 1) ptx::griddep_wait();
    return;
  }

  // ---- a record
  __shared__ int64_t at[kKeys];                // byte of the key's step in the cache, -1: no such row
  __shared__ int place[kKeys];
  __shared__ float sk[kKeys][kNb], sv[kKeys][kNb], ck[kKeys];
  __shared__ unsigned flags[4], odd_v[4];
  __shared__ uint16_t vt[kKeys * kPitch];
  const int64_t rec = blockIdx.x;
  const int j = (int)(rec % s.blocks);
  const int64_t sh = rec / s.blocks;
  const int kvh = (int)(sh % c.kv_heads), set = (int)(sh / c.kv_heads);
  const int n = set_length(s, set, s.a.err);
  if (j * kKeys >= n) return;
  if (tid < kKeys) {
    const int pos = j * kKeys + tid;
    int64_t where = -1;
    float f = s.c;
    int e_v = 0;
    bool some_v = false;  // some v of the row is not finite
    if (pos < n) {
      const unsigned u = (unsigned)pos / kCachePageUnit;
      const int pi = (int)((u * s.page_magic) >> 38);
      const int page = s.prefix ? s.a.prefix_table[pi] : s.a.s.table[set * s.a.s.table_stride + pi];
      place[tid] = pos - pi * c.page_size;
      if (page >= 0 && page < c.pages) {
        const uint8_t* step = cache_step(c, page, kvh, place[tid]);
        where = step - c.data;
        if constexpr (kFmt != BQ4_CACHE_F16) {
          const uint16_t* sc = reinterpret_cast<const uint16_t*>(step + 32 * kRow) + (place[tid] & 15) * 2 * kNb;
          float ktop = 0.0f, most = 0.0f;
          bool odd = false;  // the row's scores are NaN
#pragma unroll
          for (int e = 0; e < kNb; ++e) {
            sk[tid][e] = __uint_as_float((uint32_t)sc[e] << 16);
            float w = __uint_as_float((uint32_t)sc[kNb + e] << 16);
            odd |= !(sk[tid][e] <= 3.402823466e38f);
            if (!(w <= 3.402823466e38f)) {
              w = 0.0f;
              (kFmt == BQ4_CACHE_Q8 ? odd : some_v) = true;
            }
            sv[tid][e] = w;
            ktop = fmaxf(ktop, sk[tid][e]);
            most = fmaxf(most, w);
          }
          if constexpr (kFmt == BQ4_CACHE_Q8) {
            f *= ktop;
          } else {
            // the power of two above the row's k scales (its inverse normal too)
            const float up = fminf(fmaxf(__uint_as_float((__float_as_uint(ktop) & 0x7f800000u) + 0x00800000u),
                                         0x1p-120f), 0x1p120f);
            f *= up;
#pragma unroll
            for (int e = 0; e < kNb; ++e) sk[tid][e] = odd ? 0.0f : sk[tid][e] * (1.0f / up);
          }
          if (odd) f = __int_as_float(0x7fc00000);
          // |v| < 2^15 after the factor 2^-e
          most *= kFmt == BQ4_CACHE_Q8 ? 127.0f : 7.0f;
          if (most >= 0x1p15f) e_v = min((int)(__float_as_uint(most) >> 23) - 127 + 1 - 15, 120);
#pragma unroll
          for (int e = 0; e < kNb; ++e) sv[tid][e] *= __uint_as_float((uint32_t)(127 - e_v) << 23);
        }
      } else {
        atomicCAS(s.a.err, 0, (int)BQ4_EINVAL_ARG);
      }
    }
    at[tid] = where;
    ck[tid] = where < 0 ? 0.0f : f;
    s.consts[rec].lv[tid] = where < 0 ? -INFINITY : (float)e_v;
    s.consts[rec].w[tid] = __uint_as_float((uint32_t)(127 - e_v) << 23);
    const bool weighted = __any_sync(0xffffffffu, e_v > 0), partial = __any_sync(0xffffffffu, where < 0);
    const unsigned marked = __ballot_sync(0xffffffffu, some_v);
    if ((tid & 31) == 0) {
      flags[tid >> 5] = weighted ? 3 : partial ? 1 : 0;
      odd_v[tid >> 5] = marked;
    }
  }
  __syncthreads();

  uint8_t* kd = s.k + rec * kTile;
#pragma unroll 4
  for (int p = tid; p < kKeys * kCh; p += 256) {
    const int key = p / kCh, ch = p % kCh;
    uint32_t kw[4] = {0, 0, 0, 0}, vw[4] = {0, 0, 0, 0};  // 8 halves of k and v
    const int64_t where = at[key];
    if (where >= 0) {
      const uint8_t* kr = c.data + where;
      const uint8_t* vr = kr + 16 * kRow;
      const int pl = place[key] & 15;
      if constexpr (kFmt == BQ4_CACHE_F16) {
        const uint4 a = *reinterpret_cast<const uint4*>(kr + cache_swizzle(0, kRow, pl, 16 * ch));
        const uint4 b = *reinterpret_cast<const uint4*>(vr + cache_swizzle(1, kRow, pl, 16 * ch));
        kw[0] = a.x, kw[1] = a.y, kw[2] = a.z, kw[3] = a.w;
        vw[0] = b.x, vw[1] = b.y, vw[2] = b.z, vw[3] = b.w;
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((vw[e] & 0x7c00u) == 0x7c00u) odd = true, vw[e] &= 0xffff0000u;
          if ((vw[e] & 0x7c000000u) == 0x7c000000u) odd = true, vw[e] &= 0xffffu;
        }
        if (odd) atomicOr(&odd_v[key >> 5], 1u << (key & 31));
      } else {
        float kx[8], vx[8];
        if constexpr (kFmt == BQ4_CACHE_Q8) {
          const uint2 a = *reinterpret_cast<const uint2*>(kr + cache_swizzle(0, kRow, pl, 8 * ch));
          const uint2 b = *reinterpret_cast<const uint2*>(vr + cache_swizzle(1, kRow, pl, 8 * ch));
          const float w = sv[key][0];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            kx[e] = (float)((int)((e < 4 ? a.x : a.y) >> 8 * (e & 3) & 255) - 128);
            vx[e] = (float)((int)((e < 4 ? b.x : b.y) >> 8 * (e & 3) & 255) - 128) * w;
          }
        } else {
          const int blk = ch >> 2;
          const uint32_t a =
              *reinterpret_cast<const uint32_t*>(kr + cache_swizzle(0, kRow, pl, 4 * ((ch & 3) * kNb + blk)));
          const float wk = sk[key][blk], wv = sv[key][blk];
          uint32_t b = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            b |= (uint32_t)*reinterpret_cast<const uint16_t*>(
                     vr + cache_swizzle(1, kRow, pl, 2 * (((2 * ch + h) & 7) * kNb + blk)))
                 << 16 * h;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            kx[e] = (float)((int)(a >> (4 * (e >> 1) + 16 * (e & 1)) & 15) - 8) * wk;
            vx[e] = (float)((int)(b >> 4 * e & 15) - 8) * wv;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __half2 hk = __floats2half2_rn(kx[2 * e], kx[2 * e + 1]);
          const __half2 hv = __floats2half2_rn(vx[2 * e], vx[2 * e + 1]);
          kw[e] = *reinterpret_cast<const uint32_t*>(&hk);
          vw[e] = *reinterpret_cast<const uint32_t*>(&hv);
        }
      }
    }
    *reinterpret_cast<uint4*>(kd + (ch >> 3) * (kKeys * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4)) =
        make_uint4(kw[0], kw[1], kw[2], kw[3]);
    uint32_t* vs = reinterpret_cast<uint32_t*>(vt + key * kPitch + 8 * ch);
#pragma unroll
    for (int e = 0; e < 4; ++e) vs[e] = vw[e];
  }
  __syncthreads();
  if (tid < kKeys) s.consts[rec].ck[tid] = ck[tid];
  if (tid < 4) s.consts[rec].odd[tid] = odd_v[tid];
  if (tid == 0)
    s.consts[rec].flags = flags[0] | flags[1] | flags[2] | flags[3] |
                          ((odd_v[0] | odd_v[1] | odd_v[2] | odd_v[3]) ? 4 : 0);

  // ---- v transposed: 8 lanes write the 8 pieces (8 keys each) of one value's 64 keys
  uint8_t* vd = s.v + rec * kTile;
  for (int p = tid; p < 16 * (kHP / 2); p += 256) {
    const int kc = (p & 7) + 8 * (p / (8 * (kHP / 2))), d = 2 * ((p >> 3) % (kHP / 2));
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(vt + (8 * kc + 2 * u) * kPitch + d);
      const uint32_t y = *reinterpret_cast<const uint32_t*>(vt + (8 * kc + 2 * u + 1) * kPitch + d);
      lo[u] = __byte_perm(x, y, 0x5410);
      hi[u] = __byte_perm(x, y, 0x7632);
    }
    uint8_t* base = vd + (kc >> 3) * (kHP * 128) + d * 128;
    *reinterpret_cast<uint4*>(base + (((kc & 7) ^ (d & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    *reinterpret_cast<uint4*>(base + 128 + (((kc & 7) ^ ((d + 1) & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  }
}

// ---------------------------------------------------------------- the products

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 64 raw scores of keys from `key0` of the record -> y in place; returns their
// maximum.  kPlain: every key exists and is seen; else those from `valid` are not.
template <bool kPlain>
__device__ __forceinline__ float scores64(uint32_t (&r)[64], const Consts* k, int key0, int valid) {
  float mp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&k->ck[key0 + i]);
    uint64_t y0 = attn_pack2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    uint64_t y1 = attn_pack2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
    if constexpr (kPlain) {
      y0 = mul2(y0, f.x);
      y1 = mul2(y1, f.y);
    } else {
      const ulonglong2 z = *reinterpret_cast<const ulonglong2*>(&k->lv[key0 + i]);
      y0 = attn_fma2(y0, f.x, z.x);
      y1 = attn_fma2(y1, f.y, z.y);
    }
    float y[4];
    attn_unpack2(y0, y[0], y[1]);
    attn_unpack2(y1, y[2], y[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!kPlain && key0 + i + e >= valid) y[e] = -INFINITY;
      r[i + e] = __float_as_uint(y[e]);
    }
    mp[0] = attn_max3(mp[0], y[0], y[1]);
    mp[1] = attn_max3(mp[1], y[2], y[3]);
  }
  return fmaxf(mp[0], mp[1]);
}

// p = 2^(y + shift) of 64 keys as f16 pairs into 32 TMEM columns; returns their sum, of
// kWeighted each times its key's w.
template <bool kWeighted>
__device__ __forceinline__ float probs64(const uint32_t (&r)[64], float shift, uint32_t t_p, const float* w) {
  const uint64_t s2 = attn_pack2(shift, shift);
  uint64_t acc[2] = {0, 0};
#pragma unroll
  for (int cc = 0; cc < 4; ++cc) {
    uint32_t pk[8];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float x0, x1;
      attn_unpack2(attn_add2(attn_pack2(__uint_as_float(r[16 * cc + i]), __uint_as_float(r[16 * cc + i + 1])), s2),
                   x0, x1);
      const float p0 = attn_ex2(x0), p1 = attn_ex2(x1);
      if constexpr (kWeighted)
        acc[(i >> 1) & 1] = attn_fma2(attn_pack2(p0, p1), *reinterpret_cast<const uint64_t*>(w + 16 * cc + i),
                                      acc[(i >> 1) & 1]);
      else
        acc[(i >> 1) & 1] = attn_add2(acc[(i >> 1) & 1], attn_pack2(p0, p1));
      const __half2 hp = __floats2half2_rn(p0, p1);
      pk[i >> 1] = *reinterpret_cast<const uint32_t*>(&hp);
    }
    ptx::tmem_st_32x32b_x8(t_p + cc * 8, pk);
  }
  float a, b, c, d;
  attn_unpack2(acc[0], a, b);
  attn_unpack2(acc[1], c, d);
  return (a + b) + (c + d);
}

template <int kHP>
struct TileSmem {
  static constexpr uint32_t kTile = 128 * kHP * 2;
  static constexpr uint32_t kSubV = kHP * 128;                      // 64 keys of the v tile
  static constexpr uint32_t kOffConsts = (2 + 2 * kRing) * kTile;   // q, k, v before them
  static constexpr uint32_t kOffBars = kOffConsts + kRing * kConsts;
  static constexpr uint32_t kBytes = kOffBars + 256;
};

// Adds the v values that are not finite of the keys that a row sees, among nblk records, to its
// results: out_row of the output or (finish not set) slot of the partial ones.
__device__ __noinline__ void add_not_finite(const TileArgs& s, int set, int kvh, int j0, int nblk, int see,
                                            int64_t out_row, int64_t slot) {
  const CacheView& c = s.a.c;
  const int32_t* table = s.prefix ? s.a.prefix_table : s.a.s.table + set * s.a.s.table_stride;
  const Consts* k = s.consts + ((int64_t)set * c.kv_heads + kvh) * s.blocks + j0;
  for (int j = 0; j < nblk; ++j, ++k) {
    if (!(k->flags & 4)) continue;
    for (int i = 0; i < kKeys; ++i) {
      const int pos = (j0 + j) * kKeys + i;
      if (!(k->odd[i >> 5] >> (i & 31) & 1) || pos >= see) continue;
      const int pi = pos / c.page_size, place = pos - pi * c.page_size;
      const uint8_t* step = cache_step(c, table[pi], kvh, place);
      for (int d = 0; d < c.head_dim; ++d) {
        float x;
        if (c.format == BQ4_CACHE_F16)
          x = __half2float(*reinterpret_cast<const __half*>(step + 16 * c.row_bytes +
                                                            cache_swizzle(1, c.row_bytes, place & 15, 2 * d)));
        else
          x = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(
                                  step + 32 * c.row_bytes)[((place & 15) * 2 + 1) * c.nb + d / kCacheBlock] << 16);
        if (fabsf(x) <= 3.402823466e38f) continue;
        if (s.finish) {
          __half* o = reinterpret_cast<__half*>(s.a.out) + out_row * c.head_dim + d;
          *o = __float2half_rn(__half2float(*o) + x);
        } else {
          s.part[slot * c.hp + d] += x;
        }
      }
    }
  }
}

template <int kHP>
__global__ void __launch_bounds__(kTThreads, 1) cache_tile_kernel(const __grid_constant__ TileArgs s) {
  using M = TileSmem<kHP>;
  constexpr uint32_t kTile = M::kTile, kColO = 256;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (ptx::smem_u32(smem_raw) & 1023) {  // uniform: every thread leaves before any barrier
    if (threadIdx.x == 0) atomicCAS(s.a.err, 0, (int)BQ4_EALIGN);
    return;
  }
  const CacheAttnCall& a = s.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ptx::griddep_launch_dependents();

  // ---- which rows and records
  unsigned item = blockIdx.x;
  const int chunk = (int)(item % (unsigned)s.chunks);
  item /= (unsigned)s.chunks;
  const int kvh = (int)(item % (unsigned)a.c.kv_heads);
  item /= (unsigned)a.c.kv_heads;
  const int rt = s.tiles - 1 - (int)(item % (unsigned)s.tiles);  // late rows see the most keys: first
  const int set = (int)(item / (unsigned)s.tiles);
  const int rows = (s.prefix ? a.s.batch : 1) * a.tokens * s.group;
  const bool causal = !s.prefix && a.causal;
  const int n = set_length(s, set, a.err);
  const int last_i = (min(rt * 256 + 256, rows) - 1) / s.group;
  const int end = max(0, causal ? n - a.tokens + last_i + 1 : n);
  const int j0 = chunk * s.span, nblk = min((end + kKeys - 1) / kKeys - j0, s.span);
  const int nt = rows - rt * 256 > 128 ? 2 : 1;
  const int64_t head = (int64_t)set * a.c.kv_heads + kvh;
  auto out_row = [&](int r) {  // row r of the set in the output
    int b = set;
    if (s.prefix) {
      b = r / (a.tokens * s.group);
      r -= b * a.tokens * s.group;
    }
    const int i = r / s.group;
    return ((int64_t)b * a.tokens + i) * a.q_heads + kvh * s.group + (r - i * s.group);
  };
  if (nblk <= 0) {
    ptx::griddep_wait();  // no CTA ends before the kernel that this grid was launched beside
    if (s.finish) {  // rows that see nothing
      for (int p = threadIdx.x; p < 256 * (kHP / 8); p += kTThreads) {
        const int r = rt * 256 + p / (kHP / 8), d = 8 * (p % (kHP / 8));
        if (r < rows && d < a.c.head_dim)
          *reinterpret_cast<uint4*>(a.out + out_row(r) * a.c.head_dim + d) = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }

  uint8_t* qs = smem_raw;
  uint8_t* ks = qs + 2 * kTile;
  uint8_t* vs = ks + kRing * kTile;
  Consts* consts = reinterpret_cast<Consts*>(smem_raw + M::kOffConsts);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem_raw + M::kOffBars);
  uint64_t* k_full = q_full + 1;        // [kRing]
  uint64_t* k_empty = k_full + kRing;   // [kRing]
  uint64_t* v_full = k_empty + kRing;   // [kRing]: v and consts
  uint64_t* v_empty = v_full + kRing;   // [kRing]
  uint64_t* s_full = v_empty + kRing;   // [tile]
  uint64_t* p_half = s_full + 2;        // [tile]: P of keys 64..127 stored
  uint64_t* p_full = p_half + 2;        // [tile]: P of keys 0..63 stored
  uint64_t* o_done = p_full + 2;        // the last P v has completed
  uint64_t* drain = o_done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  if (threadIdx.x == 0) {
    ptx::mbar_init(q_full, 1);
    for (int i = 0; i < kRing; ++i) {
      ptx::mbar_init(&k_full[i], 1);
      ptx::mbar_init(&k_empty[i], 1);
      ptx::mbar_init(&v_full[i], 1);
      ptx::mbar_init(&v_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&s_full[t], 1);
      ptx::mbar_init(&p_half[t], 4);
      ptx::mbar_init(&p_full[t], 4);
    }
    ptx::mbar_init(o_done, 1);
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // the records and q tiles of the kernel before: every role waits for it here, since the bounded
  // waits below would count its time (and that of a kernel it was launched beside) as theirs
  ptx::griddep_wait();

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ copies
      ptx::mbar_arrive_expect_tx(q_full, nt * kTile);
      for (int t = 0; t < nt; ++t)
        ptx::bulk_load(qs + t * kTile, s.q + (head * 2 * s.tiles + 2 * rt + t) * kTile, kTile, q_full);
      const int64_t rec0 = head * s.blocks + j0;
      int k_issued = 0, v_issued = 0;
      for (int j = 0; j < nblk; ++j) {
        const int st = j % kRing;
        const uint32_t ph = (j / kRing) & 1;
        if (!attn_wait(&k_empty[st], ph ^ 1, abort_flag, a.err)) break;
        ptx::mbar_arrive_expect_tx(&k_full[st], kTile);
        ptx::bulk_load(ks + st * kTile, s.k + (rec0 + j) * kTile, kTile, &k_full[st]);
        k_issued = j + 1;
        if (!attn_wait(&v_empty[st], ph ^ 1, abort_flag, a.err)) break;
        ptx::mbar_arrive_expect_tx(&v_full[st], kTile + kConsts);
        ptx::bulk_load(&consts[st], &s.consts[rec0 + j], kConsts, &v_full[st]);
        ptx::bulk_load(vs + st * kTile, s.v + (rec0 + j) * kTile, kTile, &v_full[st]);
        v_issued = j + 1;
      }
      // every copy this thread started has landed before the CTA may exit
      attn_drain(q_full, 0);
      for (int j = (k_issued > kRing ? k_issued - kRing : 0); j < k_issued; ++j)
        attn_drain(&k_full[j % kRing], (j / kRing) & 1);
      for (int j = (v_issued > kRing ? v_issued - kRing : 0); j < v_issued; ++j)
        attn_drain(&v_full[j % kRing], (j / kRing) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------ MMA issuer
      constexpr uint32_t idesc_s = ptx::umma_idesc_f16(128, 128), idesc_o = ptx::umma_idesc_f16(128, kHP);
      const uint32_t q_a = ptx::smem_u32(qs);
      const int last = nt - 1;
      bool ok = attn_wait(q_full, 0, abort_flag, a.err);
      auto issue_s = [&](int t, int j) -> bool {
        const int st = j % kRing;
        if (t == 0 && !attn_wait(&k_full[st], (j / kRing) & 1, abort_flag, a.err)) return false;
        ptx::tc_fence_after();
        const uint32_t k_a = ptx::smem_u32(ks + st * kTile), qa = q_a + (uint32_t)t * kTile;
#pragma unroll
        for (int kk = 0; kk < kHP / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk >> 2) * (128 * 128) + (uint32_t)(kk & 3) * 32;
          ptx::mma_f16_ss(tmem + (uint32_t)t * 128, ptx::umma_desc_sw128(qa + off), ptx::umma_desc_sw128(k_a + off),
                          idesc_s, kk > 0 ? 1u : 0u);
        }
        ptx::mma_commit(&s_full[t]);
        if (t == last) ptx::mma_commit(&k_empty[st]);
        return true;
      };
      // O_t (+)= P_t v in two halves, keys 64..127 first (the order in which P is stored)
      auto issue_pv = [&](int t, int j, int half) -> bool {
        const int st = j % kRing;
        if (!attn_wait_poll(half ? &p_full[t] : &p_half[t], j & 1, abort_flag, a.err)) return false;
        if (t == 0 && !half && !attn_wait(&v_full[st], (j / kRing) & 1, abort_flag, a.err)) return false;
        ptx::tc_fence_after();
        const uint32_t v_a = ptx::smem_u32(vs + st * kTile);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kk = half ? i : 4 + i;
          const uint32_t off = (uint32_t)(kk >> 2) * M::kSubV + (uint32_t)(kk & 3) * 32;
          ptx::mma_f16_ts(tmem + kColO + (uint32_t)t * 128, tmem + (uint32_t)t * 128 + 64 + (uint32_t)kk * 8,
                          ptx::umma_desc_sw128(v_a + off), idesc_o, (j > 0 || half || i > 0) ? 1u : 0u);
        }
        if (t == last && half) {
          ptx::mma_commit(&v_empty[st]);
          if (j == nblk - 1) ptx::mma_commit(o_done);
        }
        return true;
      };
      for (int t = 0; ok && t < nt; ++t) ok = issue_s(t, 0);
      for (int j = 0; ok && j < nblk; ++j)
        for (int t = 0; ok && t < nt; ++t) {
          ok = issue_pv(t, j, 0) && issue_pv(t, j, 1);
          if (ok && j + 1 < nblk) ok = issue_s(t, j + 1);
        }
      // every MMA this thread issued has completed before TMEM is released
      ptx::mma_commit(drain);
      attn_drain(drain, 0);
    }
  } else if (warp >= 4 && (warp - 4) >> 2 < nt) {
    // ------------------------------------------------ softmax: one thread per query row of tile t
    const int t = (warp - 4) >> 2, q = warp & 3;
    const int local = t * 128 + q * 32 + lane, r0 = rt * 256 + local;
    const int see = causal ? n - a.tokens + min(r0, rows - 1) / s.group + 1 : n;
    const uint32_t t_lane = tmem + ((uint32_t)(q * 32) << 16);
    const uint32_t t_s = t_lane + (uint32_t)t * 128, t_o = t_lane + kColO + (uint32_t)t * 128;
    float m = kTNone, l = 0.0f;
    bool ok = true;
    int seen_flags = 0;
    uint32_t r[64];
    for (int j = 0; j < nblk && ok; ++j) {
      const int st = j % kRing;
      ok = __all_sync(0xffffffffu, attn_wait(&v_full[st], (j / kRing) & 1, abort_flag, a.err) &&
                                       attn_wait(&s_full[t], j & 1, abort_flag, a.err));
      if (!ok) break;
      ptx::tc_fence_after();
      const Consts* k = &consts[st];
      const int valid = see - (j0 + j) * kKeys;
      const int flags = k->flags;
      const bool weighted = flags & 2;
      seen_flags |= flags;
      const bool plain = !(flags & 1) && __all_sync(0xffffffffu, valid >= kKeys);
      attn_ld64(t_s, r);
      float top = plain ? scores64<true>(r, k, 0, valid) : scores64<false>(r, k, 0, valid);
#pragma unroll
      for (int i = 0; i < 64; i += 16)  // y of keys 0..63 goes back over S until the P pass
        ptx::tmem_st_32x32b_x16(t_s + i, *reinterpret_cast<uint32_t(*)[16]>(r + i));
      attn_ld64(t_s + 64, r);  // kept for the P pass
      top = fmaxf(top, plain ? scores64<true>(r, k, 64, valid) : scores64<false>(r, k, 64, valid));
      const bool jump = top > m + kTJump;
      const float m_use = jump ? top - kTHead : m;
      const float alpha = jump ? attn_ex2(m - m_use) : 1.0f;
      if (j > 0 && __any_sync(0xffffffffu, jump)) {
        // O_t holds P_t(j-1) v_{j-1} (s_full's commit for S_t(j) covered it)
#pragma unroll
        for (int cc = 0; cc < kHP / 16; ++cc) {
          uint32_t o[16];
          ptx::tmem_ld_32x32b_x16(t_o + cc * 16, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          ptx::tmem_st_32x32b_x16(t_o + cc * 16, o);
        }
      }
      // keys 64..127 -> P columns 96..127 (S columns already read): their half of P v may start
      float sum = weighted ? probs64<true>(r, -m_use, t_s + 96, k->w + 64)
                           : probs64<false>(r, -m_use, t_s + 96, nullptr);
      ptx::tmem_st_wait();  // P (and a rescaled O) in TMEM before the MMA reads them
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&p_half[t]);
      // keys 0..63 (y stored above, and the wait for P's stores since) -> P columns 64..95
      attn_ld64(t_s, r);
      sum += weighted ? probs64<true>(r, -m_use, t_s + 64, k->w) : probs64<false>(r, -m_use, t_s + 64, nullptr);
      l = l * alpha + sum;
      m = m_use;
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&p_full[t]);
    }
    if (ok) ok = __all_sync(0xffffffffu, attn_wait(o_done, 0, abort_flag, a.err));
    if (ok) {
      ptx::tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t slot = ((((int64_t)set * s.tiles + rt) * a.c.kv_heads + kvh) * s.chunks + chunk) * 256 + local;
      const int64_t row = r0 < rows ? out_row(r0) : 0;
#pragma unroll
      for (int half = 0; half < kHP / 64; ++half) {
        __syncwarp();
        attn_ld64(t_o + half * 64, r);
        if (r0 < rows && s.finish) {
#pragma unroll
          for (int i = 0; i < 64; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const __half2 h = __floats2half2_rn(__uint_as_float(r[i + 2 * u]) * inv,
                                                  __uint_as_float(r[i + 2 * u + 1]) * inv);
              w[u] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if (half * 64 + i < a.c.head_dim)
              *reinterpret_cast<uint4*>(a.out + row * a.c.head_dim + half * 64 + i) =
                  make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (r0 < rows) {
#pragma unroll
          for (int i = 0; i < 64; i += 4)
            *reinterpret_cast<uint4*>(s.part + slot * kHP + half * 64 + i) =
                make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      }
      if (!s.finish && r0 < rows) s.ml[slot] = make_float2(m, l);
      if ((seen_flags & 4) && r0 < rows) add_not_finite(s, set, kvh, j0, nblk, see, row, slot);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <int kHP>
cudaError_t launch_tile(const TileArgs& s, unsigned grid, cudaStream_t stream) {
  static std::atomic<uint64_t> ready{0};  // a bit for each device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    cudaError_t e = cudaFuncSetAttribute(cache_tile_kernel<kHP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)TileSmem<kHP>::kBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kTThreads);
  cfg.dynamicSmemBytes = TileSmem<kHP>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cache_tile_kernel<kHP>, s);
}

template <int kFmt>
cudaError_t launch_widen(const TileArgs& s, unsigned grid, bool beside, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, s.a.c.hp == 64 ? cache_widen_kernel<kFmt, 64> : cache_widen_kernel<kFmt, 128>, s);
}

}  // namespace

bool plan_cache_tile(const CacheAttnCall& a, bool prefix, int sms, size_t room, CacheTilePlan* p) {
  p->workspace_bytes = 0;
  const int group = a.q_heads / a.c.kv_heads;
  const int64_t rows = (int64_t)a.tokens * group * (prefix ? a.s.batch : 1);
  const int64_t keys = prefix ? (int64_t)a.prefix_width * a.c.page_size : a.max_length;
  const int64_t sets = prefix ? 1 : a.s.batch;
  const int64_t blocks = (keys + kKeys - 1) / kKeys, tiles = (rows + 255) / 256;
  const int64_t heads = sets * a.c.kv_heads;
  if (blocks == 0 || heads * blocks > 0x3fffffff || heads * tiles > 0x00ffffff) return false;
  p->prefix = prefix;
  p->sets = (int)sets;
  p->tiles = (int)tiles;
  p->blocks = (int)blocks;
  p->records = heads * blocks;
  p->q_tiles = heads * 2 * tiles;
  if (p->records + p->q_tiles > 0x7fffffff) return false;
  const size_t tile = (size_t)kKeys * a.c.hp * 2;
  p->tile_bytes = up256((size_t)p->records * tile);
  p->consts_bytes = up256((size_t)p->records * kConsts);
  p->q_bytes = up256((size_t)p->q_tiles * 128 * a.c.hp * 2);
  auto bytes = [&](int64_t chunks) {  // with so many chunks of a tile
    p->slots = heads * tiles * chunks * 256;
    p->part_bytes = up256((size_t)p->slots * a.c.hp * 4);
    p->ml_bytes = up256((size_t)p->slots * 8);
    return 2 * p->tile_bytes + p->consts_bytes + p->q_bytes + p->part_bytes + p->ml_bytes;
  };
  // chunks of a tile: as many as make waves of the GPU's SMs fullest, a chunk's start and end
  // costing about as much as three records
  double best = 0.0;
  p->span = (int)blocks;
  for (int64_t ch = 1; ch <= std::min<int64_t>(blocks, 64); ++ch) {
    const int64_t span = (blocks + ch - 1) / ch, chunks = (blocks + span - 1) / span;
    const int64_t waves = (heads * tiles * chunks + sms - 1) / sms;
    const double cost = (double)waves * (span + 3) + (ch > 1 ? 2.0 : 0.0);
    if (ch == 1 || (cost < best && heads * tiles * chunks <= 0x7fffffff && bytes(chunks) <= room))
      best = cost, p->span = (int)span;
  }
  p->chunks = (int)((blocks + p->span - 1) / p->span);
  p->workspace_bytes = bytes(p->chunks);
  return p->workspace_bytes <= room;
}

bq4_status run_cache_tile(const CacheAttnCall& a, const CacheTilePlan& p, bool finish, bool beside, void* workspace,
                          CacheJoinSource* source, cudaStream_t stream) {
  TileArgs s;
  s.a = a;
  s.c = a.scale * 1.4426950408889634f;  // log2(e)
  s.group = a.q_heads / a.c.kv_heads;
  s.prefix = p.prefix;
  s.sets = p.sets;
  s.tiles = p.tiles;
  s.blocks = p.blocks;
  s.span = p.span;
  s.chunks = p.chunks;
  s.q_vec = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride[0] % 8 == 0 && a.q_stride[1] % 8 == 0 &&
            a.q_stride[2] % 8 == 0;
  s.finish = finish;
  const uint64_t unit = (uint64_t)(a.c.page_size / kCachePageUnit);
  s.page_magic = ((1ull << 38) + unit - 1) / unit;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  s.k = ws;
  s.v = s.k + p.tile_bytes;
  s.consts = reinterpret_cast<Consts*>(s.v + p.tile_bytes);
  s.q = s.v + p.tile_bytes + p.consts_bytes;
  s.part = reinterpret_cast<float*>(s.q + p.q_bytes);
  s.ml = reinterpret_cast<float2*>(s.q + p.q_bytes + p.part_bytes);
  const unsigned widen = (unsigned)(p.records + p.q_tiles);
  cudaError_t e = a.c.format == BQ4_CACHE_F16  ? launch_widen<BQ4_CACHE_F16>(s, widen, beside, stream)
                  : a.c.format == BQ4_CACHE_Q8 ? launch_widen<BQ4_CACHE_Q8>(s, widen, beside, stream)
                                               : launch_widen<BQ4_CACHE_Q4>(s, widen, beside, stream);
  note_launch();
  if (e != cudaSuccess) return check_cuda(e, "cache widening launch");
  const unsigned grid = (unsigned)((int64_t)p.sets * p.tiles * a.c.kv_heads * p.chunks);
  e = a.c.hp == 64 ? launch_tile<64>(s, grid, stream) : launch_tile<128>(s, grid, stream);
  note_launch();
  source->part = s.part;
  source->ml = s.ml;
  source->pieces = nullptr;
  source->tile_rows = 256;
  source->tiles = p.tiles;
  source->span = p.span * kKeys;
  source->chunks = p.chunks;
  source->first_range = 0;
  return check_cuda(e, "cache attention tile launch");
}

}  // namespace bq4
