// bq4_cache_attn.cu -- attention over the paged key/value cache: out =
// softmax(scale q K^T + mask) V for the newest tokens of every sequence, the
// keys being a prefix that the whole batch shares (if any) and the
// sequence's own rows.
//
// The keys of a sequence (or of the prefix) are cut into chunks; one CTA takes
// one chunk, one kv head and a tile of 8 kNT query rows (the tokens and
// grouped heads that read this kv head; for the prefix those of the whole
// batch, so that it is read once).  It keeps a running maximum m, sum l and
// product O in f32 (O = sum_j 2^(x_j - m) v_j, x in log2 units), and a second
// kernel joins the chunks: O = sum_c 2^(m_c - M) O_c, l likewise.
//
// cache_split_kernel: four warps, each its own 16-key steps.
//   * Keys are the M side of the tensor core's m16n8k16 (f16 in, f32 out) and
//     the query rows its N side: S^T = K Q^T, then O^T = V^T P^T.  A group of 4
//     query heads fills half of N = 8, not a quarter of M = 16, and the widened
//     cache values (A) are made once for all rows.
//   * A lane (g = lane / 4, t = lane % 4) copies exactly the bytes that its
//     fragments need, 16 at a time (cp.async), into its own slots of a ring in
//     shared memory: k rows g and g + 8 at quarter t, v rows 2t, 2t + 1,
//     2t + 8, 2t + 9 at eighth g.  No lane reads what another copied, so the
//     loop has no barrier, and any order of the head's values inside a
//     fragment is as good as another as long as q follows it.
//   * Stored values are whole numbers u = q + 128 (q + 8).  Zero-extended to
//     16 bits they are the subnormal halves u 2^-24, exact in the tensor core:
//     widening a pair of k values is one byte permute (q8) or mask (q4).  The
//     offset leaves the scores through the accumulator's start value -128
//     2^-24 sum(q) (f32; q4: for each scale's 32 values); v, whose products
//     are summed over many keys, is made signed (one add a pair), since there
//     an offset would cost the sum its low bits.
//   * k scales multiply the f32 scores.  v scales multiply the probabilities,
//     over a running power of two that is at least the largest of them, so
//     that the f16 rounding of p s_v is a relative one (2^-11; the only
//     rounding to fewer than 32 bits besides the result's).
//   * m only moves when a score passes it by 2^14 (a vote, no shuffles in the
//     common step): p <= 2^14 fits f16, and m starts 2^6 below the first
//     maximum so that small probabilities keep f16's range below them.
//
// What bounds it: HBM for a few rows (each byte of the chunk is read once),
// instruction issue for 4-bit caches, the tensor core's legacy path when the
// row tiles are many.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "bq4_cache.h"
#include "sm100_ptx.cuh"

namespace bq4 {
namespace {

constexpr int kSWarps = 4;
constexpr int kSThreads = 32 * kSWarps;
constexpr int kStep = 16;                     // keys of a warp's step
constexpr int kMinChunk = kStep * kSWarps;    // one step a warp
constexpr int kMaxChunk = 32 * kMinChunk;     // a lane holds one page id of its warp's 32 steps
constexpr float kNone = -1e30f;               // the maximum of no score (finite: differences stay defined)
constexpr float kHead = 6.0f, kJump = 14.0f;  // log2 units; see above

template <int kN>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? kN : 0;  // 0: the bytes are filled with zeros
  if constexpr (kN == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kN), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// kWords 32-bit words from this lane's slot in shared memory.
template <int kWords>
__device__ __forceinline__ void lds(uint32_t at, uint32_t (&w)[kWords]) {
  if constexpr (kWords == 4)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else if constexpr (kWords == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D += A B: A 16 x 16 (rows g, g + 8; columns 2t.., 2t + 8..), B 16 x 8.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 x 8 transpose of 16-bit values: lane (g, t) gives [g][2t, 2t + 1] and gets [2t, 2t + 1][g].
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t add_h2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Sizes that follow from the format and the padded head.
template <int kFmt, int kHP>
struct Layout {
  static constexpr bool kQ = kFmt != BQ4_CACHE_F16;
  static constexpr int kRow = kFmt == BQ4_CACHE_F16 ? 2 * kHP : kFmt == BQ4_CACHE_Q8 ? kHP : kHP / 2;
  static constexpr int kNb = kFmt == BQ4_CACHE_Q8 ? 1 : kFmt == BQ4_CACHE_Q4 ? kHP / 32 : 0;
  static constexpr int kKS = kHP / 16;               // k16 steps of q k
  static constexpr int kMT = kHP / 16;               // 16-value tiles of the output
  static constexpr int kKLane = kRow / 4;            // bytes of one k row that a lane takes
  static constexpr int kKPiece = kKLane < 16 ? kKLane : 16;
  static constexpr int kKPieces = kKLane / kKPiece;  // piece c of lane t lies at (4 c + t) kKPiece
  static constexpr int kVLane = kRow / 8;
  static constexpr int kVPiece = kVLane < 16 ? kVLane : 16;
  static constexpr int kVPieces = kVLane / kVPiece;  // piece c of lane g lies at (8 c + g) kVPiece
  static constexpr int kScale = 4 * kNb;             // bytes of a token's scales, k then v
  // a stage: [k row g, g + 8][piece], [v row][piece], [row g, g + 8] scales; 32 lanes' slots each
  static constexpr int kOffV = 2 * kKPieces * kKPiece * 32;
  static constexpr int kOffS = kOffV + 4 * kVPieces * kVPiece * 32;
  static constexpr int kStage = kOffS + (kQ ? 2 * kScale * 32 : 0);
  static constexpr int kStages = kFmt == BQ4_CACHE_F16 ? (kHP == 128 ? 2 : 3) : kFmt == BQ4_CACHE_Q8 ? 3 : 4;
  // value d of the head that element e (0..3) of k step ks holds in lane t: at + e
  __device__ static int qd(int ks, int t) {
    return kFmt == BQ4_CACHE_Q8 ? 64 * (ks >> 2) + 16 * t + 4 * (ks & 3) : 32 * (ks >> 1) + 8 * t + 4 * (ks & 1);
  }
  // value d of row g of output tile mt; row g + 8 holds d + 1
  __device__ static int od(int mt, int g) {
    if constexpr (kFmt == BQ4_CACHE_F16) return 64 * (mt >> 2) + 8 * g + 2 * (mt & 3);
    if constexpr (kFmt == BQ4_CACHE_Q8) return kVLane * g + 2 * mt;
    return 32 * (mt >> 1) + 4 * g + 2 * (mt & 1);
  }
};

struct SplitArgs {
  CacheAttnCall a;
  uint64_t page_magic;   // floor(u / (page_size / 16)) = u * page_magic >> 38
  int64_t page_stride;   // bytes of a page
  float c;               // scale * log2(e)
  int group;             // query heads of a kv head
  int p_tiles, s_tiles;  // row tiles of the prefix and of one sequence
  int p_chunk, s_chunk, p_chunks, s_chunks;
  unsigned p_items;      // CTAs of the prefix, first in the grid
  int q_vec;             // q rows lie on 8-byte boundaries
  int direct;            // one chunk in all: rows are finished here
  float* part;           // [row][p_chunks + s_chunks][hp]
  float2* ml;            // [row][p_chunks + s_chunks]: m, l
};

// Query row r of a tile's space: its sequence, token and head.
struct Row {
  int b, i, h;
};
__device__ __forceinline__ Row row_of(const SplitArgs& s, bool prefix, int b, int kvh, int r) {
  Row o;
  o.b = b;
  if (prefix) {
    o.b = r / (s.a.tokens * s.group);
    r -= o.b * s.a.tokens * s.group;
  }
  o.i = r / s.group;
  o.h = kvh * s.group + (r - o.i * s.group);
  return o;
}

__device__ __forceinline__ int clamp_length(int n, int64_t cap, int* err) {
  if (n >= 0 && n <= cap) return n;
  atomicCAS(err, 0, (int)BQ4_EINVAL_ARG);
  return n < 0 ? 0 : (int)cap;
}

__device__ __forceinline__ int own_length(const CacheAttnCall& a, int b) {
  return clamp_length(a.s.lengths[b], min((int64_t)a.max_length, (int64_t)a.s.table_width * a.c.page_size), a.err);
}
__device__ __forceinline__ int prefix_rows(const CacheAttnCall& a) {
  return a.prefix_length ? clamp_length(a.prefix_length[0], (int64_t)a.prefix_width * a.c.page_size, a.err) : 0;
}

template <int kFmt, int kHP, int kNT>
__global__ void __launch_bounds__(kSThreads, kNT == 1 ? 4 : 2) cache_split_kernel(const __grid_constant__ SplitArgs s) {
  using Y = Layout<kFmt, kHP>;
  extern __shared__ __align__(16) uint8_t smem[];
  const CacheAttnCall& a = s.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  ptx::griddep_launch_dependents();

  // ---- which chunk, kv head and rows
  const bool prefix = blockIdx.x < s.p_items;
  unsigned item = prefix ? blockIdx.x : blockIdx.x - s.p_items;
  const int tiles = prefix ? s.p_tiles : s.s_tiles;
  const int tile = (int)(item % (unsigned)tiles);
  item /= (unsigned)tiles;
  const int kvh = (int)(item % (unsigned)a.c.kv_heads);
  item /= (unsigned)a.c.kv_heads;
  const int b = prefix ? 0 : (int)(item % (unsigned)a.s.batch);
  const int chunk = prefix ? (int)item : (int)(item / (unsigned)a.s.batch);
  const int len = prefix ? s.p_chunk : s.s_chunk, key0 = chunk * len;
  const int rows = (prefix ? a.s.batch : 1) * a.tokens * s.group;
  const int row0 = tile * 8 * kNT;
  const bool causal = !prefix && a.causal;
  const int n = prefix ? prefix_rows(a) : own_length(a, b);
  // the keys that the tile's last row sees
  const int last_i = (min(row0 + 8 * kNT, rows) - 1) / s.group;
  const int end = min(key0 + len, causal ? n - a.tokens + last_i + 1 : n);
  if (end <= key0 && !s.direct) return;
  const int32_t* table = prefix ? a.prefix_table : a.s.table + b * a.s.table_stride;

  // ---- page of this warp's step `lane` (-1: none)
  const int steps = end <= key0 ? 0 : (end - key0 + kStep - 1) / kStep;
  const int mine = steps > warp ? (steps - warp + kSWarps - 1) / kSWarps : 0;
  int page = -1, place = 0;
  if (lane < mine) {
    const unsigned u = (unsigned)(key0 / kStep) + (unsigned)(warp + kSWarps * lane);
    const int pi = (int)((u * s.page_magic) >> 38);
    page = table[pi];
    place = (int)u * kStep - pi * a.c.page_size;
    if (page < 0 || page >= a.c.pages) {
      atomicCAS(a.err, 0, (int)BQ4_EINVAL_ARG);
      page = -1;
    }
  }

  // ---- copies of one step into stage st of this warp's ring
  const uint32_t ring = ptx::smem_u32(smem) + warp * Y::kStages * Y::kStage;
  const int64_t head_at = (int64_t)kvh * 2 * a.c.kv_bytes;
  auto fetch = [&](int j) {
    if (j < mine) {
      const int pg = __shfl_sync(0xffffffffu, page, j), pl = __shfl_sync(0xffffffffu, place, j);
      const int left = pg < 0 ? 0 : end - (key0 + (warp + kSWarps * j) * kStep);  // valid keys of the step
      const uint8_t* k = a.c.values + (int64_t)max(pg, 0) * s.page_stride + head_at + pl * Y::kRow;
      const uint8_t* v = k + a.c.kv_bytes;
      const uint32_t st = ring + (j % Y::kStages) * Y::kStage;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < Y::kKPieces; ++c)
          copy_async<Y::kKPiece>(st + ((r * Y::kKPieces + c) * 32 + lane) * Y::kKPiece,
                                 k + (g + 8 * r) * Y::kRow + (4 * c + t) * Y::kKPiece, g + 8 * r < left);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 2 * t + (r & 1) + 8 * (r >> 1);
#pragma unroll
        for (int c = 0; c < Y::kVPieces; ++c)
          copy_async<Y::kVPiece>(st + Y::kOffV + ((r * Y::kVPieces + c) * 32 + lane) * Y::kVPiece,
                                 v + key * Y::kRow + (8 * c + g) * Y::kVPiece, key < left);
      }
      if constexpr (Y::kQ) {
        const uint8_t* sc = reinterpret_cast<const uint8_t*>(a.c.scales) +
                            (((int64_t)max(pg, 0) * a.c.kv_heads + kvh) * a.c.page_size + pl) * Y::kScale;
#pragma unroll
        for (int r = 0; r < 2; ++r)
          copy_async<Y::kScale>(st + Y::kOffS + (r * 32 + lane) * Y::kScale, sc + (g + 8 * r) * Y::kScale,
                                g + 8 * r < left);
      }
    }
    copy_commit();  // an empty group past the end keeps the count
  };
#pragma unroll
  for (int j = 0; j < Y::kStages - 1; ++j) fetch(j);

  // ---- q fragments; the offset's start values; what each row sees
  uint32_t q[kNT][Y::kKS][2];
  constexpr int kOffs = kFmt == BQ4_CACHE_Q4 ? Y::kNb : 1;  // start values of a row
  float off[kNT][kOffs][2];
  int see[kNT][2];
  int see_all = 0x7fffffff;
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
    const int r = row0 + 8 * nt + g;
    const Row w = row_of(s, prefix, b, kvh, min(r, rows - 1));
    const __half* p = reinterpret_cast<const __half*>(a.q) + w.b * a.q_stride[0] + w.i * a.q_stride[1] +
                      w.h * a.q_stride[2];
#pragma unroll
    for (int ks = 0; ks < Y::kKS; ++ks) {
      const int d = Y::qd(ks, t);
      uint2 u = make_uint2(0, 0);
      if (r < rows && d < a.c.head_dim) {
        if (s.q_vec) {
          u = *reinterpret_cast<const uint2*>(p + d);
        } else {
          const unsigned short* e = reinterpret_cast<const unsigned short*>(p + d);
          u = make_uint2(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16);
        }
      }
      q[nt][ks][0] = u.x;
      q[nt][ks][1] = u.y;
    }
    if constexpr (Y::kQ) {
#pragma unroll
      for (int o = 0; o < kOffs; ++o) {
        float sum = 0.0f;
#pragma unroll
        for (int ks = o * Y::kKS / kOffs; ks < (o + 1) * Y::kKS / kOffs; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[nt][ks][e]));
            sum += f.x + f.y;
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);  // of row g, in all its lanes
        constexpr float kZero = kFmt == BQ4_CACHE_Q8 ? -128.0f : -8.0f;
        off[nt][o][0] = __shfl_sync(0xffffffffu, sum, 8 * t) * (kZero * 0x1p-24f);
        off[nt][o][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4) * (kZero * 0x1p-24f);
      }
    } else {
      off[nt][0][0] = off[nt][0][1] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = row0 + 8 * nt + 2 * t + e;
      see[nt][e] = !causal ? end : rr < rows ? min(end, n - a.tokens + rr / s.group + 1) : end;
      see_all = min(see_all, see[nt][e]);
    }
  }
  // the keys that every row of the tile sees (the same for the whole warp)
  see_all = min(see_all, __shfl_xor_sync(0xffffffffu, see_all, 1));
  see_all = min(see_all, __shfl_xor_sync(0xffffffffu, see_all, 2));

  float m[kNT][2], l[kNT][2], o[kNT][Y::kMT][4];
  float vs = 0.0f, inv_vs = 0.0f;  // power of two above the v scales so far
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
    m[nt][0] = m[nt][1] = kNone;
    l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
    for (int mt = 0; mt < Y::kMT; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
  }
  const float c = Y::kQ ? s.c * 0x1p24f : s.c;

  for (int j = 0; j < mine; ++j) {
    fetch(j + Y::kStages - 1);
    copy_wait<Y::kStages - 1>();
    const uint32_t st = ring + (j % Y::kStages) * Y::kStage;
    const int at = key0 + (warp + kSWarps * j) * kStep;
    if (__shfl_sync(0xffffffffu, page, j) < 0) continue;  // a bad page holds nothing

    // ---- scales of keys g, g + 8
    float sk[2][Y::kQ ? Y::kNb : 1], sv[2][Y::kQ ? Y::kNb : 1];
    if constexpr (Y::kQ) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t w[Y::kNb];
        lds(st + Y::kOffS + (r * 32 + lane) * Y::kScale, w);
        if constexpr (kFmt == BQ4_CACHE_Q8) {
          sk[r][0] = __uint_as_float(w[0] << 16);
          sv[r][0] = __uint_as_float(w[0] & 0xffff0000u);
        } else {
#pragma unroll
          for (int e = 0; e < Y::kNb; ++e) {
            const uint32_t kw = w[e >> 1], vw = w[(Y::kNb + e) >> 1];
            sk[r][e] = __uint_as_float(e & 1 ? kw & 0xffff0000u : kw << 16);
            sv[r][e] = __uint_as_float(e & 1 ? vw & 0xffff0000u : vw << 16);
          }
        }
      }
    }

    // ---- scores x of keys g (c0, c1) and g + 8 (c2, c3) with rows 2t, 2t + 1
    float x[kNT][4];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      x[nt][0] = x[nt][2] = kFmt == BQ4_CACHE_Q4 ? 0.0f : off[nt][0][0];
      x[nt][1] = x[nt][3] = kFmt == BQ4_CACHE_Q4 ? 0.0f : off[nt][0][1];
    }
#pragma unroll
    for (int p = 0; p < Y::kKPieces; ++p) {
      uint32_t w0[Y::kKPiece / 4], w1[Y::kKPiece / 4];
      lds(st + (p * 32 + lane) * Y::kKPiece, w0);
      lds(st + ((Y::kKPieces + p) * 32 + lane) * Y::kKPiece, w1);
      if constexpr (kFmt == BQ4_CACHE_F16) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
            mma16816(x[nt], w0[2 * h], w1[2 * h], w0[2 * h + 1], w1[2 * h + 1], q[nt][2 * p + h][0],
                     q[nt][2 * p + h][1]);
      } else if constexpr (kFmt == BQ4_CACHE_Q8) {
#pragma unroll
        for (int e = 0; e < Y::kKPiece / 4; ++e) {
          const uint32_t a0 = __byte_perm(w0[e], 0, 0x4140), a2 = __byte_perm(w0[e], 0, 0x4342);
          const uint32_t a1 = __byte_perm(w1[e], 0, 0x4140), a3 = __byte_perm(w1[e], 0, 0x4342);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
            mma16816(x[nt], a0, a1, a2, a3, q[nt][4 * p + e][0], q[nt][4 * p + e][1]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < Y::kNb; ++e) {
          float y[kNT][4];
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            y[nt][0] = y[nt][2] = off[nt][e][0];
            y[nt][1] = y[nt][3] = off[nt][e][1];
          }
          constexpr uint32_t kPair = 0x000F000Fu;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = (w0[e] >> 8 * h) & kPair, a2 = (w0[e] >> (8 * h + 4)) & kPair;
            const uint32_t a1 = (w1[e] >> 8 * h) & kPair, a3 = (w1[e] >> (8 * h + 4)) & kPair;
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
              mma16816(y[nt], a0, a1, a2, a3, q[nt][2 * e + h][0], q[nt][2 * e + h][1]);
          }
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int u = 0; u < 4; ++u) x[nt][u] = fmaf(y[nt][u], sk[u >> 1][e], x[nt][u]);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int u = 0; u < 4; ++u) x[nt][u] *= kFmt == BQ4_CACHE_Q8 ? sk[u >> 1][0] * c : c;

    // ---- mask; a step below see_all has none
    const bool edge = at + kStep > see_all;
    if (edge) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (at + g + 8 * (u >> 1) >= see[nt][u & 1]) x[nt][u] = -INFINITY;
    }

    // ---- running maximum and v scale
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) move |= fmaxf(x[nt][e], x[nt][e + 2]) > m[nt][e] + kJump;
    float sv_top = 0.0f;
    if constexpr (Y::kQ) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < Y::kNb; ++e) sv_top = fmaxf(sv_top, sv[r][e]);
      move |= sv_top > vs;
    }
    if (__any_sync(0xffffffffu, move)) {
      float beta = 1.0f;
      if constexpr (Y::kQ) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sv_top = fmaxf(sv_top, __shfl_xor_sync(0xffffffffu, sv_top, w));
        if (sv_top > vs) {
          // the next power of two, kept where 1 / vs is a normal number too
          const float up = __uint_as_float((__float_as_uint(sv_top) & 0x7f800000u) + 0x00800000u);
          const float next = fminf(fmaxf(up, 0x1p-120f), 0x1p120f);
          beta = vs / next;
          vs = next;
          inv_vs = 1.0f / next;
        }
      }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(x[nt][e], x[nt][e + 2]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          float alpha = 1.0f;
          if (top > m[nt][e] + kJump) {
            alpha = ex2(m[nt][e] - (top - kHead));
            m[nt][e] = top - kHead;
          }
          l[nt][e] *= alpha;
#pragma unroll
          for (int mt = 0; mt < Y::kMT; ++mt) {
            o[nt][mt][e] *= alpha * beta;
            o[nt][mt][e + 2] *= alpha * beta;
          }
        }
    }

    // ---- p = 2^(x - m), its sum, and p (s_v / vs) as f16 in the B layout
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[nt][u] = ex2(x[nt][u] - m[nt][u & 1]);
        l[nt][u & 1] += x[nt][u];
      }
    }
    uint32_t pb[kNT][2];
    auto weigh = [&](int e) {
      if constexpr (Y::kQ) {
        const float f0 = sv[0][e] * inv_vs, f1 = sv[1][e] * inv_vs;
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float y[4] = {x[nt][0] * f0, x[nt][1] * f0, x[nt][2] * f1, x[nt][3] * f1};
          if (edge) {
            // a masked key's scale may be NaN
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (at + g + 8 * (u >> 1) >= see[nt][u & 1]) y[u] = 0.0f;
          }
          pb[nt][0] = transpose8(pack_h2(y[0], y[1]));
          pb[nt][1] = transpose8(pack_h2(y[2], y[3]));
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          pb[nt][0] = transpose8(pack_h2(x[nt][0], x[nt][1]));
          pb[nt][1] = transpose8(pack_h2(x[nt][2], x[nt][3]));
        }
      }
    };

    // ---- O^T += V^T P^T
    uint32_t v[4][Y::kVPieces][Y::kVPiece / 4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int p = 0; p < Y::kVPieces; ++p)
        lds(st + Y::kOffV + ((r * Y::kVPieces + p) * 32 + lane) * Y::kVPiece, v[r][p]);
    if constexpr (kFmt == BQ4_CACHE_F16) {
      weigh(0);
#pragma unroll
      for (int p = 0; p < Y::kVPieces; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t f[4] = {__byte_perm(v[0][p][e], v[1][p][e], 0x5410), __byte_perm(v[0][p][e], v[1][p][e], 0x7632),
                           __byte_perm(v[2][p][e], v[3][p][e], 0x5410), __byte_perm(v[2][p][e], v[3][p][e], 0x7632)};
          const int mt = 4 * p + e;
          if (edge) {
            // A key that some row does not see may hold infinities or NaN: they leave the
            // product, which would carry 0 * NaN into that row, and reach the rows that
            // see the key one by one.  f[r]: keys 2t, 2t + 1 (r < 2) or + 8, value d + (r & 1).
            bool odd = false;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t lo = f[r] & 0x00007c00u, hi = f[r] & 0x7c000000u;
              odd |= lo == 0x00007c00u || hi == 0x7c000000u;
            }
            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint32_t bad = ((f[r] & 0x00007c00u) == 0x00007c00u ? f[r] & 0xffffu : 0) |
                                     ((f[r] & 0x7c000000u) == 0x7c000000u ? f[r] & 0xffff0000u : 0);
                if ((f[r] & 0x00007c00u) == 0x00007c00u) f[r] &= 0xffff0000u;
                if ((f[r] & 0x7c000000u) == 0x7c000000u) f[r] &= 0x0000ffffu;
                for (int w = 0; w < 4; ++w) {  // lane t = w of this g holds keys 2w, 2w + 1 (+ 8)
                  const uint32_t from = __shfl_sync(0xffffffffu, bad, 4 * g + w);
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const uint32_t bits = from >> 16 * h & 0xffffu;
                    const int key = at + 2 * w + h + 8 * (r >> 1);
                    const float add = __half2float(__ushort_as_half((unsigned short)bits));
                    if (bits) {
#pragma unroll
                      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                        for (int e2 = 0; e2 < 2; ++e2)
                          if (key < see[nt][e2]) o[nt][mt][e2 + 2 * (r & 1)] += add;
                    }
                  }
                }
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
            mma16816(o[nt][mt], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
        }
    } else if constexpr (kFmt == BQ4_CACHE_Q8) {
      weigh(0);
      constexpr uint32_t kZero = 0x80808080u;  // two halves of -128 2^-24
#pragma unroll
      for (int e = 0; e < Y::kVPiece / 4; ++e)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t y0 = __byte_perm(v[0][0][e], v[1][0][e], h ? 0x7632 : 0x5410);
          const uint32_t y1 = __byte_perm(v[2][0][e], v[3][0][e], h ? 0x7632 : 0x5410);
          const uint32_t f0 = add_h2(y0 & 0x00ff00ffu, kZero), f1 = add_h2(__byte_perm(y0, 0, 0x4341), kZero);
          const uint32_t f2 = add_h2(y1 & 0x00ff00ffu, kZero), f3 = add_h2(__byte_perm(y1, 0, 0x4341), kZero);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) mma16816(o[nt][2 * e + h], f0, f1, f2, f3, pb[nt][0], pb[nt][1]);
        }
    } else {
      constexpr uint32_t kPair = 0x000F000Fu, kZero = 0x80088008u, kZero16 = 0x80808080u;
#pragma unroll
      for (int e = 0; e < Y::kNb; ++e) {
        weigh(e);
        const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
        const uint32_t y0 = __byte_perm(v[0][0][e >> 1], v[1][0][e >> 1], sel);
        const uint32_t y1 = __byte_perm(v[2][0][e >> 1], v[3][0][e >> 1], sel);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // the odd value's nibble is taken where it lies, 16 times too large; undone at the end
          const uint32_t z0 = y0 >> 8 * h, z1 = y1 >> 8 * h;
          const uint32_t f0 = add_h2(z0 & kPair, kZero), f1 = add_h2(z0 & kPair << 4, kZero16);
          const uint32_t f2 = add_h2(z1 & kPair, kZero), f3 = add_h2(z1 & kPair << 4, kZero16);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) mma16816(o[nt][2 * e + h], f0, f1, f2, f3, pb[nt][0], pb[nt][1]);
        }
      }
    }
  }

  // ---- join the four warps through shared memory, in warp order
  copy_wait<0>();
  __syncthreads();
  float* om = reinterpret_cast<float*>(smem);                                  // [warp][row][kHP + 4]
  float2* mlw = reinterpret_cast<float2*>(om + kSWarps * 8 * kNT * (kHP + 4));  // [warp][row]
  const float unit = Y::kQ ? vs * 0x1p24f : 1.0f;
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      const int r = (warp * kNT + nt) * 8 + 2 * t + e;
      if (g == 0) mlw[r] = make_float2(m[nt][e], sum);
#pragma unroll
      for (int mt = 0; mt < Y::kMT; ++mt) {
        const float hi = kFmt == BQ4_CACHE_Q4 ? unit * 0.0625f : unit;
        *reinterpret_cast<float2*>(om + r * (kHP + 4) + Y::od(mt, g)) =
            make_float2(o[nt][mt][e] * unit, o[nt][mt][e + 2] * hi);
      }
    }
  __syncthreads();
  const int slots = s.p_chunks + s.s_chunks, slot = prefix ? chunk : s.p_chunks + chunk;
  for (int i = threadIdx.x; i < 8 * kNT * (kHP / 4); i += kSThreads) {
    const int r = i / (kHP / 4), d = 4 * (i - r * (kHP / 4));
    if (row0 + r >= rows) break;
    float top = kNone;
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) top = fmaxf(top, mlw[w * 8 * kNT + r].x);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) {
      const float2 e = mlw[w * 8 * kNT + r];
      const float f = ex2(e.x - top);
      const float4 y = *reinterpret_cast<const float4*>(om + (w * 8 * kNT + r) * (kHP + 4) + d);
      lsum += f * e.y;
      sum.x += f * y.x, sum.y += f * y.y, sum.z += f * y.z, sum.w += f * y.w;
    }
    const Row w = row_of(s, prefix, b, kvh, row0 + r);
    const int64_t row = ((int64_t)w.b * a.tokens + w.i) * a.q_heads + w.h;
    if (s.direct) {
      if (d < a.c.head_dim) {
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
        const uint2 u = make_uint2(pack_h2(sum.x * inv, sum.y * inv), pack_h2(sum.z * inv, sum.w * inv));
        *reinterpret_cast<uint2*>(a.out + row * a.c.head_dim + d) = u;
      }
    } else {
      *reinterpret_cast<float4*>(s.part + (row * slots + slot) * kHP + d) = sum;
      if (d == 0) s.ml[row * slots + slot] = make_float2(top, lsum);
    }
  }
}

// Joins a row's chunks in their order: one warp a row, four values a lane.
__global__ void __launch_bounds__(kSThreads) cache_join_kernel(const __grid_constant__ SplitArgs s, unsigned rows) {
  const CacheAttnCall& a = s.a;
  const unsigned row = blockIdx.x * kSWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, d = 4 * lane;
  ptx::griddep_wait();
  if (row >= rows) return;
  const unsigned bi = row / (unsigned)a.q_heads;
  const unsigned b = bi / (unsigned)a.tokens;
  int n = own_length(a, (int)b);
  if (a.causal) n = n - a.tokens + (int)(bi - b * a.tokens) + 1;
  const int np = (prefix_rows(a) + s.p_chunk - 1) / s.p_chunk;
  const int nc = np + (max(n, 0) + s.s_chunk - 1) / s.s_chunk;
  const int64_t at = (int64_t)row * (s.p_chunks + s.s_chunks);
  auto slot = [&](int i) { return at + (i < np ? i : s.p_chunks + i - np); };
  float top = kNone;
  for (int i = lane; i < nc; i += 32) top = fmaxf(top, s.ml[slot(i)].x);
#pragma unroll
  for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float lsum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < nc; ++i) {
    const float2 e = s.ml[slot(i)];
    const float f = ex2(e.x - top);
    lsum += f * e.y;
    if (d < a.c.hp) {
      const float4 y = *reinterpret_cast<const float4*>(s.part + slot(i) * a.c.hp + d);
      sum.x += f * y.x, sum.y += f * y.y, sum.z += f * y.z, sum.w += f * y.w;
    }
  }
  if (d < a.c.head_dim) {
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
    const uint2 u = make_uint2(pack_h2(sum.x * inv, sum.y * inv), pack_h2(sum.z * inv, sum.w * inv));
    *reinterpret_cast<uint2*>(a.out + (int64_t)row * a.c.head_dim + d) = u;
  }
}

// ------------------------------------------------------------------ host side

struct SplitPlan {
  int nt, p_tiles, s_tiles, p_chunk, s_chunk, p_chunks, s_chunks;
  int64_t p_items, s_items, slots, rows;
  size_t part_bytes, ml_bytes;
};

// Chunks of `keys` keys for `units` (kv head, row tile) pairs: as long as they
// leave three CTAs for every one that the GPU holds at a time (four an SM),
// so that sequences of unequal length even out.
int pick_chunk(int64_t keys, int64_t units, int sms) {
  const int64_t want = 3LL * 4 * sms;
  const int64_t per = keys * units / want / kMinChunk * kMinChunk;
  return (int)std::min<int64_t>(std::max<int64_t>(per, kMinChunk), kMaxChunk);
}

bool plan_split(const CacheAttnCall& a, int sms, SplitPlan* p) {
  const int group = a.q_heads / a.c.kv_heads;
  const int64_t own = (int64_t)a.tokens * group, all = own * a.s.batch;
  const int64_t prefix = (int64_t)a.prefix_width * a.c.page_size;
  p->nt = (prefix > 0 ? all : own) > 8 ? 2 : 1;
  const int tile = 8 * p->nt;
  p->s_tiles = (int)((own + tile - 1) / tile);
  p->p_tiles = (int)((all + tile - 1) / tile);
  p->s_chunk = pick_chunk(a.max_length, (int64_t)a.s.batch * a.c.kv_heads * p->s_tiles, sms);
  p->p_chunk = pick_chunk(prefix, (int64_t)a.c.kv_heads * p->p_tiles, sms);
  p->s_chunks = (int)(((int64_t)a.max_length + p->s_chunk - 1) / p->s_chunk);
  p->p_chunks = (int)((prefix + p->p_chunk - 1) / p->p_chunk);
  if (p->s_chunks + p->p_chunks == 0) p->s_chunks = 1;  // no keys at all: the rows are still written
  p->s_items = (int64_t)p->s_chunks * a.s.batch * a.c.kv_heads * p->s_tiles;
  p->p_items = (int64_t)p->p_chunks * a.c.kv_heads * p->p_tiles;
  p->slots = (int64_t)p->s_chunks + p->p_chunks;
  p->rows = (int64_t)a.s.batch * a.tokens * a.q_heads;
  if (p->s_items + p->p_items > 0x7fffffff || p->rows * p->slots > ((int64_t)1 << 40)) return false;
  const bool direct = p->slots == 1;
  p->part_bytes = direct ? 0 : (size_t)(p->rows * p->slots) * a.c.hp * 4;
  p->ml_bytes = direct ? 0 : (size_t)(p->rows * p->slots) * 8;
  return true;
}

template <int kFmt, int kHP, int kNT>
cudaError_t launch_split(const SplitArgs& s, unsigned grid, cudaStream_t stream) {
  using Y = Layout<kFmt, kHP>;
  constexpr int kRing = kSWarps * Y::kStages * Y::kStage;
  constexpr int kJoin = kSWarps * 8 * kNT * (kHP + 4) * 4 + kSWarps * 8 * kNT * 8;
  constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
  auto kernel = cache_split_kernel<kFmt, kHP, kNT>;
  static std::atomic<uint64_t> ready{0};  // a bit for each device
  int dev = 0;
  cudaGetDevice(&dev);
  if (kSmem > 48 * 1024 && (dev < 0 || dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  kernel<<<grid, kSThreads, kSmem, stream>>>(s);
  return cudaGetLastError();
}

template <int kFmt, int kHP>
cudaError_t launch_rows(const SplitArgs& s, int nt, unsigned grid, cudaStream_t stream) {
  return nt == 1 ? launch_split<kFmt, kHP, 1>(s, grid, stream) : launch_split<kFmt, kHP, 2>(s, grid, stream);
}

template <int kFmt>
cudaError_t launch_head(const SplitArgs& s, int nt, unsigned grid, cudaStream_t stream) {
  return s.a.c.hp == 64 ? launch_rows<kFmt, 64>(s, nt, grid, stream) : launch_rows<kFmt, 128>(s, nt, grid, stream);
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

bq4_status cache_attn_workspace(const CacheAttnCall& a, int sms, size_t* bytes) {
  SplitPlan p;
  if (!plan_split(a, sms, &p))
    return set_error(BQ4_EINVAL_SHAPE, "cache attention: too many rows and chunks for one launch");
  *bytes = up256(p.part_bytes) + up256(p.ml_bytes);
  return BQ4_OK;
}

bq4_status run_cache_attn(const CacheAttnCall& a, int sms, void* workspace, cudaStream_t stream) {
  SplitPlan p;
  if (!plan_split(a, sms, &p))
    return set_error(BQ4_EINVAL_SHAPE, "cache attention: too many rows and chunks for one launch");
  SplitArgs s;
  s.a = a;
  const uint64_t unit = (uint64_t)(a.c.page_size / kStep);
  s.page_magic = ((1ull << 38) + unit - 1) / unit;
  s.page_stride = (int64_t)a.c.kv_heads * 2 * a.c.kv_bytes;
  s.c = a.scale * 1.4426950408889634f;  // log2(e)
  s.group = a.q_heads / a.c.kv_heads;
  s.p_tiles = p.p_tiles;
  s.s_tiles = p.s_tiles;
  s.p_chunk = p.p_chunk;
  s.s_chunk = p.s_chunk;
  s.p_chunks = p.p_chunks;
  s.s_chunks = p.s_chunks;
  s.p_items = (unsigned)p.p_items;
  s.q_vec = reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && a.q_stride[0] % 4 == 0 && a.q_stride[1] % 4 == 0 &&
            a.q_stride[2] % 4 == 0;
  s.direct = p.slots == 1;
  s.part = static_cast<float*>(workspace);
  s.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + up256(p.part_bytes));
  const unsigned grid = (unsigned)(p.p_items + p.s_items);
  cudaError_t e = a.c.format == BQ4_CACHE_F16  ? launch_head<BQ4_CACHE_F16>(s, p.nt, grid, stream)
                  : a.c.format == BQ4_CACHE_Q8 ? launch_head<BQ4_CACHE_Q8>(s, p.nt, grid, stream)
                                               : launch_head<BQ4_CACHE_Q4>(s, p.nt, grid, stream);
  note_launch();
  if (e != cudaSuccess) return check_cuda(e, "cache attention launch");
  if (s.direct) return BQ4_OK;
  // the join is launched ahead and waits on the device for the chunks
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.rows + kSWarps - 1) / kSWarps));
  cfg.blockDim = dim3(kSThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, cache_join_kernel, s, (unsigned)p.rows);
  note_launch();
  return check_cuda(e, "cache attention join launch");
}

}  // namespace bq4
