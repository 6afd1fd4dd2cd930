// bq4_cache_attn.cu -- attention over the paged key/value cache: out =
// softmax(scale q K^T + mask) V for the newest tokens of every sequence, the
// keys being a prefix that the whole batch shares (if any) and the
// sequence's own rows.
//
// The work is a line of units of 64 keys: for every kv head and tile of 8 kNT
// query rows (the tokens and grouped heads that read this kv head; for the
// prefix those of the whole batch, so that it is read once) the units of the
// prefix, then those of each sequence, each such range with four empty units
// ahead for what its start and end cost (without them the CTAs of short
// sequences end late: 64 ragged sequences in 4 bits 91.3 us, 86.6 with them).
// The lengths are on the device, so every CTA adds them up itself and takes one
// share of the line, as many units as every other: one wave, whatever the
// lengths.  A share is cut where one (head, tile)'s keys end; each such piece
// keeps a running maximum, sum l and product O in f32.  Rows that one piece
// covers are finished at once; cache_join_kernel joins the others: O = sum_c
// 2^(m_c - M) O_c, l likewise, pieces in their order, so that a call gives the
// same bits every time.  Calls with many rows a kv head run the kernels of
// bq4_cache_tile.cu instead (plan_cache).
//
// cache_split_kernel: four warps, each its own 16-key steps.
//   * Keys are the M side of the tensor core's m16n8k16 (f16 in, f32 out) and
//     the query rows its N side: S^T = K Q^T, then O^T = V^T P^T.  A group of 4
//     query heads fills half of N = 8, not a quarter of M = 16, and the widened
//     cache values (A) are made once for all rows.
//   * The 16 rows of a step lie together in their page (k, v and scales): one
//     lane brings them to a ring of the warp's own with one bulk copy, some
//     steps ahead; an mbarrier says when they are there.  No warp waits for
//     another in the loop.
//   * Lane (g = lane / 4, t = lane % 4) reads quarter t of k rows g and g + 8
//     and eighth g of v rows 2t, 2t + 1, 2t + 8, 2t + 9, 16 bytes at a time.  Any
//     order of the head's values inside a fragment is as good as another as
//     long as q follows it.
//   * Stored values are whole numbers u = q + 128 (q + 8).  Zero-extended to
//     16 bits they are the subnormal halves u 2^-24, exact in the tensor core:
//     widening a pair of k values is one byte permute (q8) or mask (q4, every
//     second pair 16 times too large, against a sixteenth of q).  The
//     offset leaves the scores through the accumulator's start value -128
//     2^-24 sum(q) (f32; q4: for each scale's 32 values).  v is made signed, one
//     add a pair: in O = sum p v, over many keys, an offset would cost the sum
//     its low bits (taking it out in every step, by a product with A = -128
//     2^-24, left values of q = 0 up to 2^-17 of the offset away from 0).
//   * k scales multiply the f32 scores.  v scales multiply the probabilities,
//     p s_v as f16 (off by 2^-11 of it; the only rounding to fewer than 32 bits
//     besides the result's).  To fill f16's range p is 2^(x - base), where base
//     is 2^6 below the running maximum of s_v 2^x; l and O are both relative to
//     it.
//   * base only moves when some p s_v would pass 2^14 (a vote, no shuffles in
//     the common step).
//   * Steps that every row sees whole run without any mask.
//
// What bounds it (148 SMs, 6.57 TB/s copied): for f16 rows HBM, and the start and
// end of the one wave (16 sequences of 3000 to 4352 rows of 64 values, 118 MB:
// 26.7 us, 0.67 of the copy rate); for 4 bits dependent instructions at low
// occupancy (64 sequences of 300 to 8192 rows, 314 MB: 85 us, 0.56; some 350
// instructions a warp and step of 2304 bytes, of which 50 widen k, 70 v and 40
// weigh p for the four v scales, 0.54 of the issue slots with 2.8 warps a
// scheduler, which mostly wait for an instruction before); latency for one short
// sequence (1000 rows: 7.6 us, of which 3 are two launches' starts).
// Taken on the way, device time: one warp a row 692 / 8502 us for one sequence
// of 1000 rows / the 64 sequences; these tiles with 16-byte copies by each lane
// 21.5 / 109; equal shares and bulk copies 16 / 120; a join with its loads in
// flight 8.2; steps without masks 7.5 / 99; one copy a step 93.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "bq4_cache.h"
#include "cache_bounds.h"
#include "sm100_ptx.cuh"

namespace bq4 {
namespace {

constexpr int kSWarps = 4;
constexpr int kSThreads = 32 * kSWarps;
constexpr int kStep = 16;                     // keys of a warp's step
constexpr int kUnit = kStep * kSWarps;        // one step a warp
constexpr int kLead = 4;                      // units that a range counts for its start and end
constexpr float kNone = -1e30f;               // the maximum of no score (finite: differences stay defined)
constexpr float kHead = 6.0f, kJump = 14.0f;  // log2 units: where base leaves p s_v, and where it moves

// kWords 32-bit words from shared memory.
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

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// CTAs of the split kernel that an SM holds: 384 threads leave 168 registers
// each, 512 leave 128.  16 rows a warp of 128 values spill at 168 (28 bytes stored
// for f16, 52 for 8 bits, 164 for 4) and still gain (a draft of 24 rows, 8 bits,
// 32.0 -> 28.5 us against two CTAs of 255); 8 rows of 4 bits keep their start values
// in registers at 168 (93.0 -> 91.3 us); f16's ring allows three; 24 rows take 255,
// and spill 20 bytes for f16 and 208 for 4 bits.
constexpr int split_per_sm(int format, int hp, int nt) {
  if (nt == 3) return 2;
  if (nt == 2) return 3;
  return format != BQ4_CACHE_Q8 && hp == 128 ? 3 : 4;
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
  // a stage: 16 k rows, 16 v rows, 16 tokens' scales
  static constexpr int kOffV = kStep * kRow;
  static constexpr int kOffS = 2 * kStep * kRow;
  static constexpr int kStage = kOffS + kStep * kScale;
  // CTAs of an SM, by registers and by the ring
  static constexpr int per_sm(int nt) { return split_per_sm(kFmt, kHP, nt); }
  static constexpr int kRing = (per_sm(1) == 3 ? 72 : 54) * 1024;  // bytes, about
  static constexpr int kStages = kRing / (kSWarps * kStage) < 8 ? kRing / (kSWarps * kStage) : 8;
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
  float c;               // scale * log2(e)
  int group;             // query heads of a kv head
  int p_tiles, s_tiles;  // row tiles of the prefix and of one sequence
  int q_vec;             // q rows lie on 8-byte boundaries
  int finish;            // rows of one piece are finished (there is no other source)
  float* part;           // [grid + ranges][8 kNT][hp]: O of piece (CTA + range)
  float2* ml;            // [grid + ranges][8 kNT]: m, l
  int2* pieces;          // [ranges]: first and last CTA with keys of the range
};

// A range is the line's units of one (kv head, row tile): prefix ranges
// [kv_heads][p_tiles] first, then [batch][kv_heads][s_tiles].  Piece CTA +
// range is unique: from one piece to the next one of them grows.

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
// Units of the line that a range of n keys takes.
__device__ __forceinline__ unsigned units_of(int n) { return n > 0 ? (unsigned)(n + kUnit - 1) / kUnit + kLead : 0; }

__device__ __forceinline__ int prefix_rows(const CacheAttnCall& a) {
  return a.prefix_length ? clamp_length(a.prefix_length[0], (int64_t)a.prefix_width * a.c.page_size, a.err) : 0;
}

template <int kFmt, int kHP, int kNT>
__global__ void __launch_bounds__(kSThreads, Layout<kFmt, kHP>::per_sm(kNT))
    cache_split_kernel(const __grid_constant__ SplitArgs s) {
  using Y = Layout<kFmt, kHP>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned before[kSThreads + 1];
  __shared__ unsigned warp_sum[kSWarps];
  __shared__ __align__(8) uint64_t bars[kSWarps * Y::kStages];
  __shared__ int abort_flag;
  const CacheAttnCall& a = s.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  ptx::griddep_launch_dependents();
  if (threadIdx.x < kSWarps * Y::kStages) ptx::mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) abort_flag = 0;
  ptx::fence_mbar_init();

  // ---- the line: units before each sequence (a thread adds up `per` of them; the host
  // bounds the line by 2^31)
  const int n_prefix = prefix_rows(a);
  const unsigned per_p = units_of(n_prefix);
  const unsigned line_p = per_p * (unsigned)(a.c.kv_heads * s.p_tiles);
  const unsigned heads_tiles = (unsigned)(a.c.kv_heads * s.s_tiles);
  const int per = (a.s.batch + kSThreads - 1) / kSThreads;
  {
    unsigned sum = 0;
    for (int i = 0; i < per; ++i) {
      const int sb = (int)threadIdx.x * per + i;
      if (sb < a.s.batch) sum += units_of(own_length(a, sb));
    }
    sum *= heads_tiles;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, sum, w);
      if (lane >= w) sum += y;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    for (int w = 0; w < warp; ++w) sum += warp_sum[w];
    before[threadIdx.x + 1] = line_p + sum;
    if (threadIdx.x == 0) before[0] = line_p;
    __syncthreads();
  }
  const unsigned line = before[kSThreads], share = (line + gridDim.x - 1) / gridDim.x;
  unsigned at_unit = blockIdx.x * share;  // below line + share
  const unsigned to_unit = min(line, at_unit + share);
  if (at_unit >= to_unit) return;

  // ---- the range that holds at_unit
  bool prefix = at_unit < line_p;
  int b = 0, tile, kvh, n;
  unsigned units, first;  // of the range, along the line
  if (prefix) {
    const int r = (int)(at_unit / per_p);
    tile = r % s.p_tiles;
    kvh = r / s.p_tiles;
    first = (unsigned)r * per_p;
    n = n_prefix;
    units = per_p;
  } else {
    int lo = 0, hi = kSThreads;  // before[lo] <= at_unit < before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= at_unit) lo = mid; else hi = mid;
    }
    first = before[lo];
    b = lo * per;
    for (;; ++b) {
      n = own_length(a, b);
      units = units_of(n);
      if (at_unit < first + units * heads_tiles) break;
      first += units * heads_tiles;
    }
    const int r = (int)((at_unit - first) / units);
    tile = r % s.s_tiles;
    kvh = r / s.s_tiles;
    first += (unsigned)r * units;
  }

  // this warp's ring: the stages to fill and to take next, and the parity of the latter
  const uint32_t ring = ptx::smem_u32(smem) + warp * Y::kStages * Y::kStage;
  uint64_t* full = bars + warp * Y::kStages;
  int put = 0, get = 0;
  uint32_t parity = 0;
  // lane offsets of its pieces in a stage; k rows g, g + 8 and v rows 2t (+ 8), 2t + 1 (+ 8) lie alike
  const uint32_t k_at = cache_swizzle(0, Y::kRow, g, t * Y::kKPiece);
  const uint32_t v_at0 = Y::kOffV + cache_swizzle(1, Y::kRow, 2 * t, g * Y::kVPiece);
  const uint32_t v_at1 = Y::kOffV + cache_swizzle(1, Y::kRow, 2 * t + 1, g * Y::kVPiece);

  for (;;) {  // a piece a turn
    const int range = prefix ? kvh * s.p_tiles + tile
                             : a.c.kv_heads * s.p_tiles + (b * a.c.kv_heads + kvh) * s.s_tiles + tile;
    const unsigned piece_to = min(to_unit, first + units);
    const int key0 = max((int)(at_unit - first) - kLead, 0) * kUnit;
    const int piece_end = ((int)(piece_to - first) - kLead) * kUnit;  // not above 0: only the lead
    const int rows = (prefix ? a.s.batch : 1) * a.tokens * s.group;
    const int row0 = tile * 8 * kNT;
    const bool causal = !prefix && a.causal;
    // the keys that the tile's last row sees
    const int last_i = (min(row0 + 8 * kNT, rows) - 1) / s.group;
    const int end = min(min(n, piece_end), causal ? n - a.tokens + last_i + 1 : n);
    const bool whole = key0 == 0 && piece_to == first + units;
    if (key0 == 0 && piece_end > 0 && threadIdx.x == 0)  // the range's first keys
      s.pieces[range] = make_int2((int)blockIdx.x, (int)((first + units - 1) / share));
    const int32_t* table = prefix ? a.prefix_table : a.s.table + b * a.s.table_stride;

    if (piece_end > 0) {
    // ---- steps of this warp; lane j % 32 knows where step j lies, for the 32 steps fetched last
    const int steps = end <= key0 ? 0 : (end - key0 + kStep - 1) / kStep;
    const int mine = steps > warp ? (steps - warp + kSWarps - 1) / kSWarps : 0;
    const int at0 = key0 + warp * kStep;  // first key of step 0; step j lies kUnit j on
    const uint8_t* src = nullptr;
    unsigned held = 0, held_before = 0;   // bit j % 32: step j's page exists; of the 32 steps before them
    int plain = mine;                     // steps below it have a page and no mask
    auto locate = [&](int j) {
      bool ok = true;
      if (j + lane < mine) {
        const unsigned u = (unsigned)(at0 / kStep + kSWarps * (j + lane));
        const int pi = (int)((u * s.page_magic) >> 38);
        int page = table[pi];
        const int place = (int)u * kStep - pi * a.c.page_size;
        ok = page >= 0 && page < a.c.pages;
        if (!ok) {
          atomicCAS(a.err, 0, (int)BQ4_EINVAL_ARG);
          page = 0;
        }
        src = cache_step(a.c, page, kvh, place);
      }
      held_before = held;
      held = __ballot_sync(0xffffffffu, ok);
      if (held != 0xffffffffu) plain = min(plain, j);
    };
    // one bulk copy brings step j, by the lane that knows it (of a step without a page, page 0's
    // rows: they are masked)
    auto fetch = [&](int j) {
      if (j >= mine) return;
      if ((j & 31) == 0) locate(j);
      if (lane == (j & 31)) {
        ptx::mbar_arrive_expect_tx(&full[put], Y::kStage);
        ptx::bulk_load(smem + (warp * Y::kStages + put) * Y::kStage, src, Y::kStage, &full[put]);
      }
      put = put + 1 == Y::kStages ? 0 : put + 1;
    };
    for (int j = 0; j < Y::kStages - 1; ++j) fetch(j);

    // ---- q fragments; the offset's start values; what each row sees
    uint32_t q[kNT][Y::kKS][2];
    constexpr int kOffs = kFmt == BQ4_CACHE_Q4 ? Y::kNb : 1;  // start values of a row
    float off[kNT][kOffs][2];
    float unit[kNT][2];  // 4 bits: log2-unit scores of rows 2t, 2t + 1 from their sums
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
      if constexpr (kFmt == BQ4_CACHE_Q4) {
        // q times a power of two that brings the row's largest into [2^9, 2^10): then every second
        // pair can be divided by 16 (below) without leaving f16's range
        uint32_t most = 0;
#pragma unroll
        for (int ks = 0; ks < Y::kKS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            most = max(most, max(q[nt][ks][e] & 0x7fffu, q[nt][ks][e] >> 16 & 0x7fffu));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));  // of row g
        const float top = __half2float(__ushort_as_half((unsigned short)most));
        const int lift = most ? 9 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;  // [-7, 33]
        const float up = __uint_as_float((uint32_t)(127 + lift) << 23);
        const float down = __uint_as_float((uint32_t)(127 - lift) << 23);
        unit[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t) * (s.c * 0x1p24f);
        unit[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4) * (s.c * 0x1p24f);
#pragma unroll
        for (int ks = 0; ks < Y::kKS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[nt][ks][e]));
            q[nt][ks][e] = pack_h2(f.x * up, f.y * up);
          }
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
        if constexpr (kFmt == BQ4_CACHE_Q4) {
#pragma unroll
          for (int ks = 0; ks < Y::kKS; ++ks) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[nt][ks][1]));
            q[nt][ks][1] = pack_h2(f.x * 0.0625f, f.y * 0.0625f);
          }
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
    plain = min(plain, max(0, (see_all - at0 + kUnit - kStep) / kUnit));

    float base[kNT][2], l[kNT][2], o[kNT][Y::kMT][4];  // p = 2^(x - base)
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      base[nt][0] = base[nt][1] = kNone;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < Y::kMT; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
    }
    const float c = Y::kQ ? s.c * 0x1p24f : s.c;

    // One step: false when its rows did not come.  kEdge: some row does not see some key, or
    // the step has no page.
    auto step = [&](auto edge_tag, int j) -> bool {
      constexpr bool kEdge = decltype(edge_tag)::value;
      __syncwarp();  // the slot that is filled next has been read by every lane
      fetch(j + Y::kStages - 1);
      const int at = at0 + kUnit * j;
      const uint32_t st = ring + get * Y::kStage;
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[get], parity, &abort_flag))) return false;
      if (++get == Y::kStages) get = 0, parity ^= 1;
      int limit[kNT][2];  // keys of this step that a row sees, less this lane's g
      if constexpr (kEdge) {
        // the fetches are kStages - 1 steps ahead, perhaps among the next 32 already
        const bool next = (min(j + Y::kStages - 1, mine - 1) >> 5) != (j >> 5);
        const bool none = !((next ? held_before : held) >> (j & 31) & 1);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) limit[nt][e] = none ? -16 : see[nt][e] - at - g;
      }

      // ---- scales of keys g, g + 8
      float sk[2][Y::kQ ? Y::kNb : 1] = {}, sv[2][Y::kQ ? Y::kNb : 1] = {};
      if constexpr (Y::kQ) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t w[Y::kNb];
          lds(st + Y::kOffS + (g + 8 * r) * Y::kScale, w);
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
          if constexpr (kEdge) {  // rows behind the end hold anything
            if (at + g + 8 * r >= end)
#pragma unroll
              for (int e = 0; e < Y::kNb; ++e) sv[r][e] = 0.0f;
          }
        }
      }

      // ---- scores of keys g (0, 1) and g + 8 (2, 3) with rows 2t, 2t + 1
      float x[kNT][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        x[nt][0] = x[nt][2] = kFmt == BQ4_CACHE_Q4 ? 0.0f : off[nt][0][0];
        x[nt][1] = x[nt][3] = kFmt == BQ4_CACHE_Q4 ? 0.0f : off[nt][0][1];
      }
#pragma unroll
      for (int p = 0; p < Y::kKPieces; ++p) {
        uint32_t w0[Y::kKPiece / 4], w1[Y::kKPiece / 4];
        const uint32_t from = st + (k_at ^ p << 6);  // 4 pieces of 16 bytes on; the swizzle is in bit 6
        lds(from, w0);
        lds(from + 8 * Y::kRow, w1);
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
              // every second pair is taken where it lies, 16 times too large, against q / 16
              const uint32_t z0 = w0[e] >> 8 * h, z1 = w1[e] >> 8 * h;
              const uint32_t a0 = z0 & kPair, a2 = z0 & kPair << 4, a1 = z1 & kPair, a3 = z1 & kPair << 4;
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

      // ---- z = x - base, x in log2 units; a masked key's is -inf
      const float c0 = kFmt == BQ4_CACHE_Q8 ? sk[0][0] * c : c, c1 = kFmt == BQ4_CACHE_Q8 ? sk[1][0] * c : c;
      // log2 of the keys' largest v scales; not below -64, so that beside a v of 0 the sum of 2^30
      // p of at most 2^(14 + 64) stays in f32 (scales below that are 0 in an f16 result)
      float lg[2] = {0.0f, 0.0f};
      if constexpr (Y::kQ) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = sv[r][0];
#pragma unroll
          for (int e = 1; e < Y::kNb; ++e) top = fmaxf(top, sv[r][e]);
          lg[r] = fmaxf(lg2(top), -64.0f);
        }
      }
      float z[kNT][4];
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          z[nt][u] = fmaf(x[nt][u], kFmt == BQ4_CACHE_Q4 ? unit[nt][u & 1] : u < 2 ? c0 : c1, -base[nt][u & 1]);
          if (kEdge && limit[nt][u & 1] <= 8 * (u >> 1)) z[nt][u] = -INFINITY;
        }
        move |= fmaxf(fmaxf(z[nt][0], z[nt][1]) + lg[0], fmaxf(z[nt][2], z[nt][3]) + lg[1]) > kJump;
      }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x0 = x[nt][e] * (kFmt == BQ4_CACHE_Q4 ? unit[nt][e] : c0);
            float x1 = x[nt][e + 2] * (kFmt == BQ4_CACHE_Q4 ? unit[nt][e] : c1);
            if (kEdge && limit[nt][e] <= 0) x0 = -INFINITY;
            if (kEdge && limit[nt][e] <= 8) x1 = -INFINITY;
            float top = fmaxf(x0 + lg[0], x1 + lg[1]);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            float alpha = 1.0f;
            if (top - base[nt][e] > kJump) {
              alpha = ex2(base[nt][e] - (top - kHead));
              base[nt][e] = top - kHead;
            }
            z[nt][e] = x0 - base[nt][e];
            z[nt][e + 2] = x1 - base[nt][e];
            l[nt][e] *= alpha;
#pragma unroll
            for (int mt = 0; mt < Y::kMT; ++mt) {
              o[nt][mt][e] *= alpha;
              o[nt][mt][e + 2] *= alpha;
            }
          }
      }

      // ---- p, its sum, and p s_v as f16 in the B layout
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          z[nt][u] = ex2(z[nt][u]);
          l[nt][u & 1] += z[nt][u];
        }
      uint32_t pb[kNT][2];
      auto weigh = [&](int e) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            y[u] = Y::kQ ? z[nt][u] * sv[u >> 1][Y::kQ ? e : 0] : z[nt][u];
            // a masked key's scale may be NaN
            if (kEdge && Y::kQ && limit[nt][u & 1] <= 8 * (u >> 1)) y[u] = 0.0f;
          }
          pb[nt][0] = transpose8(pack_h2(y[0], y[1]));
          pb[nt][1] = transpose8(pack_h2(y[2], y[3]));
        }
      };

      // ---- O^T += V^T P^T
      uint32_t v[4][Y::kVPieces][Y::kVPiece / 4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int p = 0; p < Y::kVPieces; ++p)
          lds(st + (r & 1 ? v_at1 : v_at0) + (r >> 1) * 8 * Y::kRow + p * 128, v[r][p]);
      if constexpr (kFmt == BQ4_CACHE_F16) {
        weigh(0);
#pragma unroll
        for (int p = 0; p < Y::kVPieces; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t f[4] = {__byte_perm(v[0][p][e], v[1][p][e], 0x5410), __byte_perm(v[0][p][e], v[1][p][e], 0x7632),
                             __byte_perm(v[2][p][e], v[3][p][e], 0x5410), __byte_perm(v[2][p][e], v[3][p][e], 0x7632)};
            const int mt = 4 * p + e;
            if constexpr (kEdge) {
              // A key that some row does not see may hold infinities or NaN: they leave the
              // product, which would carry 0 * NaN into that row, and reach the rows that
              // see the key one by one.  f[r]: keys 2t, 2t + 1 (r < 2) or + 8, value d + (r & 1).
              bool odd = false;
#pragma unroll
              for (int r = 0; r < 4; ++r)
                odd |= (f[r] & 0x00007c00u) == 0x00007c00u || (f[r] & 0x7c000000u) == 0x7c000000u;
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
                      const int key = 2 * w + h + 8 * (r >> 1);
                      const float add = __half2float(__ushort_as_half((unsigned short)bits));
                      if (bits) {
#pragma unroll
                        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                          for (int e2 = 0; e2 < 2; ++e2)
                            if (key < limit[nt][e2] + g) o[nt][mt][e2 + 2 * (r & 1)] += add;
                      }
                    }
                  }
                }
              }
            }
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma16816(o[nt][mt], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
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
      return true;
    };
    int j = 0;
    while (j < plain && step(std::false_type{}, j)) ++j;
    if (j >= plain)
      while (j < mine && step(std::true_type{}, j)) ++j;
    if (j < mine && lane == 0) {  // rows that did not come
      abort_flag = 1;
      atomicCAS(a.err, 0, (int)BQ4_ETIMEOUT);
    }

    // ---- join the four warps through shared memory, in warp order
    __syncthreads();
    if (abort_flag) {
      // wait once more for the copies under way (put == get may mean none or a full ring), then leave
      __shared__ int never;
      if (threadIdx.x == 0) never = 0;
      __syncthreads();
      for (int left = cache_pending(j, mine, Y::kStages); left > 0; --left) {
        ptx::mbar_wait(&full[get], parity, &never);
        if (++get == Y::kStages) get = 0, parity ^= 1;
      }
      return;
    }
    float* om = reinterpret_cast<float*>(smem);                                  // [warp][row][kHP + 4]
    float2* mlw = reinterpret_cast<float2*>(om + kSWarps * 8 * kNT * (kHP + 4));  // [warp][row]
    constexpr float kLo = Y::kQ ? 0x1p24f : 1.0f, kHi = kFmt == BQ4_CACHE_Q4 ? 0x1p20f : kLo;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const int r = (warp * kNT + nt) * 8 + 2 * t + e;
        if (g == 0) mlw[r] = make_float2(base[nt][e], sum);
#pragma unroll
        for (int mt = 0; mt < Y::kMT; ++mt)
          *reinterpret_cast<float2*>(om + r * (kHP + 4) + Y::od(mt, g)) =
              make_float2(o[nt][mt][e] * kLo, o[nt][mt][e + 2] * kHi);
      }
    __syncthreads();
    const int64_t piece = ((int64_t)blockIdx.x + range) * 8 * kNT;
    const bool finish = whole && s.finish && line_p == 0;
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
      if (finish) {
        if (d < a.c.head_dim) {
          const Row w = row_of(s, prefix, b, kvh, row0 + r);
          const int64_t row = ((int64_t)w.b * a.tokens + w.i) * a.q_heads + w.h;
          const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
          const uint2 u = make_uint2(pack_h2(sum.x * inv, sum.y * inv), pack_h2(sum.z * inv, sum.w * inv));
          *reinterpret_cast<uint2*>(a.out + row * a.c.head_dim + d) = u;
        }
      } else {
        *reinterpret_cast<float4*>(s.part + (piece + r) * kHP + d) = sum;
        if (d == 0) s.ml[piece + r] = make_float2(top, lsum);
      }
    }

    ptx::fence_proxy_async_smem();  // the copies write where the warps were joined
    }

    // ---- the next range of the line
    at_unit = piece_to;
    if (at_unit >= to_unit) return;
    __syncthreads();
    first += units;
    if (++tile == (prefix ? s.p_tiles : s.s_tiles)) {
      tile = 0;
      if (++kvh == a.c.kv_heads) {
        kvh = 0;
        b = prefix ? 0 : b + 1;
        prefix = false;
        for (;; ++b) {
          n = own_length(a, b);
          units = units_of(n);
          if (units) break;
        }
      }
    }
  }
}

struct JoinArgs {
  CacheAttnCall a;
  CacheJoinSource p, s;  // of the prefix and of the sequences' own keys
  int group, have_p, finish;
  int first;  // sequences before a's in the batch whose rows the prefix's partial results are
};

// Slots of row r (of `rows`) of kv head kvh that sees `see` keys: first and number.
__device__ __forceinline__ int2 slots_of(const JoinArgs& g, const CacheJoinSource& s, int set, int kvh, int r, int rows,
                                         int keys, bool causal) {
  const int tile = r / s.tile_rows;
  if (s.pieces) {
    const int range = s.first_range + (set * g.a.c.kv_heads + kvh) * s.tiles + tile;
    if (keys <= 0) return make_int2(0, 0);
    const int2 cta = s.pieces[range];
    const CacheSlots c = cache_slots(cta.x, cta.y, range, s.grid);
    return make_int2(c.first, c.count);
  }
  const int last_i = (min((tile + 1) * s.tile_rows, rows) - 1) / g.group;
  const int end = max(0, causal ? keys - g.a.tokens + last_i + 1 : keys);
  const int range = (set * s.tiles + tile) * g.a.c.kv_heads + kvh;
  return make_int2(range * s.chunks, (((end + 127) / 128) * 128 + s.span - 1) / s.span);
}

// Joins a row's partial results, the prefix's and then its own in their order.
// kWarps warps of a CTA take turns at a row's slots (four when the rows are few:
// what a row takes then is the latency of its loads; 17 slots 16.7 us one load
// after the other, 4.4 us so), four values a lane and four slots' loads in flight;
// the first joins what each has.
template <int kWarps>
__global__ void __launch_bounds__(kSThreads) cache_join_kernel(const __grid_constant__ JoinArgs g, unsigned rows) {
  constexpr int kAhead = 4;
  const CacheAttnCall& a = g.a;
  const int warp = (threadIdx.x >> 5) % kWarps, lane = threadIdx.x & 31, d = 4 * lane;
  const unsigned row = blockIdx.x * (kSWarps / kWarps) + (threadIdx.x >> 5) / kWarps;
  ptx::griddep_wait();
  if (row >= rows) return;  // a CTA of four warps a row has one row: all leave
  const int bi = (int)(row / (unsigned)a.q_heads), h = (int)row - bi * a.q_heads;
  const int b = bi / a.tokens, kvh = h / g.group, per = a.tokens * g.group;
  const int own = (bi - b * a.tokens) * g.group + h - kvh * g.group;  // row among the sequence's
  const int all = (g.first + b) * per + own;                         // among the prefix's
  int2 sp = make_int2(0, 0);
  if (g.have_p) sp = slots_of(g, g.p, 0, kvh, all, a.s.batch * per, prefix_rows(a), false);
  const int2 ss = slots_of(g, g.s, b, kvh, own, per, own_length(a, b), a.causal);
  if (g.finish && sp.y == 0 && ss.y == 1) return;  // finished by its one piece
  float top = kNone, lsum = 0.0f;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto take = [&](const CacheJoinSource& s, int2 slots, int local) {
    const int64_t first = (int64_t)slots.x * s.tile_rows + local;
    const float2* ml = s.ml + first;
    const float* part = s.part + first * a.c.hp + d;
    for (int i = warp; i < slots.y; i += kWarps * kAhead) {
      float2 e[kAhead];
      float4 y[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = i + u * kWarps;
        e[u] = make_float2(kNone, 0.0f);
        y[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < slots.y) {
          e[u] = __ldcg(ml + (int64_t)k * s.tile_rows);
          if (d < a.c.hp) y[u] = __ldcg(reinterpret_cast<const float4*>(part + (int64_t)k * s.tile_rows * a.c.hp));
        }
      }
      float next = top;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) next = fmaxf(next, e[u].x);
      const float f = ex2(top - next);
      top = next;
      lsum *= f;
      sum.x *= f, sum.y *= f, sum.z *= f, sum.w *= f;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float w = ex2(e[u].x - top);
        lsum += w * e[u].y;
        sum.x += w * y[u].x, sum.y += w * y[u].y, sum.z += w * y[u].z, sum.w += w * y[u].w;
      }
    }
  };
  if (sp.y) take(g.p, sp, all % g.p.tile_rows);
  take(g.s, ss, own % g.s.tile_rows);
  if constexpr (kWarps > 1) {
    __shared__ float4 sums[kWarps][32];
    __shared__ float2 mls[kWarps];
    sums[warp][lane] = sum;
    if (lane == 0) mls[warp] = make_float2(top, lsum);
    __syncthreads();
    if (warp) return;
    top = kNone;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, mls[w].x);
    lsum = 0.0f;
    sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(mls[w].x - top);
      const float4 y = sums[w][lane];
      lsum += f * mls[w].y;
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

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct SplitPlan {
  int nt, p_tiles, s_tiles, grid;
  size_t part_bytes, ml_bytes, pieces_bytes, bytes;
};

// The plan with nt eights of rows a warp: CTAs are what the GPU holds at a time, or fewer
// where the lengths' bounds give fewer units.
bool plan_rows(const CacheAttnCall& a, int nt, int sms, SplitPlan* p) {
  const int group = a.q_heads / a.c.kv_heads;
  const int64_t own = (int64_t)a.tokens * group, all = own * a.s.batch;
  const int64_t prefix = (int64_t)a.prefix_width * a.c.page_size;
  p->nt = nt;
  const int tile = 8 * p->nt;
  p->s_tiles = (int)((own + tile - 1) / tile);
  p->p_tiles = prefix > 0 ? (int)((all + tile - 1) / tile) : 0;
  const int64_t ranges = ((int64_t)p->p_tiles + (int64_t)a.s.batch * p->s_tiles) * a.c.kv_heads;
  const int64_t per = a.max_length ? ((int64_t)a.max_length + kUnit - 1) / kUnit + kLead : 0;
  const int64_t per_p = prefix ? (prefix + kUnit - 1) / kUnit + kLead : 0;
  const int64_t most = (int64_t)split_per_sm(a.c.format, a.c.hp, p->nt) * sms;
  const int64_t units = std::min(most, per_p * p->p_tiles * a.c.kv_heads) +
                        std::min(most, per * std::min(most, (int64_t)a.s.batch * p->s_tiles * a.c.kv_heads));
  p->grid = (int)std::max<int64_t>(1, std::min(most, units));
  const int64_t slots = (ranges + p->grid) * tile;
  // the line's units and the ranges are counted in 32 bits
  if (ranges > 0x3fffffff || per_p * p->p_tiles * a.c.kv_heads > 0x3fffffff ||
      (per > 0 && (int64_t)a.s.batch * p->s_tiles * a.c.kv_heads > 0x3fffffff / per))
    return false;
  p->part_bytes = up256((size_t)slots * a.c.hp * 4);
  p->ml_bytes = up256((size_t)slots * 8);
  p->pieces_bytes = up256((size_t)ranges * 8);
  p->bytes = p->part_bytes + p->ml_bytes + p->pieces_bytes;
  return true;
}

// Rows of a warp, in eights: a step costs about as much for its widening as for
// 16 rows, so the tiles are those that cost least together, over the keys of the
// prefix and of the sequences (24 rows as one tile 25.5 us, as two of 16 27.1; 128
// single tokens on 2000 rows in 4 bits behind 16 shared ones, where the prefix's 512
// rows alone would take three, 205 -> 91), among those that `room` bytes hold.
bool plan_split(const CacheAttnCall& a, int sms, size_t room, SplitPlan* p) {
  constexpr double kStart = kLead * kUnit;  // keys that a range's start and end count for
  const double own_keys = a.max_length ? a.s.batch * (a.max_length + kStart) : 0.0;
  const double prefix_keys = a.prefix_width ? (double)a.prefix_width * a.c.page_size + kStart : 0.0;
  bool found = false;
  double least = 0.0;
  for (int nt = 1; nt <= 3; ++nt) {
    SplitPlan t;
    if (!plan_rows(a, nt, sms, &t) || t.bytes > room) continue;
    const int64_t all = ((int64_t)a.tokens * (a.q_heads / a.c.kv_heads) * a.s.batch + 8 * nt - 1) / (8 * nt);
    const double cost = (2.0 + nt) * ((double)t.s_tiles * own_keys + (double)all * prefix_keys);
    if (!found || cost < least) found = true, least = cost, *p = t;
  }
  return found;
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
  // (the static part comes on top)
  if (kSmem > 46 * 1024 && (dev < 0 || dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  kernel<<<grid, kSThreads, kSmem, stream>>>(s);
  return cudaGetLastError();
}

template <int kFmt, int kHP>
cudaError_t launch_rows(const SplitArgs& s, int nt, unsigned grid, cudaStream_t stream) {
  return nt == 1   ? launch_split<kFmt, kHP, 1>(s, grid, stream)
         : nt == 2 ? launch_split<kFmt, kHP, 2>(s, grid, stream)
                   : launch_split<kFmt, kHP, 3>(s, grid, stream);
}

template <int kFmt>
cudaError_t launch_head(const SplitArgs& s, int nt, unsigned grid, cudaStream_t stream) {
  return s.a.c.hp == 64 ? launch_rows<kFmt, 64>(s, nt, grid, stream) : launch_rows<kFmt, 128>(s, nt, grid, stream);
}

// Which kernels take the prefix's and the sequences' own keys, and their workspaces.
struct CachePlan {
  bool tile_p, tile_s;
  CacheTilePlan p, s;  // s: of `slice` sequences, one slice after the other
  int slice;
  SplitPlan split;
  CacheAttnCall call;  // of the split kernel: without a prefix that the tile kernel takes
  size_t bytes;
};

// The tile kernels widen a key set once for all its rows and then take 256 rows
// at a time; the split kernel widens it for every 8 to 24 rows.  Their times in
// us, fitted to calls of 16 to 256 rows on 300 to 4000 keys (`keys` over all
// sets and kv heads, as both take them):
//   split  9 + 2.6e-6 rows (keys + 256 a set and head)
//   tile  14 + (230e-6 + 35e-6 ceil(rows / 128)) keys, and 7 for every wave of
//         256-row tiles after the first
// Measured, 8 kv heads of 8 bits, split against tile: one sequence of 1000 keys,
// 256 rows 18.0 / 21.4; of 4000 keys 96 rows 20.5 / 21.0, 256 rows 32.6 / 30.5; 16
// sequences of 1000 keys 64 rows 40.5 / 46.8, 96 rows 51.7 / 47.2; of 4000 keys
// 96 rows 132 / 152, 128 rows 191 / 152.
struct CacheCost {
  double split, tile;  // without the 9 and 14 of the launches
};
constexpr double kSplitStart = 9.0, kTileStart = 14.0;
CacheCost cost_of(const CacheAttnCall& a, bool prefix, int64_t rows, int64_t keys, int sms) {
  const double heads = (double)a.c.kv_heads * (prefix ? 1 : a.s.batch), all = heads * (double)keys;
  const double waves = std::ceil(heads * (double)((rows + 255) / 256) / sms);
  CacheCost c;
  c.split = 2.6e-6 * (double)rows * (all + 256.0 * heads);
  c.tile = (230e-6 + 35e-6 * (double)((rows + 127) / 128)) * all + 7.0 * (waves - 1.0);
  return c;
}

// What the tile kernels may widen at a time.  A batch whose own keys take more runs in slices of its
// sequences, one after the other in one workspace: 24 sequences of 512 tokens on 8192 rows, 32 / 8
// heads of 8 bits, take 2.3 ms so, 7.3 on the split kernel; 64 sequences 5.6 and 20.4.
constexpr size_t kTileWorkspace = (size_t)1 << 30;

// The plan of the largest equal slices of the batch that fit; false: not even one sequence does.
bool plan_slices(const CacheAttnCall& a, int sms, size_t room, CacheTilePlan* t, int* slice) {
  const int64_t batch = a.s.batch;
  CacheAttnCall part = a;
  for (int64_t n = 1;;) {
    *slice = part.s.batch = (int)((batch + n - 1) / n);
    if (plan_cache_tile(part, false, sms, room, t)) return true;
    if (part.s.batch == 1) return false;
    const int64_t more = t->workspace_bytes && room ? n * (int64_t)std::min<size_t>((t->workspace_bytes + room - 1) / room, batch) : 2 * n;
    n = std::min(batch, std::max(n + 1, more));
  }
}

// With a prefix a call is one of: the split kernel for every key; the tile kernels for the prefix and
// the split kernel, beside their widening, for the sequences' own keys; the tile kernels for both.
// The one of the least time as a whole is taken, each launch's start counted once: neither does a
// short prefix keep long own keys from the tile kernels, nor do those take a prefix that does not
// gain the launches that they add.  Measured over 432 calls (32 / 8 heads; 1 to 128 sequences of 1
// to 200 tokens, 8 to 8192 own rows, 16 to 16384 shared ones) the rule's choice takes 1.015 times
// the best one's time, at most 1.36 times (a rule for each part by itself: 1.046, 1.68).  The three
// in us, 8 bits: 200 tokens on 8192 rows behind 16 shared ones 147 / 144 / 87; 72 x 5 on 8 behind 16
// 38 / 46 / 70; 8 x 20 on 200 behind 300 28 / 44 / 44; 32 x 8 on 200 behind 4096 107 / 65 / 82; 128 x 1
// on 8 behind 1000, one of those that the rule misses, 35 / 31 / 99.
//
// The plan is the best one that a workspace of `room` bytes holds.  That of the best plan for a
// bound of the lengths holds one for every smaller bound too: with the same kernels, row tile,
// chunks and slices each part takes no more.
bq4_status plan_cache(const CacheAttnCall& a, int sms, size_t room, CachePlan* p) {
  const int group = a.q_heads / a.c.kv_heads;
  const int64_t own = (int64_t)a.tokens * group, all = own * a.s.batch;
  const int64_t prefix = (int64_t)a.prefix_width * a.c.page_size;
  const CacheCost cs = cost_of(a, false, own, a.max_length, sms), cp = cost_of(a, true, all, prefix, sms);
  const bool has_p = prefix > 0;
  struct Option {
    double cost;
    bool tile_p, tile_s;
  } options[3];
  int count = 0;
  auto option = [&](double cost, bool tile_p, bool tile_s) {
    int at = count++;
    for (; at > 0 && cost < options[at - 1].cost; --at) options[at] = options[at - 1];
    options[at] = {cost, tile_p, tile_s};
  };
  // BQ4_CACHE_TILE (tests): 0 none, p for the prefix alone, else wherever they can
  const char* f = getenv("BQ4_CACHE_TILE");
  auto cost = [&](double fitted, double forced) { return f ? forced : fitted; };
  const bool none = f && f[0] == '0', half = f && f[0] == 'p';
  option(cost(kSplitStart + cs.split + (has_p ? cp.split : 0.0), none ? 0.0 : 3.0), false, false);
  if (has_p) option(cost(kSplitStart + kTileStart + cs.split + cp.tile, none ? 3.0 : half ? 0.0 : 2.0), true, false);
  // Slices are cut by the bound of the lengths.  Where that is only the page table's width and the
  // lengths are far below it, each still costs a slice's 40 us with most SMs idle, and the split kernel
  // follows the lengths: 16 sequences of 128 tokens in tables 65536 rows wide take 335 us so and 146
  // there with 500 rows each, 1396 and 1159 with 8000; of 256 tokens 387 and 274, 1472 and 2243.  So
  // without a bound slices have to gain four times by the fit.
  const int64_t records = (int64_t)a.s.batch * a.c.kv_heads * ((a.max_length + 127) / 128);
  const bool slices = records * (128 * 4 * a.c.hp) > (int64_t)kTileWorkspace;
  if (a.max_length > 0)
    option(cost(kTileStart + cs.tile * (slices && !a.bounded ? 4.0 : 1.0) + (has_p ? kTileStart + cp.tile : 0.0),
                none || half ? 3.0 : 1.0), has_p, true);
  for (int i = 0; i < count; ++i) {
    size_t left = room;
    p->tile_p = options[i].tile_p;
    p->tile_s = options[i].tile_s;
    p->call = a;
    p->bytes = 0;
    if (p->tile_p) {
      if (!plan_cache_tile(a, true, sms, std::min(left, kTileWorkspace), &p->p)) continue;
      p->bytes = p->p.workspace_bytes;
      left -= p->bytes;
      p->call.prefix_width = 0, p->call.prefix_table = nullptr, p->call.prefix_length = nullptr;
    }
    if (p->tile_s) {
      if (!plan_slices(a, sms, std::min(left, kTileWorkspace), &p->s, &p->slice)) continue;
      p->bytes += p->s.workspace_bytes;
    } else {
      if (!plan_split(p->call, sms, left, &p->split)) continue;
      p->bytes += p->split.bytes;
    }
    return BQ4_OK;
  }
  if (room == SIZE_MAX) return set_error(BQ4_EINVAL_SHAPE, "cache attention: too many rows and keys for one launch (max_length bounds the keys)");
  bq4_status st = plan_cache(a, sms, SIZE_MAX, p);
  return st ? st : set_error(BQ4_EWORKSPACE, "workspace of %zu bytes; cache attention needs %zu", room, p->bytes);
}

bq4_status run_split(const CacheAttnCall& a, const SplitPlan& p, bool finish, void* workspace, CacheJoinSource* prefix,
                     CacheJoinSource* own, cudaStream_t stream) {
  SplitArgs s;
  s.a = a;
  const uint64_t unit = (uint64_t)(a.c.page_size / kStep);
  s.page_magic = ((1ull << 38) + unit - 1) / unit;
  s.c = a.scale * 1.4426950408889634f;  // log2(e)
  s.group = a.q_heads / a.c.kv_heads;
  s.p_tiles = p.p_tiles;
  s.s_tiles = p.s_tiles;
  s.q_vec = reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && a.q_stride[0] % 4 == 0 && a.q_stride[1] % 4 == 0 &&
            a.q_stride[2] % 4 == 0;
  s.finish = finish;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  s.part = reinterpret_cast<float*>(ws);
  s.ml = reinterpret_cast<float2*>(ws + p.part_bytes);
  s.pieces = reinterpret_cast<int2*>(ws + p.part_bytes + p.ml_bytes);
  const unsigned grid = (unsigned)p.grid;
  cudaError_t e = a.c.format == BQ4_CACHE_F16  ? launch_head<BQ4_CACHE_F16>(s, p.nt, grid, stream)
                  : a.c.format == BQ4_CACHE_Q8 ? launch_head<BQ4_CACHE_Q8>(s, p.nt, grid, stream)
                                               : launch_head<BQ4_CACHE_Q4>(s, p.nt, grid, stream);
  note_launch();
  own->part = prefix->part = s.part;
  own->ml = prefix->ml = s.ml;
  own->pieces = prefix->pieces = s.pieces;
  own->grid = prefix->grid = p.grid;
  own->tile_rows = prefix->tile_rows = 8 * p.nt;
  prefix->tiles = p.p_tiles;
  prefix->first_range = 0;
  own->tiles = p.s_tiles;
  own->first_range = a.c.kv_heads * p.p_tiles;
  return check_cuda(e, "cache attention launch");
}

bq4_status run_join(const JoinArgs& g, cudaStream_t stream) {
  // launched ahead: it waits on the device for the partial results
  cudaLaunchConfig_t cfg = {};
  const unsigned rows = (unsigned)((int64_t)g.a.s.batch * g.a.tokens * g.a.q_heads);
  const bool few = rows <= 1024;
  cfg.gridDim = dim3(few ? rows : (rows + kSWarps - 1) / kSWarps);
  cfg.blockDim = dim3(kSThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, few ? cache_join_kernel<kSWarps> : cache_join_kernel<1>, g, rows);
  note_launch();
  return check_cuda(e, "cache attention join launch");
}

}  // namespace

bq4_status cache_attn_workspace(const CacheAttnCall& a, int sms, size_t* bytes) {
  CachePlan p;
  bq4_status st = plan_cache(a, sms, SIZE_MAX, &p);
  if (st) return st;
  *bytes = p.bytes;
  return BQ4_OK;
}

bq4_status run_cache_attn(const CacheAttnCall& a, int sms, void* workspace, size_t workspace_bytes,
                          cudaStream_t stream) {
  CachePlan p;
  bq4_status st = plan_cache(a, sms, workspace ? workspace_bytes : 0, &p);
  if (st) return st;
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return set_error(BQ4_EALIGN, "workspace not 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  JoinArgs g = {};
  g.a = a;
  g.group = a.q_heads / a.c.kv_heads;
  g.have_p = a.prefix_length && a.prefix_width > 0;
  const bool alone = !p.tile_p;  // the split kernel has every source, or there is one
  if (!p.tile_s) {
    g.finish = alone;
    CacheJoinSource gp = {};
    st = run_split(p.call, p.split, alone, ws, &gp, &g.s, stream);
    if (st) return st;
    if (alone) g.p = gp;
    ws += p.split.bytes;
  }
  if (p.tile_p) {
    // the prefix's keys are widened while the sequences' own CTAs end: 128 sequences behind 16384
    // rows 99 -> 95 us
    st = run_cache_tile(a, p.p, false, !p.tile_s, ws, &g.p, stream);
    if (st) return st;
    ws += p.p.workspace_bytes;
  }
  if (!p.tile_s) return run_join(g, stream);
  const bool finish = alone && p.s.chunks == 1;
  for (; g.first < a.s.batch; g.first += p.slice) {
    CacheTilePlan t = p.s;
    g.a.s.batch = t.sets = std::min(p.slice, a.s.batch - g.first);
    t.records = (int64_t)t.sets * a.c.kv_heads * t.blocks;
    t.q_tiles = (int64_t)t.sets * a.c.kv_heads * 2 * t.tiles;
    g.a.s.table = a.s.table + g.first * a.s.table_stride;
    g.a.s.lengths = a.s.lengths + g.first;
    g.a.q = a.q + g.first * a.q_stride[0];
    g.a.out = a.out + (int64_t)g.first * a.tokens * a.q_heads * a.c.head_dim;
    st = run_cache_tile(g.a, t, finish, false, ws, &g.s, stream);
    if (!st && !finish) st = run_join(g, stream);
    if (st) return st;
  }
  return BQ4_OK;
}

}  // namespace bq4
