// bq4_cache.h -- layout of the paged key/value cache, shared by its kernels.
//
// One page holds page_size consecutive tokens of one sequence, for every kv
// head.  Rows are padded to HP = 64 or 128 values (head_dim rounded up).  The 16
// tokens of a step lie together, so that one bulk copy brings them:
//   data u8 [pages][kv_heads][page_size / 16][step bytes], a step being
//     k rows [16][row bytes], v rows [16][row bytes],
//     scales u16 [16][2 (k, v)][nb] (bf16 bits)
// Rows:
//   f16: 2 HP bytes, no scales.
//   q8:  byte d holds q_d + 128; one scale for the row (nb = 1).
//   q4:  a nibble holds q + 8; one scale for each 32 values (nb = HP / 32).
//        The nibbles are placed for the lanes that feed the tensor core:
//        k: the 8 values 32 b + 8 t .. + 7 form word t nb + b; within it
//           value 2 p sits in nibble p and value 2 p + 1 in nibble p + 4, so
//           (w >> 4 p) & 0x000F000F is the pair (2 p, 2 p + 1).
//        v: the 4 values 32 b + 4 g .. + 3 form u16 g nb + b, in order.
// Padding values are q = 0 with scale 0 (f16: 0).
//
// The 16-byte pieces of a 128-byte line are permuted by the row (cache_swizzle),
// so that 16 rows copied to shared memory as they lie are read by fragments
// without bank conflicts: 8 lanes take a 16-byte piece each of either two
// adjacent k rows (4 pieces of each) or four even v rows (2 of each).
#pragma once
#include "bq4_internal.h"

namespace bq4 {

constexpr int kCacheBlock = 32;       // values under one q4 scale
constexpr int kCachePageUnit = 16;    // page sizes are multiples of this
constexpr int kCacheMaxHeadDim = 128;

struct CacheView {
  uint8_t* data;
  int32_t pages, page_size, kv_heads, head_dim;
  int32_t hp, nb, row_bytes;  // padded head, scales of a row, bytes of a row
  int32_t format;
  int32_t step_bytes;
};

struct SeqView {
  const int32_t* table;
  const int32_t* lengths;
  int64_t table_stride;
  int32_t table_width, batch;
};

inline int cache_hp(int head_dim) { return head_dim <= 64 ? 64 : 128; }
inline int cache_nb(int format, int hp) {
  return format == BQ4_CACHE_Q8 ? 1 : format == BQ4_CACHE_Q4 ? hp / kCacheBlock : 0;
}
inline int cache_row_bytes(int format, int hp) {
  return format == BQ4_CACHE_F16 ? 2 * hp : format == BQ4_CACHE_Q8 ? hp : hp / 2;
}

// Byte of the k (v) rows of a step where byte `at` of row r lies.
__host__ __device__ __forceinline__ constexpr int cache_swizzle(int kv, int row_bytes, int r, int at) {
  const int f = kv == 0 ? (row_bytes >= 128 ? 4 * (r & 1) : 0)
                        : row_bytes >= 64 ? 2 * (r >> 1 & 3) : 2 * (r >> 2 & 1);
  return (r * row_bytes + at) ^ f << 4;
}

inline int cache_step_bytes(int row_bytes, int nb) { return 16 * (2 * row_bytes + 4 * nb); }

// The step that holds `place` of (page, head).
__device__ __forceinline__ uint8_t* cache_step(const CacheView& c, int page, int head, int place) {
  const int64_t steps = ((int64_t)page * c.kv_heads + head) * (c.page_size >> 4) + (place >> 4);
  return c.data + steps * c.step_bytes;
}

// Arguments of one attention call (bq4_cache_attn.cu).
struct CacheAttnCall {
  CacheView c;
  SeqView s;
  const int32_t* prefix_table;   // null: no prefix
  const int32_t* prefix_length;  // one value on the device
  int32_t prefix_width;
  const uint16_t* q;             // f16
  int64_t q_stride[3];           // batch, token, head
  uint16_t* out;                 // f16 [batch][tokens][q_heads][head_dim]
  int32_t tokens, q_heads, causal;
  int32_t max_length;            // lengths are at most this
  bool bounded;                  // the caller said so: else it is what the page table holds
  float scale;                   // of the scores
  int* err;
};

// Where a row's partial results (m, l and O of some of its keys) lie: the
// join kernel's input, one of the prefix's and one of the sequence's own keys.
// Row r of a range (kv head, tile of tile_rows rows) is at slot * tile_rows + r:
// pieces: slots first CTA + range .. last CTA + range of the split kernel's line, of
// `grid` CTAs; else slots range * chunks .., one for each `span` keys that the tile sees.
struct CacheJoinSource {
  const float* part;
  const float2* ml;
  const int2* pieces;
  int grid, tile_rows, tiles, span, chunks, first_range;
};

// Launch plan of the many-row kernels (bq4_cache_tile.cu) for the prefix or the
// sequences' own keys.
struct CacheTilePlan {
  bool prefix;
  int sets, tiles, blocks, span, chunks;
  int64_t records, q_tiles, slots;
  size_t tile_bytes, consts_bytes, q_bytes, part_bytes, ml_bytes, workspace_bytes;
};
// The best plan that `room` bytes hold; false: none does (workspace_bytes is what one needs at
// least then), or the sizes are past the kernels' (workspace_bytes is 0).
bool plan_cache_tile(const CacheAttnCall& a, bool prefix, int sms, size_t room, CacheTilePlan* p);
// finish: there is one chunk and no other source, and the rows are finished.
// beside: the kernel before on the stream is independent, and may run at the same time.
bq4_status run_cache_tile(const CacheAttnCall& a, const CacheTilePlan& p, bool finish, bool beside, void* workspace,
                          CacheJoinSource* source, cudaStream_t stream);

bq4_status cache_attn_workspace(const CacheAttnCall& c, int sms, size_t* bytes);
bq4_status run_cache_attn(const CacheAttnCall& c, int sms, void* workspace, size_t workspace_bytes, cudaStream_t s);

}  // namespace bq4
