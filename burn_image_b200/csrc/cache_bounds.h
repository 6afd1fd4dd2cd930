// cache_bounds.h -- index arithmetic of the cache attention kernels that has to hold whatever a
// kernel that gave up on a wait left behind.  Plain C++, so that it is checked without a GPU.
#pragma once
#ifdef __CUDACC__
#define BQ4_BOTH __host__ __device__ __forceinline__
#else
#define BQ4_BOTH inline
#endif

namespace bq4 {

// Partial results of a range of the split kernel's line, in its workspace of grid + ranges slots:
// those of CTAs from..to at slot CTA + range.  A CTA that gave up has not written from and to of
// the ranges that it did not reach, and the workspace holds anything there: the slots stay among
// those that exist (the sums are wrong then, and the error word says so).
struct CacheSlots {
  int first, count;
};
BQ4_BOTH CacheSlots cache_slots(int from, int to, int range, int grid) {
  from = from < 0 ? 0 : from < grid ? from : grid - 1;
  to = to < from ? from : to < grid ? to : grid - 1;
  CacheSlots s;
  s.first = from + range;
  s.count = to - from + 1;
  return s;
}

// Copies of a warp's ring that are under way when it gives up on step j of `mine`: step j has
// asked for step j + stages - 1, and nothing from step j on has been waited for.
BQ4_BOTH int cache_pending(int j, int mine, int stages) {
  return j >= mine ? 0 : mine - j < stages ? mine - j : stages;
}

}  // namespace bq4
