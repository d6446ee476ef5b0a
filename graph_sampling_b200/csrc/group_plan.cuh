// Which rows and which tile of the result a CTA takes, for products over rows sorted by expert: found on the device from the
// experts' offsets, so that no call waits for them.
#pragma once
#include "scan.cuh"

namespace gsb {

// Experts of one launch: their table is held in shared memory.  Calls with more go in several launches.
constexpr int kPlanExperts = 1024;

struct Groups {
  const i64* offsets;  // of the launch's first expert
  int first, experts;  // this launch's share
  int all;             // the call's experts
  u32 num_rows;
  i64* counters;
  u32* ends;  // where the launch before this one left the row that its experts end at, and this one leaves its own behind it; null: nowhere
};

// begin[e] .. begin[e + 1]: rows of expert e; tile[e] .. tile[e + 1]: its row tiles.  Offsets outside the rows are brought into range and
// ones below an earlier one, of this launch or one before, raised to it, so that no row is in two experts and nothing out of range is read or written;
// both are recorded.
struct PlanTable {
  u32 begin[kPlanExperts + 1];
  u32 tile[kPlanExperts + 1];
  u32 carry[33];
};

__device__ __forceinline__ u32 clamped_offset(const Groups& g, int e) {
  const i64 at = __ldg(g.offsets + e);
  return (u32)(at < 0 ? 0 : at > (i64)g.num_rows ? (i64)g.num_rows : at);
}

// The first row that no expert of the launches before has: the largest of their offsets, brought into range.  Offsets that never fall have it right in
// front, but whether they do is known only by whoever has looked at all.  Without a place for launches to leave it (products in 8 bits, which have no
// workspace) each looks again: 65 536 experts of four rows, 64 to 64, 2.54 ms for 2.36, 4 096 141 us for 140.
template <int THREADS>
__device__ __forceinline__ u32 rows_taken(PlanTable& plan, const Groups& g) {
  if (g.first == 0) return 0;
  if (g.ends) return *(volatile const u32*)g.ends;
  i64 most = 0;
#pragma unroll 8
  for (int e = threadIdx.x; e < g.first; e += THREADS) most = max(most, __ldg(g.offsets - g.first + e));
  u32 taken = __reduce_max_sync(0xffffffffu, (u32)min(most, (i64)g.num_rows));
  if ((threadIdx.x & 31) == 0) plan.carry[threadIdx.x >> 5] = taken;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) taken = max(taken, plan.carry[w]);
  __syncthreads();
  return taken;
}

// For the launches behind this one, by the kernel that makes the results.
__device__ __forceinline__ void leave_end(const PlanTable& plan, const Groups& g) {
  if (g.ends && blockIdx.x == 0 && threadIdx.x == 0) g.ends[1] = plan.begin[g.experts];
}

// All THREADS threads of the CTA; ends with a barrier.  An expert without rows gets `at_least` tiles.
template <int THREADS>
__device__ __forceinline__ void make_plan(PlanTable& plan, const Groups& g, u32 tile_rows, u32 at_least) {
  static_assert(THREADS % 32 == 0 && THREADS <= 1024, "whole warps");
  const u32 taken = rows_taken<THREADS>(plan, g);
  if (g.experts < 32) {  // a warp, and one barrier: half a microsecond sooner
    if (threadIdx.x < 32) {
      const int e = threadIdx.x;
      u32 begin = 0;
      if (e <= g.experts) {
        const i64 at = __ldg(g.offsets + e);
        begin = max(taken, clamped_offset(g, e));
        const bool bad = at < 0 || at > (i64)g.num_rows || (e < g.experts && __ldg(g.offsets + e + 1) < at);
        if (bad && blockIdx.x == 0) raise_error(g.counters, GSB_ERR_INDEX_RANGE, g.first + e);
      }
      for (int o = 1; o < 32; o <<= 1) {
        const u32 up = __shfl_up_sync(0xffffffffu, begin, o);
        if (e >= o) begin = max(begin, up);
      }
      const u32 end = __shfl_down_sync(0xffffffffu, begin, 1);
      const u32 tiles = e < g.experts ? max((end - begin + tile_rows - 1) / tile_rows, at_least) : 0;
      u32 upto = tiles;
      for (int o = 1; o < 32; o <<= 1) {
        const u32 up = __shfl_up_sync(0xffffffffu, upto, o);
        if (e >= o) upto += up;
      }
      if (e <= g.experts) {
        plan.begin[e] = begin;
        plan.tile[e] = upto - tiles;
      }
    }
    __syncthreads();
    return;
  }
  constexpr int kEach = (kPlanExperts + THREADS - 1) / THREADS;
  const int t = threadIdx.x;
  for (int e = t; e <= g.experts; e += THREADS) {
    const i64 at = __ldg(g.offsets + e);
    plan.begin[e] = max(taken, clamped_offset(g, e));
    const bool bad = at < 0 || at > (i64)g.num_rows || (e < g.experts && __ldg(g.offsets + e + 1) < at);
    if (bad && blockIdx.x == 0) raise_error(g.counters, GSB_ERR_INDEX_RANGE, g.first + e);
  }
  __syncthreads();
  u32 most = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (t * kEach + i <= g.experts) most = max(most, plan.begin[t * kEach + i]);
  for (int o = 1; o < 32; o <<= 1) {
    const u32 up = __shfl_up_sync(0xffffffffu, most, o);
    if ((t & 31) >= o) most = max(most, up);
  }
  if ((t & 31) == 31) plan.carry[t >> 5] = most;
  most = __shfl_up_sync(0xffffffffu, most, 1);
  if ((t & 31) == 0) most = 0;
  __syncthreads();
  for (int w = 0; w < (t >> 5); ++w) most = max(most, plan.carry[w]);
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (t * kEach + i <= g.experts) plan.begin[t * kEach + i] = most = max(most, plan.begin[t * kEach + i]);
  if (t == THREADS - 1 && THREADS * kEach == g.experts) plan.begin[g.experts] = max(most, plan.begin[g.experts]);
  __syncthreads();
  u32 own[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = t * kEach + i;
    u32 tiles = 0;
    if (e < g.experts) {
      tiles = (plan.begin[e + 1] - plan.begin[e] + tile_rows - 1) / tile_rows;
      if (tiles < at_least) tiles = at_least;
    }
    own[i] = sum;
    sum += tiles;
  }
  u32 scan = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const u32 up = __shfl_up_sync(0xffffffffu, scan, o);
    if ((t & 31) >= o) scan += up;
  }
  if ((t & 31) == 31) plan.carry[t >> 5] = scan;
  __syncthreads();
  u32 before = scan - sum;
  for (int w = 0; w < (t >> 5); ++w) before += plan.carry[w];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = t * kEach + i;
    if (e <= g.experts) plan.tile[e] = before + own[i];
  }
  if (t == THREADS - 1 && THREADS * kEach == g.experts) plan.tile[g.experts] = before + sum;
  __syncthreads();
}

// The expert whose row tiles hold number `tile` (below plan.tile[experts]).
__device__ __forceinline__ int expert_of_tile(const PlanTable& plan, int experts, u32 tile) {
  int low = 0, high = experts;  // plan.tile[low] <= tile < plan.tile[high]
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (plan.tile[mid] <= tile) low = mid;
    else high = mid;
  }
  return low;
}

}  // namespace gsb
