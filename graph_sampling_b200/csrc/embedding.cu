// Embedding rows: lookup by id with scaling, and the gradient of the table.
//
// Lookup: out[i, :] = scale * table[ids[i], :], one rounding.
// Gradient: total[v, :] = scale * (sum of grad[i, :] over the positions i with ids[i] == v), summed in float in the order of the
// positions within pieces that depend on sizes and types alone, so the same inputs give the same bits; one rounding.  The positions are
// sorted by id (key_sort.cuh); the sorted list is cut into chunks of equal length whoever the ids are, so a frequent id is
// shared by many groups of lanes.  A sum that begins and ends inside a chunk is written at once; what reaches over a chunk's
// ends goes to `part` and is added up by k_join_rows.  Rows without a sum are cleared beside the sort, or, where that would write
// much twice, by k_join_rows.
#include <atomic>
#include <type_traits>

#include "key_sort.cuh"
#include "launch.cuh"
#include "row_values.cuh"
#include "scan.cuh"

namespace gsb {

constexpr int kLookupThreads = 256;

// Narrow units: more rows (by two units a lane a million rows of 602 bf16 435 us for 474), but not with four (1.3 M of 50 bf16 53 for 56).
constexpr int lookup_rows(int unit, int steps) { return unit < 16 && steps < 4 ? 4 : rows_ahead(steps); }

struct LookupArgs {
  const i64* ids;
  u32 n;
  int units, lanes;
  i64 num_rows, stride;  // stride in units
  i64 padding;
  bool has_padding;
  float scale;
  i64* counters;
};

// LANES: 32, or 0 for a.lanes.  Known, and with rows that are copied as they are apart, they pay where a unit is one value of 16 bits (a
// million rows of 101 values 124 us for 180, of 251 255 for 321), but not where there are fewer to take (500 000 of 1 434 748 for 555).
//
// A group of lanes takes neighbouring rows of the result, a tile of their columns at a time: all its reads are on their way before
// anything is written.  Bound by DRAM with rows in no order: 1 000 000 rows of 1 204 bytes out of 2.45 M in 422 us, 5.7 TB/s of what
// is read and written.
template <class T, int BYTES, int STEPS, int LANES>
__global__ void __launch_bounds__(kLookupThreads) k_lookup_rows(const LookupArgs a, const Unit<T, BYTES>* __restrict__ table,
                                                                Unit<T, BYTES>* __restrict__ out) {
  constexpr int kRows = lookup_rows(BYTES, STEPS), N = Unit<T, BYTES>::N;
  await_previous();
  const int lanes = LANES > 0 ? LANES : a.lanes, lane = threadIdx.x & (lanes - 1);
  const u32 step = gridDim.x * (kLookupThreads / lanes) * kRows;
  for (u32 i = (blockIdx.x * kLookupThreads + threadIdx.x) / lanes * kRows; i < a.n; i += step) {
    const Unit<T, BYTES>* from[kRows];  // null: zeros
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      from[r] = nullptr;
      if (i + r >= a.n) continue;
      const i64 id = __ldg(a.ids + i + r);
      if (a.has_padding && id == a.padding) continue;
      if ((u64)id < (u64)a.num_rows) from[r] = table + id * a.stride;
      else if (lane == 0 && blockIdx.y == 0) raise_error(a.counters, GSB_ERR_INDEX_RANGE, i + r);
    }
    Unit<T, BYTES>* to = out + (i64)i * a.units;
    bool plain = LANES > 0 && a.scale == 1.f && i + kRows <= a.n;  // copied as they are
#pragma unroll
    for (int r = 0; r < kRows; ++r) plain = plain && from[r];
    if (plain) {
      const Unit<T, BYTES>* p[kRows];
      Unit<T, BYTES>* q[kRows];
      int j = blockIdx.y * lanes * STEPS + lane;
      const int stride = gridDim.y * lanes * STEPS;
#pragma unroll
      for (int r = 0; r < kRows; ++r) p[r] = from[r] + j, q[r] = to + (i64)r * a.units + j;
      for (; j < a.units; j += stride) {
        Unit<T, BYTES> v[kRows][STEPS];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
            if (j + s * lanes < a.units) v[r][s] = load_unit(p[r] + s * lanes);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
            if (j + s * lanes < a.units) store_unit(q[r] + s * lanes, v[r][s]);
#pragma unroll
        for (int r = 0; r < kRows; ++r) p[r] += stride, q[r] += stride;
      }
      continue;
    }
    for (int j = blockIdx.y * lanes * STEPS + lane; j < a.units; j += gridDim.y * lanes * STEPS) {
      Unit<T, BYTES> v[kRows][STEPS];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          v[r][s].clear();
          if (from[r] && j + s * lanes < a.units) v[r][s] = load_unit(from[r] + j + s * lanes);
        }
      if (a.scale != 1.f)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          if (from[r])
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
              float f[N];
              v[r][s].get(f);
#pragma unroll
              for (int q = 0; q < N; ++q) f[q] *= a.scale;
              v[r][s].set(f);
            }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (i + r < a.n)
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
            if (j + s * lanes < a.units) store_unit(to + (i64)r * a.units + j + s * lanes, v[r][s]);
    }
  }
}

// Rows of 16-bit values that begin off the 4-byte boundaries, where a unit is one value: a warp copies the next rows into shared
// memory in units of 16 bytes, from the boundary before a row to the one behind it, and writes whole units of the result, each out
// of two that it straddles.  A short row's steps cost more than it gains, and so do few rows, which come out of L2 (rows in no order
// out of twice as many, bf16): 500 000 of 601 values 243 us for 352, 80 000 of 401 57 for 64, 53 000 of 601 26 for 28, 11 000 of 1 433
// 11 for 19, 8 000 of 2 047 11.4 for 11.7, but 106 000 of 301 74 for 62, 40 000 of 401 18 for 15, 27 000 of 601 14 for 12.  (Where units
// of 4 bytes fit, nothing is gained: a million rows of 1 204 bytes 479 us for 422.)
constexpr int kStagedThreads = 128, kStages = 3;
constexpr i64 kMostStagedBytes = 8192;
static bool staged(i64 row_bytes, i64 n) {
  return row_bytes >= 800 && row_bytes <= kMostStagedBytes && n * row_bytes >= (row_bytes < 1600 ? 64000000 : 32000000);
}
static u32 stage_bytes(i64 row_bytes) { return (u32)((row_bytes + 15) / 16 * 16 + 16); }
static size_t staged_smem(u32 stage) { return (size_t)(kStagedThreads / 32) * kStages * stage; }

struct StagedArgs {
  const char* begin;  // of the table
  const char* end;
  u32 stage;          // bytes
  u32 per_warp;       // rows
  int row_bytes;
};

template <class T>
__global__ void __launch_bounds__(kStagedThreads) k_lookup_staged(const LookupArgs a, const StagedArgs s, T* __restrict__ out) {
  typedef Unit<T, (int)sizeof(T)> Value;
  typedef Unit<T, 16> Wide;
  extern __shared__ __align__(16) char smem[];
  await_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  char* ring = smem + (size_t)warp * kStages * s.stage;
  const u32 first = (blockIdx.x * (kStagedThreads / 32) + warp) * s.per_warp, rows = first < a.n ? min(s.per_warp, a.n - first) : 0;
  // lane l: the row in the table, or -1 for zeros, of rows 32 q + l (`now`) and of the next 32 (`then`)
  auto look = [&](u32 r) {
    if (r >= rows) return (i64)-1;
    const i64 id = __ldg(a.ids + first + r);
    if (a.has_padding && id == a.padding) return (i64)-1;
    if ((u64)id < (u64)a.num_rows) return id;
    raise_error(a.counters, GSB_ERR_INDEX_RANGE, first + r);
    return (i64)-1;
  };
  i64 now = look(lane), then = look(32 + lane);
  auto from_of = [&](u32 r, u32 base) {  // null: zeros
    const i64 id = __shfl_sync(0xffffffffu, r - base < 32 ? now : then, (int)(r & 31));
    return id < 0 ? nullptr : s.begin + id * a.stride;
  };
  auto start = [&](u32 r, u32 base) {
    const char* from = from_of(r, base);
    if (r < rows && from) {
      const char* at = (const char*)((uintptr_t)from & ~(uintptr_t)15);
      const int units = (int)((from + s.row_bytes - at + 15) >> 4);
      char* to = ring + (r % kStages) * s.stage;
      if (at >= s.begin && at + units * 16 <= s.end) {
        u32 there = (u32)__cvta_generic_to_shared(to) + lane * 16;
        at += lane * 16;
#pragma unroll 4
        for (int q = lane; q < units; q += 32, at += 512, there += 512)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(there), "l"(at) : "memory");
      } else {  // the table's first or last row, which has nothing in front of it or behind it
        const int shift = (int)(from - at);
        for (int h = 2 * lane; h < s.row_bytes; h += 64) *(unsigned short*)(to + shift + h) = __ldg((const unsigned short*)(from + h));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  u32 base = 0;
#pragma unroll
  for (u32 r = 0; r < kStages - 1; ++r) start(r, 0);
  for (u32 r = 0; r < rows; ++r) {
    if (r - base == 32) {
      base += 32;
      now = then;
      then = look(base + 32 + lane);
    }
    start(r + kStages - 1, base);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const char* from = from_of(r, base);
    T* to = out + (i64)(first + r) * a.units;
    const char* row = ring + (r % kStages) * s.stage + ((uintptr_t)from & 15);
    auto put = [&](auto u, auto* at) {
      if (from && a.scale != 1.f) {
        float f[decltype(u)::N];
        u.get(f);
#pragma unroll
        for (int q = 0; q < decltype(u)::N; ++q) f[q] *= a.scale;
        u.set(f);
      }
      store_unit(at, u);
    };
    // whole units of 16 bytes of the result, and the values in front of them and behind them
    const int head = min(a.units, (int)((0 - (uintptr_t)to & 15) / sizeof(T))), wide = (a.units - head) / Wide::N, behind = head + wide * Wide::N;
    const int one = lane < 16 ? (lane < head ? lane : -1) : behind + lane - 16 < a.units ? behind + lane - 16 : -1;
    if (one >= 0) {
      Value v;
      v.clear();
      if (from) v = ((const Value*)row)[one];
      put(v, (Value*)to + one);
    }
    Wide* wide_to = (Wide*)(to + head);
    row += head * sizeof(T);
    if (!from) {
      Wide zero;
      zero.clear();
      for (int j = lane; j < wide; j += 32) put(zero, wide_to + j);
    } else {
      const uint4* of = (const uint4*)((uintptr_t)row & ~(uintptr_t)15);
      const u32 shift = (u32)((uintptr_t)row & 3) * 8;
      auto go = [&](auto word) {  // a unit begins in this word of one of the row's units in shared memory
        constexpr int W = decltype(word)::value;
#pragma unroll 2
        for (int j = lane; j < wide; j += 32) {
          const uint4 x = of[j], y = of[j + 1];
          const u32 w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          Wide u;
          u.w = make_uint4(__funnelshift_r(w[W], w[W + 1], shift), __funnelshift_r(w[W + 1], w[W + 2], shift),
                           __funnelshift_r(w[W + 2], w[W + 3], shift), __funnelshift_r(w[W + 3], w[W + 4], shift));
          put(u, wide_to + j);
        }
      };
      const int word = (int)((uintptr_t)row >> 2 & 3);
      if (word == 0) go(std::integral_constant<int, 0>{});
      else if (word == 1) go(std::integral_constant<int, 1>{});
      else if (word == 2) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 3>{});
    }
    __syncwarp();  // before the stage is written again
  }
}

// Once per device: the kernel may use as much shared memory as the longest rows need.  (The limit is the function's, not the launch's:
// set call by call, one thread would lower it between another's setting and launch.)
template <class T>
static cudaError_t prepare_staged(gsb_ctx* ctx) {
  static std::atomic<bool> known[64];
  const int device = ctx_device(ctx);
  if (device >= 0 && device < 64 && known[device]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(k_lookup_staged<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)staged_smem(stage_bytes(kMostStagedBytes)));
  if (e == cudaSuccess && device >= 0 && device < 64) known[device] = true;
  return e;
}

// N values of `to`, 16 bytes at a time where they are that many.
template <class O, int N>
__device__ __forceinline__ void store_values(O* to, const float* v, float scale) {
  constexpr int kBytes = N * (int)sizeof(O), kUnit = kBytes > 16 ? 16 : kBytes, kPer = kUnit / (int)sizeof(O);
#pragma unroll
  for (int p = 0; p < N / kPer; ++p) {
    float f[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) f[q] = v[p * kPer + q] * scale;
    Unit<O, kUnit> u;
    u.set(f);
    store_unit((Unit<O, kUnit>*)(to + p * kPer), u);
  }
}

constexpr int kSumThreads = 128;

struct SumArgs {
  u32 n;         // sorted positions
  u32 chunk;     // positions per group of lanes
  u32 num_rows;  // of the result: a position whose row is not below that belongs to no sum
  int lanes;     // per group, a power of two
  int units;     // per row
  i64 stride;    // of `grad`, in units
  float scale;
  u32* summed;  // a bit per row of the result: it has a sum; null: they are not asked for
};
__device__ __forceinline__ bool usable(const SumArgs& a, u64 pair) {
  return pair_key(pair) < a.num_rows && pair_at(pair) < a.n;
}

// One group of lanes per chunk and column tile (blockIdx.y) of lanes * STEPS units.  Bound by DRAM: 3.65 M rows of 512 bytes summed
// into 1.3 M in 428 us, 5.9 TB/s; 900 000 rows of 256 bytes into 0.79 M in 80, 5.4 TB/s.
// MARK: a.summed is wanted.
template <class T, class O, int BYTES, int STEPS, bool MARK>
__global__ void __launch_bounds__(kSumThreads) k_sum_rows(const SumArgs a, const Unit<T, BYTES>* __restrict__ grad,
                                                          const u64* __restrict__ sorted, O* __restrict__ out,
                                                          float* __restrict__ part) {
  constexpr int N = Unit<T, BYTES>::N;
  constexpr int kAhead = 2;  // rows on their way; with four, rows of 200 bytes took 86 us for 82
  await_previous();
  const u32 chunk = (u32)(((u64)blockIdx.x * kSumThreads + threadIdx.x) / a.lanes);
  const u64 at = (u64)chunk * a.chunk;
  if (at >= a.n) return;
  const u32 begin = (u32)at, end = min(begin + a.chunk, a.n);
  const int first = blockIdx.y * a.lanes * STEPS + (threadIdx.x & (a.lanes - 1));
  bool in[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) in[s] = first + s * a.lanes < a.units;
  const i64 width = (i64)a.units * N;
  grad += first;
  out += (i64)first * N;
  part += 2 * (i64)chunk * width + (i64)first * N;
  float sum[STEPS][N] = {};
  auto put = [&](auto* to, float scale) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (in[s]) store_values<std::remove_pointer_t<decltype(to)>, N>(to + s * a.lanes * N, sum[s], scale);
#pragma unroll
      for (int q = 0; q < N; ++q) sum[s][q] = 0.f;
    }
  };
  sorted += begin;
  const u32 left = a.n - begin, mine = end - begin;  // positions up to the list's end, and the chunk's
  bool head = begin > 0 && pair_key(__ldg(sorted - 1)) == pair_key(__ldg(sorted));
  u64 p[kAhead + 1], next[kAhead + 1];
#pragma unroll
  for (int u = 0; u <= kAhead; ++u) p[u] = u < left ? __ldg(sorted + u) : ~0ull;
  u32 bits = 0;  // of the rows that ended and have the latest one's word
  for (u32 j = 0; j < mine; j += kAhead) {
    Unit<T, BYTES> v[kAhead][STEPS];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + u >= mine || !usable(a, p[u])) continue;
      const Unit<T, BYTES>* from = grad + (i64)pair_at(p[u]) * a.stride;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (in[s]) v[u][s] = load_unit_once(from + s * a.lanes);
    }
    next[0] = p[kAhead];
#pragma unroll
    for (int u = 1; u <= kAhead; ++u) next[u] = j + kAhead + u < left ? __ldg(sorted + j + kAhead + u) : ~0ull;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + u >= mine || !usable(a, p[u])) return;  // the sorted list ends with the positions that belong to no row
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (in[s]) {
          float f[N];
          v[u][s].get(f);
#pragma unroll
          for (int q = 0; q < N; ++q) sum[s][q] += f[q];
        }
      const u32 row = pair_key(p[u]);
      const bool ends = pair_key(p[u + 1]) != row;
      if (ends && !head) put(out + (i64)row * width, a.scale);
      else if (ends || j + u + 1 == mine) put(part + (head ? 0 : width), 1.f);
      if (ends) head = false;
      if (!MARK) continue;
      const u32 after = pair_key(p[u + 1]);
      if (ends) bits |= 1u << (row & 31);
      if (bits != 0 && (j + u + 1 == mine || after >= a.num_rows || after >> 5 != row >> 5)) {
        if (first == 0) atomicOr(a.summed + (row >> 5), bits);
        bits = 0;
      }
    }
#pragma unroll
    for (int u = 0; u <= kAhead; ++u) p[u] = next[u];
  }
}

// Where the last sum of a chunk began there and goes on: its part and those of the chunks behind.  A warp looks at kJoinSpan chunks,
// a lane each, and then takes the sums that begin there one after the other, kJoinColumns columns (blockIdx.y).  It adds up to
// kJoinShort parts in their order, with the next ones on their way; longer runs (a hub's, a frequent token's) are shared by
// the CTA's warps, whose sums are added in the warps' order.
constexpr int kJoinThreads = 512, kJoinWarps = kJoinThreads / 32, kJoinSpan = 4, kJoinSteps = 4, kJoinColumns = 32 * kJoinSteps;
constexpr int kJoinShort = 32;

// Rows without a sum, 16 bytes at a time, by warps: 32 rows each, or a piece of their columns.
struct ClearArgs {
  uint4* out;
  u32 units;    // of 16 bytes, per row
  u32 pieces;   // of kClearPiece units, per row
  u32 per_row;  // 2^32 / units, rounded up
};
constexpr u32 kClearPiece = 1024;

__device__ __forceinline__ void clear_rows(const ClearArgs& c, const u32* __restrict__ summed, u32 num_rows, i64 number, i64 of) {
  const int lane = threadIdx.x & 31;
  const i64 all = (i64)((num_rows - 1) / 32 + 1) * c.pieces;
  for (i64 item = number; item < all; item += of) {
    const u32 word = (u32)(c.pieces == 1 ? item : item / c.pieces), used = __ldg(summed + word), rows = min(32u, num_rows - word * 32);
    if (used == 0xffffffffu) continue;
    uint4* to = c.out + (i64)word * 32 * c.units;
    if (c.units < 32) {  // several rows at a time
      for (u32 q = lane; q < rows * c.units; q += 32)
        if (!(used >> __umulhi(q, c.per_row) & 1u)) to[q] = make_uint4(0, 0, 0, 0);
    } else {
      const u32 begin = (u32)(item - (i64)word * c.pieces) * kClearPiece, end = min(c.units, begin + kClearPiece);
      for (u32 r = 0; r < rows; ++r)
        if (!(used >> r & 1u))
          for (u32 q = begin + lane; q < end; q += 32) to[(i64)r * c.units + q] = make_uint4(0, 0, 0, 0);
    }
  }
}

template <class O>
__global__ void __launch_bounds__(kJoinThreads) k_join_rows(const SumArgs a, const ClearArgs clear, i64 width, i64 chunks,
                                                            const u64* __restrict__ sorted, const float* __restrict__ part,
                                                            O* __restrict__ out) {
  __shared__ int s_long;
  __shared__ i64 s_chunk[kJoinWarps * kJoinSpan], s_run[kJoinWarps * kJoinSpan];
  __shared__ u32 s_row[kJoinWarps * kJoinSpan];
  __shared__ float s_sum[kJoinWarps][kJoinColumns];
  await_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const i64 column = (i64)blockIdx.y * kJoinColumns + lane;
  if (threadIdx.x == 0) s_long = 0;
  __syncthreads();
  if (a.summed) {
    const i64 number = ((i64)blockIdx.y * gridDim.x + blockIdx.x) * kJoinWarps + warp, of = (i64)gridDim.x * gridDim.y * kJoinWarps;
    clear_rows(clear, a.summed, a.num_rows, number, of);
  }
  float sum[kJoinSteps];
  auto add = [&](i64 from, i64 n, i64 step) {  // head parts of n chunks, `step` apart
#pragma unroll 8
    for (i64 q = 0; q < n; ++q) {
      const float* row = part + 2 * (from + q * step) * width;
#pragma unroll
      for (int s = 0; s < kJoinSteps; ++s)
        if (column + 32 * s < width) sum[s] += __ldg(row + column + 32 * s);
    }
  };
  // lane l: chunk c + l, and the first key of the chunk behind it; the lanes from kJoinSpan on only look ahead
  const i64 c = ((i64)blockIdx.x * kJoinWarps + warp) * kJoinSpan + lane, end = (c + 1) * (i64)a.chunk;
  const bool inner = c + 1 < chunks;
  const u32 behind = inner ? pair_key(__ldg(sorted + end)) : kNoRow;
  u32 last = kNoRow, before = kNoRow;
  if (inner && lane < kJoinSpan) {
    last = pair_key(__ldg(sorted + end - 1));
    if (c > 0) before = pair_key(__ldg(sorted + end - a.chunk - 1));
  }
  u32 starts = __ballot_sync(0xffffffffu, lane < kJoinSpan && last < a.num_rows && behind == last && before != last);
  for (; starts != 0; starts &= starts - 1) {
    const int l = __ffs(starts) - 1;
    const u32 row = __shfl_sync(0xffffffffu, last, l);
    const i64 chunk = __shfl_sync(0xffffffffu, c, l);
    const u32 other = __ballot_sync(0xffffffffu, behind != row) & ~((1u << l) - 1u);  // lanes whose next chunk begins with another
    i64 run = other ? __ffs(other) - 1 - l : 32 - l;  // chunks behind that go on with it
    // beyond the lanes' view: the keys ascend, so 32 probes at a time narrow the end down to a 32nd
    i64 lo = chunk + 1 + run, hi = other ? lo : chunks;  // chunks before lo go on with it, from hi on none does
    while (lo < hi) {
      const i64 step = (hi - lo + 31) / 32, probe = lo + lane * step;
      const u32 not_row = __ballot_sync(0xffffffffu, probe >= hi || pair_key(__ldg(sorted + probe * (i64)a.chunk)) != row);
      const int with = not_row ? __ffs(not_row) - 1 : 32;  // probes that go on with it
      if (with < 32) hi = min(hi, lo + with * step);
      if (with > 0) lo += (with - 1) * step + 1;
    }
    run = lo - chunk - 1;
    if (run > kJoinShort) {
      if (lane == 0) {
        const int at = atomicAdd(&s_long, 1);
        s_chunk[at] = chunk;
        s_run[at] = run;
        s_row[at] = row;
      }
      continue;
    }
#pragma unroll
    for (int s = 0; s < kJoinSteps; ++s) sum[s] = column + 32 * s < width ? __ldg(part + (2 * chunk + 1) * width + column + 32 * s) : 0.f;
    add(chunk + 1, run, 1);
#pragma unroll
    for (int s = 0; s < kJoinSteps; ++s)
      if (column + 32 * s < width) out[(i64)row * width + column + 32 * s] = from_float<O>(sum[s] * a.scale);
  }
  __syncthreads();
  for (int f = 0; f < s_long; ++f) {
    const i64 chunk = s_chunk[f], run = s_run[f];
#pragma unroll
    for (int s = 0; s < kJoinSteps; ++s)
      sum[s] = warp == 0 && column + 32 * s < width ? __ldg(part + (2 * chunk + 1) * width + column + 32 * s) : 0.f;
    add(chunk + 1 + warp, run > warp ? (run - warp + kJoinWarps - 1) / kJoinWarps : 0, kJoinWarps);
#pragma unroll
    for (int s = 0; s < kJoinSteps; ++s) s_sum[warp][lane + 32 * s] = sum[s];
    __syncthreads();
    if (threadIdx.x < kJoinColumns && (i64)blockIdx.y * kJoinColumns + threadIdx.x < width) {
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) all += s_sum[w][threadIdx.x];
      out[(i64)s_row[f] * width + (i64)blockIdx.y * kJoinColumns + threadIdx.x] = from_float<O>(all * a.scale);
    }
    __syncthreads();
  }
}

// Positions per chunk: as many groups of lanes as make two waves of warps, so that hubs and frequent ids are shared by many, and no
// more: each chunk's ends, two sums, are written and read once more (200 000 rows of 512 bf16 133 us, with half the chunk 141).
static i64 sum_chunk(i64 n, int lanes, i64 tiles) {
  const i64 c = n * tiles * max(lanes, 8) / 32 / (kNumSMs * 64);
  return c < 8 ? 8 : c > 128 ? 128 : c;
}

struct GradPlan {
  size_t sort_bytes, total_bytes;
  i64 most_chunks;  // that there is room for
  size_t words;     // a bit per row of the result, where they may be wanted
};

static bool may_clear_behind(i64 n, i64 num_rows, i64 row_bytes) { return min(n, num_rows) * row_bytes >= 200000000; }

static GradPlan grad_plan(i64 n, i64 num_rows, i64 row_len) {
  GradPlan g;
  // what the units of the call, which are not known here, make of a row is at least this
  const i64 chunk = sum_chunk(n, row_len >= 512 ? 32 : row_len >= 256 ? 16 : 8, (row_len + 511) / 512);
  g.most_chunks = (n + chunk - 1) / chunk;
  g.sort_bytes = key_sort_bytes(n, num_rows);
  Pieces p(nullptr);
  p.take<char>(g.sort_bytes);
  p.take<float>((size_t)g.most_chunks * 2 * (size_t)row_len);
  g.words = may_clear_behind(n, num_rows, row_len * 4) ? ((size_t)num_rows + 31) / 32 : 0;
  p.take<u32>(g.words);
  g.total_bytes = p.used;
  return g;
}

// Positions per chunk of a call: a matter of sizes and types, not of the addresses and strides that decide about the unit, since it
// decides about the order of the sums.  That of the unit that fits rows at the best addresses.
static u32 chunk_of(i64 n, i64 row_bytes, i64 most_chunks) {
  const int unit = unit_bytes(row_bytes, 0);
  const i64 units = row_bytes / unit;
  const RowShape shape = row_shape(units, sum_steps(unit), sum_wide(unit));
  return (u32)max(sum_chunk(n, shape.lanes, grid_for(units, shape.lanes * shape.steps)), (n + most_chunks - 1) / most_chunks);
}

// Leaves the shape and the chunks in `a`.
template <class T, class O, int BYTES>
static void launch_sum(cudaStream_t stream, SumArgs& a, i64 most_chunks, const void* grad, i64 stride_bytes, i64 row_bytes,
                       const u64* sorted, void* out, float* part) {
  a.units = (int)(row_bytes / BYTES);
  a.stride = stride_bytes / BYTES;
  const RowShape shape = row_shape(a.units, sum_steps(BYTES), sum_wide(BYTES));
  a.lanes = shape.lanes;
  const int tiles = grid_for(a.units, shape.lanes * shape.steps);
  const i64 n = a.n;
  a.chunk = chunk_of(n, row_bytes, most_chunks);
  with_steps(shape.steps, [&](auto steps) {
    const dim3 grid(grid_for((n + a.chunk - 1) / a.chunk * a.lanes, kSumThreads), tiles);
    constexpr int S = decltype(steps)::value;
    auto kernel = k_sum_rows<T, O, BYTES, S, false>;
    if constexpr (BYTES == 16)
      if (a.summed) kernel = k_sum_rows<T, O, BYTES, S, true>;
    launch_behind(stream, kernel, grid, kSumThreads, a, (const Unit<T, BYTES>*)grad, sorted, (O*)out, part);
  });
}

struct GradCall {
  const void* grad;
  int dtype;
  i64 row_len, grad_stride;
  float scale;
  void* out;
  int out_dtype;
};

// The gradient's rows are read and the result's written in units of this many bytes of the former.
static int unit_of(const GradCall& c) {
  const int size = value_bytes(c.dtype), out_size = value_bytes(c.out_dtype);
  int unit = unit_bytes(c.row_len * size, (u64)(uintptr_t)c.grad | (u64)(c.grad_stride * size));
  while (unit > size && (uintptr_t)c.out % min(16, unit / size * out_size) != 0) unit /= 2;
  return unit;
}

// Whether the rows without a sum are cleared behind the sums, which mark the others; if not, the sort clears all rows on its way.
// What is saved is at most min(n, num_rows) rows; lost is what the sort hides and, of a small table, what would have stayed in L2.
// 4.05 M positions into 2.45 M rows of 512 bytes take 781 us for 931, 1 M into 2.5 M of 1 KB 0.85 of the time, into 1 M of 256 bytes
// 0.93, but 100 000 into 250 000 of 1 KB up to 1.09. Rows that share lines of 128 bytes with others cost more to clear one by
// one than together (1 M into 2.5 M of 400 bytes 1.07).
static bool clears_behind(const GradCall& c, i64 n, i64 num_rows) {
  const i64 row_bytes = c.row_len * value_bytes(c.out_dtype);
  return row_bytes % 128 == 0 && (uintptr_t)c.out % 128 == 0 && unit_of(c) == 16 && may_clear_behind(n, num_rows, row_bytes);
}

// Sums of the rows at the sorted positions, into the rows of `out` that the pairs name.
static int sum_sorted(gsb_ctx* ctx, cudaStream_t stream, const GradCall& c, const GradPlan& plan, const u64* sorted, i64 n,
                      i64 num_rows, float* part, u32* summed) {
  const int size = value_bytes(c.dtype), out_size = value_bytes(c.out_dtype);
  const i64 row_bytes = c.row_len * size, stride_bytes = c.grad_stride * size;
  const int unit = unit_of(c);
  SumArgs a{(u32)n, 0, (u32)num_rows, 0, 0, 0, c.scale, summed};
  ScopedKernelTimer timer(ctx, KID_EMBED_GRAD, stream);
  with_unit(c.dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int kBytes = decltype(bytes)::value;
    if (c.out_dtype == c.dtype)
      launch_sum<T, T, kBytes>(stream, a, plan.most_chunks, c.grad, stride_bytes, row_bytes, sorted, c.out, part);
    else
      launch_sum<T, float, kBytes>(stream, a, plan.most_chunks, c.grad, stride_bytes, row_bytes, sorted, c.out, part);
  });
  GSB_LAUNCH_OK();
  const i64 chunks = (n + a.chunk - 1) / a.chunk;
  if (chunks > 1 || summed) {
    dim3 grid(grid_for(chunks - 1, kJoinWarps * kJoinSpan), grid_for(c.row_len, kJoinColumns));
    ClearArgs clear{(uint4*)c.out, 0, 0, 0};
    if (summed) {
      clear.units = (u32)(c.row_len * out_size / 16);
      clear.pieces = (clear.units + kClearPiece - 1) / kClearPiece;
      clear.per_row = (u32)(((1ull << 32) + clear.units - 1) / clear.units);
      grid.x = max(grid.x, (unsigned)min(kNumSMs * 4, grid_for((i64)plan.words * clear.pieces, kJoinWarps)) / grid.y);
    }
    if (c.out_dtype == GSB_F32) launch_behind(stream, k_join_rows<float>, grid, kJoinThreads, a, clear, c.row_len, chunks, sorted, part, (float*)c.out);
    else if (c.out_dtype == GSB_F16) launch_behind(stream, k_join_rows<__half>, grid, kJoinThreads, a, clear, c.row_len, chunks, sorted, part, (__half*)c.out);
    else launch_behind(stream, k_join_rows<__nv_bfloat16>, grid, kJoinThreads, a, clear, c.row_len, chunks, sorted, part, (__nv_bfloat16*)c.out);
    GSB_LAUNCH_OK();
    ctx_count_launches(ctx, 1);
  }
  return GSB_OK;
}

// What the calls that sum gradients ask of their arguments.
static int check_grad(i64 n, i64 num_rows, i64 row_len, i64 grad_stride, int dtype, int out_dtype) {
  GSB_REQUIRE(n >= 0 && n < ((i64)1 << 31) && num_rows >= 0 && num_rows < 0xffffffffll, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(row_len >= 1 && row_len <= GSB_MAX_ROW_LEN && grad_stride >= 0, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(value_bytes(dtype) != 0 && (out_dtype == dtype || out_dtype == GSB_F32), GSB_ERR_INVALID_ARGUMENT);
  return GSB_OK;
}

// What they ask of addresses.
static bool aligned_grad(const void* grad, int dtype, const i64* ids, const void* out, int out_dtype, const void* workspace) {
  return aligned_to(value_bytes(dtype), (const char*)grad) && aligned_to(8, ids) && aligned_to(value_bytes(out_dtype), (const char*)out) &&
         aligned_to(256, (const char*)workspace);
}

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_embedding_lookup(gsb_ctx* ctx, void* stream_, const void* table, int dtype, int64_t num_rows,
                                    int64_t row_len, int64_t row_stride, const int64_t* ids, int64_t n, float scale,
                                    int has_padding, int64_t padding_id, void* out) {
  GSB_ENTER(ctx);
  GSB_REQUIRE(num_rows >= 0 && row_len >= 1 && row_len <= GSB_MAX_ROW_LEN && row_stride >= 0 && n >= 0 && n < ((i64)1 << 31) &&
                  value_bytes(dtype) != 0, GSB_ERR_INVALID_ARGUMENT);
  if (n == 0) return GSB_OK;
  GSB_REQUIRE((table || num_rows == 0) && ids && out, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_to(value_bytes(dtype), (const char*)table, (const char*)out) && aligned_to(8, ids), GSB_ERR_INVALID_ARGUMENT);
  const void* from = nullptr;
  bool resident = false;
  cudaError_t failed = cudaSuccess;
  if (num_rows > 0) {  // device memory, or page-locked host memory by the address that the device uses for it
    cudaPointerAttributes attr;
    GSB_CUDA_OK(cudaPointerGetAttributes(&attr, table));
    GSB_REQUIRE(attr.devicePointer != nullptr && (attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeHost ||
                                                  attr.type == cudaMemoryTypeManaged),
                GSB_ERR_INVALID_ARGUMENT);
    from = attr.devicePointer;
    resident = attr.type == cudaMemoryTypeDevice;
  }
  cudaStream_t stream = (cudaStream_t)stream_;
  const int size = value_bytes(dtype);
  const int unit = unit_bytes(row_len * size, (u64)(uintptr_t)from | (u64)(uintptr_t)out | (u64)(row_stride * size));
  {
    ScopedKernelTimer timer(ctx, KID_EMBED_LOOKUP, stream);
    with_unit(dtype, unit, [&](auto value, auto bytes) {
      typedef decltype(value) T;
      constexpr int kBytes = decltype(bytes)::value;
      const i64 units = row_len * size / kBytes;
      if constexpr (kBytes == 2) {
        const i64 row_bytes = row_len * size;
        if (resident && staged(row_bytes, n)) {
          StagedArgs s;
          s.begin = (const char*)from;
          s.end = s.begin + (num_rows - 1) * row_stride * size + row_bytes;
          s.stage = stage_bytes(row_bytes);
          s.row_bytes = (int)row_bytes;
          const size_t smem = staged_smem(s.stage);
          const i64 most = (i64)kNumSMs * min((i64)16, (i64)(227 * 1024 / (smem + 1024))) * (kStagedThreads / 32);
          s.per_warp = (u32)((n + most - 1) / most);
          const LookupArgs args{ids, (u32)n, (int)row_len, 0, num_rows, row_stride * size, padding_id, has_padding != 0, scale,
                                ctx_counters(ctx)};
          failed = prepare_staged<T>(ctx);
          if (failed == cudaSuccess)
            failed = launch_behind_with(stream, smem, k_lookup_staged<T>, grid_for((n + s.per_warp - 1) / s.per_warp, kStagedThreads / 32),
                                        kStagedThreads, args, s, (T*)out);
          return;
        }
      }
      const RowShape shape = row_shape(units, copy_steps(kBytes), copy_wide(kBytes));
      with_steps(shape.steps, [&](auto steps) {
        constexpr int S = decltype(steps)::value, kRows = lookup_rows(kBytes, S);
        // a group goes through the tiles of its rows' columns, or shares them with others where there are few rows
        const i64 ctas = grid_for((n + kRows - 1) / kRows * shape.lanes, kLookupThreads), tiles = grid_for(units, shape.lanes * S);
        const dim3 grid((unsigned)min((i64)kNumSMs * 32, ctas), (unsigned)min(tiles, max((i64)1, kNumSMs * 8 / ctas)));
        const LookupArgs args{ids, (u32)n, (int)units, shape.lanes, num_rows, row_stride * size / kBytes, padding_id, has_padding != 0,
                              scale, ctx_counters(ctx)};
        auto kernel = k_lookup_rows<T, kBytes, S, 0>;
        if constexpr (kBytes == 2)
          if (shape.lanes == 32) kernel = k_lookup_rows<T, kBytes, S, 32>;
        launch_behind(stream, kernel, grid, kLookupThreads, args, (const Unit<T, kBytes>*)from,
                      (Unit<T, kBytes>*)out);
      });
    });
  }
  GSB_CUDA_OK(failed);
  GSB_LAUNCH_OK();
  return GSB_OK;
}

extern "C" int64_t gsb_embedding_grad_workspace(int64_t n, int64_t num_rows, int64_t row_len) {
  const int st = check_grad(n, num_rows, row_len, row_len, GSB_F32, GSB_F32);
  return st != GSB_OK ? st : (int64_t)grad_plan(n, num_rows, row_len).total_bytes;
}

extern "C" int gsb_embedding_grad(gsb_ctx* ctx, void* stream_, const void* grad, int dtype, int64_t row_len,
                                  int64_t grad_stride, const int64_t* ids, int64_t n, int64_t num_rows, float scale,
                                  int has_padding, int64_t padding_id, void* out, int out_dtype, void* workspace,
                                  int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  int st = check_grad(n, num_rows, row_len, grad_stride, dtype, out_dtype);
  if (st != GSB_OK) return st;
  if (num_rows == 0 && n == 0) return GSB_OK;
  GSB_REQUIRE((out || num_rows == 0) && aligned_grad(grad, dtype, ids, out, out_dtype, workspace), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const size_t out_bytes = (size_t)num_rows * (size_t)row_len * value_bytes(out_dtype);
  if (n == 0) {
    GSB_CUDA_OK(cudaMemsetAsync(out, 0, out_bytes, stream));
    return GSB_OK;
  }
  const GradPlan plan = grad_plan(n, num_rows, row_len);
  GSB_REQUIRE(grad && ids && workspace, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(workspace_bytes >= (int64_t)plan.total_bytes, GSB_ERR_CAPACITY);
  Pieces p(workspace);
  p.take<char>(plan.sort_bytes);
  float* part = p.take<float>((size_t)plan.most_chunks * 2 * (size_t)row_len);
  u32* summed = p.take<u32>(plan.words);
  const GradCall c{grad, dtype, row_len, grad_stride, scale, out, out_dtype};
  if (!clears_behind(c, n, num_rows)) summed = nullptr;
  const u64* sorted;
  {
    ScopedKernelTimer timer(ctx, KID_KEY_SORT, stream);
    SortCall call{KeySource{ids, n, num_rows, has_padding != 0, padding_id, ctx_counters(ctx)}, SORT_PAIRS};
    call.zero = summed ? (void*)summed : out;
    call.zero_bytes = summed ? plan.words * sizeof(u32) : out_bytes;
    st = key_sort(ctx, stream, call, workspace, &sorted);
  }
  if (st != GSB_OK) return st;
  return sum_sorted(ctx, stream, c, plan, sorted, n, num_rows, part, summed);
}

extern "C" int gsb_embedding_grad_rows(gsb_ctx* ctx, void* stream_, const void* grad, int dtype, int64_t row_len,
                                       int64_t grad_stride, const int64_t* ids, int64_t n, int64_t num_rows, float scale,
                                       int has_padding, int64_t padding_id, int64_t* out_ids, void* out_rows, int out_dtype,
                                       int64_t* out_count, void* workspace, int64_t workspace_bytes, int64_t* count_host) {
  GSB_ENTER(ctx);
  int st = check_grad(n, num_rows, row_len, grad_stride, dtype, out_dtype);
  if (st != GSB_OK) return st;
  cudaStream_t stream = (cudaStream_t)stream_;
  if (count_host) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    GSB_CUDA_OK(cudaStreamIsCapturing(stream, &capture));
    GSB_REQUIRE(capture == cudaStreamCaptureStatusNone, GSB_ERR_UNSUPPORTED);
    *count_host = 0;
  }
  GSB_REQUIRE(out_count, GSB_ERR_INVALID_ARGUMENT);
  if (n == 0) {
    GSB_CUDA_OK(cudaMemsetAsync(out_count, 0, sizeof(int64_t), stream));
    return GSB_OK;
  }
  const GradPlan plan = grad_plan(n, num_rows, row_len);
  GSB_REQUIRE(grad && ids && out_ids && out_rows && workspace, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_grad(grad, dtype, ids, out_rows, out_dtype, workspace) && aligned_to(8, out_ids, out_count),
              GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(workspace_bytes >= (int64_t)plan.total_bytes, GSB_ERR_CAPACITY);
  Pieces p(workspace);
  p.take<char>(plan.sort_bytes);
  float* part = p.take<float>((size_t)plan.most_chunks * 2 * (size_t)row_len);
  const u64* sorted;
  SortCall call{KeySource{ids, n, num_rows, has_padding != 0, padding_id, ctx_counters(ctx)}, SORT_RANKS};
  call.distinct = out_ids;
  call.number = out_count;
  std::unique_lock<std::mutex> waiting;
  if (count_host) {
    waiting = std::unique_lock<std::mutex>(ctx_rows_wait(ctx));
    call.mail = ctx_mail(ctx, WAIT_ROWS);
  }
  {
    ScopedKernelTimer timer(ctx, KID_KEY_SORT, stream);
    st = key_sort(ctx, stream, call, workspace, &sorted);
  }
  if (st != GSB_OK) return st;
  st = sum_sorted(ctx, stream, GradCall{grad, dtype, row_len, grad_stride, scale, out_rows, out_dtype}, plan, sorted, n, n, part, nullptr);
  if (st != GSB_OK || !count_host) return st;
  return ctx_mail_result(ctx, stream, call.mail, 1, count_host, WAIT_ROWS);
}
