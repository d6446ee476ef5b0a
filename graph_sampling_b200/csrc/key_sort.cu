// One launch sorts: CTAs own equal stretches of the positions and go through the digits of the key, least significant first.
// Per digit a CTA counts its stretch, all counts become visible behind a barrier, every CTA adds up for itself what lies before
// its own (in place of a scan with a barrier of its own), and puts its positions where they belong.  Nothing depends on the
// order in which CTAs run.
//
// Up to 32 768 positions are sorted by one cluster of 8 CTAs in its shared memory (k_sort_cluster): counts are read and positions
// written from CTA to CTA, the barrier is the hardware's, and nothing waits for global memory between the ids and the result.
// More go through global memory (k_sort_grid), tile by tile through shared memory so that neighbouring threads write
// neighbouring words, by CTAs that are launched cooperatively and meet at a word in the workspace (grid_sync.cuh).  Digits are
// as wide as keeps the number of passes small: 11 bits where few CTAs have to read each other's counts, 10 or 9 where up to 148 do.
// A kernel for each width: with the width as an argument passes took 5 to 15 % longer (500 000 by 64 experts 16.7 us for 15.1).
//
// The launch may also clear memory (the rows of a dense gradient that no position has), with bulk copies of zeros from shared
// memory: SMs without a sorting CTA clear all the time, the others between the steps of the sort or behind it.
//
// What bounds it: instruction issue and the latencies of a pass's steps, not memory (1 000 003 positions by 27 bits, three passes
// and the ranks of the distinct keys: 64 us between two events, DRAM at 2 % of its peak, half of the issue slots used).  Ranking takes a
// third of a pass, the counts of all CTAs and the placing a quarter each, two barriers the rest.
#include "key_sort.cuh"

#include <atomic>
#include <initializer_list>

#include "grid_sync.cuh"
#include "launch.cuh"
#include "scan.cuh"

namespace gsb {

namespace {

// 32 warps hide more of a large sort's latencies, 16 have less to do for each digit of a small one.
constexpr int kClusterThreads = 512, kGridThreads = 1024;
constexpr int kRounds = 8;
constexpr int kClusterCtas = 8;
// Up to 1 024 positions one CTA sorts for itself: 17 bits of 1 024 in 6.5 us, shared by two CTAs in 7.2; of 2 048 in 8.6 and 8.2.
constexpr int kAloneShares = 2;
constexpr int kClusterBits = 11, kGridBits = 10;
// Ten bits make one pass of two for up to 1 023 keys (a million positions 23.1 us for 37.5), or save a pass of few positions (200 000 by
// 20 bits 45.4 for 47.6); of many, two wide passes cost more than three narrow ones (4 M by 20 bits 437 for 416, a million the same).
constexpr i64 kFewPositions = 600000;
constexpr int kMinBits = 5;  // a row of counts is read in pieces of 16 bytes
constexpr int kMaxBins = 1 << kClusterBits;
constexpr int kPiece = 16384;      // bytes cleared by one bulk copy
constexpr int kPiecesAtOnce = 32;  // at most, that a sorting CTA starts between two steps
constexpr u32 kAllLanes = 0xffffffffu;

struct SortArgs {
  SortCall call;
  u64 *from, *to;  // [key : 32 | position : 32], exchanged after every pass
  u32* counts;     // CTAs x bins
  int ctas;        // that sort; the others clear
  int passes;
  u32 stretch;     // positions per CTA
  int rounds;      // of a tile: a position per thread each
  bool single;     // a stretch is one tile, which stays in registers between counting and placing
  int room;        // bytes of shared memory for a tile's items
  int pieces;      // to clear, that a sorting CTA starts at a time
  GridSync sync;
};

__device__ __forceinline__ u32 key_of(const KeySource& s, u32 i, bool check) {
  const i64 id = __ldg(s.ids + i);
  if (s.has_dropped && id == s.dropped) return (u32)s.num_keys;
  if ((u64)id < (u64)s.num_keys) return (u32)id;
  if (check) raise_error(s.counters, GSB_ERR_INDEX_RANGE, i);
  return (u32)s.num_keys;
}

// (The loops over a thread's items and digits below have no `break`: with it, threads that had left came to the next barrier before
// their warp's others, and it let the CTA go on too early.)

// The CTA's pieces of the memory to clear, started by one thread.  The bytes before the first and behind the last 16-byte
// boundary are written by the first CTA's threads.
struct Clearing {
  char* base;
  size_t bytes, next, step;
  u32 zeros;

  __device__ Clearing(const SortCall& c, char* smem, size_t number, size_t of) {
    const size_t head = min(c.zero_bytes, (size_t)(0 - (uintptr_t)c.zero & 15));
    base = (char*)c.zero + head;
    bytes = (c.zero_bytes - head) / 16 * 16;
    next = number * kPiece;
    step = of * kPiece;
    zeros = (u32)__cvta_generic_to_shared(smem);
    if (c.zero_bytes == 0) return;
    for (int q = threadIdx.x; q < kPiece / 16; q += blockDim.x) ((uint4*)smem)[q] = make_uint4(0, 0, 0, 0);
    if (number == 0) {
      if (threadIdx.x < head) ((char*)c.zero)[threadIdx.x] = 0;
      const size_t tail = c.zero_bytes - head - bytes;
      if (threadIdx.x < tail) base[bytes + threadIdx.x] = 0;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
  __device__ __forceinline__ void start(int most) {
    if (threadIdx.x != 0) return;
    for (int q = 0; q < most && next < bytes; ++q, next += step)
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(base + next), "r"(zeros),
                   "r"((u32)min((size_t)kPiece, bytes - next))
                   : "memory");
  }
  __device__ __forceinline__ void finish() {
    if (threadIdx.x != 0) return;
    while (next < bytes) start(1 << 20);
    asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group 0;" ::: "memory");
  }
};

// Exclusive scan over the CTA; the total is left in s_scan[32], for whoever reads it behind the next barrier.
template <int WARPS>
__device__ __forceinline__ u32 scan_threads(u32 v, u32* s_scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u32 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u32 t = __shfl_up_sync(kAllLanes, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // s_scan may still be read
  if (lane == 31) s_scan[warp] = inc;
  __syncthreads();
  u32 w = lane < WARPS ? s_scan[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u32 t = __shfl_up_sync(kAllLanes, w, o);
    if (lane >= o) w += t;
  }
  const u32 before = __shfl_sync(kAllLanes, w, (warp + 31) & 31);
  if (threadIdx.x == 31) s_scan[32] = w;
  return (warp == 0 ? 0 : before) + inc - v;
}

// Ranks of the items that a warp holds (round by round, lane by lane) among those of the same digit; `counts`, cleared, becomes the
// warp's counts.  Lanes with the same digit are found bit by bit, by a vote each: with the match instruction 1 000 003 positions
// take 75 us for 64, 4.05 M take 191 for 156.  mine: the thread's first item, of `items`.
template <int ROUNDS, int BITS>
__device__ __forceinline__ void rank_items(const u32 (&key)[ROUNDS], u32 (&rank)[ROUNDS], unsigned short* counts, int shift,
                                           int rounds, u32 mine, u32 items) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (r >= rounds) break;
    const bool valid = mine + r * 32 < items;
    const u32 digit = (key[r] >> shift) & ((1u << BITS) - 1u);
    u32 peers = __ballot_sync(kAllLanes, valid);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const u32 bit = (digit >> b) & 1u;
      peers &= __ballot_sync(kAllLanes, bit) ^ (bit - 1u);
    }
    const u32 before = __popc(peers & ((1u << lane) - 1u));
    const u32 found = valid ? counts[digit] : 0;
    __syncwarp();
    if (valid && before == 0) counts[digit] = (unsigned short)(found + __popc(peers));
    __syncwarp();
    rank[r] = found + before;
  }
}

// Warps' counts become starts within the digit, two digits at a time; the digits' counts in the tile go to s_tile.
template <int THREADS>
__device__ __forceinline__ void warp_starts(unsigned short* s_count, u32* s_tile, int bins) {
  for (int d = threadIdx.x; d < bins / 2; d += THREADS) {
    u32* column = (u32*)s_count + d;
    u32 run = 0;
#pragma unroll
    for (int part = 0; part < THREADS / 512; ++part) {
      u32 k[16];
#pragma unroll
      for (int w = 0; w < 16; ++w) k[w] = column[(part * 16 + w) * (bins / 2)];
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        column[(part * 16 + w) * (bins / 2)] = run;
        run += k[w];  // both halves: a tile has fewer than 2^16 items
      }
    }
    s_tile[2 * d] = run & 0xffffu;
    s_tile[2 * d + 1] = run >> 16;
  }
  __syncthreads();
}

// offsets[q] = row for q in [from, to), a range per lane of a whole warp: long ones (experts without a slot lie in between) by all lanes.
// By one thread each, an order of one slot by 65 536 experts took 308 us.
__device__ __forceinline__ void fill_offsets(i64* offsets, u32 from, u32 to, u32 row) {
  const int lane = threadIdx.x & 31;
  const bool is_long = to > from + 32;
  if (!is_long)
    for (; from < to; ++from) offsets[from] = row;
  for (u32 left = __ballot_sync(kAllLanes, is_long); left != 0; left &= left - 1) {
    const int l = __ffs(left) - 1;
    const u32 begin = __shfl_sync(kAllLanes, from, l), end = __shfl_sync(kAllLanes, to, l), value = __shfl_sync(kAllLanes, row, l);
    for (u32 q = begin + lane; q < end; q += 32) offsets[q] = value;
  }
}

// Addresses in another CTA's shared memory.
__device__ __forceinline__ u32 in_cta(const void* p, u32 cta) {
  u32 there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((u32)__cvta_generic_to_shared(p)), "r"(cta));
  return there;
}
__device__ __forceinline__ u32 load_far(u32 address) {
  u32 v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ uint4 load_far4(u32 address) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ void store_far(u32 address, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(address), "l"(v) : "memory");
}

template <int DIGIT>
__global__ void __launch_bounds__(kClusterThreads, 1) k_sort_cluster(const SortArgs a) {
  constexpr int kThreads = kClusterThreads, kWarps = kThreads / 32, kPer = (1 << kClusterBits) / kThreads;
  extern __shared__ __align__(128) char smem[];
  __shared__ u32 s_scan[33], s_heads;
  await_previous();
  const SortCall& c = a.call;
  const u32 cta = blockIdx.x;
  if (cta >= (u32)a.ctas) {
    if (cta < kClusterCtas) return;
    Clearing clearing(c, smem, cta - kClusterCtas, gridDim.x - kClusterCtas);
    clearing.finish();
    return;
  }
  constexpr int bins = 1 << DIGIT;
  const int rounds = a.rounds;
  u64* s_items = (u64*)smem;                                   // the stretch: written by all CTAs
  u32* s_tile = (u32*)(s_items + rounds * kThreads);           // its counts: read by all CTAs
  u32* s_base = s_tile + bins;                                 // where the CTA's items of a digit begin
  unsigned short* s_count = (unsigned short*)(s_base + bins);  // kWarps x bins
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u32 n = (u32)c.source.n, lo = cta * a.stretch, items = min(a.stretch, n - lo);
  const u32 mine = warp * (rounds * 32) + lane;                // the thread's first item of the stretch
  const bool alone = a.ctas == 1;
  u32 key[kRounds], at[kRounds], rank[kRounds];
  auto barrier = [&] {
    if (alone) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  };
  auto load = [&](bool ids) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const u32 i = mine + r * 32;
      key[r] = kNoRow;
      if (r >= rounds || i >= items) continue;
      if (ids) {
        key[r] = key_of(c.source, lo + i, true);
        at[r] = lo + i;
      } else {
        const u64 pair = s_items[i];
        key[r] = pair_key(pair);
        at[r] = pair_at(pair);
      }
    }
  };

  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * DIGIT;
    load(pass == 0);
    for (int q = threadIdx.x; q < kWarps * bins / 8; q += kThreads) ((uint4*)s_count)[q] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    rank_items<kRounds, DIGIT>(key, rank, s_count + warp * bins, shift, rounds, mine, items);
    __syncthreads();
    warp_starts<kThreads>(s_count, s_tile, bins);
    barrier();
    {
      constexpr int per = bins > kThreads ? bins / kThreads : 1;  // digits of a thread
      static_assert(kPer == 4, "four digits are one access");
      u32 all[kPer] = {}, before[kPer] = {};
#pragma unroll
      for (int g = 0; g < kClusterCtas; ++g) {
        if (g >= a.ctas) continue;
        u32 v[kPer] = {};
        if (per == kPer) {
          const uint4 w = load_far4(in_cta(s_tile + threadIdx.x * kPer, g));
          v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (q < per && threadIdx.x * per + q < bins) v[q] = load_far(in_cta(s_tile + threadIdx.x * per + q, g));
        }
#pragma unroll
        for (int q = 0; q < kPer; ++q) all[q] += v[q], before[q] += g < (int)cta ? v[q] : 0;
      }
      const u32 sum = all[0] + all[1] + all[2] + all[3];
      u32 start = scan_threads<kWarps>(sum, s_scan);
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int e = threadIdx.x * per + q;
        if (q >= per || e >= bins) continue;
        s_base[e] = start + before[q];
        if (c.result == SORT_ORDER && a.passes == 1 && cta == 0 && e <= c.source.num_keys) c.offsets[e] = start;
        start += all[q];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (r >= rounds || mine + r * 32 >= items) continue;
      const u32 digit = (key[r] >> shift) & (bins - 1);
      const u32 spot = s_base[digit] + s_count[warp * bins + digit] + rank[r], to = spot / a.stretch;
      const u64 pair = (u64)key[r] << 32 | at[r];
      if (spot >= n) continue;  // never, unless memory was overwritten
      if (alone) s_items[spot] = pair;
      else store_far(in_cta(s_items + (spot - to * a.stretch), to), pair);
    }
    barrier();
  }

  if (c.result == SORT_PAIRS) {
    for (u32 i = threadIdx.x; i < items; i += kThreads) a.to[lo + i] = s_items[i];
    return;  // nobody reads this CTA's memory any more
  }
  // the key before the CTA's first
  u32 before = kNoRow;
  if (cta > 0) before = load_far(in_cta((const u32*)(s_items + a.stretch - 1) + 1, cta - 1));
  if (c.result == SORT_ORDER) {
    const u32 experts = (u32)c.source.num_keys;
    for (u32 base = 0; base < items; base += kThreads) {
      const u32 i = base + threadIdx.x, j = lo + i;
      u32 from = 0, to = 0, behind = 0;
      if (i < items) {
        const u64 pair = s_items[i];
        const u32 e = pair_key(pair);
        c.order_source[j] = pair_at(pair);
        c.place[pair_at(pair)] = e < experts ? (i64)j : ~(i64)j;
        from = j == 0 ? 0 : (i > 0 ? pair_key(s_items[i - 1]) : before) + 1;
        to = e + 1;
        if (j == n - 1) behind = experts + 1;
      }
      if (a.passes == 1) continue;
      fill_offsets(c.offsets, from, to, j);
      fill_offsets(c.offsets, to, behind, n);
    }
    barrier();  // until everybody has read the key before his first
    return;
  }
  // SORT_RANKS
  const u32 none = (u32)c.source.num_keys;
  load(false);
  u32 heads[kRounds], of_warp = 0;
  {
    u32 left_key = warp == 0 ? before : mine - lane < items ? pair_key(s_items[mine - lane - 1]) : kNoRow;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      u32 left = __shfl_up_sync(kAllLanes, key[r], 1);
      if (lane == 0) left = left_key;
      left_key = __shfl_sync(kAllLanes, key[r], 31);
      heads[r] = __ballot_sync(kAllLanes, key[r] < none && key[r] != left);
      of_warp += __popc(heads[r]);
    }
  }
  u32 next = scan_threads<kWarps>(lane == 0 ? of_warp : 0, s_scan);
  __syncthreads();
  const u32 of_cta = s_scan[32];
  if (threadIdx.x == 0) s_heads = of_cta;
  barrier();
  u32 others = 0;
  if (!alone)
#pragma unroll
    for (int g = 0; g < kClusterCtas; ++g)
      if (g < (int)cta) others += load_far(in_cta(&s_heads, g));
  next = __shfl_sync(kAllLanes, next, 0) + others;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const u32 i = mine + r * 32, my = next + __popc(heads[r] & ((2u << lane) - 1u)) - 1u;  // of the latest head up to here
    if (r < rounds && i < items) {
      if (heads[r] >> lane & 1u) c.distinct[my] = key[r];
      a.to[lo + i] = (u64)(key[r] < none ? my : kNoRow) << 32 | at[r];
    }
    next += __popc(heads[r]);
  }
  if (cta == (u32)a.ctas - 1 && threadIdx.x == 0) {
    c.number[0] = others + of_cta;
    mail_post(c.mail, 0, others + of_cta, c.source.counters);
  }
  barrier();  // until everybody has read s_heads
}

// The word that the sorting CTAs meet at.
__global__ void k_clear_word(u64* word) {
  await_previous();
  *word = 0;
}

template <int DIGIT>
__global__ void __launch_bounds__(kGridThreads, 1) k_sort_grid(const SortArgs a) {
  constexpr int kThreads = kGridThreads, kWarps = kThreads / 32;
  static_assert((1 << kGridBits) <= kThreads, "a digit per thread");
  extern __shared__ __align__(128) char smem[];
  __shared__ u32 s_scan[33];
  await_previous();
  const SortCall& c = a.call;
  const u32 cta = blockIdx.x;
  constexpr int bins = 1 << DIGIT;
  char* s_zeros = smem;                                        // kPiece
  u64* s_items = (u64*)(smem + (c.zero_bytes > 0 ? kPiece : 0));  // a tile; also the partial sums of the counts
  u32* s_base = (u32*)((char*)s_items + a.room);               // where the next item of a digit goes
  u32* s_tile = s_base + bins;                                 // where a digit starts in the tile
  unsigned short* s_count = (unsigned short*)(s_tile + bins);  // kWarps x bins
  Clearing clearing(c, s_zeros, cta, gridDim.x);
  if (cta >= (u32)a.ctas) {
    clearing.finish();
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u32 n = (u32)c.source.n, lo = cta * a.stretch, hi = min(lo + a.stretch, n);
  const bool single = a.single;
  const int rounds = a.rounds;
  const u32 tile = (u32)rounds * kThreads, mine = warp * (rounds * 32) + lane;  // the thread's first item of a tile
  const u64* from = a.from;
  u64* to = a.to;
  u32 key[kRounds], at[kRounds], rank[kRounds];

  auto give_up = [&] {  // results that are wrong but within range
    if (c.result == SORT_RANKS) c.number[0] = 0;
    if (c.result == SORT_ORDER)
      for (u32 q = cta; q < max(n, (u32)c.source.num_keys + 1); q += a.ctas) {
        if (q <= (u32)c.source.num_keys) c.offsets[q] = 0;
        if (q < n) c.order_source[q] = q, c.place[q] = ~(i64)q;
      }
    clearing.finish();
  };
  u32 met = 0;
  auto barrier = [&] {
    ++met;
    grid_barrier(a.sync, met, give_up, (u32)a.ctas);
  };
  auto load_tile = [&](u32 base, bool ids, bool check) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const u32 i = base + mine + r * 32;
      key[r] = kNoRow;
      if (r >= rounds || i >= hi) continue;
      if (ids) {
        key[r] = key_of(c.source, i, check);
        at[r] = i;
      } else {
        const u64 pair = __ldcg(from + i);
        key[r] = pair_key(pair);
        at[r] = pair_at(pair);
      }
    }
  };
  // Ranks of a tile's items, and the warps' starts.
  auto rank_tile = [&](u32 base, int shift) {
    for (int q = threadIdx.x; q < kWarps * bins / 8; q += kThreads) ((uint4*)s_count)[q] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    rank_items<kRounds, DIGIT>(key, rank, s_count + warp * bins, shift, rounds, mine, hi - base);
    __syncthreads();
    warp_starts<kThreads>(s_count, s_tile, bins);
  };

  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * DIGIT;
    const bool ids = pass == 0, last = pass == a.passes - 1;
    // counts of the stretch
    u32* row = a.counts + (size_t)cta * bins;
    if (single) {
      load_tile(lo, ids, true);
      rank_tile(lo, shift);
    } else {
      for (int d = threadIdx.x; d < bins; d += kThreads) s_tile[d] = 0;
      __syncthreads();
      for (u32 base = lo; base < hi; base += tile) {
        load_tile(base, ids, true);
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
          if (r < rounds && base + mine + r * 32 < hi) atomicAdd(&s_tile[(key[r] >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
    }
    if ((int)threadIdx.x < bins) row[threadIdx.x] = s_tile[threadIdx.x];
    clearing.start(a.pieces);
    barrier();
    // all counts: of each digit, and of each digit in the CTAs before this one; groups of threads share the rows
    const int e = threadIdx.x;  // the thread's digit
    {
      const int per_row = bins / 4, groups = min(min(kThreads / per_row, a.ctas), 16), group = threadIdx.x / per_row;
      const int d = (threadIdx.x % per_row) * 4;
      u32* s_total = (u32*)s_items;  // groups x bins
      u32* s_before = s_total + groups * bins;
      if (group < groups) {
        uint4 total = make_uint4(0, 0, 0, 0), less = total;
        constexpr int kBatch = 6;  // rows on their way
        for (int g0 = group; g0 < a.ctas; g0 += kBatch * groups) {
          uint4 v[kBatch];
#pragma unroll
          for (int q = 0; q < kBatch; ++q) {
            const int g = g0 + q * groups;
            v[q] = g < a.ctas ? __ldcg((const uint4*)(a.counts + (size_t)g * bins + d)) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int q = 0; q < kBatch; ++q) {
            total.x += v[q].x, total.y += v[q].y, total.z += v[q].z, total.w += v[q].w;
            if (g0 + q * groups < (int)cta) less.x += v[q].x, less.y += v[q].y, less.z += v[q].z, less.w += v[q].w;
          }
        }
        *(uint4*)(s_total + group * bins + d) = total;
        *(uint4*)(s_before + group * bins + d) = less;
      }
      __syncthreads();
      u32 all = 0, before = 0;
      if (e < bins)
        for (int g = 0; g < groups; ++g) all += s_total[g * bins + e], before += s_before[g * bins + e];
      const u32 start = scan_threads<kWarps>(all, s_scan);
      if (e < bins) {
        s_base[e] = start + before;
        if (c.result == SORT_ORDER && a.passes == 1 && cta == 0 && e <= c.source.num_keys) c.offsets[e] = start;
      }
      __syncthreads();
    }
    // to their places
    if (!single) load_tile(lo, ids, false);
    for (u32 base = lo; base < hi; base += tile) {
      if (!single) {
        rank_tile(base, shift);
      }
      // s_tile: counts -> starts in the tile; s_base: where the tile's first item of a digit goes, less its place in the tile
      const u32 count = e < bins ? s_tile[e] : 0, start = scan_threads<kWarps>(count, s_scan);
      if (e < bins) {
        s_tile[e] = start;
        s_base[e] -= start;
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        if (r >= rounds || base + mine + r * 32 >= hi) continue;
        const u32 digit = (key[r] >> shift) & (bins - 1);
        const u32 spot = s_tile[digit] + s_count[warp * bins + digit] + rank[r];
        s_items[spot] = (u64)key[r] << 32 | at[r];
        if (c.result == SORT_ORDER && last) {
          const u32 row_of = s_base[digit] + spot;
          if (row_of >= n || at[r] >= n) continue;  // never, unless memory was overwritten
          c.place[at[r]] = key[r] < (u32)c.source.num_keys ? (i64)row_of : ~(i64)row_of;
        }
      }
      if (base + tile < hi) load_tile(base + tile, ids, false);  // on its way while this tile is written
      __syncthreads();
      clearing.start(a.pieces);
      const u32 items = min(tile, hi - base);
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const u32 j = r * kThreads + threadIdx.x;
        if (j >= items) continue;
        const u64 item = s_items[j];
        const u32 spot = s_base[(pair_key(item) >> shift) & (bins - 1)] + j;
        if (spot >= n) continue;  // as above
        if (c.result == SORT_ORDER && last) c.order_source[spot] = pair_at(item);
        if (c.result != SORT_ORDER || a.passes > 1) to[spot] = item;
      }
      __syncthreads();
      if (e < bins) s_base[e] += start + count;
    }
    u64* free = const_cast<u64*>(from);
    from = to;
    to = free;
    if (!last || c.result == SORT_RANKS || (c.result == SORT_ORDER && a.passes > 1)) barrier();
  }

  if (c.result == SORT_ORDER && a.passes > 1) {
    for (u32 base = lo; base < hi; base += kThreads) {
      const u32 j = base + threadIdx.x;
      u32 begin = 0, end = 0, behind = 0;
      if (j < hi) {
        end = pair_key(__ldcg(from + j)) + 1;
        begin = j > 0 ? pair_key(__ldcg(from + j - 1)) + 1 : 0;
        if (j == n - 1) behind = (u32)c.source.num_keys + 1;
      }
      fill_offsets(c.offsets, begin, end, j);
      fill_offsets(c.offsets, end, behind, n);
    }
  }
  if (c.result == SORT_RANKS) {
    const u32 none = (u32)c.source.num_keys;
    // the tile's items, and which of them are the first of their key; returns how many of the warp's are
    u32 (&heads)[kRounds] = rank;
    auto find_heads = [&](u32 base) {
      load_tile(base, false, false);
      const u32 begin = base + warp * (rounds * 32);
      u32 before = begin > 0 && begin < hi ? pair_key(__ldcg(from + begin - 1)) : kNoRow, all = 0;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        u32 left = __shfl_up_sync(kAllLanes, key[r], 1);
        if (lane == 0) left = before;
        before = __shfl_sync(kAllLanes, key[r], 31);
        heads[r] = __ballot_sync(kAllLanes, key[r] < none && key[r] != left);
        all += __popc(heads[r]);
      }
      return all;
    };
    u32 of_thread = 0, of_tile = 0;
    for (u32 base = lo; base < hi; base += tile) of_thread += of_tile = find_heads(base);
    scan_threads<kWarps>(lane == 0 ? of_thread : 0, s_scan);
    __syncthreads();
    if (threadIdx.x == 0) a.counts[cta] = s_scan[32];
    barrier();
    u32 others = threadIdx.x < cta ? __ldcg(a.counts + threadIdx.x) : 0;  // cta < kThreads
    scan_threads<kWarps>(others, s_scan);
    __syncthreads();
    u32 before = s_scan[32];
    for (u32 base = lo; base < hi; base += tile) {
      if (!single) of_tile = find_heads(base);
      u32 next = before + scan_threads<kWarps>(lane == 0 ? of_tile : 0, s_scan);
      next = __shfl_sync(kAllLanes, next, 0);
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const u32 i = base + mine + r * 32, my = next + __popc(heads[r] & ((2u << lane) - 1u)) - 1u;  // of the latest head up to here
        if (r < rounds && i < hi) {
          if (heads[r] >> lane & 1u) c.distinct[my] = key[r];
          to[i] = (u64)(key[r] < none ? my : kNoRow) << 32 | at[r];
        }
        next += __popc(heads[r]);
      }
      __syncthreads();
      before += s_scan[32];
    }
    if (cta == (u32)a.ctas - 1 && threadIdx.x == 0) {
      c.number[0] = before;
      mail_post(c.mail, 0, before, c.source.counters);
    }
  }
  clearing.finish();
}

// Of both kernels: a full tile, the widest digits, and zeros to copy.
constexpr int kMostShared = kPiece + kGridThreads * kRounds * 8 + kMaxBins * (8 + kClusterThreads / 32 * 2);
static_assert(kMostShared <= 227 * 1024, "");

struct Plan {
  bool cluster, single;
  int ctas, passes, digit, rounds;
  u32 stretch;
  int threads() const { return cluster ? kClusterThreads : kGridThreads; }
  int bins() const { return 1 << digit; }
  int room() const {  // for a tile's items, and for the partial sums of the counts: 2 words x groups x bins
    return max(rounds * threads() * 8, cluster ? 0 : 2 * 4 * min(16 * bins(), 4 * threads()));
  }
  size_t smem(bool clears) const {
    const int sort = room() + bins() * 8 + threads() / 32 * bins() * 2;
    return (size_t)(cluster ? max(sort, clears ? kPiece : 0) : sort + (clears ? kPiece : 0));
  }
};

Plan plan_of(i64 n, i64 num_keys, int most = kNumSMs) {  // most: CTAs of a large sort
  Plan p;
  int bits = 1;  // of the largest key, num_keys itself
  while (bits < 32 && (num_keys >> bits) != 0) ++bits;
  // The cluster's passes are short and may be fewer, the grid has more SMs to rank with: one pass over 32 768 positions takes 11.0
  // us in the grid and 14.7 in the cluster, over 16 384 12.4 and 12.4; two passes and the ranks over 32 768 31.3 and 29.5; and by 11
  // bits, of which the grid makes two passes, 20.8 and 17.9.
  p.cluster = n <= (i64)kClusterCtas * kClusterThreads * (bits <= kGridBits ? kRounds / 2 : kRounds);
  const i64 threads = p.threads(), shares = (n + threads - 1) / threads;
  const i64 most_ctas = !p.cluster ? most : shares <= kAloneShares ? 1 : kClusterCtas;
  const i64 per = (shares + most_ctas - 1) / most_ctas;
  p.stretch = (u32)(per * threads);
  p.ctas = (int)((shares + per - 1) / per);
  p.single = per <= kRounds;
  const i64 tiles = (per + kRounds - 1) / kRounds;  // of a stretch, about equal
  p.rounds = (int)((per + tiles - 1) / tiles);
  const int widest = p.cluster ? kClusterBits : bits <= kGridBits || n <= kFewPositions ? kGridBits : kGridBits - 1;
  p.passes = (bits + widest - 1) / widest;
  p.digit = (bits + p.passes - 1) / p.passes;
  if (p.digit < kMinBits) p.digit = kMinBits;
  return p;
}

// By the width of a digit; null where a kernel does not use it.
const void* kernel_of(bool cluster, int digit) {
  static const void* const in_cluster[] = {(const void*)k_sort_cluster<5>, (const void*)k_sort_cluster<6>, (const void*)k_sort_cluster<7>,
                                           (const void*)k_sort_cluster<8>, (const void*)k_sort_cluster<9>, (const void*)k_sort_cluster<10>,
                                           (const void*)k_sort_cluster<11>};
  static const void* const in_grid[] = {(const void*)k_sort_grid<5>, (const void*)k_sort_grid<6>, (const void*)k_sort_grid<7>,
                                        (const void*)k_sort_grid<8>, (const void*)k_sort_grid<9>, (const void*)k_sort_grid<10>};
  static_assert(kMinBits == 5 && kClusterBits == 11 && kGridBits == 10, "the lists above");
  if (digit < kMinBits || digit > (cluster ? kClusterBits : kGridBits)) return nullptr;
  return cluster ? in_cluster[digit - kMinBits] : in_grid[digit - kMinBits];
}

// Once per device: the kernels may use as much shared memory as they need, and how many clusters are resident at once (15 on a
// B200, two per GPC but one): a cluster that clears and has to wait for the one that sorts comes behind it (16 384 positions and 134
// MB in 38 us for 23).
int prepare(gsb_ctx* ctx, int* clusters) {
  static std::atomic<int> known[64];
  const int device = ctx_device(ctx);
  if (device >= 0 && device < 64 && known[device] > 0) {
    *clusters = known[device];
    return GSB_OK;
  }
  for (int digit = kMinBits; digit <= kClusterBits + kGridBits; ++digit) {
    const void* kernel = digit <= kClusterBits ? kernel_of(true, digit) : kernel_of(false, digit - kClusterBits);
    if (kernel) GSB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kNumSMs / kClusterCtas * kClusterCtas);
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = kMostShared;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kClusterCtas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  GSB_CUDA_OK(cudaOccupancyMaxActiveClusters(clusters, kernel_of(true, kClusterBits), &cfg));
  if (*clusters < 2) *clusters = 2;  // one that clears there has to be
  if (device >= 0 && device < 64) known[device] = *clusters;
  return GSB_OK;
}

int launch(gsb_ctx* ctx, cudaStream_t stream, SortArgs& a, bool cluster, int digit, int grid, size_t smem) {
  const void* kernel = kernel_of(cluster, digit);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(cluster ? kClusterThreads : kGridThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  if (cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kClusterCtas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  } else {
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
  }
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  void* args[] = {&a};
  GSB_CUDA_OK(cudaLaunchKernelExC(&cfg, kernel, args));
  return GSB_OK;
}

}  // namespace

size_t key_sort_bytes(i64 n, i64 num_keys) {
  if (n <= 0) return 256;
  const Plan p = plan_of(n, num_keys);
  Pieces w(nullptr);
  w.take<u64>(32);
  w.take<u32>((size_t)p.ctas << p.digit);
  w.take<u64>((size_t)n);
  w.take<u64>((size_t)n);
  return w.used;
}

int key_sort(gsb_ctx* ctx, cudaStream_t stream, const SortCall& call, void* workspace, const u64** pairs, int most_ctas) {
  const i64 n = call.source.n;
  int clusters = 0;
  const int st = prepare(ctx, &clusters);
  if (st != GSB_OK) return st;
  static int resident[64];
  const int most = min(most_ctas, ctx_resident_ctas(ctx, kernel_of(false, kGridBits), kGridThreads, kMostShared, resident));
  const Plan p = plan_of(n, call.source.num_keys, max(1, most));  // fewer CTAs need less of the workspace
  GSB_REQUIRE(p.cluster || most > 0, GSB_ERR_UNSUPPORTED);
  Pieces w(workspace);
  u64* word = w.take<u64>(32);
  SortArgs a;
  a.call = call;
  a.counts = w.take<u32>((size_t)p.ctas << p.digit);
  a.from = w.take<u64>((size_t)n);
  a.to = w.take<u64>((size_t)n);
  a.ctas = p.ctas;
  a.passes = p.passes;
  a.stretch = p.stretch;
  a.rounds = p.rounds;
  a.single = p.single;
  a.room = p.room();
  int barriers = 2 * p.passes - 1;
  if (call.result == SORT_RANKS) barriers += 2;
  if (call.result == SORT_ORDER && p.passes > 1) barriers += 1;
  a.sync = GridSync{word, 0, (u32)barriers, call.source.counters, (int)ctx_option(ctx, GSB_OPT_MAX_POLLS)};
  if (pairs) *pairs = p.cluster || ((p.passes + (call.result == SORT_RANKS ? 1 : 0)) & 1) ? a.to : a.from;
  const i64 pieces = (i64)((call.zero_bytes + kPiece - 1) / kPiece);
  const size_t smem = p.smem(pieces > 0);
  // A sorting CTA with one tile clears as it goes, its share of the pieces over the steps of its passes (500 000 positions and 256
  // MB 73 us, with all of it behind the sort 76).  With more tiles the writes hold the sort up by as much as they take (4.05 M
  // and 1.25 GB 382 us, 371 with all of it behind).
  const i64 steps = p.passes * 2;
  a.pieces = p.single ? (int)min((i64)kPiecesAtOnce, (pieces / kNumSMs + steps - 1) / steps) : 0;
  if (p.cluster) {  // CTAs that clear come in clusters too, as many as the GPU holds beside the one that sorts
    const i64 more = min((pieces + kClusterCtas - 1) / kClusterCtas, (i64)(clusters - 1)) * kClusterCtas;
    return launch(ctx, stream, a, true, p.digit, (int)(kClusterCtas + more), smem);
  }
  GSB_CUDA_OK(launch_behind(stream, k_clear_word, dim3(1), 1, word));
  ctx_count_launches(ctx, 1);
  return launch(ctx, stream, a, false, p.digit, (int)(p.ctas + min(pieces, (i64)(most - p.ctas))), smem);
}

}  // namespace gsb
