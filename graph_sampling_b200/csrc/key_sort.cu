// One launch sorts: CTAs own equal stretches of the positions and go through the digits of the key, least significant first.
// Per digit a CTA counts its stretch, all counts become visible behind a barrier, every CTA adds up for itself what lies before
// its own (G CTAs x bins words from L2, in place of a scan with a barrier of its own), and puts its positions where they
// belong, tile by tile through shared memory so that neighbouring threads write neighbouring words.  Nothing depends on the
// order in which CTAs run.
//
// Up to 8 CTAs (32 768 positions) are one cluster: its barrier is the hardware's, needs no word in memory and no bound.  More
// are launched cooperatively and meet at a word in the workspace (grid_sync.cuh).  Digits are as wide as keeps the number of
// passes small: 11 bits where few CTAs have to read each other's counts, 9 where up to 148 do.
//
// The launch may also clear memory (the rows of a dense gradient that no position has): CTAs beyond the sorting ones do that
// at the same time, the sort being bound by latency and the clearing by HBM.
#include "key_sort.cuh"

#include "grid_sync.cuh"
#include "scan.cuh"

namespace gsb {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kRounds = 8;
constexpr int kTile = kThreads * kRounds;
constexpr int kClusterCtas = 8;
constexpr int kClusterBits = 11, kGridBits = 9;
constexpr int kMaxBins = 1 << kClusterBits;
constexpr size_t kZeroPiece = 1 << 16;

struct SortArgs {
  SortCall call;
  u64 *from, *to;  // [key : 32 | position : 32], exchanged after every pass
  u32* counts;     // CTAs x bins
  int ctas;        // that sort; the others clear
  int bits, passes, digit;
  i64 stretch;     // positions per CTA
  int rounds;      // of a tile: kThreads positions each
  bool single;     // a stretch is one tile, which stays in registers between counting and placing
  u64* next_piece;   // of the memory to clear (cooperative launches); null: pieces by CTA number
  GridSync sync;
};

__device__ __forceinline__ u32 key_of(const KeySource& s, i64 i, bool check) {
  const i64 id = __ldg(s.ids + i);
  if (s.has_dropped && id == s.dropped) return (u32)s.num_keys;
  if ((u64)id < (u64)s.num_keys) return (u32)id;
  if (check) raise_error(s.counters, GSB_ERR_INDEX_RANGE, i);
  return (u32)s.num_keys;
}

__device__ __forceinline__ void clear_piece(char* p, size_t bytes) {
  const size_t head = min(bytes, (size_t)(0 - (uintptr_t)p & 15));
  for (size_t q = threadIdx.x; q < head; q += kThreads) p[q] = 0;
  uint4* w = (uint4*)(p + head);
  const size_t words = (bytes - head) / 16;
  for (size_t q = threadIdx.x; q < words; q += kThreads) __stcs(w + q, make_uint4(0, 0, 0, 0));
  for (size_t q = head + words * 16 + threadIdx.x; q < bytes; q += kThreads) p[q] = 0;
}

__device__ __forceinline__ size_t pieces_of(const SortCall& c) { return (c.zero_bytes + kZeroPiece - 1) / kZeroPiece; }

__device__ void clear_by_number(const SortCall& c, size_t number, size_t of) {
  for (size_t q = number; q < pieces_of(c); q += of)
    clear_piece((char*)c.zero + q * kZeroPiece, min(kZeroPiece, c.zero_bytes - q * kZeroPiece));
}

__device__ void clear_rest(const SortCall& c, u64* next) {
  __shared__ u64 s_piece;
  for (;;) {
    __syncthreads();
    if (threadIdx.x == 0) s_piece = atomicAdd((unsigned long long*)next, 1ull);
    __syncthreads();
    const size_t q = (size_t)s_piece;
    if (q >= pieces_of(c)) return;
    clear_piece((char*)c.zero + q * kZeroPiece, min(kZeroPiece, c.zero_bytes - q * kZeroPiece));
  }
}

// Exclusive scan of bins values, kMaxBins / kThreads per thread at most; returns the total through s_scan.
__device__ __forceinline__ u32 scan_threads(u32 v, u32* s_scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u32 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u32 t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // s_scan may still be read
  if (lane == 31) s_scan[warp] = inc;
  __syncthreads();
  u32 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const u32 t = s_scan[w];
    if (w < warp) before += t;
    all += t;
  }
  if (threadIdx.x == 0) s_scan[kWarps] = all;
  return before + inc - v;
}

template <bool CLUSTER>
struct Barrier {
  const SortArgs& a;
  u32 index = 0;
  template <class F>
  __device__ __forceinline__ void operator()(F give_up) {
    ++index;
    if constexpr (CLUSTER) {
      asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
      grid_barrier(a.sync, index, give_up, (u32)a.ctas);
    }
  }
};

struct Tile {
  u64 item[kRounds];
  u32 rank[kRounds];
};

template <bool CLUSTER>
__global__ void __launch_bounds__(kThreads) k_sort_keys(const SortArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ u32 s_scan[kWarps + 1];
  const SortCall& c = a.call;
  const int cta = blockIdx.x;
  if (cta >= a.ctas) {
    if (!CLUSTER) clear_rest(c, a.next_piece);
    else if (cta >= kClusterCtas) clear_by_number(c, cta - kClusterCtas, gridDim.x - kClusterCtas);
    return;
  }
  const i64 n = c.source.n;
  const int bins = 1 << a.digit;
  u64* s_items = (u64*)smem;                           // kTile, also the partial sums of the counts
  u32* s_base = (u32*)(s_items + kTile);               // where the next item of a digit goes
  u32* s_tile = s_base + bins;                         // where a digit starts in the tile
  unsigned short* s_count = (unsigned short*)(s_tile + bins);  // kWarps x bins
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const i64 lo = (i64)cta * a.stretch, hi = min(lo + a.stretch, n);
  const bool single = a.single;
  const int rounds = a.rounds, tile = rounds * kThreads;
  Barrier<CLUSTER> barrier{a};
  auto give_up = [&] {
    if (c.result == SORT_RANKS) c.number[0] = 0;
    if (c.result == SORT_ORDER)
      for (i64 q = cta; q < max(n, c.source.num_keys + 1); q += a.ctas) {
        if (q <= c.source.num_keys) c.offsets[q] = 0;
        if (q < n) c.order_source[q] = q, c.place[q] = ~q;
      }
  };
  const u64* from = a.from;
  u64* to = a.to;
  Tile t;

  auto item_at = [&](i64 i, int pass, bool check) {
    return pass == 0 ? (u64)key_of(c.source, i, check) << 32 | (u64)i : __ldcg(from + i);
  };
  auto load_tile = [&](i64 base, int pass, bool check) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const i64 i = base + warp * (rounds * 32) + r * 32 + lane;
      t.item[r] = r < rounds && i < hi ? item_at(i, pass, check) : ~0ull;
    }
  };
  // Ranks of a tile's items among those of the same digit in their warp; s_count = the warps' counts.  Lanes with the same digit
  // are found bit by bit (a vote each; the match instruction takes as long as there are different digits: 6 us for eight
  // rounds of 16 warps, where all votes of 9 bits take 2).
  auto rank_tile = [&](i64 base, int shift) {
    for (int q = threadIdx.x; q < kWarps * bins / 8; q += kThreads) ((uint4*)s_count)[q] = make_uint4(0, 0, 0, 0);
    u32 peers[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      peers[r] = __ballot_sync(0xffffffffu, r < rounds && base + warp * (rounds * 32) + r * 32 + lane < hi);
    for (int b = 0; b < a.digit; ++b) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const bool bit = (pair_key(t.item[r]) >> (shift + b)) & 1u;
        const u32 with = __ballot_sync(0xffffffffu, bit);
        peers[r] &= bit ? with : ~with;
      }
    }
    __syncthreads();
    unsigned short* mine = s_count + warp * bins;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (r >= rounds) break;
      const bool valid = base + warp * (rounds * 32) + r * 32 + lane < hi;
      const u32 digit = (pair_key(t.item[r]) >> shift) & (bins - 1);
      const u32 before = __popc(peers[r] & ((1u << lane) - 1u));
      const u32 found = valid ? mine[digit] : 0;
      __syncwarp();
      if (valid && before == 0) mine[digit] = (unsigned short)(found + __popc(peers[r]));
      __syncwarp();
      t.rank[r] = found + before;
    }
    __syncthreads();
  };
  // Warps' counts become starts within the digit; returns the digit's count in the tile.
  auto warp_starts = [&](int digit) {
    u32 k[kWarps], run = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) k[w] = s_count[w * bins + digit];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      s_count[w * bins + digit] = (unsigned short)run;
      run += k[w];
    }
    return run;
  };

  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.digit;
    const bool last = pass == a.passes - 1;
    // counts of the stretch
    u32* row = a.counts + (size_t)cta * bins;
    if (single) {
      load_tile(lo, pass, true);
      rank_tile(lo, shift);
      for (int d = threadIdx.x; d < bins; d += kThreads) row[d] = s_tile[d] = warp_starts(d);
    } else {
      for (int d = threadIdx.x; d < bins; d += kThreads) s_tile[d] = 0;
      __syncthreads();
      for (i64 i = lo + threadIdx.x; i < hi; i += 4 * kThreads) {
        u64 item[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i + q * kThreads < hi) item[q] = item_at(i + q * kThreads, pass, true);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i + q * kThreads < hi) atomicAdd(&s_tile[(pair_key(item[q]) >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
      for (int d = threadIdx.x; d < bins; d += kThreads) row[d] = s_tile[d];
    }
    barrier(give_up);
    // all counts: of each digit, and of each digit in the CTAs before this one; `groups` groups of threads share the rows
    {
      const int per_row = min(bins / 4, kThreads), groups = min(min(kThreads / per_row, a.ctas), 16), group = threadIdx.x / per_row;
      const int d = (threadIdx.x % per_row) * 4;
      u32* s_total = (u32*)s_items;                    // groups x bins
      u32* s_before = s_total + groups * bins;
      uint4 total = make_uint4(0, 0, 0, 0), before = total;
      if (group < groups) {
#pragma unroll 8
      for (int g = group; g < a.ctas; g += groups) {
        const uint4 v = __ldcg((const uint4*)(a.counts + (size_t)g * bins + d));
        total.x += v.x, total.y += v.y, total.z += v.z, total.w += v.w;
        if (g < cta) before.x += v.x, before.y += v.y, before.z += v.z, before.w += v.w;
      }
      *(uint4*)(s_total + group * bins + d) = total;
      *(uint4*)(s_before + group * bins + d) = before;
      }
      __syncthreads();
      const int per = (bins + kThreads - 1) / kThreads;  // digits per thread, 1 .. 4
      u32 sum = 0;
      for (int q = 0; q < per; ++q) {
        const int e = threadIdx.x * per + q;
        if (e < bins)
          for (int g = 0; g < groups; ++g) sum += s_total[g * bins + e];
      }
      u32 start = scan_threads(sum, s_scan);
      for (int q = 0; q < per; ++q) {
        const int e = threadIdx.x * per + q;
        if (e >= bins) break;
        u32 all = 0, mine = 0;
        for (int g = 0; g < groups; ++g) all += s_total[g * bins + e], mine += s_before[g * bins + e];
        s_base[e] = start + mine;
        if (c.result == SORT_ORDER && a.passes == 1 && cta == 0 && e <= c.source.num_keys) c.offsets[e] = start;
        start += all;
      }
      __syncthreads();
    }
    // to their places
    if (!single) load_tile(lo, pass, false);
    for (i64 base = lo; base < hi; base += tile) {
      if (!single) {
        rank_tile(base, shift);
        for (int d = threadIdx.x; d < bins; d += kThreads) s_tile[d] = warp_starts(d);
      }
      __syncthreads();
      // s_tile: counts -> starts in the tile; s_base: where the tile's first item of a digit goes, less its place in the tile
      const int per = (bins + kThreads - 1) / kThreads;
      u32 count[kMaxBins / kThreads], sum = 0;
#pragma unroll
      for (int q = 0; q < kMaxBins / kThreads; ++q) {
        const int e = threadIdx.x * per + q;
        count[q] = q < per && e < bins ? s_tile[e] : 0;
        sum += count[q];
      }
      u32 start = scan_threads(sum, s_scan);
#pragma unroll
      for (int q = 0; q < kMaxBins / kThreads; ++q) {
        const int e = threadIdx.x * per + q;
        if (q >= per || e >= bins) break;
        s_tile[e] = start;
        s_base[e] -= start;
        start += count[q];
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const i64 i = base + warp * (rounds * 32) + r * 32 + lane;
        if (r < rounds && i < hi) {
          const u32 digit = (pair_key(t.item[r]) >> shift) & (bins - 1);
          const u32 at = s_tile[digit] + s_count[warp * bins + digit] + t.rank[r];
          s_items[at] = t.item[r];
          if (c.result == SORT_ORDER && last) {
            const i64 row_of = (i64)(s_base[digit] + at);
            if (row_of >= n || pair_at(t.item[r]) >= n) continue;  // never, unless memory was overwritten
            c.place[pair_at(t.item[r])] = pair_key(t.item[r]) < c.source.num_keys ? row_of : ~row_of;
          }
        }
      }
      if (base + tile < hi) load_tile(base + tile, pass, false);  // on its way while this tile is written
      __syncthreads();
      const int items = (int)min((i64)tile, hi - base);
      for (int j = threadIdx.x; j < items; j += kThreads) {
        const u64 item = s_items[j];
        const i64 at = (i64)(u32)(s_base[(pair_key(item) >> shift) & (bins - 1)] + (u32)j);
        if (at >= n) continue;  // as above
        if (c.result == SORT_ORDER && last) c.order_source[at] = pair_at(item);
        if (c.result != SORT_ORDER || a.passes > 1) to[at] = item;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kMaxBins / kThreads; ++q) {
        const int e = threadIdx.x * per + q;
        if (q < per && e < bins) s_base[e] += s_tile[e] + count[q];
      }
    }
    u64* free = const_cast<u64*>(from);
    from = to;
    to = free;
    if (!last || c.result == SORT_RANKS || (c.result == SORT_ORDER && a.passes > 1)) barrier(give_up);
  }

  if (c.result == SORT_ORDER && a.passes > 1) {
    const i64 experts = c.source.num_keys;
    for (i64 j = lo + threadIdx.x; j < hi; j += kThreads) {
      const i64 e = pair_key(__ldcg(from + j)), before = j > 0 ? (i64)pair_key(__ldcg(from + j - 1)) : -1;
      for (i64 q = before + 1; q <= e; ++q) c.offsets[q] = j;
      if (j == n - 1)
        for (i64 q = e + 1; q <= experts; ++q) c.offsets[q] = n;
    }
  }
  if (c.result == SORT_RANKS) {
    const u32 none = (u32)c.source.num_keys;
    // the tile's items, and which of them are the first of their key; returns how many of the warp's are
    u32 first[kRounds];
    auto find_heads = [&](i64 base) {
      const i64 begin = base + warp * (rounds * 32);
      u32 before = begin > 0 && begin < hi ? pair_key(__ldcg(from + begin - 1)) : kNoRow, all = 0;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const i64 i = begin + r * 32 + lane;
        t.item[r] = r < rounds && i < hi ? __ldcg(from + i) : (u64)kNoRow << 32;
      }
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const u32 key = pair_key(t.item[r]);
        u32 left = __shfl_up_sync(0xffffffffu, key, 1);
        if (lane == 0) left = before;
        before = __shfl_sync(0xffffffffu, key, 31);
        first[r] = __ballot_sync(0xffffffffu, key < none && key != left);
        all += __popc(first[r]);
      }
      return all;
    };
    u32 mine = 0, heads = 0;
    for (i64 base = lo; base < hi; base += tile) mine += heads = find_heads(base);
    scan_threads(lane == 0 ? mine : 0, s_scan);
    __syncthreads();
    if (threadIdx.x == 0) a.counts[cta] = s_scan[kWarps];
    barrier(give_up);
    u32 others = 0;
    for (int g = threadIdx.x; g < cta; g += kThreads) others += __ldcg(a.counts + g);
    scan_threads(others, s_scan);
    __syncthreads();
    u32 before = s_scan[kWarps];
    for (i64 base = lo; base < hi; base += tile) {
      if (!single) heads = find_heads(base);
      u32 rank = before + scan_threads(lane == 0 ? heads : 0, s_scan);
      rank = __shfl_sync(0xffffffffu, rank, 0);
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const i64 i = base + warp * (rounds * 32) + r * 32 + lane;
        const u32 key = pair_key(t.item[r]), my = rank + __popc(first[r] & (2u << lane) - 1u) - 1u;  // of the latest head up to here
        if (r < rounds && i < hi) {
          if (first[r] >> lane & 1u) c.distinct[my] = key;
          to[i] = (u64)(key < none ? my : kNoRow) << 32 | pair_at(t.item[r]);
        }
        rank += __popc(first[r]);
      }
      __syncthreads();
      before += s_scan[kWarps];
    }
    if (cta == a.ctas - 1 && threadIdx.x == 0) {
      c.number[0] = before;
      mail_post(c.mail, 0, before, c.source.counters);
    }
  }
  if (!CLUSTER && c.zero_bytes > 0) clear_rest(c, a.next_piece);
}

int key_bits(i64 num_keys) {  // of the largest key, num_keys itself
  int bits = 1;
  while (bits < 32 && (num_keys >> bits) != 0) ++bits;
  return bits;
}

struct Plan {
  bool cluster;
  int ctas, bits, passes, digit, rounds;
  bool single;
  i64 stretch;
  size_t smem() const {
    const size_t bins = (size_t)1 << digit;
    return kTile * 8 + bins * 8 + kWarps * bins * 2;
  }
};

// With memory to clear, half of the SMs sort and the others clear.
Plan plan_of(i64 n, i64 num_keys, bool clears) {
  Plan p;
  p.cluster = n <= (i64)kClusterCtas * kTile;
  const i64 most_ctas = p.cluster ? kClusterCtas : clears ? kNumSMs / 2 : kNumSMs;
  const i64 shares = (n + kThreads - 1) / kThreads, per = (shares + most_ctas - 1) / most_ctas;
  p.stretch = per * kThreads;
  p.ctas = (int)((shares + per - 1) / per);
  p.single = per <= kRounds;
  p.rounds = p.single ? (int)per : kRounds;
  p.bits = key_bits(num_keys);
  const int most = p.cluster ? kClusterBits : kGridBits;
  p.passes = (p.bits + most - 1) / most;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  if (p.digit < 5) p.digit = 5;  // a row of counts is read in pieces of 16 bytes
  return p;
}

template <bool CLUSTER>
int launch(gsb_ctx* ctx, cudaStream_t stream, SortArgs& a, int grid, size_t smem) {
  const void* kernel = (const void*)k_sort_keys<CLUSTER>;
  static bool known[64] = {};
  const int device = ctx_device(ctx);
  if (device < 0 || device >= 64 || !known[device]) {
    const size_t most = kTile * 8 + (size_t)kMaxBins * (8 + kWarps * 2);
    GSB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    if (device >= 0 && device < 64) known[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  if (CLUSTER) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kClusterCtas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  } else {
    attr.id = cudaLaunchAttributeCooperative;
    attr.val.cooperative = 1;
  }
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  void* args[] = {&a};
  GSB_CUDA_OK(cudaLaunchKernelExC(&cfg, kernel, args));
  return GSB_OK;
}

}  // namespace

size_t key_sort_bytes(i64 n, i64 num_keys) {
  if (n <= 0) return 256;
  const Plan p = plan_of(n, num_keys, false);  // the larger of the two
  Pieces w(nullptr);
  w.take<u64>(32);
  w.take<u32>((size_t)p.ctas << p.digit);
  w.take<u64>((size_t)n);
  w.take<u64>((size_t)n);
  return w.used;
}

int key_sort(gsb_ctx* ctx, cudaStream_t stream, const SortCall& call, void* workspace, const u64** pairs) {
  const i64 n = call.source.n;
  const Plan p = plan_of(n, call.source.num_keys, call.zero_bytes > 0);
  Pieces w(workspace);
  u64* words = w.take<u64>(32);
  SortArgs a;
  a.call = call;
  a.counts = w.take<u32>((size_t)p.ctas << p.digit);
  a.from = w.take<u64>((size_t)n);
  a.to = w.take<u64>((size_t)n);
  a.ctas = p.ctas;
  a.bits = p.bits;
  a.passes = p.passes;
  a.digit = p.digit;
  a.stretch = p.stretch;
  a.rounds = p.rounds;
  a.single = p.single;
  a.next_piece = words + 16;
  int barriers = 2 * p.passes - 1;
  if (call.result == SORT_RANKS) barriers += 2;
  if (call.result == SORT_ORDER && p.passes > 1) barriers += 1;
  a.sync = GridSync{words, 0, (u32)barriers, call.source.counters, (int)ctx_option(ctx, GSB_OPT_MAX_POLLS)};
  if (pairs) *pairs = ((p.passes + (call.result == SORT_RANKS ? 1 : 0)) & 1) ? a.to : a.from;
  const i64 pieces = (i64)((call.zero_bytes + kZeroPiece - 1) / kZeroPiece);
  if (p.cluster) {
    // CTAs that clear come in clusters too
    const i64 more = min((pieces + kClusterCtas - 1) / kClusterCtas, (i64)(kNumSMs / kClusterCtas - 1)) * kClusterCtas;
    return launch<true>(ctx, stream, a, (int)(kClusterCtas + more), p.smem());
  }
  GSB_CUDA_OK(cudaMemsetAsync(words, 0, 32 * sizeof(u64), stream));
  const i64 more = min(pieces, (i64)kNumSMs - p.ctas);
  return launch<false>(ctx, stream, a, (int)(p.ctas + more), p.smem());
}

}  // namespace gsb
