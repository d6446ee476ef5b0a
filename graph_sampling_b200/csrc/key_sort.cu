#include "key_sort.cuh"

#include "scan.cuh"

namespace gsb {

constexpr int kThreads = 256;
constexpr int kRounds = 8;
constexpr int kTile = kThreads * kRounds;
constexpr int kBins = 256;
constexpr int kScanThreads = 1024;

__device__ u32 checked_key_of(const KeySource& s, i64 i) {
  const i64 id = __ldg(s.ids + i);
  if (s.has_dropped && id == s.dropped) return (u32)s.num_keys;
  if ((u64)id < (u64)s.num_keys) return (u32)id;
  raise_error(s.counters, GSB_ERR_INDEX_RANGE, i);
  return (u32)s.num_keys;
}

template <bool FIRST>
__global__ void __launch_bounds__(kThreads) k_key_count(const KeySource source, const u32* __restrict__ keys, i64 n, int shift,
                                                        u32* __restrict__ count, int tiles) {
  __shared__ u32 s_count[kBins];
  s_count[threadIdx.x] = 0;
  __syncthreads();
  const i64 base = (i64)blockIdx.x * kTile;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const i64 i = base + r * kThreads + threadIdx.x;
    if (i < n) atomicAdd(&s_count[((FIRST ? checked_key_of(source, i) : keys[i]) >> shift) & (kBins - 1)], 1u);
  }
  __syncthreads();
  count[(i64)threadIdx.x * tiles + blockIdx.x] = s_count[threadIdx.x];
}

// Exclusive scan of all tiles' counts by one CTA.
__global__ void __launch_bounds__(kScanThreads) k_key_scan(u32* __restrict__ count, i64 n) {
  __shared__ i64 s_scan[33];
  i64 before = 0;
  for (i64 base = 0; base < n; base += kScanThreads) {
    const i64 i = base + threadIdx.x;
    const u32 mine = i < n ? count[i] : 0;
    i64 total;
    const i64 excl = block_exclusive_scan<kScanThreads>((i64)mine, s_scan, &total);
    if (i < n) count[i] = (u32)(before + excl);
    before += total;
  }
}

template <bool FIRST>
__global__ void __launch_bounds__(kThreads) k_key_place(const KeySource source, const u32* __restrict__ keys,
                                                        const u32* __restrict__ at, i64 n, int shift,
                                                        const u32* __restrict__ start, int tiles, u32* __restrict__ out_keys,
                                                        u32* __restrict__ out_at) {
  constexpr int kWarps = kThreads / 32;
  __shared__ u32 s_count[kWarps][kBins];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int q = threadIdx.x; q < kWarps * kBins; q += kThreads) (&s_count[0][0])[q] = 0;
  __syncthreads();
  const i64 base = (i64)blockIdx.x * kTile + warp * (kRounds * 32);
  u32 key[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const i64 i = base + r * 32 + lane;
    const bool valid = i < n;
    key[r] = valid ? (FIRST ? key_of(source, i) : keys[i]) : 0;
    const u32 digit = valid ? (key[r] >> shift) & (kBins - 1) : kBins;
    const u32 peers = __match_any_sync(0xffffffffu, digit);
    const u32 before = __popc(peers & ((1u << lane) - 1u));
    u32 found = 0;
    if (valid) found = s_count[warp][digit];
    __syncwarp();
    if (valid && before == 0) s_count[warp][digit] = found + __popc(peers);
    __syncwarp();
    rank[r] = found + before;
  }
  __syncthreads();
  {
    u32 run = start[(i64)threadIdx.x * tiles + blockIdx.x];  // kThreads == kBins
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const u32 c = s_count[w][threadIdx.x];
      s_count[w][threadIdx.x] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const i64 i = base + r * 32 + lane;
    if (i < n) {
      const u32 to = s_count[warp][(key[r] >> shift) & (kBins - 1)] + rank[r];
      out_keys[to] = key[r];
      out_at[to] = FIRST ? (u32)i : at[i];
    }
  }
}

static int key_bits(i64 num_keys) {
  int bits = 1;
  while (bits < 32 && (num_keys >> bits) != 0) ++bits;
  return bits;
}

size_t key_sort_bytes(i64 n, i64 num_keys) {
  (void)num_keys;
  const i64 tiles = (n + kTile - 1) / kTile;
  Pieces p(nullptr);
  for (int q = 0; q < 4; ++q) p.take<u32>((size_t)n);
  p.take<u32>((size_t)(tiles * kBins));
  return p.used;
}

int key_sort(gsb_ctx* ctx, cudaStream_t stream, const KeySource& source, void* workspace, SortedKeys* out) {
  const i64 n = source.n;
  const int tiles = grid_for(n, kTile);
  Pieces p(workspace);
  u32 *keys = p.take<u32>((size_t)n), *at = p.take<u32>((size_t)n), *keys_out = p.take<u32>((size_t)n),
      *at_out = p.take<u32>((size_t)n);
  u32* count = p.take<u32>((size_t)tiles * kBins);
  const int bits = key_bits(source.num_keys);
  for (int shift = 0; shift < bits; shift += 8) {
    if (shift == 0) k_key_count<true><<<tiles, kThreads, 0, stream>>>(source, nullptr, n, shift, count, tiles);
    else k_key_count<false><<<tiles, kThreads, 0, stream>>>(source, keys, n, shift, count, tiles);
    GSB_LAUNCH_OK();
    k_key_scan<<<1, kScanThreads, 0, stream>>>(count, (i64)tiles * kBins);
    GSB_LAUNCH_OK();
    if (shift == 0) k_key_place<true><<<tiles, kThreads, 0, stream>>>(source, nullptr, nullptr, n, shift, count, tiles, keys_out, at_out);
    else k_key_place<false><<<tiles, kThreads, 0, stream>>>(source, keys, at, n, shift, count, tiles, keys_out, at_out);
    GSB_LAUNCH_OK();
    ctx_count_launches(ctx, 3);
    u32* t = keys; keys = keys_out; keys_out = t;
    t = at; at = at_out; at_out = t;
  }
  *out = SortedKeys{keys, at, keys_out};
  return GSB_OK;
}

}  // namespace gsb
