// Stable sort of positions by a small integer key: ids of table rows, numbers of experts.
//
// The key of position i is ids[i] where that is in [0, num_keys), and num_keys (sorted last) where it is `dropped` (when
// there is such a value) or out of range; the latter records GSB_ERR_INDEX_RANGE.  Everything lives in memory that the caller
// provides, so that calls on several streams and captured calls have nothing in common.
#pragma once
#include "common.cuh"

namespace gsb {

struct KeySource {
  const i64* ids;
  i64 n;         // 1 .. 2^31 - 1
  i64 num_keys;  // below 2^32 - 1
  bool has_dropped;
  i64 dropped;
  i64* counters;
};

// A sorted position: [key, or what stands for it : 32 | position : 32].
__host__ __device__ inline u32 pair_key(u64 p) { return (u32)(p >> 32); }
__host__ __device__ inline u32 pair_at(u64 p) { return (u32)p; }

constexpr u32 kNoRow = 0xffffffffu;

// What a sort leaves behind.
enum SortResult {
  SORT_PAIRS,  // [key, position] in order
  SORT_RANKS,  // [rank of the key among the distinct ones, kNoRow for num_keys; position], the distinct keys, their number
  SORT_ORDER   // source, place and offsets of expert_rows.cu
};

struct SortCall {
  KeySource source;
  int result;
  // bytes set to zero on the way: the rows of a dense gradient
  void* zero = nullptr;
  size_t zero_bytes = 0;
  // SORT_RANKS
  i64* distinct = nullptr;
  i64* number = nullptr;
  Mail mail = Mail{nullptr, 0};
  // SORT_ORDER
  i64 *offsets = nullptr, *order_source = nullptr, *place = nullptr;
};

size_t key_sort_bytes(i64 n, i64 num_keys);
// *pairs: the sorted pairs in `workspace` (SORT_PAIRS, SORT_RANKS).  A sort that is given up (a bounded wait ran out) leaves
// anything at all there: what reads them checks both halves.
// most_ctas: of a large sort; no more than are resident at once.
int key_sort(gsb_ctx* ctx, cudaStream_t stream, const SortCall& call, void* workspace, const u64** pairs, int most_ctas = kNumSMs);

// A caller's memory in pieces that start on 256-byte boundaries.
struct Pieces {
  char* base;
  size_t used = 0;
  explicit Pieces(void* p) : base((char*)p) {}
  template <class T>
  T* take(size_t n) {
    T* p = (T*)(base + used);
    used += (n * sizeof(T) + 255) & ~(size_t)255;
    return p;
  }
};

}  // namespace gsb
