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
  i64 n;
  i64 num_keys;  // below 2^32 - 1
  bool has_dropped;
  i64 dropped;
  i64* counters;
};

__device__ __forceinline__ u32 key_of(const KeySource& s, i64 i) {
  const i64 id = __ldg(s.ids + i);
  return (u64)id < (u64)s.num_keys && !(s.has_dropped && id == s.dropped) ? (u32)id : (u32)s.num_keys;
}
// The same, and an id out of range is recorded.
__device__ u32 checked_key_of(const KeySource& s, i64 i);

// Sorted: position at[j] has the j-th smallest key, equal keys in the order of their positions.
struct SortedKeys {
  u32* key;
  u32* at;
  u32* spare;  // n words that the sort needs no longer
};

size_t key_sort_bytes(i64 n, i64 num_keys);
int key_sort(gsb_ctx* ctx, cudaStream_t stream, const KeySource& source, void* workspace, SortedKeys* out);

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
