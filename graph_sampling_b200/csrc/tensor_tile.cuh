// The tensor cores of sm_100a as the products use them: barriers in shared memory, tiles moved by TMA, matrix instructions of a pair
// of CTAs with their sums in tensor memory.
//
// Layouts.  A tile's operand is held in blocks of 128-byte lines, 16-byte pieces of line i exchanged by i % 8 (the 128-byte swizzle, which
// TMA writes and the matrix instructions read).  With the reduced index along the lines ("along"), line i is row i of the tile.  With it
// across the lines ("across"), line i is the i-th reduced index and holds 64 rows' values; 64 more rows are the next block.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "scan.cuh"

namespace gsb {

constexpr int kLineBytes = 128;

__device__ __forceinline__ u32 smem_address(const void* p) { return (u32)__cvta_generic_to_shared(p); }
__device__ __forceinline__ u32 rank_in_pair() {
  u32 r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The same place in another CTA of the cluster.
__device__ __forceinline__ u32 address_in(u32 smem, u32 rank) {
  u32 r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- barriers ----
__device__ __forceinline__ void barrier_init(u32 bar, u32 count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void barriers_ready() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void barrier_expect(u32 bar, u32 bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(u32 bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// At a barrier of either CTA.  What it tells of is in this CTA's shared memory or in tensor memory, behind a fence of its own
// (written_for_tensor_cores, sums_fence_before), so the arrival does not publish this thread's other writes to the cluster, which took 1 250
// cycles each time.
__device__ __forceinline__ void barrier_arrive_at(u32 cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ bool barrier_try(u32 bar, u32 parity) {
  u32 done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// What was written to shared memory before is seen by matrix instructions that are issued behind a barrier this thread arrives at next.
__device__ __forceinline__ void written_for_tensor_cores() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// How long a wait may last, in nanoseconds, and what one that lasts longer does: the CTA notes it in `stop`, its other waits end too, and the
// error is recorded.
struct Patience {
  u64 limit;
  volatile int* stop;
  i64* counters;
};
__device__ __forceinline__ u64 nanoseconds() {
  u64 t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
static __device__ __noinline__ bool barrier_wait_long(u32 bar, u32 parity, Patience p) {
  const u64 start = nanoseconds();
  while (!barrier_try(bar, parity)) {
    if (*p.stop) return false;
    if (nanoseconds() - start > p.limit) {
      *p.stop = 1;
      raise_error(p.counters, GSB_ERR_LOOKBACK_TIMEOUT, blockIdx.x);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool barrier_wait(u32 bar, u32 parity, const Patience& p) {
  for (int i = 0; i < 16; ++i)
    if (barrier_try(bar, parity)) return true;
  return barrier_wait_long(bar, parity, p);
}

// ---- tiles by TMA ----
// Into this CTA's shared memory, with the arrival counted at a barrier of either CTA of the pair.
__device__ __forceinline__ void load_tile(u32 to, const CUtensorMap* map, u32 cluster_bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
               "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void load_tile(u32 to, const CUtensorMap* map, u32 cluster_bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(to),
               "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// Lines one behind the other, not exchanged, with the arrival at a barrier of this CTA's.
__device__ __forceinline__ void load_own_tile(u32 to, const CUtensorMap* map, u32 bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to), "l"(map),
               "r"(bar), "r"(c0), "r"(c1), "r"(0)
               : "memory");
}
// Rows of 64 bytes out of shared memory, 16-byte pieces of row i exchanged by i / 2 % 4 (the 64-byte swizzle).  What lies outside the array is
// not written.
__device__ __forceinline__ void store_tile(const CUtensorMap* map, u32 from, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(from), "r"(c0), "r"(c1) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// All but the last LEFT stores of this thread have read what they write.
template <int LEFT>
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---- matrix instructions ----
// One warp of each CTA of the pair.
__device__ __forceinline__ void sums_alloc(u32 smem_to, u32 columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_to), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void sums_free(u32 at, u32 columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void sums_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void sums_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Where an operand is: the block's address, the distance of 8 lines, and, across, of the next 64 rows.
__device__ __forceinline__ u64 operand(u32 smem, u32 next_block_bytes) {
  return (u64)((smem & 0x3ffffu) >> 4) | (u64)(next_block_bytes >> 4) << 16 | (u64)(8 * kLineBytes >> 4) << 32 | (u64)1 << 46 | (u64)2 << 61;
}
enum OperandType : u32 { OPERAND_F16 = 0, OPERAND_BF16 = 1, OPERAND_S8 = 2 };
__host__ __device__ constexpr u32 instruction(OperandType type, bool a_across, bool b_across, u32 m, u32 n) {
  return (type == OPERAND_S8 ? 2u : 1u) << 4 | (type == OPERAND_F16 ? 0u : 1u) << 7 | (type == OPERAND_F16 ? 0u : 1u) << 10 | (a_across ? 1u : 0u) << 15 |
         (b_across ? 1u : 0u) << 16 | (n >> 3) << 17 | (m >> 4) << 24;
}
// sums (+)= A B over one step of the reduced index (32 bytes of it), for 256 rows of A, half of them in each CTA, as are B's.
template <bool WHOLE_NUMBERS>
__device__ __forceinline__ void multiply(u32 sums, u64 a, u64 b, u32 how, bool add) {
  if constexpr (WHOLE_NUMBERS)
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(sums), "l"(a), "l"(b), "r"(how),
                 "r"((u32)add)
                 : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(sums), "l"(a), "l"(b), "r"(how),
                 "r"((u32)add)
                 : "memory");
}
// Arrives at the barrier, in both CTAs, when the instructions issued so far are done.
__device__ __forceinline__ void multiplied(u32 bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3)
               : "memory");
}
// 16 or 32 columns of sums, of the row that the lane stands for.
__device__ __forceinline__ void read_sums(u32 at, u32 (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                 "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(at));
}
__device__ __forceinline__ void read_sums(u32 at, u32 (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
        "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
        "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
}
__device__ __forceinline__ void sums_read() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- host: what a TMA load is told of an array ----
// `dims` extents, the first of neighbours in memory; strides in bytes of the others (multiples of 16, below 2^40).  False: it cannot be
// described.  Swizzled: 16-byte pieces of line i of a box are exchanged by i % 8 (the 128-byte swizzle).
bool describe_array(CUtensorMap* map, const void* base, int value_bytes, int rank, const u64* dims, const u64* strides, const u32* box,
                    bool swizzled = true);
// Of stores: `rows` rows of `width` values, one behind the other; boxes of 32 rows by 64 bytes.
bool describe_rows(CUtensorMap* map, void* base, int value_bytes, u64 width, u64 rows);

}  // namespace gsb
