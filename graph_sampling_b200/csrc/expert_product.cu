// Products of rows sorted by expert (or node type) with one matrix per expert.
//
// Rows offsets[e] .. offsets[e + 1] are those of expert e.  Product: out[r, :] = rows[r, :] W[e(r)], zeros for rows of no expert.
// Its gradient for the rows is the product of the output's gradient with the transposed matrices, the same kernel; that for the
// matrices is grad_W[e] = sum over the rows r of e of rows[r, :]^T grad[r, :].
//
// All run on the tensor cores.  float32 operands are taken apart into three bfloat16 parts, a = a0 + a1 + a2 with |a1| < 2^-7 |a| and
// |a2| <= 2^-16 |a|, and a b is the sum of the six products a_i b_j with i + j <= 2: what is left out is 2^-22 |a b| at the very most.  a0 is a
// towards zero, so that a0 b0 leaves the range of float only where a b does; a1 and a2 are to nearest.  That is exact (24 bits are 3 times 8)
// but for numbers below 2^-100, of which the parts that bfloat16 has no numbers for are lost.
#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "few_rows.cuh"
#include "group_plan.cuh"
#include "launch.cuh"
#include "row_values.cuh"
#include "tensor_tile.cuh"

namespace gsb {

// A pair of CTAs takes a tile of 256 rows of the result, 128 each, by `columns` (128 or 256); each holds half of the columns' operand.
constexpr int kPairRows = 256, kMaxStages = 8;
constexpr int kSumColumns = 512;                 // of tensor memory: two tiles' sums, so that one is written out while the next is made
constexpr int kRowsOperand = 128 * kLineBytes;   // bytes of a CTA's rows in a stage
constexpr int kAcross = 64 * kLineBytes;         // a block of 64 lines
// Warps: 0 loads by TMA, 1 (of the first CTA) issues the matrix instructions, 4 to 11 write results out, 12 to 19 read what TMA cannot, and 3
// hands over what they have read, or, of a gradient that TMA loads, the lines that an expert's rows end in.
constexpr int kWriters = 8, kFirstReader = 4 + kWriters, kReaders = 8;
constexpr int tile_threads(bool read) { return 32 * (kFirstReader + (read ? kReaders : 0)); }

// The widest access, of at most 16 bytes, that addresses with these bits allow.
__host__ __device__ __forceinline__ int unit_of(u64 bits) { return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2; }

// How rows come: by TMA; by warps, from memory; by TMA as they lie in memory, from where warps bring them into their lines.
enum { BY_TMA, BY_WARPS, SHIFTED };
// Rows that do not begin on 16-byte boundaries, for TMA: their distance in bytes times `classes` (2, 4 or 8) is a multiple of 16, so the rows number
// c, c + classes and so on are an array whose lines begin on 16-byte boundaries, the row some values behind.  A slot of shared memory holds 128
// rows, class by class, and of each the 128 bytes of two lines and those that the row may begin behind the boundary.  A box costs TMA some 140 cycles
// and a row of it 9, so two lines at a time (200 003 rows of 602, 601 and 604 fp16 to 100: 77, 82 and 75 us) do better than one (95, 128 and 80) and, for
// want of slots, than three (85, 88 and 83); two slots of two 86, four with two stages 81.  Of 608, which need none of this, 61 us.
constexpr int kMostClasses = 8, kSlots = 3, kSlotBlocks = 2, kSlotLine = kSlotBlocks * kLineBytes + 16, kSlotBytes = 128 * kSlotLine;
struct ShiftedMaps {
  CUtensorMap of_class[kMostClasses];
};
template <int READ>
using RowMaps = std::conditional_t<READ == SHIFTED, ShiftedMaps, CUtensorMap>;

// Rows as they lie in memory, for the warps that read them.
struct RawRows {
  const void* at;
  i64 stride;   // in values
  u32 width;
  int unit;     // bytes that an access may have
};

struct TileArgs {
  Groups groups;
  u32 depth, n;              // reduced index of a product; columns of the result
  u32 k;                     // rows of a gradient's result
  u32 columns;               // of a tile
  u32 chunk;                 // rows of an expert that one tile of a gradient sums, a multiple of 64
  int stages;
  int expert_step;           // 0: one matrix for all experts
  RawRows rows, grad;        // where they are read by warps
  u32 classes;               // of shifted rows
  bool by_tma;               // results may leave by TMA
  float* partial;            // gradient: sums of the chunks (null: one chunk per expert, written out)
  float* held;               // of 16-bit types: room for the sums that leave tensor memory before the last (null: none does)
  const float *row_scales, *weight_scales;  // of 8-bit operands
  u64 wait_limit;            // ns
  u32 how;
};

struct Tile {
  int e;
  u32 row0, rows;  // product: of the tile; gradient: of the chunk, counted from the expert's first
  u32 m0, n0;      // gradient: first row of the result; first column
  u32 blocks;      // steps of the reduced index, a line each
  u32 chunk;
};

template <bool GRAD>
__device__ __forceinline__ u64 number_of_tiles(const TileArgs& a, const PlanTable& plan) {
  const u32 across = (a.n + a.columns - 1) / a.columns, down = GRAD ? (a.k + kPairRows - 1) / kPairRows : 1;
  return (u64)plan.tile[a.groups.experts] * across * down;
}
template <bool GRAD, int PER_LINE>
__device__ __forceinline__ Tile tile_at(const TileArgs& a, const PlanTable& plan, u64 t) {
  Tile r;
  const u32 across = (a.n + a.columns - 1) / a.columns, down = GRAD ? (a.k + kPairRows - 1) / kPairRows : 1, each = across * down;
  r.chunk = t >> 32 ? (u32)(t / each) : (u32)t / each;
  const u32 rest = (u32)(t - (u64)r.chunk * each);
  r.n0 = rest % across * a.columns;
  r.m0 = rest / across * kPairRows;
  r.e = expert_of_tile(plan, a.groups.experts, r.chunk);
  const u32 step = GRAD ? a.chunk : kPairRows, count = plan.begin[r.e + 1] - plan.begin[r.e], from = (r.chunk - plan.tile[r.e]) * step;
  r.rows = min(step, count - from);
  r.row0 = GRAD ? from : plan.begin[r.e] + from;
  r.blocks = ((GRAD ? r.rows : a.depth) + PER_LINE - 1) / PER_LINE;
  return r;
}

// The steps of a tile alone: all of a product's have the same.
template <bool GRAD, int PER_LINE>
__device__ __forceinline__ u32 blocks_at(const TileArgs& a, const PlanTable& plan, u64 t) {
  if constexpr (GRAD) return tile_at<GRAD, PER_LINE>(a, plan, t).blocks;
  else return (a.depth + PER_LINE - 1) / PER_LINE;
}
// Lines of the reduced index that a matrix instruction takes.
constexpr u32 kStepLines = 16;
// An addition to a sum in tensor memory cuts what is left of its 16 products below the sum's last bits: of positive numbers 6.4e-9 of the result
// for each value that is summed (1 024 to 262 144 of them), 1.7e-3 over 262 144, where a float16 is rounded by 4.9e-4.  Longer sums of 16-bit types
// than 16 384 values leave tensor memory after so many, and are added in float: 1.1e-4 (2 048 rows of 65 536 to 2 048 412 us for 399).
constexpr u32 kHeldLines = 256, kHeldValues = 64 * kHeldLines;

// 64 bytes of each of 32 rows of the result, a row a lane, leave through shared memory: by TMA where all 32 rows are wanted and begin on 16-byte
// boundaries, else copied by neighbouring lanes, to `to`, `pitch` bytes apart, `bytes` of each, in accesses of `unit` bytes, which divide them.
constexpr int kStoreBytes = 64, kRoom = 32 * kStoreBytes;
template <class Word>
__device__ __forceinline__ void copy_rows_by(const char* room, int lane, char* to, i64 pitch, u32 rows, u32 bytes) {
  constexpr int W = sizeof(Word), LANES = kStoreBytes / W;  // of a row
#pragma unroll 4
  for (int i = 0; i < LANES; ++i) {
    const u32 at = i * 32 + lane, r = at / LANES, x = at % LANES * W;
    if (r < rows && x < bytes) *(Word*)(to + r * pitch + x) = *(const Word*)(room + r * kStoreBytes + ((x >> 4 ^ (r >> 1 & 3)) << 4) + (x & 15));
  }
}
static __device__ __noinline__ void copy_rows(const char* room, int lane, char* to, i64 pitch, u32 rows, u32 bytes, int unit) {
  __syncwarp();
  if (unit == 16) copy_rows_by<uint4>(room, lane, to, pitch, rows, bytes);
  else if (unit == 8) copy_rows_by<uint2>(room, lane, to, pitch, rows, bytes);
  else if (unit == 4) copy_rows_by<u32>(room, lane, to, pitch, rows, bytes);
  else copy_rows_by<unsigned short>(room, lane, to, pitch, rows, bytes);
  __syncwarp();
}
// A warp's way out: one room or two, taken in turn.  float32 has two; 16-bit types do better with one and a stage more for their loads (65 536
// rows of 2 048 to 2 048: 411 us for 433).
constexpr int rooms_of(int parts) { return parts == 3 ? 2 : 1; }
template <int ROOMS>
struct Exit {
  char* rooms;
  u32 turn;
};
template <class U, int ROOMS>
__device__ __forceinline__ void write_rows(Exit<ROOMS>& exit, int lane, const float (&v)[kStoreBytes / sizeof(U)], U* to, i64 pitch, u32 rows, u32 columns, int unit,
                                           const CUtensorMap* map, i64 row, u32 column) {
  constexpr int PER = 16 / sizeof(U);
  Unit<U, 16> w[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    float f[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) f[q] = v[p * PER + q];
    w[p].set(f);
  }
  if (rows < 32 && unit == 16 && columns >= kStoreBytes / sizeof(U)) {  // each lane its row: for a few of them that is sooner
    if ((u32)lane < rows)
#pragma unroll
      for (int p = 0; p < 4; ++p) store_unit((Unit<U, 16>*)(to + lane * pitch) + p, w[p]);
    return;
  }
  char* const room = exit.rooms + exit.turn % ROOMS * kRoom;
  ++exit.turn;
  if (lane == 0) stores_read<ROOMS - 1>();
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p) *(uint4*)(room + lane * kStoreBytes + ((p ^ (lane >> 1 & 3)) << 4)) = w[p].w;
  if (map && rows == 32) {
    written_for_tensor_cores();
    __syncwarp();
    if (lane == 0) store_tile(map, smem_address(room), (int)column, (int)row);
  } else {
    copy_rows(room, lane, (char*)to, pitch * (i64)sizeof(U), rows, columns * (u32)sizeof(U), unit);
    if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // an empty turn
  }
}

// ---- rows read by warps: rows of any address and distance, and float32, which is taken apart on the way ----------------------------
// 16-bit values: a warp reads a line at a time, two neighbouring values a lane: every eighth line of an operand, `lines` of them with values, the
// others zeros, into LINES words from FIRST on.  `valid`: of the lane's two columns; `aligned`: they are one word.
template <int FIRST, int LINES, int WORDS>
__device__ __forceinline__ void read_lines(u32 (&v)[WORDS], const unsigned short* from, i64 step, int lines, int valid, bool aligned) {
  if (aligned && valid != 1) {
    if (valid <= 0) lines = 0;
#pragma unroll
    for (int i = 0; i < LINES; ++i) v[FIRST + i] = i < lines ? __ldg((const u32*)(from + i * step)) : 0;
  } else {
#pragma unroll
    for (int i = 0; i < LINES; ++i) {
      const u32 low = i < lines && valid > 0 ? __ldg(from + i * step) : 0, high = i < lines && valid > 1 ? __ldg(from + i * step + 1) : 0;
      v[FIRST + i] = low | high << 16;
    }
  }
}
// To lines 8 apart.
template <int FIRST, int LINES, int WORDS>
__device__ __forceinline__ void write_lines(const u32 (&v)[WORDS], u32 to) {
#pragma unroll
  for (int i = 0; i < LINES; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + i * 8 * kLineBytes), "r"(v[FIRST + i]) : "memory");
}
__device__ __forceinline__ void write_line(u32 to, const u32 (&w)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// float32: 8 neighbouring values of a row, of which there are `valid`, in accesses of up to `unit` bytes.
__device__ __forceinline__ void read_eight(const float* from, int valid, int unit, float (&v)[8]) {
  if (valid >= 8 && unit == 32) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(from));
  } else if (valid >= 8 && unit == 16) {
    const float4 a = __ldg((const float4*)from), b = __ldg((const float4*)from + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = q < valid ? __ldg(from + q) : 0.f;
  }
}
// The next part of a float32 value, and what is left of it: the first towards zero, the others to nearest.  Infinities and NaN are all in the
// first part.  OF_WEIGHT: it is 0 for zeros alone, so that infinity times a weight is NaN for them alone.
template <bool OF_WEIGHT>
__device__ __forceinline__ u32 next_part(float& rest, bool is_first) {
  __nv_bfloat16 part = is_first ? __float2bfloat16_rz(rest) : __float2bfloat16_rn(rest);
  if constexpr (OF_WEIGHT)
    if (is_first && __bfloat162float(part) == 0.f && rest != 0.f) part = __ushort_as_bfloat16(rest < 0.f ? 0x8001 : 1);
  rest = fabsf(rest) <= 3.402823466e38f ? rest - __bfloat162float(part) : 0.f;
  return __bfloat16_as_ushort(part);
}
// Two parts of neighbours in a word; what is left of them stays.  Towards zero a part is the upper half, also where that is 0 and the number is
// not: looking for such numbers, of no weight but in a product with infinity, cost products 3 to 11 % (500 000 rows of 256 to 256 403 us for
// 393, their gradient 473 for 426).
template <bool IS_FIRST>
__device__ __forceinline__ u32 next_parts(float& low, float& high) {
  u32 w;
  if constexpr (IS_FIRST) w = __byte_perm(__float_as_uint(low), __float_as_uint(high), 0x7632);
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(high), "f"(low));
  low -= __uint_as_float(w << 16);
  high -= __uint_as_float(w & 0xffff0000u);
  return w;
}
// 8 values each of two lines, 32 apart, to their places, every part in an operand of its own, `apart` bytes from the one before.
__device__ __forceinline__ void write_parts(const float (&x)[8], const float (&y)[8], u32 to, u32 apart) {
  float rest[16], any = 0.f;  // what is left of an infinity and of NaN is none of the numbers
  u32 w[2][4];
#pragma unroll
  for (int q = 0; q < 8; ++q) rest[q] = x[q], rest[8 + q] = y[q];
#pragma unroll
  for (int q = 0; q < 8; ++q) w[q / 4][q % 4] = next_parts<true>(rest[2 * q], rest[2 * q + 1]);
#pragma unroll
  for (int q = 0; q < 4; ++q) any += (rest[4 * q] + rest[4 * q + 1]) + (rest[4 * q + 2] + rest[4 * q + 3]);
  if (fabsf(any) <= 3.402823466e38f) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      if (p > 0)
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q / 4][q % 4] = next_parts<false>(rest[2 * q], rest[2 * q + 1]);
      write_line(to + p * apart, w[0]);
      write_line(to + p * apart + 32 * kLineBytes, w[1]);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) rest[q] = x[q], rest[8 + q] = y[q];
#pragma unroll 1
    for (int p = 0; p < 3; ++p) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const u32 low = next_part<false>(rest[2 * q], p == 0);
        w[q / 4][q % 4] = low | next_part<false>(rest[2 * q + 1], p == 0) << 16;
      }
      write_line(to + p * apart, w[0]);
      write_line(to + p * apart + 32 * kLineBytes, w[1]);
    }
  }
}

// The lines of the reduced index that a pair of CTAs goes through, tile by tile.
template <bool GRAD, int PER_LINE>
struct Walk {
  u64 t;
  u32 b;
  Tile tile;
  __device__ __forceinline__ void settle(const TileArgs& a, const PlanTable& plan, u64 tiles, u64 step) {  // to the next tile that has lines
    while (t < tiles && (tile = tile_at<GRAD, PER_LINE>(a, plan, t)).blocks == 0) t += step;
  }
  __device__ __forceinline__ void next(const TileArgs& a, const PlanTable& plan, u64 tiles, u64 step) {
    if (++b < tile.blocks) return;
    b = 0;
    t += step;
    settle(a, plan, tiles, step);
  }
};

// PARTS: 3 for float32, else 1.  ACROSS: the second operand's lines hold the reduced index across them (a gradient's both do).  READ: how rows
// (and a gradient's both operands) come.  LONG: 16-bit types' sums may be longer than kHeldValues; what holds them would cost short calls 0.4 of 14 us.
template <class T, bool WHOLE_NUMBERS, int PARTS, bool GRAD, bool ACROSS, int READ, bool LONG>
__global__ void __launch_bounds__(tile_threads(READ), 1) k_tiles(const __grid_constant__ RowMaps<READ> map_a, const __grid_constant__ CUtensorMap map_b,
                                                                 const __grid_constant__ CUtensorMap map_out, const TileArgs a, T* __restrict__ out) {
  constexpr int kPerLine = kLineBytes / (WHOLE_NUMBERS ? 1 : 2);
  static_assert(!LONG || (PARTS == 1 && !WHOLE_NUMBERS), "of 16-bit types");
  // Sums leave tensor memory, where additions cut, after this many lines of the reduced index.  float32: over 16 instructions that is an error
  // of 2.3e-7 of the sums (rms), over 32 4.7e-7, and they are added up in registers
  constexpr u32 kDrain = PARTS > 1 ? 4 : LONG ? kHeldLines : 0xffffffffu;
  extern __shared__ char raw[];
  __shared__ PlanTable plan;
  static_assert(READ != SHIFTED || (PARTS == 1 && !GRAD && !WHOLE_NUMBERS), "a product's rows of 16-bit values");
  __shared__ __align__(8) u64 bars[4 * kMaxStages + 4 + 2 * kSlots];
  __shared__ float column_scales[WHOLE_NUMBERS ? kWriters : 1][128];
  constexpr int kRooms = rooms_of(PARTS);
  __shared__ __align__(1024) char rooms[kWriters][kRooms * kRoom];
  __shared__ u32 sums_at;
  __shared__ volatile int stop;
  const u32 stages_at = (smem_address(raw) + 1023u) & ~1023u;
  const u32 full = smem_address(bars), empty = full + 8 * kMaxStages, written = full + 16 * kMaxStages;
  const u32 sums_full = full + 24 * kMaxStages, sums_empty = sums_full + 16;
  const u32 slot_full = sums_empty + 16, slot_empty = slot_full + 8 * kSlots, cut = slot_empty + 8 * kSlots;
  const u32 rank = rank_in_pair();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const Groups& g = a.groups;
  const Patience patience{a.wait_limit, &stop, g.counters};

  if (threadIdx.x == 0) {
    stop = 0;
    for (int s = 0; s < kMaxStages; ++s) {
      barrier_init(full + 8 * s, (READ && GRAD ? 0 : 1) + (READ ? 2 : 0));
      barrier_init(written + 8 * s, READ ? kReaders : 1);
      if (GRAD && !READ) barrier_init(cut + 8 * s, 2);
      barrier_init(empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(sums_full + 8 * s, 1);
      barrier_init(sums_empty + 8 * s, 2 * kWriters);
    }
    for (int s = 0; s < kSlots; ++s) {
      barrier_init(slot_full + 8 * s, 1);
      barrier_init(slot_empty + 8 * s, kReaders);
    }
    barriers_ready();
    if (!READ) prefetch_map((const CUtensorMap*)&map_a);
    if (!READ || !GRAD) prefetch_map(&map_b);
  }
  if (warp == 2) sums_alloc(smem_address(&sums_at), kSumColumns);
  make_plan<tile_threads(READ)>(plan, g, GRAD ? a.chunk : kPairRows, GRAD ? 1 : 0);
  leave_end(plan, g);
  sums_fence_before();
  cluster_barrier();
  sums_fence_after();
  const u32 sums = sums_at;
  const u64 tiles = number_of_tiles<GRAD>(a, plan);
  const u64 first = blockIdx.x / 2, step = gridDim.x / 2;
  const u32 half = a.columns / 2, b_bytes = half * kLineBytes, stage_bytes = PARTS * (kRowsOperand + b_bytes);
  const u32 slots_at = stages_at + a.stages * stage_bytes;  // of shifted rows

  if (warp == 0 && lane == 0 && !(READ && GRAD)) {
    const u32 full_of_first = address_in(full, 0);
    u32 stage = 0, turn = 0;
    for (u64 t = first; t < tiles; t += step) {
      const Tile tile = tile_at<GRAD, kPerLine>(a, plan, t);
      const CUtensorMap *of_a = (const CUtensorMap*)&map_a, *of_b = &map_b;
      const int matrix = (g.first + tile.e) * a.expert_step;
      // A second CTA without rows loads zeros from behind the array: products that cost the least power (1 to 2 % under the power limit).  (Not the
      // least traffic: for what is out of range TMA reads as many sectors somewhere in the array.  Boxes of the 32 rows that a step has, which leave the
      // rest as it was, were slower than one of 128: 64 rows to 64 experts 30 us for 27.)
      const int first_row = rank == 0 || tile.rows > 128 ? (int)(tile.row0 + rank * 128) : (int)g.num_rows;
      const u32 loaded_bytes = 2 * PARTS * ((READ ? 0 : kRowsOperand) + b_bytes);
      const u32 cut_blocks = GRAD && tile.rows % 64 != 0 ? 1 : 0;  // the last, which warp 3 hands over
      const int grad_row = GRAD ? (int)(plan.begin[tile.e] + tile.row0) : 0;
      auto load = [&](u32 b, u32 bar) {
        const u32 at = stages_at + stage * stage_bytes;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          const u32 to_a = at + p * kRowsOperand, to_b = at + PARTS * kRowsOperand + p * b_bytes;
          if (GRAD) {
            const int row = grad_row + (int)(b * 64);
            for (int j = 0; j < 2; ++j) load_tile(to_a + j * kAcross, of_a, bar, (int)(tile.m0 + rank * 128 + j * 64), row, p);
            for (u32 j = 0; j < half / 64; ++j) load_tile(to_b + j * kAcross, of_b, bar, (int)(tile.n0 + rank * half + j * 64), row, p);
          } else {
            if (!READ) load_tile(to_a, of_a, bar, (int)(b * kPerLine), first_row, p);
            if (ACROSS)
              for (u32 j = 0; j < half / 64; ++j)
                load_tile(to_b + j * kAcross, of_b, bar, (int)(tile.n0 + rank * half + j * 64), (int)(b * kPerLine), matrix, p);
            else
              load_tile(to_b, of_b, bar, (int)(b * kPerLine), (int)(tile.n0 + rank * half), matrix, p);
          }
        }
        if (++stage == (u32)a.stages) stage = 0, turn ^= 1;
      };
      for (u32 b = 0; b + cut_blocks < tile.blocks; ++b) {
        if (!barrier_wait(empty + 8 * stage, turn ^ 1, patience)) goto loaded;
        if (rank == 0) barrier_expect(full + 8 * stage, loaded_bytes);
        load(b, full_of_first + 8 * stage);
      }
      if (GRAD && cut_blocks) {
        if (!barrier_wait(empty + 8 * stage, turn ^ 1, patience)) goto loaded;
        if (rank == 0) barrier_arrive(full + 8 * stage);  // a turn like any other
        barrier_expect(written + 8 * stage, loaded_bytes / 2);
        load(tile.blocks - 1, address_in(written, rank) + 8 * stage);
      }
    }
  loaded:;
  } else if (warp == 1 && rank == 0 && lane == 0) {
    constexpr bool A_ACROSS = GRAD, B_ACROSS = GRAD || ACROSS;
    u32 stage = 0, turn = 0, made = 0, cut_turns = 0;
    for (u64 t = first; t < tiles; t += step) {
      u32 blocks, cut_lines = 0;
      if constexpr (GRAD && !READ) {
        const Tile tile = tile_at<GRAD, kPerLine>(a, plan, t);
        blocks = tile.blocks;
        cut_lines = tile.rows % 64;
      } else {
        blocks = blocks_at<GRAD, kPerLine>(a, plan, t);
      }
      for (u32 b0 = 0; b0 < blocks; b0 += min(kDrain, blocks - b0), ++made) {
        const u32 buffer = made & 1, to = sums + buffer * 256;
        if (!barrier_wait(sums_empty + 8 * buffer, (made >> 1 & 1) ^ 1, patience)) goto issued;
        sums_fence_after();
        auto issue = [&](bool onto, u32 steps) {  // the stage's block, onto what the sums are or as the first of them
          const u32 at = stages_at + stage * stage_bytes;
          const u64 op_a = operand(at, kAcross), op_b = operand(at + PARTS * kRowsOperand, kAcross);
#pragma unroll
          for (u32 s = 0; s < 4; ++s) {
            if (s >= steps) break;
            const u64 a_s = op_a + s * ((A_ACROSS ? 16 * kLineBytes : 32) >> 4), b_s = op_b + s * ((B_ACROSS ? 16 * kLineBytes : 32) >> 4);
            const bool add = onto || s > 0;
            multiply<WHOLE_NUMBERS>(to, a_s, b_s, a.how, add);
            if (PARTS == 3) {  // the five small products have sums of their own, 2^-7 the size
              const u64 next_a = kRowsOperand >> 4, next_b = b_bytes >> 4;
              multiply<false>(to + 128, a_s, b_s + next_b, a.how, add);
              multiply<false>(to + 128, a_s + next_a, b_s, a.how, true);
              multiply<false>(to + 128, a_s + next_a, b_s + next_b, a.how, true);
              multiply<false>(to + 128, a_s, b_s + 2 * next_b, a.how, true);
              multiply<false>(to + 128, a_s + 2 * next_a, b_s, a.how, true);
            }
          }
          multiplied(empty + 8 * stage);
          if (++stage == (u32)a.stages) stage = 0, turn ^= 1;
        };
        const u32 end = b0 + min(kDrain, blocks - b0), whole_end = cut_lines > 0 && end == blocks ? end - 1 : end;
        for (u32 b = b0; b < whole_end; ++b) {
          if (!barrier_wait(full + 8 * stage, turn, patience)) goto issued;
          sums_fence_after();
          issue(b > b0, 4);
        }
        if constexpr (GRAD && !READ)
          if (whole_end < end) {  // as many instructions as have lines of the expert's
            if (!barrier_wait(cut + 8 * stage, cut_turns >> stage & 1, patience)) goto issued;
            cut_turns ^= 1u << stage;
            sums_fence_after();
            issue(whole_end > b0, (cut_lines + kStepLines - 1) / kStepLines);
          }
        multiplied(sums_full + 8 * buffer);
      }
    }
  issued:;
  } else if (READ == SHIFTED && warp == 2 && lane == 0) {
    u32 slot = 0, turn = 0;
    for (u64 t = first; t < tiles; t += step) {
      const Tile tile = tile_at<GRAD, kPerLine>(a, plan, t);
      const u32 first_row = rank == 0 || tile.rows > 128 ? tile.row0 + rank * 128 : g.num_rows;  // from behind the array: zeros
      for (u32 b = 0; b < tile.blocks; b += kSlotBlocks) {
        if (!barrier_wait(slot_empty + 8 * slot, turn ^ 1, patience)) goto brought;
        barrier_expect(slot_full + 8 * slot, kSlotBytes);
        for (u32 c = 0; c < a.classes; ++c) {
          const u32 row = first_row + ((c - first_row) & (a.classes - 1));
          load_own_tile(slots_at + slot * kSlotBytes + c * (kSlotBytes / a.classes), (const CUtensorMap*)&map_a + c, slot_full + 8 * slot, (int)(b * 64),
                        (int)(row / a.classes));
        }
        if (++slot == kSlots) slot = 0, turn ^= 1;
      }
    }
  brought:;
  } else if (GRAD && !READ && warp == 3) {
    // Behind an expert's last row are the next one's: where an instruction takes lines that are none of its own, both operands get zeros.  (Descriptions
    // that end where the expert's rows do, made on the device from the array's, are no way: TMA sends what is out of range to somewhere in the array
    // as it was first described, which from a later beginning is behind its end, up to 32 KB, and faults where memory ends there too.)  64 experts of
    // 497 rows, 1 024 to 1 024, take 72.7 us, of 512, which need none of this, 72.2.
    const u32 cut_of_first = address_in(cut, 0);
    u32 stage = 0, turns = 0;  // of which stages the next turn is an odd one
    for (u64 t = first; t < tiles; t += step) {
      const Tile tile = tile_at<GRAD, kPerLine>(a, plan, t);
      const u32 lines = tile.rows % 64, none = (kStepLines - lines % kStepLines) % kStepLines, last = (stage + tile.blocks - 1) % a.stages;
      stage = (stage + tile.blocks) % a.stages;
      if (lines == 0) continue;
      const u32 zeros[4] = {}, at = stages_at + last * stage_bytes + lines * kLineBytes;
      const bool there = barrier_wait(written + 8 * last, turns >> last & 1, patience);
      if (!__all_sync(0xffffffffu, there)) break;
      turns ^= 1u << last;
      for (u32 j = 0; j < 2 + half / 64; ++j)  // the blocks of both operands
        for (u32 piece = lane; piece < none * (kLineBytes / 16); piece += 32) write_line(at + j * kAcross + piece * 16, zeros);
      written_for_tensor_cores();
      __syncwarp();
      if (lane == 0) barrier_arrive_at(cut_of_first + 8 * last);
    }
  } else if (READ && warp == 3 && lane == 0) {
    // The readers' fence towards the tensor cores: theirs would wait for their copies that are on their way
    const u32 full_of_first = address_in(full, 0);
    u32 stage = 0, turn = 0;
    for (u64 t = first; t < tiles; t += step) {
      const u32 blocks = blocks_at<GRAD, kPerLine>(a, plan, t);
      for (u32 b = 0; b < blocks; ++b) {
        if (!barrier_wait(written + 8 * stage, turn, patience)) goto handed_over;
        written_for_tensor_cores();
        barrier_arrive_at(full_of_first + 8 * stage);
        if (++stage == (u32)a.stages) stage = 0, turn ^= 1;
      }
    }
  handed_over:;
  } else if (READ && warp >= kFirstReader) {
    // All readers take a stage together; what comes next is on its way while they write
    const u32 me = threadIdx.x - 32 * kFirstReader;
    u32 stage = 0, turn = 0;
    Walk<GRAD, kPerLine> ahead{first, 0, {}};  // what is read next
    ahead.settle(a, plan, tiles, step);
    // first of a tile's rows that the reduced index runs over (gradient), or of this CTA's (product)
    auto first_row = [&](const Tile& tile) { return GRAD ? (i64)plan.begin[tile.e] + tile.row0 : (i64)tile.row0 + rank * 128; };
    auto rows_here = [&](const Tile& tile) { return GRAD ? (int)tile.rows : (int)tile.rows - (int)rank * 128; };
    if constexpr (PARTS == 3) {
      // A lane has the same 8 values' place in lines 4 w + lane / 8, 32 behind them and so on; those of the next stage are on their way while it
      // takes this one's apart.  (Copied into shared memory meanwhile they met the matrix instructions' operands there: 460 us for 500 000
      // rows of 256 to 256 values.)
      constexpr int kPieces = GRAD ? 6 : 4;
      const u32 chunk = lane & 7, segment = me / 32 * 4 + lane / 8, place = segment * kLineBytes + ((chunk ^ (segment & 7)) << 4);
      const float *from = nullptr, *from_grad = nullptr;
      int columns = 0, grad_columns = 0, rows_left = 0;  // from this lane's first on
      auto begin_tile = [&] {
        if (ahead.t >= tiles) return;
        const Tile& tile = ahead.tile;
        const u32 c = (GRAD ? tile.m0 + rank * 128 : 0) + chunk * 8;
        from = (const float*)a.rows.at + (first_row(tile) + segment) * a.rows.stride + c;
        columns = (int)a.rows.width - (int)c;
        rows_left = rows_here(tile) - (int)segment;
        if (GRAD) {
          const u32 d = tile.n0 + rank * half + chunk * 8;
          from_grad = (const float*)a.grad.at + (first_row(tile) + segment) * a.grad.stride + d;
          grad_columns = (int)a.grad.width - (int)d;
        }
      };
      begin_tile();
      float v[kPieces][8];
      auto read = [&](int j, float(&to)[8]) {  // piece j: of the rows, lines 32 j on (a gradient's second two: the next 64 columns); of a gradient's rows
        if (ahead.t >= tiles) return;
        if (GRAD && j >= 4) read_eight(from_grad + (j - 4) * 32 * a.grad.stride, rows_left > (j - 4) * 32 ? grad_columns : 0, a.grad.unit, to);
        else if (GRAD) read_eight(from + (j & 1) * 32 * a.rows.stride + (j >> 1) * 64, rows_left > (j & 1) * 32 ? columns - (j >> 1) * 64 : 0, a.rows.unit, to);
        else read_eight(from + j * 32 * a.rows.stride, rows_left > j * 32 ? columns : 0, a.rows.unit, to);
      };
      auto go_on = [&] {
        if (ahead.t >= tiles) return;
        from += GRAD ? 64 * a.rows.stride : 64;
        if (GRAD) from_grad += 64 * a.grad.stride, rows_left -= 64;
        else columns -= 64;
        ahead.next(a, plan, tiles, step);
        if (ahead.b == 0) begin_tile();
      };
#pragma unroll
      for (int j = 0; j < kPieces; ++j) read(j, v[j]);
      bool left = ahead.t < tiles;
      go_on();
      while (left) {
        const bool free = barrier_wait(empty + 8 * stage, turn ^ 1, patience);
        if (!__all_sync(0xffffffffu, free)) break;
        const u32 at = stages_at + stage * stage_bytes + place;
#pragma unroll
        for (int j = 0; j < kPieces; j += 2) {
          const bool of_grad = GRAD && j >= 4;
          write_parts(v[j], v[j + 1], at + (of_grad ? PARTS * kRowsOperand : j * 32 * kLineBytes), of_grad ? b_bytes : kRowsOperand);
          read(j, v[j]);
          read(j + 1, v[j + 1]);
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(written + 8 * stage);
        left = ahead.t < tiles;
        go_on();
        if (++stage == (u32)a.stages) stage = 0, turn ^= 1;
      }
    } else if constexpr (READ == SHIFTED) {
      // Warp w has lines w, w + 8 and so on, all of one class
      const u32 w = me / 32, to = stages_at + w * kLineBytes + (((lane >> 2) ^ w) << 4) + (lane & 3) * 4, class_bytes = kSlotBytes / a.classes;
      u32 slot = 0, slot_turn = 0;
      for (u64 t = first; t < tiles; t += step) {
        const Tile tile = tile_at<GRAD, kPerLine>(a, plan, t);
        const u32 c = (tile.row0 + rank * 128 + w) & (a.classes - 1), behind = c * (u32)a.rows.stride & 7;  // values behind the boundary
        const u32 from = slots_at + c * class_bytes + w / a.classes * kSlotLine + behind / 2 * 4 + lane * 4, by = 8 / a.classes * kSlotLine;
        for (u32 b = 0; b < tile.blocks; ++b) {
          const u32 block = b % kSlotBlocks;
          if (block == 0 && !__all_sync(0xffffffffu, barrier_wait(slot_full + 8 * slot, slot_turn, patience))) goto shifted;
          u32 v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const u32 at = from + slot * kSlotBytes + block * kLineBytes + i * by;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[i]) : "r"(at) : "memory");
            if (behind & 1) {
              u32 next;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(next) : "r"(at + 4) : "memory");
              v[i] = __funnelshift_r(v[i], next, 16);
            }
          }
          if (!__all_sync(0xffffffffu, barrier_wait(empty + 8 * stage, turn ^ 1, patience))) goto shifted;
          write_lines<0, 16>(v, to + stage * stage_bytes);
          __syncwarp();
          const bool last = block + 1 == kSlotBlocks || b + 1 == tile.blocks;
          if (lane == 0) {
            if (last) barrier_arrive(slot_empty + 8 * slot);
            barrier_arrive(written + 8 * stage);
          }
          if (last && ++slot == kSlots) slot = 0, slot_turn ^= 1;
          if (++stage == (u32)a.stages) stage = 0, turn ^= 1;
        }
      }
    shifted:;
    } else {
      // Warp w has lines w, w + 8 and so on; those of the next stages are on their way while it writes this one's, two stages of a product's rows
      // or one of both operands of a gradient.  (200 003 rows of 602 to 100 take 106 us; of 608, which TMA loads, 58.  Asynchronous copies of four
      // bytes a lane, and twice as many warps, took 111 and 109: two requests for each line that begins between 128-byte boundaries, of which
      // L1 has so many on their way and no more.)
      constexpr int kWords = GRAD ? 32 : 16;
      const u32 w = me / 32, place = w * kLineBytes + (((lane >> 2) ^ w) << 4) + (lane & 3) * 4;
      const bool aligned = a.rows.unit >= 4, grad_aligned = a.grad.unit >= 4;
      auto lines_of = [&](int rows) { return rows > (int)w ? (rows - (int)w + kReaders - 1) / kReaders : 0; };
      const i64 rows_step = kReaders * a.rows.stride, grad_step = kReaders * a.grad.stride;
      const unsigned short *from = nullptr, *from_grad = nullptr;
      int columns = 0, grad_columns = 0, rows_left = 0;  // from this lane's first on
      auto fetch = [&](u32(&v)[kWords]) {                // whether there was anything left
        if (ahead.t >= tiles) return false;
        if (ahead.b == 0) {
          const Tile& tile = ahead.tile;
          const u32 c = (GRAD ? tile.m0 + rank * 128 : 0) + lane * 2;
          from = (const unsigned short*)a.rows.at + (first_row(tile) + w) * a.rows.stride + c;
          columns = (int)a.rows.width - (int)c;
          rows_left = rows_here(tile);
          if (GRAD) {
            const u32 d = tile.n0 + rank * half + lane * 2;
            from_grad = (const unsigned short*)a.grad.at + (first_row(tile) + w) * a.grad.stride + d;
            grad_columns = (int)a.grad.width - (int)d;
          }
        }
        const int lines = lines_of(rows_left);
        if constexpr (GRAD) {
          read_lines<0, 8>(v, from, rows_step, lines, columns, aligned);
          read_lines<8, 8>(v, from + 64, rows_step, lines, columns - 64, aligned);
          read_lines<16, 8>(v, from_grad, grad_step, lines, grad_columns, grad_aligned);
          if (half > 64) read_lines<24, 8>(v, from_grad + 64, grad_step, lines, grad_columns - 64, grad_aligned);
          from += 8 * rows_step;
          from_grad += 8 * grad_step;
          rows_left -= 64;
        } else {
          read_lines<0, 16>(v, from, rows_step, lines, columns, aligned);
          from += 64;
          columns -= 64;
        }
        ahead.next(a, plan, tiles, step);
        return true;
      };
      auto turn_over = [&](u32(&v)[kWords], bool& there) {  // false: nothing is left, or the wait was given up
        if (!there) return false;
        const bool free = barrier_wait(empty + 8 * stage, turn ^ 1, patience);
        if (!__all_sync(0xffffffffu, free)) return false;
        const u32 at = stages_at + stage * stage_bytes + place;
        write_lines<0, 16>(v, at);
        if constexpr (GRAD) {
          write_lines<16, 8>(v, at + kRowsOperand);
          if (half > 64) write_lines<24, 8>(v, at + kRowsOperand + kAcross);
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(written + 8 * stage);
        there = fetch(v);
        if (++stage == (u32)a.stages) stage = 0, turn ^= 1;
        return true;
      };
      u32 v[kWords];
      bool there = fetch(v);
      if constexpr (GRAD) {
        while (turn_over(v, there)) {
        }
      } else {
        u32 second[kWords];
        bool second_there = fetch(second);
        while (turn_over(v, there) && turn_over(second, second_there)) {
        }
      }
    }
  } else if (warp >= 4 && warp < 4 + kWriters) {
    const u32 quarter = (u32)(warp & 3) * 32;
    const u32 c0 = (u32)(warp - 4) / 4 * half;                                     // this warp's half of the columns
    const u32 sums_empty_of_first = address_in(sums_empty, 0);
    const int unit = unit_of((u64)(uintptr_t)out | (u64)a.n * sizeof(T)), unit_partial = unit_of((u64)a.n * 4);
    Exit<kRooms> exit{rooms[warp - 4], 0};
    u32 made = 0;
    for (u64 t = first; t < tiles; t += step) {
      const Tile tile = tile_at<GRAD, kPerLine>(a, plan, t);
      const u32 limit = GRAD ? a.k - tile.m0 : tile.rows, above = rank * 128 + quarter;
      const u32 valid_rows = limit > above ? min(32u, limit - above) : 0;
      const bool mine = (u32)lane < valid_rows;
      const u32 n0 = tile.n0 + c0;
      const i64 out_row = GRAD ? (i64)(a.partial ? (i64)tile.chunk : (i64)(g.first + tile.e)) * a.k + tile.m0 + above : (i64)tile.row0 + above;
      const i64 at = out_row * a.n + n0;
      // 32 values of each row, in as many steps as they are 64 bytes
      auto store = [&](u32 c, const float(&v)[32]) {
        auto write = [&](auto* to, int width) {
          typedef std::remove_pointer_t<decltype(to)> U;
          constexpr int N = kStoreBytes / sizeof(U);
#pragma unroll
          for (int x = 0; x < 32; x += N) {
            if (n0 + c + x >= a.n || valid_rows == 0) continue;
            float f[N];
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] = v[x + q];
            write_rows(exit, lane, f, to + at + c + x, a.n, valid_rows, a.n - n0 - c - x, width, a.by_tma ? &map_out : nullptr, out_row, n0 + c + x);
          }
        };
        if (GRAD && a.partial) write(a.partial, unit_partial);
        else write(out, unit);
      };
      if (tile.blocks == 0) {
        const float zeros[32] = {};
        for (u32 c = 0; c < half; c += 32) store(c, zeros);
        continue;
      }
      if constexpr (PARTS == 1) {
        float of_row = 1.f;
        if constexpr (WHOLE_NUMBERS) {
          if (mine) of_row = a.row_scales[tile.row0 + above + lane];
          __syncwarp();
          for (u32 c = lane; c < half; c += 32)
            column_scales[warp - 4][c] = n0 + c < a.n ? __ldg(a.weight_scales + (i64)(g.first + tile.e) * a.n + n0 + c) : 0.f;
          __syncwarp();
        }
        constexpr int kAtOnce = READ ? 8 : 32;  // that there are registers for
        float* const held = a.held + (i64)(blockIdx.x * kWriters + warp - 4) * half * 32 + lane;  // read by the lane that wrote it
        bool lost = false;
        for (u32 b0 = 0; b0 < tile.blocks; b0 += min(kDrain, tile.blocks - b0), ++made) {
          const u32 buffer = made & 1;
          const bool there = barrier_wait(sums_full + 8 * buffer, made >> 1 & 1, patience);
          if (!__all_sync(0xffffffffu, there)) {
            lost = true;
            break;
          }
          sums_fence_after();
          const bool last = tile.blocks - b0 <= kDrain;
          for (u32 c = 0; c < half; c += 32) {
            u32 v[32];
            __syncwarp();
            read_sums(sums + (quarter << 16) + buffer * 256 + c0 + c, v);
            sums_read();
            if (c + 32 == half) {
              sums_fence_before();
              __syncwarp();
              if (lane == 0) barrier_arrive_at(sums_empty_of_first + 8 * buffer);
            }
            float f[32];
#pragma unroll
            for (int q = 0; q < 32; ++q) {
              if constexpr (WHOLE_NUMBERS) f[q] = (float)(int)v[q] * of_row * column_scales[warp - 4][c + q];
              else f[q] = __uint_as_float(v[q]);
            }
            if constexpr (LONG) {
              if (b0 > 0 || !last)
#pragma unroll
                for (int q = 0; q < 32; q += kAtOnce) {
                  float* const at = held + (c + q) * 32;
                  if (b0 > 0)
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) f[q + i] += at[i * 32];
                  if (!last)
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) at[i * 32] = f[q + i];
                  __syncwarp();
                }
            }
            if (last) store(c, f);
          }
        }
        if (lost) break;
      } else {
        float total[2][32] = {};
        bool lost = false;
        for (u32 b0 = 0; b0 < tile.blocks; b0 += min(kDrain, tile.blocks - b0), ++made) {
          const u32 buffer = made & 1;
          const bool there = barrier_wait(sums_full + 8 * buffer, made >> 1 & 1, patience);
          if (!__all_sync(0xffffffffu, there)) {
            lost = true;
            break;
          }
          sums_fence_after();
          const u32 from = sums + (quarter << 16) + buffer * 256 + c0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int kind = 0; kind < 2; ++kind) {
              u32 v[16];
              __syncwarp();
              read_sums(from + kind * 128 + c * 16, v);
              sums_read();
#pragma unroll
              for (int q = 0; q < 16; ++q) {
                // an infinity's small products are infinity times 0: the large one has the answer
                const float f = __uint_as_float(v[q]);
                total[c / 2][c % 2 * 16 + q] += kind == 0 || fabsf(f) <= 3.402823466e38f ? f : 0.f;
              }
            }
          }
          sums_fence_before();
          __syncwarp();
          if (lane == 0) barrier_arrive_at(sums_empty_of_first + 8 * buffer);
        }
        if (lost) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) store(c * 32, total[c]);
      }
    }
    if (lane == 0) stores_done();
    if (!GRAD) {  // rows of no expert
      const i64 at = (i64)blockIdx.x * (32 * kWriters) + (threadIdx.x - 128), by = (i64)gridDim.x * (32 * kWriters);
      auto clear = [&](i64 from, i64 to) {
        if (unit == 16) {
          constexpr int N = 16 / sizeof(T);
          for (i64 i = from / N + at; i < to / N; i += by) ((uint4*)out)[i] = make_uint4(0, 0, 0, 0);
        } else {
          for (i64 i = from + at; i < to; i += by) out[i] = from_float<T>(0.f);
        }
      };
      if (g.first == 0) clear(0, (i64)plan.begin[0] * a.n);
      if (g.first + g.experts == g.all) clear((i64)plan.begin[g.experts] * a.n, (i64)g.num_rows * a.n);
    }
  }
  __syncwarp();
  if (stop) {  // given up: what is still on its way into this CTA's memory gets a moment to arrive
    const u64 since = nanoseconds();
    while (nanoseconds() - since < 1000000) __nanosleep(1000);
  }
  __syncthreads();
  __syncwarp();
  sums_fence_before();
  cluster_barrier();
  sums_fence_after();
  __syncwarp();
  if (warp == 2) sums_free(sums, kSumColumns);
}

// out[e] = the sum of the chunks of expert e, in their order.
constexpr int kAddThreads = 256;
template <class T>
__global__ void __launch_bounds__(kAddThreads) k_add_chunks(const Groups g, u32 chunk, i64 values, const float* __restrict__ partial,
                                                             T* __restrict__ out) {
  __shared__ PlanTable plan;
  await_previous();
  make_plan<kAddThreads>(plan, g, chunk, 1);
  const i64 step = (i64)gridDim.x * kAddThreads;
  for (i64 i = (i64)blockIdx.x * kAddThreads + threadIdx.x; i < values * g.experts; i += step) {
    const int e = (int)(i / values);
    const i64 at = i - e * values;
    float sum = 0.f;
#pragma unroll 8
    for (u32 c = plan.tile[e]; c < plan.tile[e + 1]; ++c) sum += __ldcs(partial + c * values + at);
    out[(i64)g.first * values + i] = from_float<T>(sum);
  }
}

// ---- operands brought into lines -------------------------------------------------------------------------------------------------
// Matrices whose rows do not begin on 16-byte boundaries are copied to where they do; float32 is cut into its parts, one array each.
template <class T, int PARTS>
__global__ void __launch_bounds__(256) k_into_lines(const T* __restrict__ from, i64 matrices, i64 matrix_stride, u32 height, i64 stride, u32 width,
                                                    u32 to_stride, int unit, unsigned short* __restrict__ to) {
  await_previous();
  const u32 pieces = to_stride / 8;
  const i64 count = matrices * height * pieces, plane = matrices * height * (i64)to_stride;
  for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < count; i += (i64)gridDim.x * 256) {
    const i64 line = i / pieces;
    const u32 x = (u32)(i - line * pieces) * 8;
    const T* row = from + line / height * matrix_stride + line % height * stride;
    if (PARTS == 1 && unit >= 4 && x + 8 <= width) {
      const u32* words = (const u32*)(row + x);
      uint4 w;
      if (unit >= 8) {
        const uint2 low = __ldg((const uint2*)words), high = __ldg((const uint2*)words + 1);
        w = make_uint4(low.x, low.y, high.x, high.y);
      } else {
        w = make_uint4(__ldg(words), __ldg(words + 1), __ldg(words + 2), __ldg(words + 3));
      }
      *(uint4*)(to + line * to_stride + x) = w;
      continue;
    }
    unsigned short v[PARTS][8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if constexpr (PARTS == 1) {
        v[0][q] = x + q < width ? ((const unsigned short*)row)[x + q] : (unsigned short)0;
      } else {
        float rest = x + q < width ? row[x + q] : 0.f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) v[p][q] = (unsigned short)next_part<true>(rest, p == 0);
      }
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      uint4 w;
      w.x = v[p][0] | (u32)v[p][1] << 16;
      w.y = v[p][2] | (u32)v[p][3] << 16;
      w.z = v[p][4] | (u32)v[p][5] << 16;
      w.w = v[p][6] | (u32)v[p][7] << 16;
      *(uint4*)(to + p * plane + line * to_stride + x) = w;
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
static i64 rounded(i64 bytes) { return (bytes + 255) / 256 * 256; }

constexpr i64 kMostStride = (i64)1 << 40;  // bytes that a description for TMA can hold

// An operand as the kernel reads it: `matrices` of `height` lines of `width` values, neighbours in memory.
struct Lines {
  const void* at;
  i64 matrices, matrix_stride, height, stride, width;
  int dtype;
  bool copied() const {
    const int size = value_bytes(dtype);
    return dtype == GSB_F32 || !aligned_to(16, (const char*)at) || (height > 1 && (stride * size % 16 != 0 || stride == 0)) ||
           (matrices > 1 && matrix_stride * size % 16 != 0) || (height > 1 && stride >= kMostStride / size) || (matrices > 1 && matrix_stride >= kMostStride / size);
  }
  // TMA can load its lines class by class
  bool shifted() const {
    return dtype != GSB_F32 && height >= kMostClasses && matrices == 1 && aligned_to(16, (const char*)at) && stride % 8 != 0 && stride >= width &&
           stride < kMostStride / (2 * kMostClasses);
  }
  u32 classes() const { return stride % 2 ? 8 : stride % 4 ? 4 : 2; }
  i64 parts() const { return dtype == GSB_F32 ? 3 : 1; }
  i64 to_stride() const { return (width + 7) / 8 * 8; }
  i64 copies() const { return matrices > 1 && matrix_stride == 0 ? 1 : matrices; }  // one matrix for all is copied once
  i64 bytes() const { return copied() ? rounded(parts() * copies() * height * to_stride() * 2) : 0; }
};

// The operand, copied first where it has to be; `room` moves on behind the copy.
static int bring(gsb_ctx* ctx, cudaStream_t stream, Lines* x, char** room) {
  if (!x->copied()) return GSB_OK;
  unsigned short* to = (unsigned short*)*room;
  *room += x->bytes();
  const i64 count = x->copies() * x->height * (x->to_stride() / 8);
  const int grid = (int)min((i64)kNumSMs * 16, (i64)grid_for(count, 256));
  const int size = value_bytes(x->dtype);
  const u64 strides = (u64)((x->height > 1 ? x->stride : 0) | (x->copies() > 1 ? x->matrix_stride : 0));
  const int unit = unit_of((u64)(uintptr_t)x->at | strides * (u64)size);
  ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
  if (x->dtype == GSB_F32)
    launch_behind(stream, k_into_lines<float, 3>, grid, 256, (const float*)x->at, x->copies(), x->matrix_stride, (u32)x->height, x->stride, (u32)x->width,
                  (u32)x->to_stride(), unit, to);
  else
    launch_behind(stream, k_into_lines<unsigned short, 1>, grid, 256, (const unsigned short*)x->at, x->copies(), x->matrix_stride, (u32)x->height, x->stride,
                  (u32)x->width, (u32)x->to_stride(), unit, to);
  GSB_LAUNCH_OK();
  x->at = to;
  x->matrix_stride = x->matrix_stride == 0 ? 0 : x->height * x->to_stride();
  x->stride = x->to_stride();
  return GSB_OK;
}

// Four extents: along a line, lines, matrices, parts.  A distance between things of which there is one is never used, but checked.
static int describe(const Lines& x, int size, u32 box_along, u32 box_lines, bool matrices, CUtensorMap* map) {
  const i64 lines = x.height > 1 ? x.stride * size : 16, step = x.copies() > 1 ? x.matrix_stride * size : 16;
  const i64 part = x.parts() > 1 ? x.copies() * x.height * x.stride * size : 16;
  const u64 dims4[4] = {(u64)x.width, (u64)x.height, (u64)x.copies(), (u64)x.parts()}, strides4[3] = {(u64)lines, (u64)step, (u64)part};
  const u64 dims3[3] = {(u64)x.width, (u64)x.height, (u64)x.parts()}, strides3[2] = {(u64)lines, (u64)part};
  const u32 box[4] = {box_along, box_lines, 1, 1};
  if (step >= kMostStride || part >= kMostStride) return GSB_ERR_UNSUPPORTED;
  return describe_array(map, x.at, size, matrices ? 4 : 3, matrices ? dims4 : dims3, matrices ? strides4 : strides3, box) ? GSB_OK : GSB_ERR_UNSUPPORTED;
}

static int describe_shifted(const Lines& x, ShiftedMaps* maps) {
  const u32 classes = x.classes();
  for (u32 c = 0; c < classes; ++c) {
    const u32 behind = (u32)(c * x.stride % 8);
    const u64 dims[3] = {(u64)(x.width + behind), (u64)((x.height - c + classes - 1) / classes), 1}, strides[2] = {(u64)(x.stride * 2 * classes), 16};
    const u32 box[3] = {kSlotLine / 2, 128 / classes, 1};
    if (!describe_array(&maps->of_class[c], (const unsigned short*)x.at + c * x.stride - behind, 2, 3, dims, strides, box, false)) return GSB_ERR_UNSUPPORTED;
  }
  return GSB_OK;
}

static int check_product(i64 num_rows, i64 k, i64 n, i64 num_experts, i64 rows_stride, const int64_t* offsets) {
  GSB_REQUIRE(num_rows >= 0 && num_rows < ((i64)1 << 31) && k >= 1 && k <= GSB_MAX_ROW_LEN && n >= 1 && n <= GSB_MAX_ROW_LEN && num_experts >= 1 &&
                  num_experts <= GSB_MAX_EXPERTS && rows_stride >= 0,
              GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(offsets && aligned_to(8, offsets), GSB_ERR_INVALID_ARGUMENT);
  return GSB_OK;
}

// One launch per kPlanExperts experts, in order.  `ends`: a word for each, or null.
template <class F>
static int by_experts(gsb_ctx* ctx, i64 num_experts, i64 num_rows, const int64_t* offsets, u32* ends, F launch) {
  for (i64 first = 0; first < num_experts; first += kPlanExperts) {
    const int some = (int)min((i64)kPlanExperts, num_experts - first);
    const int st = launch(Groups{offsets + first, (int)first, some, (int)num_experts, (u32)num_rows, ctx_counters(ctx), ends ? ends + first / kPlanExperts : nullptr});
    if (st != GSB_OK) return st;
  }
  return GSB_OK;
}
// Room for the ends of all launches, where there are several, and one word behind the last.  It is the first of a workspace.
static i64 ends_bytes(i64 num_experts) { return num_experts > kPlanExperts ? rounded((num_experts + kPlanExperts - 1) / kPlanExperts * 4 + 4) : 0; }
static u32* take_ends(i64 num_experts, char** room) {
  const i64 bytes = ends_bytes(num_experts);
  u32* const ends = bytes > 0 ? (u32*)*room : nullptr;
  *room += bytes;
  return ends;
}

// Shared memory for stages: what the fixed part (the plan, the scales, the ways out) leaves, and what is lost to their alignment.
constexpr int stages_room(int parts) { return (227 - 14) * 1024 - rooms_of(parts) * kWriters * kRoom - 1024; }
// A wait is given up after GSB_OPT_MAX_POLLS of these: two seconds by default.
constexpr u64 kNanosecondsPerPoll = 477;
// Launches pairs of CTAs: at most one CTA per SM.  In the order of the stream, with no overlap of its neighbours' ends and beginnings: with
// overlap, hundreds of copies and products queued one behind the other once came to a halt.  Why is not known.  A successor is set up only when all CTAs
// of its predecessor have begun, so it was not CTAs that wait beside pairs which have no room yet; at that time the writers also went from stores that some
// lanes made alone to warp-wide reads of tensor memory without converging, which is mended.
template <class T, bool WHOLE_NUMBERS, int PARTS, bool GRAD, bool ACROSS, int READ>
static int launch_tiles(gsb_ctx* ctx, cudaStream_t stream, const RowMaps<READ>& map_a, const CUtensorMap& map_b, TileArgs a, i64 most_tiles, i64 out_rows, T* out) {
  constexpr bool kHalves = PARTS == 1 && !WHOLE_NUMBERS;
  const bool is_long = kHalves && a.held;
  auto kernel = k_tiles<T, WHOLE_NUMBERS, PARTS, GRAD, ACROSS, READ, false>;
  if (is_long) kernel = k_tiles<T, WHOLE_NUMBERS, PARTS, GRAD, ACROSS, READ, kHalves>;
  const int stage = PARTS * (kRowsOperand + (int)a.columns / 2 * kLineBytes);
  constexpr int kSlotsRoom = READ == SHIFTED ? kSlots * kSlotBytes : 0;
  a.stages = min(kMaxStages, (stages_room(PARTS) - kSlotsRoom) / stage);
  a.how = instruction(WHOLE_NUMBERS ? OPERAND_S8 : std::is_same<T, __half>::value ? OPERAND_F16 : OPERAND_BF16, GRAD, GRAD || ACROSS, kPairRows, a.columns);
  a.wait_limit = (u64)ctx_option(ctx, GSB_OPT_MAX_POLLS) * kNanosecondsPerPoll;
  const int smem = a.stages * stage + kSlotsRoom + 1024;
  CUtensorMap map_out = {};
  const int size = a.partial ? 4 : (int)sizeof(T);
  void* const results = a.partial ? (void*)a.partial : (void*)out;
  a.by_tma = (i64)a.n * size % 16 == 0 && aligned_to(16, (const char*)results) && out_rows < ((i64)1 << 31) && describe_rows(&map_out, results, size, a.n, (u64)out_rows);
  static std::atomic<bool> allowed[2][64];  // on which devices the kernel may have all the shared memory it can ask for
  const int device = ctx_device(ctx);
  if (device >= 64 || !allowed[is_long][device]) {
    GSB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, stages_room(PARTS) + 1024));
    if (device < 64) allowed[is_long][device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * max((i64)1, min((i64)kNumSMs / 2, most_tiles))));
  cfg.blockDim = dim3(tile_threads(READ));
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
  GSB_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_out, a, out));
  return GSB_OK;
}

// Room for the sums of 16-bit types that leave tensor memory before the last, of all CTAs; it follows the launches' ends in a workspace.
static i64 held_bytes(i64 depth, int dtype, u32 columns) {
  return dtype != GSB_F32 && depth > kHeldValues ? (i64)kNumSMs * kWriters * 32 * (columns / 2) * 4 : 0;
}
static float* take_held(i64 depth, int dtype, u32 columns, char** room) {
  const i64 bytes = held_bytes(depth, dtype, columns);
  float* const held = bytes > 0 ? (float*)*room : nullptr;
  *room += bytes;
  return held;
}

// Columns of a tile: narrow ones for narrow results, for float32, whose parts need the room, and where wide ones would leave half of the pairs of
// CTAs without any (512 rows of 512 to 512 by eight experts 9.7 us for 12.6).  `row_tiles`: how many there are down the result.
static u32 tile_columns(i64 n, int dtype, i64 row_tiles) { return dtype == GSB_F32 || n <= 128 || row_tiles * ((n + 255) / 256) <= kNumSMs / 4 ? 128 : 256; }
static i64 row_tiles_of(i64 num_rows, i64 num_experts) { return num_rows / kPairRows + min(num_rows, num_experts); }
static i64 row_tiles_of_grad(i64 k, i64 num_experts) { return (k + kPairRows - 1) / kPairRows * num_experts; }

static Lines rows_operand(const void* rows, int dtype, i64 num_rows, i64 width, i64 stride) { return Lines{rows, 1, 0, num_rows, stride, width, dtype}; }
// The matrices with their rows (ACROSS) or their columns as lines, whichever are neighbours in memory.
static bool rows_are_lines(i64 k, i64 n, i64 k_stride, i64 n_stride) { return n_stride == 1 || n == 1 ? !(k_stride == 1 && n == 1 && k > 1) : false; }
static Lines matrices_operand(const void* w, int dtype, i64 experts, i64 expert_stride, i64 k, i64 k_stride, i64 n, i64 n_stride) {
  if (rows_are_lines(k, n, k_stride, n_stride)) return Lines{w, experts, experts > 1 ? expert_stride : 0, k, k_stride, n, dtype};
  return Lines{w, experts, experts > 1 ? expert_stride : 0, n, n_stride, k, dtype};
}

// Whether a product is of little work, for which the kernels without tensor cores are sooner done: by what both take, in microseconds,
// fitted to a sweep of 17 shapes with bfloat16 and float32 (1 to 16 384 rows, 1 to 200 experts, widths of 32 to 2 048).
// Few rows: 4 for the launch, one per 300 CTAs, one per 350 of the reduced index, one per 2.4 M weights that pass a CTA, 1.2 M of floats whose columns
// are runs (1 024 rows of 100 to 47 by
// three experts: 5.4 for 13.4 by tiles; 4 096 of 64 to 64 by four: 10.3 for 7.1; 32 of 1 024 floats to 2 048 by eight: 18 for 87).  Tiles: 7, the
// weights or the chain of stages, whichever is longer, and the copy of matrices that TMA cannot read.
static double few_time(i64 num_rows, i64 k, i64 n, i64 num_experts, bool slow) {
  const double tiles = (double)(num_rows / kFewRows + min(num_rows, num_experts));
  return 4. + tiles * (double)((n + kFewColumns - 1) / kFewColumns) / 300. + (double)k / 350. + tiles * (double)k * (double)n / (slow ? 1.2e6 : 2.4e6);
}
static bool few_rows(i64 num_rows, i64 k, i64 n, i64 num_experts, int size, bool across, i64 copied_bytes) {
  const double weights = (double)min(num_rows, num_experts) * (double)k * (double)n * size / 4.5e6;
  // steps one behind the other, of all tiles that a pair of CTAs takes: 0.35 us each, of float32 1.4
  const double waves = (double)(num_rows / kPairRows + min(num_rows, num_experts)) * (double)((n + 255) / 256) / (kNumSMs / 2);
  const double chain = (waves > 1. ? waves : 1.) * (double)k * size / 128. * (size == 4 ? 0.7 : 0.35);
  // the copy: read, written with its parts, and read again by the products
  const double copy = copied_bytes > 0 ? 3. + (double)copied_bytes * (size == 4 ? 10. / 6. : 2.) / 2.6e6 : 0.;
  return few_time(num_rows, k, n, num_experts, !across && size > 1) < 6. + (weights > chain ? weights : chain) + copy;
}
// The same of the weights' gradient.  Few rows: 3, one per 400 CTAs, and the rows that a CTA goes through (1 024 rows of 100 to 47 by three experts 7.5
// us for 22; one row of 1 024 to 1 024 16 for 11.6; 4 096 of 64 to 64 by four 20 for 15, of floats 14 for 26).  Tiles: 8, or 14 with chunks, 8 more for float32.
static bool few_grad(i64 num_rows, i64 k, i64 n, i64 num_experts, int size, bool chunks) {
  const double ctas = (double)num_experts * (double)((k + kFewRows - 1) / kFewRows) * (double)((n + kFewColumns - 1) / kFewColumns);
  const double few = 3. + ctas / 400. + (double)num_rows / (double)num_experts * 0.018;
  return few < (chunks ? 14. : 8.) + (size == 4 ? 8. : 0.) + (double)num_experts * (double)k * (double)n * size / 3e6;
}
static int few_grid(i64 tiles) { return (int)max((i64)1, min((i64)kNumSMs * 6, tiles)); }

// Rows of an expert that one tile of the weights' gradient sums.  All of them, unless that leaves pairs of CTAs without work.
static i64 chunk_rows(i64 num_rows, i64 k, i64 n, u32 columns, i64 num_experts) {
  const i64 tiles = (k + kPairRows - 1) / kPairRows * ((n + columns - 1) / columns);
  const i64 wanted = (3 * kNumSMs / 2 + tiles - 1) / tiles;  // chunks in all
  i64 chunk = (num_rows + wanted - 1) / wanted;
  if (num_experts >= wanted) chunk = num_rows;
  chunk = max(chunk, (i64)512);
  // Of more rows than this an expert is cut however many experts there are, where room for the chunks' sums is to be had: 600 000 rows of 256 to 256
  // values, nearly all of one of 300 experts, take 1.6 ms for 3.5 without, of experts that are even 195 us for 116
  constexpr i64 kMostRows = 262144;
  if (chunk > kMostRows && (min(num_experts, (i64)kPlanExperts) + num_rows / kMostRows) * k * n * 4 <= (i64)1 << 30) chunk = kMostRows;
  return min((chunk + 63) / 64 * 64, ((num_rows + 63) / 64) * 64);
}
static i64 most_chunks(i64 num_rows, i64 chunk, i64 num_experts) { return min(num_experts, (i64)kPlanExperts) + num_rows / max((i64)1, chunk); }

// Calls f(T, PARTS, READ).
template <class F>
static int with_type(int dtype, int read, F f) {
  using std::integral_constant;
  if (dtype == GSB_F32) return f(float{}, integral_constant<int, 3>{}, integral_constant<int, BY_WARPS>{});
  auto by_type = [&](auto reading) {
    return dtype == GSB_F16 ? f(__half{}, integral_constant<int, 1>{}, reading) : f(__nv_bfloat16{}, integral_constant<int, 1>{}, reading);
  };
  if (read == SHIFTED) return by_type(integral_constant<int, SHIFTED>{});
  return read == BY_WARPS ? by_type(integral_constant<int, BY_WARPS>{}) : by_type(integral_constant<int, BY_TMA>{});
}
// A product's 16-bit rows that TMA cannot load line by line come class by class (shifted).  Of the others (from an address off 16-byte boundaries, all one row,
// fewer than eight) and of a gradient's, for which classes are not built (a line of its operands is one row, and so of one class, too), those are read by warps
// that every tile reads once, and copied into lines those that several tiles of columns would read again (a product of 210 395 rows of 602 to 602 by 33
// experts with both gradients 950 us for 1 190).  Rows that begin on odd values, which are read value by value, are copied for a gradient (300 000 of
// 101 and 101 127 us for 254) and, where they are long, for a product.  Shifted against copied, products of 200 003 rows of 602 to 602 235 us for
// 264, of 601 240 for 283, of 602 to 2 048 591 for 548; of 100 000 of 102 to 512 42 for 62.
static bool rows_are_copied(const Lines& x, i64 readers, bool grad) {
  if (x.dtype == GSB_F32 || !x.copied()) return false;
  if (!grad && x.shifted()) return false;
  const bool odd = (((u64)(uintptr_t)x.at | (u64)(x.height > 1 ? x.stride * 2 : 0)) & 3) != 0;
  return readers > 1 || (odd && (grad || x.width > 256));
}
static i64 grad_readers(i64 k, i64 n, u32 columns) { return (k + kPairRows - 1) / kPairRows * ((n + columns - 1) / columns); }
static i64 tiles_across(i64 n, u32 columns) { return (n + columns - 1) / columns; }

// Rows for the warps that read them.
static RawRows raw_rows(const Lines& x) {
  const int size = value_bytes(x.dtype);
  const i64 stride = x.height > 1 ? x.stride : 0;
  const u64 bits = (u64)(uintptr_t)x.at | (u64)(stride * size);
  return RawRows{x.at, stride, (u32)x.width, bits % 32 == 0 ? 32 : unit_of(bits)};
}

}  // namespace gsb

using namespace gsb;

extern "C" int64_t gsb_expert_product_workspace(const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride, const void* weights,
                                                int64_t weights_expert_stride, int64_t weights_k_stride, int64_t weights_n_stride, int64_t n,
                                                int64_t num_experts) {
  if (value_bytes(dtype) == 0 || num_rows < 0 || num_rows >= ((i64)1 << 31) || k < 1 || k > GSB_MAX_ROW_LEN || n < 1 || n > GSB_MAX_ROW_LEN ||
      num_experts < 1 || num_experts > GSB_MAX_EXPERTS)
    return GSB_ERR_INVALID_ARGUMENT;
  const i64 copied = matrices_operand(weights, dtype, num_experts, weights_expert_stride, k, weights_k_stride, n, weights_n_stride).bytes();
  if (few_rows(num_rows, k, n, num_experts, value_bytes(dtype), rows_are_lines(k, n, weights_k_stride, weights_n_stride), copied)) return ends_bytes(num_experts);
  const Lines x = rows_operand(rows, dtype, num_rows, k, rows_stride);
  const u32 columns = tile_columns(n, dtype, row_tiles_of(num_rows, num_experts));
  return ends_bytes(num_experts) + held_bytes(k, dtype, columns) + copied + (rows_are_copied(x, tiles_across(n, columns), false) ? x.bytes() : 0);
}

extern "C" int gsb_expert_product(gsb_ctx* ctx, void* stream_, const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride,
                                  const void* weights, int64_t weights_expert_stride, int64_t weights_k_stride, int64_t weights_n_stride, int64_t n,
                                  const int64_t* offsets, int64_t num_experts, void* out, void* workspace, int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  int st = check_product(num_rows, k, n, num_experts, rows_stride, offsets);
  if (st != GSB_OK) return st;
  const int size = value_bytes(dtype);
  GSB_REQUIRE(size != 0 && weights_expert_stride >= 0 && weights_k_stride >= 0 && weights_n_stride >= 0, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(weights_k_stride == 1 || weights_n_stride == 1 || k == 1 || n == 1, GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0) return GSB_OK;
  GSB_REQUIRE(rows && weights && out && aligned_to(size, (const char*)rows, (const char*)weights, (const char*)out), GSB_ERR_INVALID_ARGUMENT);
  const int64_t need = gsb_expert_product_workspace(rows, dtype, num_rows, k, rows_stride, weights, weights_expert_stride, weights_k_stride,
                                                    weights_n_stride, n, num_experts);
  GSB_REQUIRE(need >= 0 && (need == 0 || workspace) && aligned_to(256, (const char*)workspace), GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(workspace_bytes >= need, GSB_ERR_CAPACITY);
  cudaStream_t stream = (cudaStream_t)stream_;
  const bool across = rows_are_lines(k, n, weights_k_stride, weights_n_stride);
  Lines x = rows_operand(rows, dtype, num_rows, k, rows_stride);
  Lines w = matrices_operand(weights, dtype, num_experts, weights_expert_stride, k, weights_k_stride, n, weights_n_stride);
  char* room = (char*)workspace;
  u32* const ends = take_ends(num_experts, &room);
  if (few_rows(num_rows, k, n, num_experts, size, across, w.bytes()))
    return by_experts(ctx, num_experts, num_rows, offsets, ends, [&](const Groups& g) {
      const i64 line = w.height > 1 ? w.stride : 0;
      const FewArgs a{g, rows, weights, rows_stride, line, w.matrix_stride, (u32)k, (u32)n, nullptr, nullptr};
      const bool wide = aligned_to(16, (const char*)weights) && line * size % 16 == 0 && w.matrix_stride * size % 16 == 0;
      const int grid = few_grid((num_rows / kFewRows + min(num_rows, (i64)g.experts)) * ((n + kFewColumns - 1) / kFewColumns));
      ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
      with_unit(dtype, size, [&](auto value, auto) {
        typedef decltype(value) T;
        auto kernel = across ? (wide ? k_few_across<T, true> : k_few_across<T, false>) : (wide ? k_few_along<T, T, true> : k_few_along<T, T, false>);
        launch_behind(stream, kernel, grid, kFewThreads, a, (T*)out);
      });
      GSB_LAUNCH_OK();
      return (int)GSB_OK;
    });
  TileArgs a = {};
  a.columns = tile_columns(n, dtype, row_tiles_of(num_rows, num_experts));
  a.held = take_held(k, dtype, a.columns, &room);
  if ((st = bring(ctx, stream, &w, &room)) != GSB_OK) return st;
  if (rows_are_copied(x, tiles_across(n, a.columns), false) && (st = bring(ctx, stream, &x, &room)) != GSB_OK) return st;
  a.rows = raw_rows(x);
  a.depth = (u32)k;
  a.n = (u32)n;
  a.expert_step = w.copies() > 1;
  CUtensorMap map_x = {}, map_w;
  ShiftedMaps shifted_x = {};
  const int read = !x.copied() ? BY_TMA : x.shifted() ? SHIFTED : BY_WARPS;
  if (read == BY_TMA && (st = describe(x, 2, 64, 128, false, &map_x)) != GSB_OK) return st;
  if (read == SHIFTED && (st = describe_shifted(x, &shifted_x)) != GSB_OK) return st;
  a.classes = read == SHIFTED ? x.classes() : 0;
  if ((st = describe(w, 2, 64, across ? 64 : a.columns / 2, true, &map_w)) != GSB_OK) return st;
  return by_experts(ctx, num_experts, num_rows, offsets, ends, [&](const Groups& g) {
    a.groups = g;
    const i64 tiles = (num_rows / kPairRows + g.experts) * ((n + a.columns - 1) / a.columns);
    return with_type(dtype, read, [&](auto value, auto parts, auto reading) {
      typedef decltype(value) T;
      constexpr int P = decltype(parts)::value;
      constexpr int R = decltype(reading)::value;
      auto launch = [&](const RowMaps<R>& map) {
        if (across) return launch_tiles<T, false, P, false, true, R>(ctx, stream, map, map_w, a, tiles, num_rows, (T*)out);
        return launch_tiles<T, false, P, false, false, R>(ctx, stream, map, map_w, a, tiles, num_rows, (T*)out);
      };
      if constexpr (R == SHIFTED) return launch(shifted_x);
      else return launch(map_x);
    });
  });
}

extern "C" int64_t gsb_expert_product_grad_workspace(const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride, const void* grad,
                                                     int64_t n, int64_t grad_stride, int64_t num_experts) {
  if (value_bytes(dtype) == 0 || num_rows < 0 || num_rows >= ((i64)1 << 31) || k < 1 || k > GSB_MAX_ROW_LEN || n < 1 || n > GSB_MAX_ROW_LEN ||
      num_experts < 1 || num_experts > GSB_MAX_EXPERTS)
    return GSB_ERR_INVALID_ARGUMENT;
  const u32 columns = tile_columns(n, dtype, row_tiles_of_grad(k, num_experts));
  const i64 chunk = chunk_rows(num_rows, k, n, columns, num_experts);
  if (few_grad(num_rows, k, n, num_experts, value_bytes(dtype), chunk < num_rows)) return ends_bytes(num_experts);
  const Lines x = rows_operand(rows, dtype, num_rows, k, rows_stride), d = rows_operand(grad, dtype, num_rows, n, grad_stride);
  const i64 readers = grad_readers(k, n, columns);
  return ends_bytes(num_experts) + held_bytes(chunk, dtype, columns) + (rows_are_copied(x, readers, true) ? x.bytes() : 0) +
         (rows_are_copied(d, readers, true) ? d.bytes() : 0) + (chunk < num_rows ? rounded(most_chunks(num_rows, chunk, num_experts) * k * n * 4) : 0);
}

extern "C" int gsb_expert_product_grad(gsb_ctx* ctx, void* stream_, const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride,
                                       const void* grad, int64_t n, int64_t grad_stride, const int64_t* offsets, int64_t num_experts, void* out,
                                       void* workspace, int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  int st = check_product(num_rows, k, n, num_experts, rows_stride, offsets);
  if (st != GSB_OK) return st;
  const int size = value_bytes(dtype);
  GSB_REQUIRE(size != 0 && grad_stride >= 0 && out && ((rows && grad) || num_rows == 0), GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_to(size, (const char*)rows, (const char*)grad, (const char*)out), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (num_rows == 0) {
    GSB_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)(num_experts * k * n * size), stream));
    return GSB_OK;
  }
  const int64_t need = gsb_expert_product_grad_workspace(rows, dtype, num_rows, k, rows_stride, grad, n, grad_stride, num_experts);
  GSB_REQUIRE(need >= 0 && (need == 0 || workspace) && aligned_to(256, (const char*)workspace), GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(workspace_bytes >= need, GSB_ERR_CAPACITY);
  char* room = (char*)workspace;
  u32* const ends = take_ends(num_experts, &room);
  if (few_grad(num_rows, k, n, num_experts, size, chunk_rows(num_rows, k, n, tile_columns(n, dtype, row_tiles_of_grad(k, num_experts)), num_experts) < num_rows))
    return by_experts(ctx, num_experts, num_rows, offsets, ends, [&](const Groups& g) {
      const FewArgs a{g, rows, grad, rows_stride, grad_stride, 0, (u32)k, (u32)n, nullptr, nullptr};
      const bool wide = aligned_to(16, (const char*)grad) && (num_rows == 1 || grad_stride * size % 16 == 0);
      const int grid = few_grid(g.experts * ((k + kFewRows - 1) / kFewRows) * ((n + kFewColumns - 1) / kFewColumns));
      ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
      with_unit(dtype, size, [&](auto value, auto) {
        typedef decltype(value) T;
        launch_behind(stream, wide ? k_few_grad<T, true> : k_few_grad<T, false>, grid, kFewThreads, a, (T*)out);
      });
      GSB_LAUNCH_OK();
      return (int)GSB_OK;
    });
  Lines x = rows_operand(rows, dtype, num_rows, k, rows_stride), d = rows_operand(grad, dtype, num_rows, n, grad_stride);
  TileArgs a = {};
  a.columns = tile_columns(n, dtype, row_tiles_of_grad(k, num_experts));
  const i64 chunk = chunk_rows(num_rows, k, n, a.columns, num_experts);
  a.held = take_held(chunk, dtype, a.columns, &room);
  for (Lines* some : {&x, &d})
    if (rows_are_copied(*some, grad_readers(k, n, a.columns), true) && (st = bring(ctx, stream, some, &room)) != GSB_OK) return st;
  a.rows = raw_rows(x);
  a.grad = raw_rows(d);
  a.k = (u32)k;
  a.n = (u32)n;
  a.chunk = (u32)chunk;
  a.partial = chunk < num_rows ? (float*)room : nullptr;
  CUtensorMap map_x = {}, map_d = {};
  const int read = x.copied() || d.copied() ? BY_WARPS : BY_TMA;
  if (!read && ((st = describe(x, 2, 64, 64, false, &map_x)) != GSB_OK || (st = describe(d, 2, 64, 64, false, &map_d)) != GSB_OK)) return st;
  return by_experts(ctx, num_experts, num_rows, offsets, ends, [&](const Groups& g) -> int {
    a.groups = g;
    const i64 tiles = (num_rows / chunk + g.experts) * ((k + kPairRows - 1) / kPairRows) * ((n + a.columns - 1) / a.columns);
    return with_type(dtype, read, [&](auto value, auto parts, auto reading) -> int {
      typedef decltype(value) T;
      constexpr int R = decltype(reading)::value == BY_TMA ? BY_TMA : BY_WARPS;
      const int launched = launch_tiles<T, false, decltype(parts)::value, true, true, R>(ctx, stream, map_x, map_d, a, tiles, (a.partial ? num_rows / chunk + g.experts : num_experts) * k, (T*)out);
      if (launched != GSB_OK || !a.partial) return launched;
      ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
      launch_behind(stream, k_add_chunks<T>, (int)min((i64)kNumSMs * 8, (i64)grid_for(k * n * g.experts, kAddThreads)), kAddThreads, g, a.chunk, k * n,
                    (const float*)a.partial, (T*)out);
      GSB_LAUNCH_OK();
      return GSB_OK;
    });
  });
}

extern "C" int gsb_expert_product_int8(gsb_ctx* ctx, void* stream_, const int8_t* values, int64_t num_rows, int64_t k, int64_t values_stride,
                                       const float* scales, const int8_t* weight_values, int64_t weight_expert_stride, int64_t weight_n_stride,
                                       const float* weight_scales, int64_t n, const int64_t* offsets, int64_t num_experts, void* out, int out_dtype) {
  GSB_ENTER(ctx);
  int st = check_product(num_rows, k, n, num_experts, values_stride, offsets);
  if (st != GSB_OK) return st;
  const int size = value_bytes(out_dtype);
  GSB_REQUIRE(size != 0 && k <= GSB_MAX_INT8_ROW_LEN && weight_expert_stride >= 0 && weight_n_stride >= 0, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_to(16, values, weight_values) && (num_rows <= 1 || (values_stride > 0 && values_stride % 16 == 0)) &&
                  (num_experts == 1 || (weight_expert_stride > 0 && weight_expert_stride % 16 == 0)) &&
                  (n == 1 || (weight_n_stride > 0 && weight_n_stride % 16 == 0)),
              GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0) return GSB_OK;
  GSB_REQUIRE(values && scales && weight_values && weight_scales && out && aligned_to(4, scales, weight_scales) && aligned_to(size, (const char*)out),
              GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (few_rows(num_rows, k, n, num_experts, 1, false, 0))
    return by_experts(ctx, num_experts, num_rows, offsets, nullptr, [&](const Groups& g) {
      const FewArgs a{g, values, weight_values, values_stride, weight_n_stride, num_experts > 1 ? weight_expert_stride : 0, (u32)k, (u32)n, scales, weight_scales};
      const int grid = few_grid((num_rows / kFewRows + min(num_rows, (i64)g.experts)) * ((n + kFewColumns - 1) / kFewColumns));
      ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
      with_unit(out_dtype, size, [&](auto value, auto) {
        typedef decltype(value) Out;
        launch_behind(stream, k_few_along<signed char, Out, true>, grid, kFewThreads, a, (Out*)out);
      });
      GSB_LAUNCH_OK();
      return (int)GSB_OK;
    });
  const Lines x{values, 1, 0, num_rows, values_stride, k, GSB_F16};
  const Lines w{weight_values, num_experts, num_experts > 1 ? weight_expert_stride : 0, n, weight_n_stride, k, GSB_F16};
  TileArgs a = {};
  a.depth = (u32)k;
  a.n = (u32)n;
  a.columns = tile_columns(n, GSB_F16, row_tiles_of(num_rows, num_experts));
  a.expert_step = num_experts > 1;
  a.row_scales = scales;
  a.weight_scales = weight_scales;
  CUtensorMap map_x, map_w;
  if ((st = describe(x, 1, 128, 128, false, &map_x)) != GSB_OK || (st = describe(w, 1, 128, a.columns / 2, true, &map_w)) != GSB_OK) return st;
  return by_experts(ctx, num_experts, num_rows, offsets, nullptr, [&](const Groups& g) {
    a.groups = g;
    const i64 tiles = (num_rows / kPairRows + g.experts) * ((n + a.columns - 1) / a.columns);
    if (out_dtype == GSB_F32) return launch_tiles<float, true, 1, false, false, BY_TMA>(ctx, stream, map_x, map_w, a, tiles, num_rows, (float*)out);
    if (out_dtype == GSB_F16) return launch_tiles<__half, true, 1, false, false, BY_TMA>(ctx, stream, map_x, map_w, a, tiles, num_rows, (__half*)out);
    return launch_tiles<__nv_bfloat16, true, 1, false, false, BY_TMA>(ctx, stream, map_x, map_w, a, tiles, num_rows, (__nv_bfloat16*)out);
  });
}
