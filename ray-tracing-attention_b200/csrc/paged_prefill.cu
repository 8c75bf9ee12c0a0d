// paged_prefill.cu -- attention of many new tokens per sequence over a paged
// K/V cache, causal, with a window and first tokens that stay visible, on the
// 5th-generation tensor cores.
//
// Rows.  The query heads that share a K/V head are rows of one matrix: row R
// of a sequence and K/V head is query R / group, head R % group.  A lane is a
// tile of 128 rows (the M of an MMA); a unit is the one (head_dim 256) or two
// lanes that read the same K and V blocks of 128 positions.  The positions a
// unit needs are the first tokens, then a run of neighbours up to its last
// row's own; they are numbered without the gap, u < firsts ? u : u + skip.
//
// Mathematics.  One pass over the blocks, in base 2: S = Q K^T, w = 2^(scale_log2
// S - m + shift), O += w V, z += sum w, with a reference m per row.  m is the
// maximum of the first positions the row sees, and stays while a block's weights
// add up to a number within Range: a row's result is O / z whatever m is, so m
// only has to keep the weights where their type is exact, and the maximum of
// later blocks is not looked for (a pass over S is bounded by its exponentials
// and conversions).  Otherwise, above the range or below it, the block is weighed
// again with its own maximum and O and z are scaled.  w enters the second product
// rounded to the cache's type (its one rounding; the sum takes w itself).
//
// Work: the blocks of all units form one list, cut evenly over the CTAs (one
// per SM) whatever the lengths are; a lane of a unit that is cut leaves a
// record (m, z, O) per CTA, which a second launch joins in order, many CTAs to a
// unit.  That launch also computes rows by themselves (see row_alone) that are not
// finite beside values they do not see: nobody waits for them there.
//
// Roles (all waits bounded):
//   softmax    four warps per lane, a thread per row: load Q, take S from
//              tensor memory, write w back over it, keep m and z, rescale O,
//              write results or records
//   MMA        one warp issues S = Q K^T (both operands in shared memory) and
//              O += w V (w from tensor memory)
//   producers  three or seven warps bring K and V blocks into a ring of stages (128
//              positions x up to 128 dimensions, 128-byte swizzle): by TMA, a
//              box of positions of one page at a time, where the page size is a
//              multiple of 32; otherwise, and for a unit's last block (its end is
//              filled with zeros), row by row with 16-byte copies
// head_dim 256: one lane, two S buffers, so that S of the next block is
// computed under this block's softmax; 64 and 128: two lanes take turns.
//
// Measured: 8192 rows of 16 / 4 heads x 256 fp16 595 us sustained (0.92 PFLOP/s
// of visible pairs; K and V come out of L2 at 128 KB per block and SM, which
// bounds it), seven ragged prompts of 32 / 8 x 128 bf16 226 us (0.73 PFLOP/s; a
// lane's chain of products and exponentials bounds it, the tensor pipe is 43 %
// active), 64 rows over 2048 positions 20 us (latency).
#include <atomic>
#include <mutex>

#include <cuda.h>

#include "paged_device.cuh"

namespace rta {
namespace paged {
namespace {

constexpr uint32_t kKeys = 128;      // positions per block
constexpr uint32_t kLaneRows = 128;  // rows per lane
constexpr uint32_t kSub = 16384;     // bytes of 128 rows x 64 dimensions

template <int HD>
struct Shape {
  static constexpr uint32_t kLanes = HD == 256 ? 1 : 2;
  static constexpr uint32_t kHalves = HD == 256 ? 2 : 1;          // stages per K or V block
  static constexpr uint32_t kSubs = HD == 64 ? 1 : 2;             // 64-dimension parts per stage
  static constexpr uint32_t kStage = kSubs * kSub;
  static constexpr uint32_t kQ = HD / 64 * kSub;                  // bytes of one lane's queries
  static constexpr uint32_t kStages = HD == 64 ? 10 : 5;
  static constexpr uint32_t kSoftmaxWarps = 4 * kLanes;
  static constexpr uint32_t kProducers = HD == 256 ? 7 : 3;
  static constexpr uint32_t kOwn = HD == 256 ? 20 : 44;           // rows of a stage per producer (the last one: the rest)
  static constexpr uint32_t kThreads = (kSoftmaxWarps + 1 + kProducers) * 32;
  static constexpr uint32_t kRows = kLanes * kLaneRows;           // rows per unit
  static constexpr uint32_t kRing = kLanes * kQ;                  // offset of the stages
  static constexpr uint32_t kBars = kRing + kStages * kStage;     // offset of the barriers
  static constexpr uint32_t kSmem = kBars + 512 + 1024;           // + alignment of the base
  static constexpr uint32_t kRecord = kLaneRows * (HD + 2);       // floats of a lane's record
};

constexpr uint32_t kTmemO = 256;  // tensor-memory column of O (S buffers at 0 and 128)

// What the second launch has to know of a CTA: the unit that begins in its range
// and ends in another's (at most one), and whether units that it wrote by itself,
// which follow one another, have rows that are not finite.
struct Cut {
  uint32_t parts;   // CTAs that hold a part of it, from this one on; 0: no such unit
  uint32_t rows;
  uint32_t second;  // this CTA's record of it is its second (the others': their first)
  uint32_t first_row, R0, kv, slot;
  int32_t past;
  uint32_t firsts, low, high;
  uint32_t bad;                           // units from the first whole one to the last with such a row; 0: none
  uint32_t whole_b, whole_kv, whole_tile;  // the first whole one
};
static_assert(sizeof(Cut) <= kCutBytes, "a description's room in the workspace");
__device__ __forceinline__ Cut& cut_of(const AttendParams& p, uint32_t cta) {
  return *reinterpret_cast<Cut*>(static_cast<uint8_t*>(p.cuts) + cta * kCutBytes);
}

// K and V as TMA sees them: (dimension, position in the page, head, page), or
// head before position where that is the order of the strides.
struct Maps {
  CUtensorMap k, v;
  uint32_t box, heads_first;  // positions per box, 0: no TMA
};

// One unit and its place in the list.
struct Unit {
  uint32_t b, kv, tile;
  uint32_t first_row, rows, tiles, slot;  // of the sequence: its rows are count * group
  int32_t past;                           // position of the sequence's first new token
  uint32_t firsts, skip, seen, blocks;
};

template <int HD>
__device__ __forceinline__ void load_sequence(const AttendParams& p, uint32_t b, Unit& u, uint32_t* err) {
  const Sequence s = sequence(p.c, b, err);  // (its loads and those of the rows run side by side)
  const uint32_t count = new_rows(p, b, u.first_row, err);
  u.b = b;
  u.rows = count * p.group;
  u.tiles = (u.rows + Shape<HD>::kRows - 1u) / Shape<HD>::kRows;
  u.slot = s.slot;
  u.past = static_cast<int32_t>(s.length) - static_cast<int32_t>(count);
}
// Last visible position + 1, numbered without the gap, of rows up to R.
__device__ __forceinline__ uint32_t seen_by(const AttendParams& p, const Unit& u, uint32_t R) {
  const int32_t t = u.past + static_cast<int32_t>(R / p.group);
  return t < 0 ? 0u : static_cast<uint32_t>(t) + 1u - u.skip;
}
__device__ __forceinline__ uint32_t blocks_of(uint32_t seen) { return seen ? (seen + kKeys - 1u) / kKeys : 1u; }
template <int HD>
__device__ __forceinline__ void set_tile(const AttendParams& p, Unit& u, uint32_t tile) {
  u.tile = tile;
  const uint32_t R0 = tile * Shape<HD>::kRows, R1 = min(R0 + Shape<HD>::kRows, u.rows);
  const int32_t t0 = u.past + static_cast<int32_t>(R0 / p.group);
  // what is read begins and ends the first tokens at whole boxes
  uint32_t low = p.window && t0 >= 0 && static_cast<uint32_t>(t0) >= p.window ? t0 - p.window + 1u : 0u;
  low -= low % p.align;
  u.firsts = min((min(p.sinks, 1u << 30) + p.align - 1u) / p.align * p.align, low);
  u.skip = low - u.firsts;
  u.seen = seen_by(p, u, R1 - 1u);
  u.blocks = blocks_of(u.seen);
}
// By a whole warp; there is a next unit.
template <int HD>
__device__ __forceinline__ void next_unit(const AttendParams& p, Unit& u) {
  if (u.tile + 1u < u.tiles) {
    set_tile<HD>(p, u, u.tile + 1u);
    return;
  }
  if (++u.kv == p.c.kv_heads) {
    u.kv = 0;
    load_sequence<HD>(p, u.b + 1u, u, nullptr);
    if (u.tiles == 0u) {  // the next sequence with new rows, a warp's 32 at a time: other roles wait meanwhile
      uint32_t b = u.b + 1u, some = 0, first;
      for (; b < p.c.batch; b += 32u) {
        const uint32_t l = b + (threadIdx.x & 31u);
        some = __ballot_sync(0xffffffffu, l < p.c.batch && new_rows(p, l, first, nullptr) != 0u);
        if (some) break;
      }
      load_sequence<HD>(p, b + __ffs(some) - 1u, u, nullptr);
    }
  }
  set_tile<HD>(p, u, 0u);
}
// Blocks of all tiles of a sequence (one K/V head), by the whole warp: a lane
// adds a short sequence's itself, the warp shares a long one's.
template <int HD>
__device__ uint64_t sequence_blocks(const AttendParams& p, Unit u) {
  uint64_t sum = 0;
  if (u.tiles <= 4u)
    for (uint32_t i = 0; i < u.tiles; ++i) {
      set_tile<HD>(p, u, i);
      sum += u.blocks;
    }
  uint32_t longs = __ballot_sync(0xffffffffu, u.tiles > 4u);
  while (longs) {
    const int from = __ffs(longs) - 1;
    longs &= longs - 1u;
    Unit v = u;
    v.rows = __shfl_sync(0xffffffffu, u.rows, from);
    v.tiles = __shfl_sync(0xffffffffu, u.tiles, from);
    v.past = __shfl_sync(0xffffffffu, u.past, from);
    uint64_t part = 0;
    for (uint32_t i = threadIdx.x & 31u; i < v.tiles; i += 32u) {
      set_tile<HD>(p, v, i);
      part += v.blocks;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
    if (static_cast<int>(threadIdx.x & 31u) == from) sum = part;
  }
  return sum;
}

// The segments of a CTA's range: blocks [a, e) of unit u, one after the other.
template <int HD>
struct Walk {
  Unit u;
  uint64_t unit0, left;     // the unit's place in the list; what is left of the range
  uint32_t entry, at, a, e;  // what a unit costs besides its blocks; place in the unit
  __device__ __forceinline__ bool step(const AttendParams& p) {
    while (left) {
      uint32_t cost = u.blocks + entry;
      if (at == cost) {
        unit0 += cost;
        at = 0;
        next_unit<HD>(p, u);
        cost = u.blocks + entry;
      }
      const uint32_t take = static_cast<uint32_t>(min(left, static_cast<uint64_t>(cost - at)));
      a = at > entry ? at - entry : 0u;
      at += take;
      e = at > entry ? at - entry : 0u;
      left -= take;
      if (e > a) return true;
    }
    return false;
  }
};

// ---- tcgen05 ----------------------------------------------------------------
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define RTA_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define RTA_W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : RTA_R8(v, 0), RTA_R8(v, 8), RTA_R8(v, 16), RTA_R8(v, 24)
      : "r"(addr));
}
// Waits for this thread's loads; the 32 registers pass through it, so nothing
// that uses them can be moved ahead.
#define RTA_X8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
__device__ __forceinline__ void tc_wait_ld(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : RTA_X8(v, 0), RTA_X8(v, 8), RTA_X8(v, 16), RTA_X8(v, 24)::"memory");
}
#undef RTA_X8
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      RTA_W8(v, 0), RTA_W8(v, 8), RTA_W8(v, 16), RTA_W8(v, 24)
      : "memory");
}
#undef RTA_R8
#undef RTA_W8

// Shared-memory matrix descriptor, 128-byte swizzle, 8-row groups 1024 bytes
// apart; `lbo` is the distance of 64-element parts of an MN-major operand (a
// K-major one does not use it).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | static_cast<uint64_t>(lbo >> 4) << 16 |
         static_cast<uint64_t>(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// kind::f16: fp32 D, M = 128; `mn` marks B as MN-major (V: dimensions run fastest)
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc(uint32_t n, bool mn) {
  const uint32_t t = Num<T>::kBf16 ? 1u : 0u;
  return 1u << 4 | t << 7 | t << 10 | (mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (128u >> 4) << 24;
}
// Four k steps, issued by a whole warp in uniform control flow under one
// election.  The first of them overwrites D when `add` is 0.
template <uint32_t ASTEP, uint32_t BSTEP>  // in descriptor units (16 bytes)
__device__ __forceinline__ void mma_ss4(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "add.u64 a1, %1, %5;\n\tadd.u64 a2, a1, %5;\n\tadd.u64 a3, a2, %5;\n\t"
      "add.u64 b1, %2, %6;\n\tadd.u64 b2, b1, %6;\n\tadd.u64 b3, b2, %6;\n\t"
      "elect.sync r|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, 1;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(add), "n"(ASTEP), "n"(BSTEP)
      : "memory");
}
template <uint32_t ASTEP, uint32_t BSTEP>  // tensor-memory columns; descriptor units
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r, a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "add.u32 a1, %1, %5;\n\tadd.u32 a2, a1, %5;\n\tadd.u32 a3, a2, %5;\n\t"
      "add.u64 b1, %2, %6;\n\tadd.u64 b2, b1, %6;\n\tadd.u64 b3, b2, %6;\n\t"
      "elect.sync r|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(add), "n"(ASTEP), "n"(BSTEP)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\telect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void store32(void* at, const uint32_t* v) {  // 32 bytes, 32-byte aligned
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {  // once this thread's copies so far have landed
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;  // volatile: exponentials, sums and conversions stay in turn as written (3 percent of a ragged batch)
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one of them is
  float y;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, %2;\n\tmax.NaN.f32 %0, t, %3;\n\t}" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// (x, y) = (x, y) * a + b and (x, y) += (a, b), two at a time
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 v, s, t;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %2};\n\tmov.b64 t, {%3, %3};\n\t"
      "fma.rn.f32x2 v, v, s, t;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 v, s;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tadd.rn.f32x2 v, v, s;\n\t"
      "mov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w,
                                     uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// Bounded wait of a whole warp; false (for all its lanes) ends the role.
// Inline to the end: a kernel that moves registers between its warps cannot
// call functions.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* err, volatile uint32_t* stop) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint64_t start = globaltimer();
  for (uint32_t spin = 1;; ++spin) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((spin & 63u) == 0u) {
      const bool late = globaltimer() - start > RTA_WAIT_NS;
      if (__any_sync(0xffffffffu, late || *stop != 0u)) {
        if (late && err) atomicOr(err, RTA_DEVERR_TIMEOUT);
        return false;
      }
    }
  }
}

// Where a block's weights may lie.  The reference weighs 2^shift; a row takes
// the block's maximum for its new one when the weights add up to `most` or more
// (each is below it), or to less than `least`.
//   fp16: weights end at 65504, are exact to 2^-12 from 2^-14 on and vanish below
//   2^-25.  shift 8 leaves 128 positions as heavy as the reference below the end,
//   and keeps positions 15 nats under it exact; `least` is 128 times 2^-14.  A
//   first token that scores far above all others and holds nearly nothing is
//   common, and then those others are the result: with shift 0 and no `least` the
//   values of 3000 positions 18 nats below it came out 15 percent off, 120 of them
//   73, now 0.02 and 0.1.  Scores that spread by three nats take new references
//   more often so (8192 rows of 256-dimension heads 580 -> 700 us; by one nat 520
//   before and after; one input over and over).
//   bf16 has fp32's exponents, and so have its values: 2^24 blocks (2^31
//   positions) below 2^-24 add up to less than 1, so O stays below the largest
//   value.  A later block may weigh 2^30 times the reference (2^20 made ragged
//   prompts 234 instead of 220 us where scores spread by five nats), and what lies
//   2^72 below it vanishes.
template <typename T>
struct Range {
  static constexpr float shift = Num<T>::kBf16 ? -54.f : 8.f;
  static constexpr float most = Num<T>::kBf16 ? 5.9604644775390625e-8f : 65504.f;  // 2^-24
  static constexpr float least = Num<T>::kBf16 ? 0.f : 0.0078125f;                 // 2^-7
  // a block that adds less than this of the sum so far is below what a result of
  // its type can show, and its reference would make O and z outgrow fp32
  static constexpr float nothing = 8.8817841970012523e-16f;  // 2^-50
};
// See the list of units: kEntry blocks for a unit's beginning and end where there
// are kFew blocks or more per CTA; without entries at least kLeast blocks per CTA.
constexpr uint32_t kEntry = 2, kFew = 4, kLeast = 2;

template <typename T, int HD>
__global__ void __launch_bounds__(Shape<HD>::kThreads, 1) prefill_kernel(const AttendParams p, const __grid_constant__ Maps maps) {
  using S = Shape<HD>;
  using N = Num<T>;
  constexpr uint32_t kLanes = S::kLanes, kStages = S::kStages, kHalves = S::kHalves;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t scan_part[S::kThreads / 32];
  __shared__ uint64_t found_at;
  __shared__ Unit found_unit;
  __shared__ uint32_t found_kv, found_tile, tmem_base, stop_word, never;
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~uintptr_t{1023});
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* const full = bars;                 // [stages] producers -> MMA
  uint64_t* const empty = bars + 10;           // [stages] MMA -> producers
  uint64_t* const q_full = bars + 20;          // [lane] softmax -> MMA
  uint64_t* const s_full = bars + 22;          // [S buffer] MMA -> softmax
  uint64_t* const p_full = bars + 24;          // [S buffer] softmax -> MMA
  uint64_t* const o_done = bars + 26;          // [lane] MMA -> softmax
  uint64_t* const drain = bars + 28;
  volatile uint32_t* const stop = &stop_word;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&full[i], S::kProducers * 32u);
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < 2u; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
    stop_word = never = 0u;
  }

  pdl_wait();
  if (threadIdx.x == 0) cut_of(p, blockIdx.x).parts = cut_of(p, blockIdx.x).bad = 0u;

  // ---- the list of units and this CTA's range --------------------------------
  uint64_t blocks = 0, tiles = 0, own = 0, own_upto = 0, own_tiles_upto = 0;  // own: this thread's (last) sequence
  uint32_t own_tiles = 0;
  Unit seq;
  for (uint32_t b0 = 0; b0 < p.c.batch; b0 += S::kThreads) {
    const uint32_t b = b0 + threadIdx.x;
    seq.tiles = 0;
    if (b < p.c.batch) load_sequence<HD>(p, b, seq, blockIdx.x == 0u ? p.err : nullptr);
    uint64_t sum;
    own = sequence_blocks<HD>(p, seq);
    own_upto = blocks + block_scan(own, scan_part, sum);
    blocks += sum;
    own_tiles = seq.tiles;
    own_tiles_upto = tiles + block_scan(own_tiles, scan_part, sum);
    tiles += sum;
  }
  if (tiles == 0u) return;
  // Filling and emptying the pipeline costs a unit about as much as kEntry
  // blocks: where the CTAs have several blocks each, a unit counts as that much
  // longer, in front.  Where they have few it counts one block longer (four
  // prompts of up to 200 rows 39 -> 32 us), or none where there are two units a
  // K/V head at most, which are alike and are cut evenly.
  const uint64_t units = tiles * p.c.kv_heads;
  const uint32_t entry = blocks * p.c.kv_heads >= static_cast<uint64_t>(kFew) * gridDim.x ? kEntry : tiles > 2u ? 1u : 0u;
  const uint64_t total = blocks * p.c.kv_heads + units * entry;
  uint64_t ctas = entry ? total : (total + kLeast - 1u) / kLeast;
  if (ctas > gridDim.x) ctas = gridDim.x;
  if (!entry && units <= gridDim.x) ctas = min((ctas + units - 1u) / units, gridDim.x / units) * units;
  if (blockIdx.x >= ctas) return;
  const uint64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1u) / ctas;
  {
    uint64_t before = 0, before_tiles = 0;
    for (uint32_t b0 = 0; b0 < p.c.batch; b0 += S::kThreads) {
      if (p.c.batch > S::kThreads) {  // otherwise the sums above are still these
        const uint32_t b = b0 + threadIdx.x;
        seq.tiles = 0;
        if (b < p.c.batch) load_sequence<HD>(p, b, seq, nullptr);
        uint64_t sum;
        own = sequence_blocks<HD>(p, seq);
        own_upto = before + block_scan(own, scan_part, sum);
        before += sum;
        own_tiles = seq.tiles;
        own_tiles_upto = before_tiles + block_scan(own_tiles, scan_part, sum);
        before_tiles += sum;
      }
      const uint64_t upto = (own_upto + own_tiles_upto * entry) * p.c.kv_heads, per_kv = own + own_tiles * entry;
      if (own_tiles && begin < upto && begin >= upto - per_kv * p.c.kv_heads) {
        const uint64_t at = begin - (upto - per_kv * p.c.kv_heads);
        found_unit = seq;
        found_kv = static_cast<uint32_t>(at / per_kv);
        found_at = at % per_kv;
      }
      if (p.c.batch <= S::kThreads || begin < (before + before_tiles * entry) * p.c.kv_heads) break;
    }
    __syncthreads();
  }
  Unit first = found_unit;
  first.kv = found_kv;
  if (warp == 0) {  // the tile that holds the offset
    uint64_t off = found_at;
    for (uint32_t i0 = 0; i0 < first.tiles; i0 += 32u) {
      Unit v = first;
      uint64_t n = 0;
      if (i0 + lane < first.tiles) {
        set_tile<HD>(p, v, i0 + lane);
        n = v.blocks + entry;
      }
      uint64_t upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint64_t o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= static_cast<uint32_t>(d)) upto += o;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, off < upto);
      if (hit) {
        const int at = __ffs(hit) - 1;
        const uint64_t past = __shfl_sync(0xffffffffu, upto - n, at);
        if (lane == 0) {
          found_tile = i0 + at;
          found_at = off - past;
        }
        break;
      }
      off -= __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (warp == kLanes * 4u) {  // the MMA warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_base;
  set_tile<HD>(p, first, found_tile);
  Walk<HD> walk;
  walk.u = first;
  walk.entry = entry;
  walk.at = static_cast<uint32_t>(found_at);
  walk.unit0 = begin - walk.at;
  walk.left = end - begin;
  const auto lane_rows = [&](const Unit& u, uint32_t L) {
    const uint32_t at = u.tile * S::kRows + L * kLaneRows;
    return u.rows > at ? min(kLaneRows, u.rows - at) : 0u;
  };
  // blocks of lane L of a segment that takes blocks [a, e) of the unit
  const auto lane_blocks = [&](const Unit& u, uint32_t L, uint32_t a, uint32_t e) {
    const uint32_t rows = lane_rows(u, L);
    if (rows == 0u) return 0u;
    const uint32_t n = min(e, blocks_of(seen_by(p, u, u.tile * S::kRows + L * kLaneRows + rows - 1u)));
    return n > a ? n - a : 0u;
  };

  if (warp < S::kSoftmaxWarps) {
    // ---------------------------------------------------------------- softmax
    // registers of the launch: 384 x 168 = 64512; two lanes: 256 x 208 + 128 x 80, one lane: 128 x 240 + 256 x 128
    if constexpr (kLanes == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 240;");
    const uint32_t L = warp >> 2, quarter = warp & 3u, r = quarter * 32u + lane;
    const uint32_t lane_addr = quarter * 32u << 16, tmem_o = tmem + lane_addr + kTmemO + L * HD;
    const uint32_t q_smem = smem_u32(smem) + L * S::kQ;
    // 0: all weights equal (the smallest number, since -inf times it is still -inf);
    // a negative one: the MMA negates the queries
    const float scale = p.scale_log2 == 0.f ? 1.4e-45f : fabsf(p.scale_log2);
    uint32_t it = 0;  // blocks of this lane
    uint32_t wholes = 0;  // units this CTA wrote by itself
    bool ok = true, first_segment = true;
    // the queries of a lane, a row at a time, 16 bytes per thread
    const auto load_queries = [&](const Unit& v) {
      constexpr uint32_t kChunks = HD / 8, kPer = 32 / kChunks;
      const uint32_t R = v.tile * S::kRows + L * kLaneRows + r;
      const bool real = r < lane_rows(v, L);
      const uint64_t off = real ? ((v.first_row + R / p.group) * p.q_row + (v.kv * p.group + R % p.group) * p.q_head) * 2u : 0u;
#pragma unroll 4
      for (uint32_t x0 = 0; x0 < 32u; x0 += kPer) {
        const uint32_t x = x0 + lane / kChunks, c = lane % kChunks, y = quarter * 32u + x;
        const uint64_t o = __shfl_sync(0xffffffffu, off, x);
        const bool on = __shfl_sync(0xffffffffu, real ? 1 : 0, x) != 0;
        cp_async16(q_smem + (c >> 3) * kSub + y * 128u + (((c & 7u) ^ (y & 7u)) << 4),
                   static_cast<const uint8_t*>(p.q) + o + c * 16u, on);
      }
      cp_commit();
    };
    const auto queries_here = [&]() {
      cp_wait<0>();
      fence_async();
      __syncwarp();
      if (lane == 0) arrive(&q_full[L]);
    };
    bool more = walk.step(p);
    if (more && lane_blocks(walk.u, L, walk.a, walk.e)) {
      load_queries(walk.u);
      queries_here();
    }
    while (more && ok) {
      const Unit u = walk.u;
      const uint32_t a = walk.a, e = walk.e;
      const uint64_t unit_last = walk.unit0 + u.blocks + walk.entry - 1u;  // the unit's last place in the list
      const uint32_t rows = lane_rows(u, L), n = lane_blocks(u, L, a, e);
      const uint32_t R = u.tile * S::kRows + L * kLaneRows + r;
      const bool real = r < rows;
      const uint32_t i = real ? R / p.group : 0u, head = u.kv * p.group + (real ? R % p.group : 0u);
      const int32_t t = real ? u.past + static_cast<int32_t>(i) : -1;
      const uint32_t row = u.first_row + i;
      // visible u of this row: u < s_hi or w_lo <= u < w_hi
      const uint32_t w_hi = t < 0 ? 0u : static_cast<uint32_t>(t) + 1u - u.skip;
      const uint32_t w_lo = p.window && t >= 0 && static_cast<uint32_t>(t) >= p.window ? t - p.window + 1u - u.skip : 0u;
      const uint32_t s_hi = min(p.sinks, w_hi);
      // blocks that every row of the lane sees whole: [clear_lo, clear_hi) in u
      const int32_t t_first = u.past + static_cast<int32_t>((u.tile * S::kRows + L * kLaneRows) / p.group);
      const int32_t t_last = rows ? u.past + static_cast<int32_t>((u.tile * S::kRows + L * kLaneRows + rows - 1u) / p.group) : -1;
      const uint32_t clear_hi = t_first < 0 ? 0u : static_cast<uint32_t>(t_first) + 1u - u.skip;
      const uint32_t clear_lo = p.window && t_last >= 0 && static_cast<uint32_t>(t_last) >= p.window ? t_last - p.window + 1u - u.skip : 0u;
      float m = t < 0 ? 0.f : -INFINITY, z = 0.f;  // a row that sees nothing needs no reference
      for (uint32_t j = 0; j < n; ++j, ++it) {
        const uint32_t sb = kLanes == 2 ? L : it & 1u;
        const uint32_t tmem_s = tmem + lane_addr + sb * 128u;
        if (!(ok = warp_wait(&s_full[sb], kLanes == 2 ? it & 1u : it >> 1 & 1u, p.err, stop))) break;
        tc_after();
        const uint32_t u0 = (a + j) * kKeys;
        uint32_t s[2][32], w[64];
        if (u0 < clear_lo || u0 + kKeys > clear_hi) {  // -inf where a row does not see, in place
          const int32_t sh = static_cast<int32_t>(s_hi) - static_cast<int32_t>(u0);
          const int32_t lo = static_cast<int32_t>(w_lo) - static_cast<int32_t>(u0), hi = static_cast<int32_t>(w_hi) - static_cast<int32_t>(u0);
#pragma unroll 1
          for (int32_t c0 = 0; c0 < 128; c0 += 32) {
            if (u0 + c0 >= clear_lo && u0 + c0 + 32u <= clear_hi) continue;
            tc_ld32(tmem_s + c0, s[0]);
            tc_wait_ld(s[0]);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(c0 + c < sh || (c0 + c >= lo && c0 + c < hi))) s[0][c] = 0xff800000u;
            tc_st32(tmem_s + c0, s[0]);
          }
          tc_wait_st();
        }
        // the largest score of the first `columns` (NaN if one of them is)
        const auto largest = [&](uint32_t columns) {
          float x = -INFINITY;
#pragma unroll 1
          for (uint32_t c = 0; c < columns; c += 32u) {
            tc_ld32(tmem_s + c, s[0]);
            tc_wait_ld(s[0]);
            float mx[4] = {x, x, x, x};
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              mx[i >> 1 & 3] = max3(mx[i >> 1 & 3], __uint_as_float(s[0][i]), __uint_as_float(s[0][i + 1]));
            x = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
          }
          return x * scale;
        };
        const float before = m;
        for (uint32_t columns = 32u; columns <= kKeys && __any_sync(0xffffffffu, m == -INFINITY); columns *= 4u) {
          const float x = largest(columns);  // 32 positions give most rows a reference, all of the block the rest
          if (m == -INFINITY) m = x;
        }
        float sum;
        for (bool again = false;;) {
          const float base = m == -INFINITY ? 0.f : Range<T>::shift - m;
          float zs[4][2] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
          tc_ld32(tmem_s, s[0]);
#pragma unroll
          for (uint32_t c = 0; c < 4u; ++c) {
            tc_wait_ld(s[c & 1u]);
            if (c < 3u) tc_ld32(tmem_s + (c + 1u) * 32u, s[(c + 1u) & 1u]);
            uint32_t(&v)[32] = s[c & 1u];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              float w0 = __uint_as_float(v[2 * x]), w1 = __uint_as_float(v[2 * x + 1]);
              fma2(w0, w1, scale, base);
              w0 = ex2(w0);
              w1 = ex2(w1);
              add2(zs[x & 3][0], zs[x & 3][1], w0, w1);
              w[c * 16u + x] = N::pack(w0, w1);
            }
          }
          sum = ((zs[0][0] + zs[0][1]) + (zs[1][0] + zs[1][1])) + ((zs[2][0] + zs[2][1]) + (zs[3][0] + zs[3][1]));
          const bool outside = !(sum < Range<T>::most) || (sum < Range<T>::least && sum > z * Range<T>::nothing);
          if (again || !__any_sync(0xffffffffu, outside)) break;
          const float x = largest(kKeys);
          if (outside) m = x;
          again = true;
        }
        if (!(m < INFINITY)) sum = NAN;  // a NaN or +inf score: the row has no weights
        const bool moved = m != before;
        const float factor = moved ? ex2(before - m) : 1.f;  // before = -inf: 0
        z = z * factor + sum;
        tc_st32(tmem_s, w);  // the weights take the place of the scores
        tc_st32(tmem_s + 32, w + 32);
        if (j) {
          // O holds the blocks before this one
          // (two lanes: S of this block was computed after O of the one before)
          if (kLanes == 1 && !(ok = warp_wait(&o_done[L], (it - 1u) & 1u, p.err, stop))) break;
          if (__any_sync(0xffffffffu, moved)) {
            tc_after();
#pragma unroll 1
            for (uint32_t c = 0; c < HD; c += 32u) {
              uint32_t o[32];
              tc_ld32(tmem_o + c, o);
              tc_wait_ld(o);
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
              tc_st32(tmem_o + c, o);
            }
          }
        }
        tc_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) arrive(&p_full[sb]);
      }
      if (!ok) break;
      // Every S of this unit has been computed, so its queries are done with:
      // the next unit's take their place, and its first S is computed while
      // this one's results are written.  (Loading them a block earlier put the
      // search for the next unit into the loop over blocks: 8 percent slower.)
      more = walk.step(p);
      const bool ahead = more && lane_blocks(walk.u, L, walk.a, walk.e);
      if (ahead) load_queries(walk.u);
      if (ahead) queries_here();
      if (n) {
        if (!(ok = warp_wait(&o_done[L], (it - 1u) & 1u, p.err, stop))) break;
        tc_after();
      }
      const bool whole = a == 0u && e == u.blocks;
      bool bad = false;
      if (whole && rows) {
        const size_t at = static_cast<size_t>(row) * p.heads + head;
        T* const out = static_cast<T*>(p.out) + at * HD;
        const float inv = 1.f / z;
        float odd[2] = {0.f, 0.f};  // NaN once a result is not finite
#pragma unroll 1  // (unrolled: 10 percent slower, the loop over blocks leaves the instruction cache)
        for (uint32_t c = 0; c < HD; c += 32u) {
          uint32_t o[32];
          tc_ld32(tmem_o + c, o);
          tc_wait_ld(o);
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            float f0 = __uint_as_float(o[2 * x]), f1 = __uint_as_float(o[2 * x + 1]);
            fma2(f0, f1, inv, 0.f);
            o[x] = t < 0 ? 0u : N::pack(f0, f1);
            fma2(f0, f1, 0.f, 0.f);
            add2(odd[0], odd[1], f0, f1);
          }
          if (real) {
            store32(out + c, o);
            store32(out + c + 16, o + 8);
          }
        }
        bad = !(odd[0] + odd[1] == 0.f);
        if (real && p.lse) p.lse[at] = t < 0 ? -INFINITY : (m - Range<T>::shift + log2f(z)) * kLn2;
      } else if (rows) {
        float* const rec = p.records + (static_cast<size_t>(blockIdx.x * 2u + (first_segment ? 0u : 1u)) * kLanes + L) * S::kRecord;
        rec[r] = m;
        rec[kLaneRows + r] = z;
        float4* const rec_o = reinterpret_cast<float4*>(rec + 2 * kLaneRows);
        if (n) {
#pragma unroll 1
          for (uint32_t c = 0; c < HD; c += 32u) {
            uint32_t o[32];
            tc_ld32(tmem_o + c, o);
            tc_wait_ld(o);
#pragma unroll
            for (int x = 0; x < 8; ++x)
              rec_o[(c / 4u + x) * kLaneRows + r] = make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                                                                __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
          }
        }
        if (a == 0u && threadIdx.x == 0u) {  // this unit begins here: what the second launch has to know of it
          Cut& cut = cut_of(p, blockIdx.x);
          cut.parts = static_cast<uint32_t>(((unit_last + 1u) * ctas - 1u) / total) - blockIdx.x + 1u;
          cut.second = first_segment ? 0u : 1u;
          cut.first_row = u.first_row;
          cut.R0 = u.tile * S::kRows;
          cut.rows = min(S::kRows, u.rows - cut.R0);
          cut.kv = u.kv;
          cut.slot = u.slot;
          cut.past = u.past;
          cut.firsts = u.firsts;
          cut.low = u.firsts + u.skip;
          cut.high = u.seen + u.skip;
        }
      }
      if (whole) {
        Cut& cut = cut_of(p, blockIdx.x);
        if (wholes == 0u && threadIdx.x == 0u) {
          cut.whole_b = u.b;
          cut.whole_kv = u.kv;
          cut.whole_tile = u.tile;
        }
        ++wholes;
        // (the second launch looks at them: alone, a row of a long history takes
        // longer than the other warps' waits are bounded by)
        if (__any_sync(0xffffffffu, bad && real && t >= 0) && lane == 0) atomicMax(&cut.bad, wholes);
      }
      first_segment = false;
    }
    if (!ok) *stop = 1u;
  } else if (warp == S::kSoftmaxWarps) {
    // -------------------------------------------------------------------- MMA
    if constexpr (kLanes == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
    const uint32_t q0 = smem_u32(smem), ring = q0 + S::kRing;
    uint32_t st = 0, it[2] = {0, 0}, segs[2] = {0, 0};  // stages consumed, blocks and segments of each lane
    bool ok = true;
    const auto wait_stage = [&](uint32_t x) {
      const bool here = warp_wait(&full[x % kStages], x / kStages & 1u, p.err, stop);
      fence_async();  // rows copied by the producers' threads are read by the MMA's proxy
      return here;
    };
    const uint64_t high = desc(0u, 16u), high_v = desc(0u, kSub);
    const uint32_t id_s = idesc<T>(kKeys, false) | (p.scale_log2 < 0.f ? 1u << 13 : 0u);
    // S (+)= Q K^T over the dimensions of one stage
    const auto qk = [&](uint32_t L, uint32_t sbuf, uint32_t x, uint32_t half) {
      const uint32_t qa = q0 + L * S::kQ + half * 2u * kSub, kb = ring + x % kStages * S::kStage;
#pragma unroll 1
      for (uint32_t k = 0; k < S::kSubs; ++k)
        mma_ss4<2, 2>(tmem + sbuf * 128u, high + ((qa + k * kSub) >> 4), high + ((kb + k * kSub) >> 4), id_s, half + k);
    };
    // O[dimensions of one stage] (+)= w V
    const auto pv = [&](uint32_t L, uint32_t sbuf, uint32_t x, uint32_t half, bool fresh) {
      const uint32_t vb = ring + x % kStages * S::kStage;
#pragma unroll 1
      for (uint32_t k = 0; k < kKeys / 16u; k += 4u)
        mma_ts4<8, 128>(tmem + kTmemO + L * HD + half * 128u, tmem + sbuf * 128u + k * 8u, high_v + ((vb + k * 2048u) >> 4),
                        idesc<T>(S::kSubs * 64u, true), fresh && k == 0u ? 0u : 1u);
    };
    while (ok && walk.step(p)) {
      const Unit& u = walk.u;
      const uint32_t a = walk.a, e = walk.e, n = e - a;
      uint32_t ln[2];
      ln[0] = lane_blocks(u, 0, a, e);
      ln[1] = kLanes == 2 ? lane_blocks(u, 1, a, e) : 0u;
#pragma unroll
      for (uint32_t L = 0; L < kLanes; ++L)
        if (ok && ln[L]) ok = warp_wait(&q_full[L], segs[L]++ & 1u, p.err, stop);
      if (!ok) break;
      if constexpr (kLanes == 2) {
        if (!(ok = wait_stage(st))) break;
        tc_after();
#pragma unroll
        for (uint32_t L = 0; L < 2u; ++L)
          if (ln[L]) {
            qk(L, L, st, 0);
            commit(&s_full[L]);
          }
        commit(&empty[st % kStages]);
        ++st;
        for (uint32_t j = 0; j < n && ok; ++j) {
          const bool more = j + 1u < n;
          const uint32_t kst = st, vst = st + (more ? 1u : 0u);
          if (!(ok = (!more || wait_stage(kst)) && wait_stage(vst))) break;
#pragma unroll
          for (uint32_t L = 0; L < 2u; ++L)
            if (ok && j < ln[L]) {
              if (!(ok = warp_wait(&p_full[L], it[L] & 1u, p.err, stop))) break;
              tc_after();
              pv(L, L, vst, 0, j == 0u);
              commit(&o_done[L]);
              ++it[L];
              if (j + 1u < ln[L]) {
                qk(L, L, kst, 0);
                commit(&s_full[L]);
              }
            }
          if (!ok) break;
          if (more) commit(&empty[kst % kStages]);
          commit(&empty[vst % kStages]);
          st = vst + 1u;
        }
      } else {
        for (uint32_t h = 0; h < kHalves && ok; ++h) {
          if (!(ok = wait_stage(st))) break;
          tc_after();
          qk(0, it[0] & 1u, st, h);
          commit(&empty[st++ % kStages]);
        }
        if (!ok) break;
        commit(&s_full[it[0] & 1u]);
        for (uint32_t j = 0; j < n && ok; ++j, ++it[0]) {
          const uint32_t sb = it[0] & 1u;
          if (j + 1u < n) {
            for (uint32_t h = 0; h < kHalves && ok; ++h) {
              if (!(ok = wait_stage(st))) break;
              tc_after();
              qk(0, sb ^ 1u, st, h);
              commit(&empty[st++ % kStages]);
            }
            if (!ok) break;
            commit(&s_full[sb ^ 1u]);
          }
          if (!(ok = warp_wait(&p_full[sb], it[0] >> 1 & 1u, p.err, stop))) break;
          for (uint32_t h = 0; h < kHalves && ok; ++h) {
            if (!(ok = wait_stage(st))) break;
            tc_after();
            pv(0, sb, st, h, j == 0u);
            commit(&empty[st++ % kStages]);
          }
          if (!ok) break;
          commit(&o_done[0]);
        }
      }
    }
    if (!ok) *stop = 1u;
    commit(drain);  // every MMA issued above has completed once this arrives
    (void)warp_wait(drain, 0u, nullptr, &never);
    __syncwarp();
  } else {
    // -------------------------------------------------------------- producers
    if constexpr (kLanes == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
    constexpr uint32_t kOwn = S::kOwn;
    const uint32_t w = warp - S::kSoftmaxWarps - 1u, row0 = w * kOwn, mine = min(kOwn, kKeys - row0);
    const uint32_t ring = smem_u32(smem) + S::kRing;
    uint32_t st = 0;  // stages issued
    bool ok = true;
    const Unit& u = walk.u;
    // Table entry of position `block * 128 + row0 + lane + 32 x`, 0 where there is
    // none; resolved to an offset a block later, when it is here.
    const auto look = [&](uint32_t block, uint32_t x) -> int32_t {
      const uint32_t l = lane + 32u * x, at = block * kKeys + row0 + l;
      if (l >= mine || at >= u.seen) return 0;
      const uint32_t pos = at < u.firsts ? at : at + u.skip;
      return p.c.table[static_cast<size_t>(u.slot) * p.c.width + page_of(p.c, pos)];
    };
    const auto resolve = [&](uint32_t block, uint32_t x, int32_t page) -> uint64_t {
      const uint32_t l = lane + 32u * x, at = block * kKeys + row0 + l;
      if (l >= mine || at >= u.seen) return ~0ull;
      if (static_cast<uint32_t>(page) >= p.c.pages) {
        atomicOr(p.err, RTA_DEVERR_PAGE);
        return ~0ull;
      }
      const uint32_t pos = at < u.firsts ? at : at + u.skip;
      return static_cast<uint64_t>(page) * p.c.page_bytes + static_cast<uint64_t>(pos - page_of(p.c, pos) * p.c.page_size) * p.c.pos_bytes +
             static_cast<uint64_t>(u.kv) * p.c.head_bytes;
    };
    const auto next_stage = [&]() {  // waits until the next stage is free
      const uint32_t s = st % kStages;
      ok = warp_wait(&empty[s], (st / kStages & 1u) ^ 1u, p.err, stop);
      return s;
    };
    // one stage by TMA: lane i of the first producer brings box i, of `page`
    const uint32_t boxes = maps.box ? kKeys / maps.box : 0u;
    const auto bring = [&](const CUtensorMap* map, int32_t page, uint32_t block, uint32_t half) {
      const uint32_t s = next_stage();
      if (!ok) return;
      if (w == 0u) {
        if (lane == 0) mbar_expect_tx(&full[s], S::kStage);  // arrives, as 31 others do here, and 32 of each other warp
        __syncwarp();
        if (lane < boxes) {
          const uint32_t at = block * kKeys + lane * maps.box, pos = at < u.firsts ? at : at + u.skip;
          const int32_t y = static_cast<int32_t>(pos - page_of(p.c, pos) * p.c.page_size), kv = static_cast<int32_t>(u.kv);
          // a page outside the pool is flagged and read as zeros, as TMA reads outside its bounds
          if (static_cast<uint32_t>(page) >= p.c.pages) {
            atomicOr(p.err, RTA_DEVERR_PAGE);
            page = static_cast<int32_t>(p.c.pages);
          }
          const uint32_t dst = ring + s * S::kStage + lane * maps.box * 128u;
#pragma unroll
          for (uint32_t x = 0; x < S::kSubs; ++x)
            tma4(dst + x * kSub, map, static_cast<int32_t>(half * 128u + x * 64u), maps.heads_first ? kv : y,
                 maps.heads_first ? y : kv, page, &full[s]);
        }
      }
      if (lane == 0) arrive(&full[s], w == 0u ? 31u : 32u);
      ++st;
    };
    const auto box_page = [&](uint32_t block) -> int32_t {
      const uint32_t at = block * kKeys + lane * maps.box;
      if (w != 0u || lane >= boxes || at >= u.seen) return 0;
      const uint32_t pos = at < u.firsts ? at : at + u.skip;
      return p.c.table[static_cast<size_t>(u.slot) * p.c.width + page_of(p.c, pos)];
    };
    // one stage row by row: dimensions [128 half, ..) of a block's K or V rows
    const auto copy = [&](const uint8_t* base, uint64_t off0, uint64_t off1, uint32_t half) {
      const uint32_t s = next_stage();
      if (!ok) return;
      const uint32_t dst = ring + s * S::kStage, c = lane & 7u;
#pragma unroll
      for (uint32_t x = 0; x < kOwn / 4u; ++x) {
        const uint32_t l = x * 4u + (lane >> 3);
        const uint64_t o = x < 8u ? __shfl_sync(0xffffffffu, off0, l) : __shfl_sync(0xffffffffu, off1, l - 32u);
        const uint32_t row = row0 + l;
        if (l < mine) {
          const uint8_t* src = base + (o == ~0ull ? 0ull : o) + half * 256u + c * 16u;
          const uint32_t to = dst + row * 128u + ((c ^ (row & 7u)) << 4);
#pragma unroll
          for (uint32_t y = 0; y < S::kSubs; ++y) cp_async16(to + y * kSub, src + y * 128u, o != ~0ull);
        }
      }
      cp_arrive(&full[s]);  // when this thread's copies have landed
      ++st;
    };
    while (ok && walk.step(p)) {
      const uint32_t a = walk.a, e = walk.e;
      // blocks [a, whole) lie inside the sequence and come by TMA
      const uint32_t whole = maps.box ? min(e, max(a, u.seen / kKeys)) : a;
      int32_t kp = box_page(a), np = box_page(a + 1u), vp = 0;  // pages of this K block, the next, and the V block
      uint64_t k0 = 0, k1 = 0, v0 = 0, v1 = 0;
      int32_t n0 = 0, n1 = 0;
      if (whole < a + 2u) {
        n0 = look(whole, 0);
        n1 = look(whole, 1);
      }
      for (uint32_t j = a; j <= e && ok; ++j) {  // K of block j, then V of block j - 1
        v0 = k0;
        v1 = k1;
        if (j < e) {
          if (j < whole) {
            for (uint32_t h = 0; h < kHalves && ok; ++h) bring(&maps.k, kp, j, h);
          } else {
            k0 = resolve(j, 0, n0);
            k1 = resolve(j, 1, n1);
            for (uint32_t h = 0; h < kHalves && ok; ++h) copy(p.c.k, k0, k1, h);
          }
          if (j + 1u >= whole) {
            n0 = look(j + 1u, 0);
            n1 = look(j + 1u, 1);
          }
        }
        if (j > a && ok) {
          if (j - 1u < whole) {
            for (uint32_t h = 0; h < kHalves && ok; ++h) bring(&maps.v, vp, j - 1u, h);
          } else {
            for (uint32_t h = 0; h < kHalves && ok; ++h) copy(p.c.v, v0, v1, h);
          }
        }
        vp = kp;
        kp = np;
        np = box_page(j + 2u);
      }
    }
    if (!ok) {
      *stop = 1u;
      if (w == 0u)  // boxes still on their way have landed before the CTA exits (bounded)
        for (uint32_t x = st > kStages ? st - kStages : 0u; x < st; ++x)
          (void)warp_wait(&full[x % kStages], x / kStages & 1u, nullptr, &never);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == S::kSoftmaxWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Rows of a CTA's whole units that are not finite, by row_alone: a warp per row.
template <typename T, int HD>
__device__ __forceinline__ void look_again(const AttendParams& p, const volatile Cut& cut, uint32_t units) {
  using S = Shape<HD>;
  const uint32_t lane = threadIdx.x & 31u;
  Unit u;
  load_sequence<HD>(p, cut.whole_b, u, nullptr);
  u.kv = cut.whole_kv;
  set_tile<HD>(p, u, cut.whole_tile);
  for (uint32_t k = 0;;) {
    const uint32_t R0 = u.tile * S::kRows, rows = min(S::kRows, u.rows - R0);
    for (uint32_t y = blockIdx.y * 8u + (threadIdx.x >> 5); y < rows; y += gridDim.y * 8u) {
      const uint32_t i = (R0 + y) / p.group, row = u.first_row + i, head = u.kv * p.group + (R0 + y) % p.group;
      const int32_t t = u.past + static_cast<int32_t>(i);
      if (t < 0) continue;
      float o[HD / 32];
      load_dims<T, HD>(static_cast<const T*>(p.out) + (static_cast<size_t>(row) * p.heads + head) * HD, lane, o);
      bool bad = false;
#pragma unroll
      for (int x = 0; x < HD / 32; ++x) bad |= !isfinite(o[x]);
      if (__any_sync(0xffffffffu, bad) &&
          spoiled<T, HD>(p, u.slot, u.kv, u.firsts, u.firsts + u.skip, u.seen + u.skip, static_cast<uint32_t>(t)))
        row_alone<T, HD>(p, u.slot, u.kv, head, row, static_cast<uint32_t>(t));
    }
    if (++k == units) return;
    next_unit<HD>(p, u);
  }
}

// Joins the records of cut units: blockIdx.x is the CTA in whose range the unit
// begins, blockIdx.y some of its rows.  O = sum_j 2^(m_j - max m) O_j over
// sum_j 2^(m_j - max m) z_j.  It is bound by latency: every possible piece has a
// CTA of its own (CTAs that share out the pieces: 25 us for a ragged batch where
// this takes 7), and a row's O is on its way while its weights are worked out.
template <int HD>
constexpr uint32_t join_rows() { return 2048u / HD; }  // a thread for eight dimensions of a row
template <typename T, int HD>
__device__ __forceinline__ void join_cut(const AttendParams& p, const Cut& cut) {
  using S = Shape<HD>;
  using N = Num<T>;
  constexpr uint32_t kRows = join_rows<HD>();
  constexpr uint32_t kPer = 256 / kRows;      // threads that work out a row's weights
  constexpr uint32_t kOwn = kMaxCtas / kPer;  // parts of each
  constexpr uint32_t kAhead = 4;
  __shared__ float weight[kMaxCtas][kRows];
  __shared__ uint32_t bad_rows;
  const uint32_t y0 = blockIdx.y * kRows;  // first row within the unit
  if (cut.parts == 0u || y0 >= cut.rows) return;
  const uint32_t L = y0 / kLaneRows, r0 = y0 % kLaneRows;
  const auto record = [&](uint32_t j) {
    return p.records + (static_cast<size_t>((blockIdx.x + j) * 2u + (j == 0u ? cut.second : 0u)) * S::kLanes + L) * S::kRecord;
  };
  const auto place = [&](uint32_t y, uint32_t& row, uint32_t& head, int32_t& t) {
    const uint32_t R = cut.R0 + y;
    row = cut.first_row + R / p.group;
    head = cut.kv * p.group + R % p.group;
    t = cut.past + static_cast<int32_t>(R / p.group);
  };
  const uint32_t x = threadIdx.x % kRows, d8 = threadIdx.x / kRows;  // eight dimensions of a row
  float4 lo[kAhead], hi[kAhead];
  const auto load = [&](uint32_t j0) {
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j)
      if (j0 + j < cut.parts) {
        const float4* o = reinterpret_cast<const float4*>(record(j0 + j) + 2 * kLaneRows) + 2u * d8 * kLaneRows + r0 + x;
        lo[j] = __ldcg(o);
        hi[j] = __ldcg(o + kLaneRows);
      }
  };
  load(0u);
  if (threadIdx.x == 0) bad_rows = 0u;
  {
    const uint32_t wx = threadIdx.x / kPer, k = threadIdx.x % kPer;
    float m[kOwn], z[kOwn], mm = -INFINITY, zz = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
      const uint32_t j = i * kPer + k;
      m[i] = j < cut.parts ? record(j)[r0 + wx] : -INFINITY;
      z[i] = j < cut.parts ? record(j)[kLaneRows + r0 + wx] : 0.f;
    }
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) mm = fmaxf(mm, m[i]);
#pragma unroll
    for (int d = kPer / 2; d >= 1; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
      m[i] = ex2(m[i] - base);
      if (m[i] != 0.f) zz += m[i] * z[i];
    }
#pragma unroll
    for (int d = kPer / 2; d >= 1; d >>= 1) zz += __shfl_xor_sync(0xffffffffu, zz, d);
    const float inv = 1.f / zz;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i)
      if (i * kPer + k < cut.parts) weight[i * kPer + k][wx] = m[i] * inv;
    if (p.lse && k == 0u && y0 + wx < cut.rows) {
      uint32_t row, head;
      int32_t t;
      place(y0 + wx, row, head, t);
      p.lse[static_cast<size_t>(row) * p.heads + head] = t < 0 ? -INFINITY : (mm - Range<T>::shift + log2f(zz)) * kLn2;
    }
  }
  __syncthreads();
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
  for (uint32_t j0 = 0; j0 < cut.parts; j0 += kAhead) {
    if (j0) load(j0);
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) {
      const float f = j0 + j < cut.parts ? weight[j0 + j][x] : 0.f;
      if (f == 0.f) continue;  // an empty part has no O: what was loaded is not used
      a.x += f * lo[j].x;
      a.y += f * lo[j].y;
      a.z += f * lo[j].z;
      a.w += f * lo[j].w;
      b.x += f * hi[j].x;
      b.y += f * hi[j].y;
      b.z += f * hi[j].z;
      b.w += f * hi[j].w;
    }
  }
  if (y0 + x < cut.rows) {
    uint32_t row, head;
    int32_t t;
    place(y0 + x, row, head, t);
    uint4 w = make_uint4(N::pack(a.x, a.y), N::pack(a.z, a.w), N::pack(b.x, b.y), N::pack(b.z, b.w));
    if (t < 0)
      w = make_uint4(0u, 0u, 0u, 0u);
    else if (!isfinite(a.x) || !isfinite(a.y) || !isfinite(a.z) || !isfinite(a.w) || !isfinite(b.x) || !isfinite(b.y) ||
             !isfinite(b.z) || !isfinite(b.w))
      atomicOr(&bad_rows, 1u << x);
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (static_cast<size_t>(row) * p.heads + head) * HD + d8 * 8u) = w;
  }
  __syncthreads();
  for (uint32_t bx = threadIdx.x >> 5; bx < kRows; bx += 8u) {  // see row_alone
    if (!(bad_rows >> bx & 1u)) continue;
    uint32_t row, head;
    int32_t t;
    place(y0 + bx, row, head, t);
    if (spoiled<T, HD>(p, cut.slot, cut.kv, cut.firsts, cut.low, cut.high, static_cast<uint32_t>(t)))
      row_alone<T, HD>(p, cut.slot, cut.kv, head, row, static_cast<uint32_t>(t));
  }
}

// (Registers for three or two blocks per SM: with the compiler's own choice what is
// on its way was spilled, 64 rows over 2048 positions took 33 us instead of 20; for
// two where three fit, ragged batches of 128-dimension heads 214 instead of 211.)
template <typename T, int HD>
__global__ void __launch_bounds__(256, HD == 64 ? 2 : 3) prefill_join_kernel(const AttendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const Cut cut = cut_of(p, blockIdx.x);
  join_cut<T, HD>(p, cut);
  if (cut.bad) look_again<T, HD>(p, *const_cast<volatile Cut*>(&cut_of(p, blockIdx.x)), cut.bad);
}

// Tensor maps of the call's layer, if pages hold whole boxes of at least 32
// positions and the strides are of the kind that TMA takes; otherwise box = 0 and
// rows are copied.  A box costs about as much to issue whatever its size: boxes of
// 16 positions made 8192 rows of 256-dimension heads 886 us where copied rows took
// 676, boxes of 32 and 64 positions saved 4 and 2 percent of ragged batches.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}
template <typename T>
void encode(const AttendParams& p, Maps& maps) {
  maps.box = 0;
  maps.heads_first = p.c.head_bytes < p.c.pos_bytes ? 1u : 0u;
  uint32_t box = 128;
  while (p.c.page_size % box) box /= 2u;
  const EncodeFn fn = encoder();
  if (box < 32u || !fn) return;
  // a dimension of extent 1 is never stepped over: give it the stride that its neighbours ask for
  uint64_t pos = p.c.pos_bytes, head = p.c.head_bytes, page = p.c.page_bytes;
  const uint64_t row = p.c.head_dim * 2u;
  if (p.c.kv_heads == 1u) {
    maps.heads_first = 0u;
    head = pos * p.c.page_size;
  }
  if (p.c.pages == 1u) page = maps.heads_first ? pos * p.c.page_size : head * p.c.kv_heads;
  if (pos < row || head < row || page < row) return;
  const uint64_t a = maps.heads_first ? p.c.kv_heads : p.c.page_size, b = maps.heads_first ? p.c.page_size : p.c.kv_heads;
  const cuuint64_t dims[4] = {p.c.head_dim, a, b, p.c.pages};
  const cuuint64_t strides[3] = {maps.heads_first ? head : pos, maps.heads_first ? pos : head, page};
  const cuuint32_t boxes[4] = {64u, maps.heads_first ? 1u : box, maps.heads_first ? box : 1u, 1u}, steps[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = Num<T>::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  for (int i = 0; i < 2; ++i)
    if (fn(i ? &maps.v : &maps.k, type, 4, const_cast<uint8_t*>(i ? p.c.v : p.c.k), dims, strides, boxes, steps,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return;
  maps.box = box;
}

template <typename T, int HD>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  static std::atomic<int> sms_of[64];
  static std::mutex m;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  int sms = sms_of[dev].load(std::memory_order_acquire);
  if (sms <= 0) {
    std::lock_guard<std::mutex> lock(m);
    e = cudaFuncSetAttribute(prefill_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(Shape<HD>::kSmem));
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (sms <= 0) return cudaErrorInvalidDevice;
    sms_of[dev].store(sms, std::memory_order_release);
  }
  const uint32_t ctas = static_cast<uint32_t>(sms) < kMaxCtas ? static_cast<uint32_t>(sms) : kMaxCtas;
  Maps maps = {};
  AttendParams q = p;
  encode<T>(p, maps);
  q.align = maps.box ? maps.box : 1u;
  e = launch_early(prefill_kernel<T, HD>, dim3(ctas), dim3(Shape<HD>::kThreads), Shape<HD>::kSmem, s, q, maps);
  if (e != cudaSuccess) return e;
  return launch_early(prefill_join_kernel<T, HD>, dim3(ctas, Shape<HD>::kRows / join_rows<HD>()), dim3(256), 0, s, q);
}
template <typename T>
cudaError_t by_dim(const AttendParams& p, cudaStream_t s) {
  switch (p.c.head_dim) {
    case 64: return launch<T, 64>(p, s);
    case 128: return launch<T, 128>(p, s);
    default: return launch<T, 256>(p, s);
  }
}

}  // namespace

size_t prefill_record_bytes() {
  const size_t one = Shape<256>::kRecord, two = 2 * Shape<128>::kRecord;
  return static_cast<size_t>(kMaxCtas) * 2u * (one > two ? one : two) * 4u;
}

cudaError_t launch_prefill(const AttendParams& p, int fmt, cudaStream_t s) {
  return fmt == kF16 ? by_dim<__half>(p, s) : by_dim<__nv_bfloat16>(p, s);
}

}  // namespace paged
}  // namespace rta
