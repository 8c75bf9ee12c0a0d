// pages.cu -- writes of new K/V rows into a paged cache, and the bookkeeping
// of its pages: reserve, fork, free, compact, copy.
//
// Everything is decided on the device (no call waits for the host): one block
// plans -- it ranks free pages, holes and movers with block-wide sums, so the
// choice is the lowest page first, whatever the order of threads -- and a
// launch over the whole device moves the data.  What a call checks is checked
// before anything is written.  The moves of a plan have disjoint sources and
// destinations, so they run in any order.
//
// The moves are bound by HBM (freeing half of 64 sequences and compacting, 1.85 GB
// of reads and writes, takes 316 us with its plan; pages of 64 to 128 positions are
// copied at 6.3 TB/s; pieces of 4 KB per warp keep eight loads in flight per lane,
// 2 and 8 KB were slower), the plans by the latency of one block (8 - 15 us over
// some thousand pages, more over larger pools), appended rows by HBM when they are
// many (17,000 rows of 8 x 128 in 33 us with reserve).
#include "paged_device.cuh"

namespace rta {
namespace paged {
namespace {

// ------------------------------------------------------------------ append
// A block takes `block_rows` new rows.  Its threads load 16-byte pieces of their K
// and V (neighbouring threads neighbouring pieces, whatever head_dim is), and
// while these are on their way its warps find the rows' places in the pool
// (17,200 rows of 8 x 128 bf16 24 us, 5.9 TB/s; 28 with the places found first).
template <typename X>
struct Eight {  // numbers, as they lie in memory
  uint4 v[sizeof(X) / 2];
  __device__ __forceinline__ void load(const X* src) {
#pragma unroll
    for (uint32_t k = 0; k < sizeof(X) / 2; ++k) v[k] = __ldcs(reinterpret_cast<const uint4*>(src) + k);
  }
};
template <typename T>
__device__ __forceinline__ uint4 as(const Eight<T>& x) {
  return x.v[0];
}
template <typename T>
__device__ __forceinline__ uint4 as(const Eight<float>& x) {
  const auto f = [](uint32_t u) { return __uint_as_float(u); };
  const uint4 a = x.v[0], b = x.v[1];
  return make_uint4(Num<T>::pack(f(a.x), f(a.y)), Num<T>::pack(f(a.z), f(a.w)), Num<T>::pack(f(b.x), f(b.y)),
                    Num<T>::pack(f(b.z), f(b.w)));
}

constexpr uint32_t kBlockRows = 64;  // at most
constexpr uint32_t kAhead = 2;       // pieces per thread at a time (those rows: 29 us with 1, 25 with 3, 31 with 8)

template <typename T, typename X>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  __shared__ uint64_t place[kBlockRows];
  constexpr uint64_t kNowhere = ~0ull;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t lane = threadIdx.x & 31u, row0 = blockIdx.x * p.block_rows;
  const uint32_t rows = min(p.block_rows, p.rows - row0);
  const uint32_t per_head = p.c.head_dim / 8u, per_row = 2u * p.c.kv_heads * per_head;  // pieces: K and V side by side
  const uint32_t pieces = rows * per_row;
  for (uint32_t i0 = threadIdx.x; i0 - threadIdx.x < pieces; i0 += 256u * kAhead) {
    Eight<X> piece[kAhead];
    uint32_t of[kAhead];  // rows
    uint8_t* to[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      const uint32_t i = i0 + k * 256u, r = i / per_row, x = i % per_row, h = x / (2u * per_head), y = x % (2u * per_head);
      const bool is_v = y >= per_head;
      const uint32_t d = (is_v ? y - per_head : y) * 8u;
      of[k] = r;
      to[k] = const_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + h * p.c.head_bytes + d * 2u;
      if (i < pieces) piece[k].load(static_cast<const X*>(is_v ? p.v : p.k) + (row0 + r) * p.row_stride + h * p.head_stride + d);
    }
    if (i0 == threadIdx.x) {
      for (uint32_t r = threadIdx.x >> 5; r < rows; r += 8u) {
        const uint32_t row = row0 + r;
        // the sequence: how many of starts[1 .. batch] are <= row
        uint32_t b = 0;
        for (uint32_t i = 0; i < p.c.batch; i += 32u)
          b += __popc(__ballot_sync(0xffffffffu, i + lane < p.c.batch && static_cast<uint32_t>(p.starts[i + lane + 1u]) <= row));
        if (lane) continue;
        uint64_t off = kNowhere;
        if (b < p.c.batch) {
          const Sequence s = sequence(p.c, b, p.err);
          const uint32_t first = static_cast<uint32_t>(p.starts[b]), count = static_cast<uint32_t>(p.starts[b + 1u]) - first;
          const int64_t at = static_cast<int64_t>(s.length) - count + (row - first);
          if (at < 0 || at >= s.length)
            atomicOr(p.err, RTA_DEVERR_SLOT);
          else if (!locate(p.c, s.slot, static_cast<uint32_t>(at), off)) {
            atomicOr(p.err, RTA_DEVERR_PAGE);
            off = kNowhere;
          }
        } else {
          atomicOr(p.err, RTA_DEVERR_SLOT);
        }
        place[r] = off;
      }
      __syncthreads();
    }
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k)
      if (i0 + k * 256u < pieces && place[of[k]] != kNowhere) *reinterpret_cast<uint4*>(to[k] + place[of[k]]) = as<T>(piece[k]);
  }
}

// ------------------------------------------------------------------ plans
// Scratch words of a plan: [0] moves, [1] live pages, [8 ..] what the blocks of a
// compact's look over the map have found; then per move source page, destination
// page and positions, then the free-page list, or for compact the map of moved
// pages.
constexpr uint32_t kLookBlocks = 296, kPlanHead = 8 + kLookBlocks;
struct Plan {
  uint32_t *moves, *found, *src, *dst, *held, *list;
  __device__ __forceinline__ Plan(uint32_t* w, uint32_t pages, uint32_t slots) {
    const uint32_t most = pages > slots ? pages : slots;
    moves = w;
    found = w + 8;
    src = w + kPlanHead;
    dst = src + most;
    held = dst + most;
    list = held + most;
  }
};

constexpr uint32_t kPlanThreads = 1024;

// The first `want` free pages, ascending, into list (at most `want` of them);
// returns how many there are.
__device__ uint32_t list_free(const int32_t* refs, uint32_t pages, uint32_t want, uint32_t* list, uint64_t* part) {
  uint64_t found = 0;
  for (uint32_t p0 = 0; p0 < pages && found < want; p0 += kPlanThreads * 4u) {
    const uint32_t p = p0 + threadIdx.x * 4u;
    uint32_t free_mask = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k)
      if (p + k < pages && refs[p + k] == 0) free_mask |= 1u << k;
    uint64_t sum;
    const uint32_t n = __popc(free_mask);
    uint64_t at = found + block_scan(n, part, sum) - n;
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k)
      if (free_mask >> k & 1u) {
        if (at < want) list[at] = p + k;
        ++at;
      }
    found += sum;
  }
  __syncthreads();
  return static_cast<uint32_t>(found < want ? found : want);
}

// A plan on another map's copy: where that is small, its block copies it itself
// (a launch less); MapArrays.refs is null when there is nothing to copy.
constexpr uint64_t kCopyWords = 32768;
__device__ void copy_map(const PagesParams& p) {
  if (!p.from.refs) return;
  const uint64_t cells = static_cast<uint64_t>(p.slot_count) * p.width;
#pragma unroll 8
  for (uint64_t i = threadIdx.x; i < cells; i += kPlanThreads) p.map.table[i] = p.from.table[i];
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < p.pages; i += kPlanThreads) p.map.refs[i] = p.from.refs[i];
  for (uint32_t i = threadIdx.x; i < p.slot_count; i += kPlanThreads) p.map.lengths[i] = p.from.lengths[i];
  __syncthreads();
}

__global__ void map_copy_kernel(MapArrays from, MapArrays to, uint32_t pages, uint32_t slots, uint64_t cells) {
  pdl_wait();
  pdl_launch_dependents();
  const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x;
  const uint64_t t = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (uint64_t i = t; i < cells; i += stride) to.table[i] = from.table[i];
  for (uint64_t i = t; i < pages; i += stride) to.refs[i] = from.refs[i];
  for (uint64_t i = t; i < slots; i += stride) to.lengths[i] = from.lengths[i];
}

__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(const PagesParams p) {
  pdl_wait();
  pdl_launch_dependents();
  copy_map(p);
  __shared__ uint64_t part[32];
  const Plan plan(p.plan, p.pages, p.slot_count);
  constexpr uint32_t kUnclaimed = 0xffffffffu;
  uint64_t total = 0;
  bool bad = false;
  for (uint32_t i0 = 0; i0 < p.count; i0 += kPlanThreads) {
    const uint32_t i = i0 + threadIdx.x;
    uint64_t need = 0, sum;
    if (i < p.count) {
      const int32_t slot = p.a ? p.a[i] : static_cast<int32_t>(i), add = p.b[i];
      plan.dst[i] = kUnclaimed;
      if (slot < 0 || static_cast<uint32_t>(slot) >= p.slot_count || add < 0) {
        bad = true;
      } else {
        // a slot list may name a slot twice: the length is taken by one of them
        const int64_t n = p.map.lengths[slot];
        if (n < 0 || n + add > static_cast<int64_t>(p.width) * p.page_size ||
            (p.a && atomicCAS(&p.map.lengths[slot], static_cast<int32_t>(n), -1) != n)) {
          bad = true;
        } else {
          plan.dst[i] = static_cast<uint32_t>(n);
          need = (n + add + p.page_size - 1) / p.page_size - (n + p.page_size - 1) / p.page_size;
        }
      }
    }
    const uint64_t first = total + block_scan(need, part, sum) - need;
    if (i < p.count) plan.src[i] = static_cast<uint32_t>(first);
    total += sum;
  }
  uint32_t wrong = __syncthreads_or(bad ? 1 : 0) ? RTA_DEVERR_SLOT : 0u;
  if (!wrong && (total > p.pages ||
                 list_free(p.map.refs, p.pages, static_cast<uint32_t>(total), plan.list, part) < total))
    wrong = RTA_DEVERR_POOL;
  if (wrong) {  // give the lengths back
    if (p.a)
      for (uint32_t i = threadIdx.x; i < p.count; i += kPlanThreads)
        if (plan.dst[i] != kUnclaimed) p.map.lengths[p.a[i]] = static_cast<int32_t>(plan.dst[i]);
    if (threadIdx.x == 0) atomicOr(p.err, wrong);
    return;
  }
  for (uint32_t k = threadIdx.x; k < total; k += kPlanThreads) p.map.refs[plan.list[k]] = 1;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  for (uint32_t i = warp; i < p.count; i += kPlanThreads / 32u) {
    const uint32_t slot = p.a ? p.a[i] : i;
    const uint32_t n = plan.dst[i], grown = n + p.b[i];
    const uint32_t have = (n + p.page_size - 1u) / p.page_size, need = (grown + p.page_size - 1u) / p.page_size;
    for (uint32_t j = have + lane; j < need; j += 32u)
      p.map.table[static_cast<size_t>(slot) * p.width + j] = static_cast<int32_t>(plan.list[plan.src[i] + j - have]);
    if (lane == 0u) p.map.lengths[slot] = static_cast<int32_t>(grown);
  }
}

// Whether the first `held` entries of a row name pages of the pool that are in
// use, by a warp.
__device__ bool row_good(const PagesParams& p, const int32_t* row, uint32_t held) {
  constexpr uint32_t kMany = 8;  // entries per lane and step
  bool good = true;
  for (uint32_t j0 = threadIdx.x & 31u; j0 < held; j0 += 32u * kMany) {
    int32_t page[kMany], refs[kMany];
#pragma unroll
    for (uint32_t k = 0; k < kMany; ++k) page[k] = j0 + k * 32u < held ? row[j0 + k * 32u] : row[j0];
#pragma unroll
    for (uint32_t k = 0; k < kMany; ++k) refs[k] = static_cast<uint32_t>(page[k]) < p.pages ? p.map.refs[page[k]] : 0;
#pragma unroll
    for (uint32_t k = 0; k < kMany; ++k) good &= refs[k] > 0;
  }
  return __all_sync(0xffffffffu, good);
}

// Claims the destinations, looks at the sources' pages, ranks the partly filled
// last ones, takes a page for each; the launch after it shares the full pages and
// copies the rest.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const PagesParams p) {
  pdl_wait();
  pdl_launch_dependents();
  copy_map(p);
  __shared__ uint64_t part[32];
  __shared__ uint32_t fault;
  const Plan plan(p.plan, p.pages, p.slot_count);
  if (threadIdx.x == 0) {
    *plan.moves = 0u;
    fault = 0u;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < p.count; i += kPlanThreads) {
    const int32_t dst = p.b[i];
    if (dst < 0 || static_cast<uint32_t>(dst) >= p.slot_count ||
        atomicCAS(&p.map.lengths[dst], 0, -1 - static_cast<int32_t>(i)) != 0)
      atomicOr(&fault, RTA_DEVERR_SLOT);
  }
  __syncthreads();
  uint64_t total = 0;
  for (uint32_t i0 = 0; i0 < p.count; i0 += kPlanThreads) {
    const uint32_t i = i0 + threadIdx.x;
    uint64_t need = 0, sum;
    if (i < p.count) {
      const int32_t src = p.a[i];
      const int32_t n = src >= 0 && static_cast<uint32_t>(src) < p.slot_count ? p.map.lengths[src] : -1;
      if (n < 0 || static_cast<uint32_t>(n) > p.width * p.page_size) {
        atomicOr(&fault, RTA_DEVERR_SLOT);
      } else {
        const uint32_t rest = static_cast<uint32_t>(n) % p.page_size;
        if (rest) {
          plan.src[i] = static_cast<uint32_t>(p.map.table[static_cast<size_t>(src) * p.width + static_cast<uint32_t>(n) / p.page_size]);
          need = 1u;
        }
        plan.held[i] = rest;
      }
    }
    const uint64_t first = total + block_scan(need, part, sum) - need;
    if (i < p.count) plan.dst[i] = static_cast<uint32_t>(first);
    total += sum;
  }
  __syncthreads();
  if (!fault) {  // every source is a sequence
    __syncthreads();
    for (uint32_t i = threadIdx.x >> 5; i < p.count; i += kPlanThreads / 32u) {
      const uint32_t src = p.a[i], held = (static_cast<uint32_t>(p.map.lengths[src]) + p.page_size - 1u) / p.page_size;
      if (!row_good(p, p.map.table + static_cast<size_t>(src) * p.width, held)) atomicOr(&fault, RTA_DEVERR_PAGE);
    }
  }
  __syncthreads();
  uint32_t wrong = fault;
  if (!wrong && (total > p.pages ||
                 list_free(p.map.refs, p.pages, static_cast<uint32_t>(total), plan.list, part) < total))
    wrong = RTA_DEVERR_POOL;
  if (wrong) {  // give the claimed slots back
    for (uint32_t i = threadIdx.x; i < p.count; i += kPlanThreads) {
      const int32_t dst = p.b[i];
      if (dst >= 0 && static_cast<uint32_t>(dst) < p.slot_count)
        atomicCAS(&p.map.lengths[dst], -1 - static_cast<int32_t>(i), 0);
    }
    if (threadIdx.x == 0) atomicOr(p.err, wrong);
    return;
  }
  for (uint32_t k = threadIdx.x; k < total; k += kPlanThreads) p.map.refs[plan.list[k]] = 1;
  for (uint32_t i = threadIdx.x; i < p.count; i += kPlanThreads) {
    plan.dst[i] = plan.held[i] ? plan.list[plan.dst[i]] : 0u;
    p.map.lengths[p.b[i]] = p.map.lengths[p.a[i]];
  }
  if (threadIdx.x == 0) *plan.moves = p.count;
}

// Before a compact: whether every entry of the tables names a page of the pool
// that is in use (each block notes what it has found), and the copy of the map
// where the result goes into another one.
__global__ void __launch_bounds__(256) compact_look_kernel(const PagesParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const Plan plan(p.plan, p.pages, p.slot_count);
  const bool copy = p.from.refs != nullptr;
  const MapArrays from = copy ? p.from : p.map;
  const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x, cells = static_cast<uint64_t>(p.slot_count) * p.width;
  const uint64_t t = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  bool bad = false;
#pragma unroll 4
  for (uint64_t i = t; i < cells; i += stride) {
    const int32_t page = from.table[i];
    if (copy) p.map.table[i] = page;
    if (page >= 0) bad |= static_cast<uint32_t>(page) >= p.pages || from.refs[page] <= 0;
  }
  if (copy) {
    for (uint64_t i = t; i < p.pages; i += stride) p.map.refs[i] = from.refs[i];
    for (uint64_t i = t; i < p.slot_count; i += stride) p.map.lengths[i] = from.lengths[i];
  }
  const uint32_t any = __syncthreads_or(bad);
  if (threadIdx.x == 0) plan.found[blockIdx.x] = any;
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagesParams p, const uint32_t look_blocks) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint64_t part[32];
  const Plan plan(p.plan, p.pages, p.slot_count);
  const bool wrong = __syncthreads_or(threadIdx.x < look_blocks && plan.found[threadIdx.x]);
  uint64_t mine = 0, live;
  for (uint32_t i = threadIdx.x; i < p.pages; i += kPlanThreads) mine += p.map.refs[i] > 0 ? 1u : 0u;
  block_scan(mine, part, live);
  if (wrong) {
    if (threadIdx.x == 0) {
      *plan.moves = 0u;
      if (p.live) *p.live = static_cast<uint32_t>(live);
      atomicOr(p.err, RTA_DEVERR_PAGE);
    }
    return;
  }
  uint64_t holes = 0, movers = 0;
  for (uint32_t p0 = 0; p0 < p.pages; p0 += kPlanThreads * 4u) {
    const uint32_t i = p0 + threadIdx.x * 4u;
    uint32_t hole = 0, mover = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k)
      if (i + k < p.pages) {
        const bool used = p.map.refs[i + k] > 0;
        if (!used && i + k < live) hole |= 1u << k;
        if (used && i + k >= live) mover |= 1u << k;
      }
    uint64_t sum;  // both ranks in one scan: holes in the low half, movers in the high half
    const uint64_t n = __popc(hole) | static_cast<uint64_t>(__popc(mover)) << 32;
    const uint64_t before = block_scan(n, part, sum) - n;
    uint32_t h = static_cast<uint32_t>(holes + (before & 0xffffffffu)), m = static_cast<uint32_t>(movers + (before >> 32));
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k) {
      if (hole >> k & 1u) plan.dst[h++] = i + k;
      if (mover >> k & 1u) plan.src[m++] = i + k;
    }
    holes += sum & 0xffffffffu;
    movers += sum >> 32;
  }
  __syncthreads();  // holes == movers: both count the pages in use from `live` on
  for (uint32_t k = threadIdx.x; k < movers; k += kPlanThreads) {
    const uint32_t s = plan.src[k], d = plan.dst[k];
    plan.list[s] = d;
    plan.held[k] = p.page_size;
    p.map.refs[d] = p.map.refs[s];
    p.map.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    plan.moves[0] = static_cast<uint32_t>(movers);
    plan.moves[1] = static_cast<uint32_t>(live);
    if (p.live) *p.live = static_cast<uint32_t>(live);
  }
}

__global__ void __launch_bounds__(kPlanThreads) copy_plan_kernel(const PagesParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const Plan plan(p.plan, p.pages, p.slot_count);
  bool bad = false;
  for (uint32_t i = threadIdx.x; i < p.count; i += kPlanThreads) {
    const uint32_t s = p.a[i], d = p.b[i];
    bad |= s >= p.pages || d >= p.pages;
    plan.src[i] = s;
    plan.dst[i] = d;
    plan.held[i] = p.page_size;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    *plan.moves = bad ? 0u : p.count;
    if (bad) atomicOr(p.err, RTA_DEVERR_PAGE);
  }
}

// ------------------------------------------------------------------ moves
enum { kMoveFork = 0, kMoveCompact = 1, kMoveCopy = 2 };
constexpr uint32_t kPiece = 4096;  // bytes one warp moves per step: eight 16-byte loads in flight per lane

template <int KIND>
__global__ void __launch_bounds__(256) move_kernel(const PagesParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const Plan plan(p.plan, p.pages, p.slot_count);
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t warps = static_cast<uint64_t>(gridDim.x) * 8u;
  const uint64_t me = static_cast<uint64_t>(blockIdx.x) * 8u + (threadIdx.x >> 5);
  const uint32_t moves = *plan.moves;
  if (KIND == kMoveFork) {
    for (uint64_t i = me; i < moves; i += warps) {  // share the full pages (the plan has looked at them), end the row
      const uint32_t src = p.a[i], dst = p.b[i], rest = plan.held[i];
      const uint32_t full = static_cast<uint32_t>(p.map.lengths[src]) / p.page_size;
      const int32_t* from = p.map.table + static_cast<size_t>(src) * p.width;
      int32_t* to = p.map.table + static_cast<size_t>(dst) * p.width;
      for (uint32_t j = lane; j < p.width; j += 32u) {
        int32_t page = -1;
        if (j < full) {
          page = from[j];
          atomicAdd(&p.map.refs[page], 1);
        } else if (j == full && rest) {
          page = static_cast<int32_t>(plan.dst[i]);
        }
        to[j] = page;
      }
    }
  }
  if (KIND == kMoveCompact && moves) {
    const uint32_t live = plan.moves[1];
    const uint64_t cells = static_cast<uint64_t>(p.slot_count) * p.width;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < cells; i += warps * 32u) {
      const int32_t page = p.map.table[i];
      if (page >= 0 && static_cast<uint32_t>(page) >= live) p.map.table[i] = static_cast<int32_t>(plan.list[page]);  // a moved one
    }
  }
  // (move, layer, K or V, head, piece of the head's positions)
  const uint32_t pieces = (p.page_size * p.row_bytes + kPiece - 1u) / kPiece;
  const uint64_t items = static_cast<uint64_t>(moves) * p.layers * 2u * p.kv_heads * pieces;
  const uint32_t per_row = p.row_bytes / 16u;
  for (uint64_t it = me; it < items; it += warps) {
    uint64_t x = it;
    const uint32_t piece = static_cast<uint32_t>(x % pieces);
    x /= pieces;
    const uint32_t head = static_cast<uint32_t>(x % p.kv_heads);
    x /= p.kv_heads;
    const uint32_t is_v = static_cast<uint32_t>(x & 1u);
    x >>= 1;
    const uint32_t layer = static_cast<uint32_t>(x % p.layers), i = static_cast<uint32_t>(x / p.layers);
    const uint32_t chunks = plan.held[i] * per_row, c0 = piece * (kPiece / 16u);
    if (c0 >= chunks) continue;
    uint8_t* const base = (is_v ? p.v : p.k) + layer * p.layer_bytes + head * p.head_bytes;
    const uint8_t* const from = base + plan.src[i] * p.page_bytes;
    uint8_t* const to = base + plan.dst[i] * p.page_bytes;
    uint4 v[kPiece / 512u];
#pragma unroll
    for (uint32_t k = 0; k < kPiece / 512u; ++k) {
      const uint32_t c = c0 + k * 32u + lane;
      if (c < chunks) v[k] = __ldcs(reinterpret_cast<const uint4*>(from + c / per_row * p.pos_bytes + c % per_row * 16u));
    }
#pragma unroll
    for (uint32_t k = 0; k < kPiece / 512u; ++k) {
      const uint32_t c = c0 + k * 32u + lane;
      if (c < chunks) *reinterpret_cast<uint4*>(to + c / per_row * p.pos_bytes + c % per_row * 16u) = v[k];
    }
  }
}

// Every block looks over all of the call's slots before it frees its own, so none
// is freed where one is bad: a bad slot or length is not written by any block, and
// a length that another block has set to 0 already is a good one.
constexpr uint32_t kFreeBlocks = 592;  // at most, four per SM
__global__ void __launch_bounds__(256) free_kernel(const PagesParams p) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int32_t length;
  bool bad = false;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < p.count; i += blockDim.x) {
    const int32_t slot = p.a[i];
    const bool real = slot >= 0 && static_cast<uint32_t>(slot) < p.slot_count;
    const int32_t n = real ? p.map.lengths[slot] : -1;
    bad |= n < 0 || static_cast<uint32_t>(n) > p.width * p.page_size;
  }
  if (__syncthreads_or(bad)) {
    if (blockIdx.x == 0u && threadIdx.x == 0) atomicOr(p.err, RTA_DEVERR_SLOT);
    return;
  }
  for (uint32_t i = blockIdx.x; i < p.count; i += gridDim.x) {
    const int32_t slot = p.a[i];
    if (threadIdx.x == 0) length = atomicExch(&p.map.lengths[slot], 0);  // a slot named twice is freed once
    __syncthreads();
    const uint32_t held = (static_cast<uint32_t>(length) + p.page_size - 1u) / p.page_size;
    for (uint32_t j = threadIdx.x; j < held; j += blockDim.x) {
      int32_t* cell = p.map.table + static_cast<size_t>(slot) * p.width + j;
      const int32_t page = *cell;
      *cell = -1;
      if (static_cast<uint32_t>(page) >= p.pages) {
        atomicOr(p.err, RTA_DEVERR_PAGE);
      } else if (atomicSub(&p.map.refs[page], 1) <= 0) {
        atomicAdd(&p.map.refs[page], 1);
        atomicOr(p.err, RTA_DEVERR_PAGE);
      }
    }
    __syncthreads();  // length has been read
  }
}

// Blocks of a move: a warp per piece, at most eight rounds of the four blocks
// that each of the 148 SMs holds.  Compacting 1.85 GB took 341 us with a round and
// a half, 326 with four, 310 with eight, 305 with sixteen, forking 0.21 GB 49, 44,
// 44, 45 us (one input over and over; changing ones take 316 and 48 with eight); a
// block without work costs 0.8 ns, so a call that can move little launches few.
uint32_t move_blocks(const PagesParams& p, uint64_t most_moves) {
  const uint64_t pieces = (p.page_size * p.row_bytes + kPiece - 1u) / kPiece;
  const uint64_t blocks = (most_moves * p.layers * 2u * p.kv_heads * pieces + 7u) / 8u;
  constexpr uint64_t kLeast = 148, kMost = 148 * 32;
  return static_cast<uint32_t>(blocks < kLeast ? kLeast : blocks > kMost ? kMost : blocks);
}

}  // namespace

size_t plan_bytes(uint32_t pages, uint32_t slots) {
  const size_t most = pages > slots ? pages : slots;
  return (kPlanHead + 4u * most) * 4u;
}

cudaError_t launch_append(const AppendParams& in, int fmt, int in_fmt, cudaStream_t s) {
  if (in.rows == 0u) return cudaSuccess;
  AppendParams p = in;
  // kAhead pieces per thread, fewer while that leaves SMs (148, two blocks each) idle
  const uint32_t per_row = p.c.kv_heads * p.c.head_dim / 4u;
  p.block_rows = per_row >= 256u * kAhead ? 1u : 256u * kAhead / per_row;
  if (p.block_rows > kBlockRows) p.block_rows = kBlockRows;
  while (p.block_rows > 1u && p.rows / p.block_rows < 296u) p.block_rows /= 2u;
  const dim3 grid((p.rows + p.block_rows - 1u) / p.block_rows);
  if (fmt == kF16 && in_fmt == kF32)
    return launch_early(append_kernel<__half, float>, grid, dim3(256), 0, s, p);
  if (fmt == kF16)
    return launch_early(append_kernel<__half, __half>, grid, dim3(256), 0, s, p);
  if (in_fmt == kF32)
    return launch_early(append_kernel<__nv_bfloat16, float>, grid, dim3(256), 0, s, p);
  return launch_early(append_kernel<__nv_bfloat16, __nv_bfloat16>, grid, dim3(256), 0, s, p);
}

bool plan_copies(uint32_t pages, uint32_t slots, uint32_t width) {
  return static_cast<uint64_t>(slots) * width + pages <= kCopyWords;
}
cudaError_t launch_map_copy(const MapArrays& from, const MapArrays& to, uint32_t pages, uint32_t slots,
                            uint32_t width, cudaStream_t s) {
  const uint64_t cells = static_cast<uint64_t>(slots) * width;
  const uint64_t most = cells > pages ? cells : pages;
  const uint64_t blocks = (most + 1023u) / 1024u;
  return launch_early(map_copy_kernel, dim3(static_cast<uint32_t>(blocks < 592u ? (blocks ? blocks : 1u) : 592u)), dim3(256),
                      0, s, from, to, pages, slots, cells);
}
cudaError_t launch_reserve(const PagesParams& p, cudaStream_t s) {
  return launch_early(reserve_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
}
cudaError_t launch_fork(const PagesParams& p, cudaStream_t s) {
  const cudaError_t e = launch_early(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
  if (e != cudaSuccess) return e;
  return launch_early(move_kernel<kMoveFork>, dim3(move_blocks(p, p.count)), dim3(256), 0, s, p);
}
cudaError_t launch_free(const PagesParams& p, cudaStream_t s) {
  return launch_early(free_kernel, dim3(p.count < kFreeBlocks ? p.count : kFreeBlocks), dim3(256), 0, s, p);
}
cudaError_t launch_compact(const PagesParams& p, cudaStream_t s) {
  const uint64_t blocks = (static_cast<uint64_t>(p.slot_count) * p.width + 1023u) / 1024u;  // four entries a thread
  const uint32_t look = static_cast<uint32_t>(blocks < kLookBlocks ? blocks : kLookBlocks);
  cudaError_t e = launch_early(compact_look_kernel, dim3(look), dim3(256), 0, s, p);
  if (e != cudaSuccess) return e;
  e = launch_early(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, look);
  if (e != cudaSuccess) return e;
  return launch_early(move_kernel<kMoveCompact>, dim3(move_blocks(p, p.pages / 2u)), dim3(256), 0, s, p);
}
cudaError_t launch_copy(const PagesParams& p, cudaStream_t s) {
  const cudaError_t e = launch_early(copy_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
  if (e != cudaSuccess) return e;
  return launch_early(move_kernel<kMoveCopy>, dim3(move_blocks(p, p.count)), dim3(256), 0, s, p);
}

}  // namespace paged
}  // namespace rta
