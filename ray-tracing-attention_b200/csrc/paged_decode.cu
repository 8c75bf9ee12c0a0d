// paged_decode.cu -- attention of one new token per sequence over a paged K/V
// cache: o = sum_p softmax_p(scale q . k_p) v_p over the positions the token
// sees (all, or a window and the first tokens).
//
// One pass over K and V with a reference m and a sum z per head: a tile of 16
// positions gives scores s, a reference m' >= s, o' = o 2^(m - m') + sum
// 2^(s - m') v, z' likewise; partial results (m, z, o) of the same head add up
// the same way, so the positions are cut anywhere.  m' is max(m, s), but with
// fp16 weights a tile far below m takes its own maximum (see Num), and o and z
// grow by 2^(m - m').
//
// Work: the tiles of all (sequence, K/V head, head block) units form one list;
// every CTA takes an equal contiguous range of it, whatever the lengths are
// (they are read on the device, so a step graph replays with them).  A unit
// that lies inside one range is written at once; one that is cut leaves a
// record per CTA, which a second launch joins, a CTA per head.
//
// The kernel is bound by HBM, so everything else has to stay out of the way of
// the copies: each warp owns a ring of tiles (of its dimensions) that it fills by
// 16-byte copies two tiles ahead, across the ends of units; the page of a tile is looked up
// one tile before its copies; the next unit's queries are copied while this
// one's tiles are read.  Measured: 64 sequences of 128 to 8192 positions, 16 / 4
// heads x 256 fp16, 177 us (1.1 GB at 6.2 TB/s, 95 % of a copy's rate), 100
// windowed ones, 32 / 8 x 128 bf16, 233 us (99 %); one of 32768 positions 33 us,
// of which about 10 are the way to the first tile and the joining launch.
#include <atomic>
#include <mutex>

#include "paged_device.cuh"

namespace rta {
namespace paged {
namespace {

constexpr uint32_t kTile = 16;         // positions per warp tile (the k extent of one value MMA)
constexpr uint32_t kHeadsMax = 16;     // rows of the MMA: 16 heads, or 8 as fp16 pairs (hi, lo)
constexpr uint32_t kRecHeader = 2 * kHeadsMax;  // m and z of a record's heads

__host__ __device__ constexpr uint32_t record_floats(uint32_t hd) { return kRecHeader + kHeadsMax * hd; }

// A unit that begins in a CTA's range and ends in another's: at most one per CTA.
struct Cut {
  uint32_t parts;   // CTAs that hold a part of it, from this one on; 0: no such unit
  uint32_t heads;
  uint32_t second;  // this CTA's record of it is its second (the others': their first)
  uint32_t b, head0;
};
__device__ __forceinline__ Cut& cut_of(const AttendParams& p, uint32_t cta) {
  return *reinterpret_cast<Cut*>(static_cast<uint8_t*>(p.cuts) + cta * kCutBytes);
}

// PAIR: rows g and g + 8 of the MMA are the two 16-bit halves of head g's
// operand (x = T(x) + T(x - T(x))), so weights, and fp32 queries, enter with
// about twice the bits of T at no extra MMA; up to 8 heads per unit.  fp32
// queries are scaled first, by the power of two that puts a warp's largest of a
// head at 2^14 to 2^15 (their scores by its inverse): both halves are then within
// fp16's range whatever the queries' size is, with 22 bits down to 2^-18 of it.
// Otherwise 16 heads per unit and the weights' lower half is a second MMA.
template <typename T, typename Q, int HD, int WARPS, int STAGES, bool PAIR>
struct Shape {
  static constexpr uint32_t kHeads = PAIR ? 8 : 16;
  // Warps that share a tile, each with 128 of its dimensions: its part of the
  // scores, which the two exchange, and its part of the values.  (One warp for
  // 256 dimensions, four per SM, was bound by its own instructions: 64 ragged
  // sequences 205 us.)
  static constexpr uint32_t kParts = HD == 256 ? 2 : 1;
  static constexpr uint32_t kGroups = WARPS / kParts;  // tiles in work at a time
  static constexpr uint32_t kWide = HD / kParts;       // dimensions of a warp
  static constexpr uint32_t kRow = kWide * 2;          // bytes of one K or V row of a warp
  static constexpr uint32_t kChunks = kRow / 16;       // 16-byte chunks per row
  static constexpr uint32_t kStage = 2 * kTile * kRow; // K rows then V rows
  static constexpr uint32_t kRing = WARPS * STAGES * kStage;
  static constexpr uint32_t kQueries = kHeads * HD * sizeof(Q);  // one unit's
  // two CTAs of four warps share an SM (one's units begin and end under the
  // other's copies), or one of eight with 256 dimensions (its rings fill the SM)
  static constexpr uint32_t kPerSm = WARPS == 4 ? 2 : 1;
  // the warps' results are added a part of the dimensions at a time
  static constexpr uint32_t kRoom = kPerSm == 2 ? 8192 : 16384;
  static constexpr uint32_t kPasses = WARPS * kHeads * kWide * 4 / kRoom ? WARPS * kHeads * kWide * 4 / kRoom : 1;
  static constexpr uint32_t kJoin = WARPS * kHeads * (kWide / kPasses) * 4;
  static constexpr uint32_t kSwap = PAIR ? 4 : 8;      // scores per lane that two warps exchange
  static constexpr uint32_t kSmem = kRing + 2 * kQueries + kJoin;
};

struct Unit {  // one (sequence, K/V head, head block)
  uint32_t b, pr;  // sequence of the call; K/V head * head blocks + head block
  uint32_t slot, seen, first, skip;  // visible positions: u < first ? u : u + skip for u < seen
  uint32_t tiles;
};

__device__ __forceinline__ void visible(const AttendParams& p, const Sequence& s, Unit& u) {
  const uint32_t n = s.length;
  const uint32_t low = p.window && n > p.window ? n - p.window : 0u;
  u.slot = s.slot;
  u.first = min(p.sinks, low);
  u.skip = low - u.first;
  u.seen = n - u.skip;
  u.tiles = (u.seen + kTile - 1u) / kTile;
}

__device__ __forceinline__ float2 two(const float* q) { return *reinterpret_cast<const float2*>(q); }
__device__ __forceinline__ float2 two(const __half* q) { return __half22float2(*reinterpret_cast<const __half2*>(q)); }
__device__ __forceinline__ float2 two(const __nv_bfloat16* q) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(q));
}

__device__ __forceinline__ void store4(float* dst, float4 v) { *reinterpret_cast<float4*>(dst) = v; }
__device__ __forceinline__ void store4(__half* dst, float4 v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(Num<__half>::pack(v.x, v.y), Num<__half>::pack(v.z, v.w));
}
__device__ __forceinline__ void store4(__nv_bfloat16* dst, float4 v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(Num<__nv_bfloat16>::pack(v.x, v.y), Num<__nv_bfloat16>::pack(v.z, v.w));
}

template <typename T, typename Q, int HD, int WARPS, int STAGES, bool PAIR>
__global__ void __launch_bounds__(WARPS * 32, Shape<T, Q, HD, WARPS, STAGES, PAIR>::kPerSm) decode_kernel(const AttendParams p) {
  using S = Shape<T, Q, HD, WARPS, STAGES, PAIR>;
  using N = Num<T>;
  constexpr uint32_t kThreads = WARPS * 32, kSteps = S::kWide / 16, kParts = S::kParts, kGroups = S::kGroups;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t scan_part[WARPS];
  __shared__ uint32_t found_b;
  __shared__ uint64_t found_at;
  __shared__ float join_m[WARPS][S::kHeads], join_z[WARPS][S::kHeads];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t4 = lane & 3u;
  const uint32_t group = warp / kParts, part = warp % kParts;
  const uint32_t blocks = (p.group + S::kHeads - 1u) / S::kHeads;  // head blocks per K/V head
  const uint32_t per_seq = p.c.kv_heads * blocks;
  Q* const out = static_cast<Q*>(p.out);
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x == 0) cut_of(p, blockIdx.x).parts = 0u;

  // ---- the list of units: its length, and this CTA's range ------------------
  uint64_t tiles = 0, own = 0, own_upto = 0;  // this thread's (last) sequence in the list
  uint32_t some = 0;                          // sequences that have anything to see
  for (uint32_t b0 = 0; b0 < p.c.batch; b0 += kThreads) {
    const uint32_t b = b0 + threadIdx.x;
    uint64_t mine = 0, sum;
    if (b < p.c.batch) {
      Unit u;
      visible(p, sequence(p.c, b, blockIdx.x == 0u ? p.err : nullptr), u);
      mine = u.tiles;
      if (u.seen == 0u && b % gridDim.x == blockIdx.x) {  // nothing to see: zeros
        for (uint32_t i = 0; i < p.heads * HD; i += 4u)
          store4(out + static_cast<size_t>(b) * p.heads * HD + i, make_float4(0.f, 0.f, 0.f, 0.f));
        if (p.lse)
          for (uint32_t h = 0; h < p.heads; ++h) p.lse[static_cast<size_t>(b) * p.heads + h] = -INFINITY;
      }
    }
    some += __syncthreads_count(mine != 0u);
    own = mine;
    own_upto = tiles + block_scan(mine, scan_part, sum);
    tiles += sum;
  }
  if (tiles == 0u) return;
  tiles *= per_seq;
  // Beginning and ending a unit costs a CTA about as much as some tiles (3.3 us
  // measured, a tile of 16 KB 0.4 us), so each unit counts as that much longer,
  // in front: four tiles per group of warps where the CTAs have a tile per group
  // or more (64 ragged sequences 209 -> 185 us, 100 windowed ones 244 -> 232 us,
  // 37 of up to 300 positions 33 -> 16 us), two where they have less (ten of up to
  // 300 positions 21 -> 12 us), none for one sequence alone, whose units are
  // alike and are cut evenly, a tile per group.
  const uint32_t entry = tiles / gridDim.x >= kGroups ? 4u * kGroups : some > 1u ? 2u * kGroups : 0u;
  const uint64_t units = static_cast<uint64_t>(some) * per_seq, total = tiles + units * entry;
  uint64_t ctas = (total + kGroups - 1u) / kGroups;
  if (ctas > gridDim.x) ctas = gridDim.x;
  if (!entry && units <= gridDim.x) ctas = min((ctas + units - 1u) / units, gridDim.x / units) * units;
  if (blockIdx.x >= ctas) return;
  const uint64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1u) / ctas;
  const auto owner = [&](uint64_t t) { return static_cast<uint32_t>(((t + 1u) * ctas - 1u) / total); };

  // ---- the unit at its beginning --------------------------------------------
  {
    uint64_t base = 0;
    for (uint32_t b0 = 0; b0 < p.c.batch; b0 += kThreads) {
      const uint32_t b = b0 + threadIdx.x;
      uint64_t mine = own, upto = own_upto, sum = tiles;
      if (p.c.batch > kThreads) {  // otherwise the sums above are still these
        mine = 0;
        if (b < p.c.batch) {
          Unit u;
          visible(p, sequence(p.c, b, nullptr), u);
          mine = u.tiles;
        }
        upto = block_scan(mine, scan_part, sum);
      }
      // sequences with anything to see before this one, for their entries
      uint64_t sum_entries = 0;
      const uint32_t before = entry ? static_cast<uint32_t>(block_scan(mine ? 1u : 0u, scan_part, sum_entries)) : 0u;
      const uint64_t cost = mine ? (mine + entry) * per_seq : 0u;
      const uint64_t last = p.c.batch > kThreads ? base + (upto + static_cast<uint64_t>(before) * entry) * per_seq
                                                 : (upto + static_cast<uint64_t>(before) * entry) * per_seq;
      if (mine && begin < last && begin >= last - cost) {
        found_b = b;
        found_at = begin - (last - cost);
      }
      base += (sum + sum_entries * entry) * per_seq;
      if (p.c.batch <= kThreads || begin < base) break;
    }
    __syncthreads();
  }
  // ---- segments: tiles [a, e) of one unit, one after the other --------------
  struct Segment {
    Unit u;
    uint32_t a, e;
    uint64_t unit0;  // the unit's place in the list
  };
  uint64_t at = begin;  // place in the list behind the segments taken so far
  // s.u is set, and its place `from` on is this CTA's; false: it holds no tile
  const auto take = [&](Segment& s, uint32_t from) {
    s.unit0 = at - from;
    const uint32_t to = static_cast<uint32_t>(min(static_cast<uint64_t>(s.u.tiles + entry), from + (end - at)));
    at += to - from;
    s.a = from > entry ? from - entry : 0u;
    s.e = to > entry ? to - entry : 0u;
    return s.e > s.a;
  };
  const auto follow = [&](const Segment& s, Segment& next) {  // false: there is none
    next.u = s.u;
    while (at < end) {
      if (++next.u.pr == per_seq) {
        next.u.pr = 0;
        visible(p, sequence(p.c, ++next.u.b, nullptr), next.u);
        if (next.u.tiles == 0u) {  // the next sequence with anything to see, a warp's 32 at a time
          uint32_t b = next.u.b + 1u, some = 0;
          for (; b < p.c.batch; b += 32u) {
            some = __ballot_sync(0xffffffffu, b + lane < p.c.batch && sequence(p.c, b + lane, nullptr).length != 0u);
            if (some) break;
          }
          next.u.b = b + __ffs(some) - 1u;
          visible(p, sequence(p.c, next.u.b, nullptr), next.u);
        }
      }
      if (take(next, 0u)) return true;
    }
    return false;
  };
  const auto first_head = [&](const Unit& u) { return u.pr / blocks * p.group + u.pr % blocks * S::kHeads; };
  const auto heads_of = [&](const Unit& u) { return min(S::kHeads, p.group - u.pr % blocks * S::kHeads); };
  const auto copy_queries = [&](const Unit& u, uint32_t to) {  // rows past the unit's heads become zeros
    constexpr uint32_t kPer = HD * sizeof(Q) / 16;
    const uint32_t heads = heads_of(u);
    const Q* q = static_cast<const Q*>(p.q) + static_cast<size_t>(u.b) * p.q_row + static_cast<size_t>(first_head(u)) * p.q_head;
    const uint32_t dst = smem_u32(smem + S::kRing + to * S::kQueries);
    for (uint32_t i = threadIdx.x; i < S::kHeads * kPer; i += kThreads) {
      const uint32_t h = i / kPer;
      cp_async16(dst + i * 16u, q + (h < heads ? h * p.q_head : 0u) + i % kPer * (16u / sizeof(Q)), h < heads);
    }
  };

  Segment cur, next;
  cur.u.b = found_b;
  visible(p, sequence(p.c, cur.u.b, nullptr), cur.u);
  cur.u.pr = static_cast<uint32_t>(found_at / (cur.u.tiles + entry));
  if (!take(cur, static_cast<uint32_t>(found_at % (cur.u.tiles + entry)))) {
    next = cur;
    if (!follow(next, cur)) return;
  }
  next = cur;

  // ---- this warp's tiles: group, group + groups, .. of every segment --------
  const uint32_t ring = smem_u32(smem) + warp * STAGES * S::kStage;
  uint32_t issued = 0, consumed = 0;  // tiles; tile n lies in stage n % STAGES
  // the next tile to issue: lane r < 16 holds the page of its position r and
  // the bytes inside the page
  bool in_next = false, have = false;
  uint32_t tile = cur.a + group;
  int32_t page = -1;
  uint32_t real = 0;
  uint64_t inside = 0;
  const auto look = [&](const Segment& s) {
    const uint32_t n = tile * kTile + (lane & 15u);
    real = n < s.u.seen ? 1u : 0u;
    const uint32_t pos = n < s.u.first ? n : n + s.u.skip;
    const uint32_t j = real ? page_of(p.c, pos) : 0u;
    page = real ? p.c.table[static_cast<size_t>(s.u.slot) * p.c.width + j] : 0;
    inside = static_cast<uint64_t>(pos - j * p.c.page_size) * p.c.pos_bytes + static_cast<uint64_t>(s.u.pr / blocks) * p.c.head_bytes +
             part * S::kRow;
  };
  const auto find = [&](bool more) {  // the tile at or after `tile`, in this segment or the next
    have = false;
    if (!in_next) {
      if (tile < cur.e) {
        have = true;
        look(cur);
        return;
      }
      if (!more) return;
      in_next = true;
      tile = next.a + group;
    }
    if (tile < next.e) {
      have = true;
      look(next);
    }
  };
  const auto issue = [&](bool more) {
    const bool good = static_cast<uint32_t>(page) < p.c.pages;
    if (real && !good) atomicOr(p.err, RTA_DEVERR_PAGE);
    const uint32_t ok = real && good ? 1u : 0u;  // 0: the position becomes zeros
    const uint64_t off = ok ? static_cast<uint64_t>(static_cast<uint32_t>(page)) * p.c.page_bytes + inside : 0u;
    constexpr uint32_t kPer = 32 / S::kChunks;  // rows per warp instruction
    const uint32_t st = ring + issued % STAGES * S::kStage;
#pragma unroll
    for (uint32_t r0 = 0; r0 < kTile; r0 += kPer) {
      const uint32_t r = r0 + lane / S::kChunks, c = lane % S::kChunks;
      const uint64_t o = __shfl_sync(0xffffffffu, off, r) + c * 16u;
      const bool on = __shfl_sync(0xffffffffu, ok, r) != 0u;
      const uint32_t dst = st + r * S::kRow + ((c ^ (r & 7u)) << 4);
      cp_async16(dst, p.c.k + o, on);
      cp_async16(dst + kTile * S::kRow, p.c.v + o, on);
    }
    cp_commit();
    ++issued;
    tile += kGroups;
    find(more);
  };

  find(false);
  copy_queries(cur.u, 0);
  bool more = follow(cur, next);
  if (!have) find(more);
  while (have && issued < STAGES - 1u) issue(more);
  if (issued == 0u) cp_commit();
  cp_wait<0>();
  __syncthreads();  // the queries are there
  for (uint32_t segment = 0;; ++segment) {
    const Unit u = cur.u;
    const uint32_t a = cur.a, e = cur.e, head0 = first_head(u), heads = heads_of(u);
    if (more) copy_queries(next.u, (segment + 1u) & 1u);  // part of the next group of copies

    // Query fragments (A operand: rows are heads, k is the dimension).
    uint32_t qa[kSteps][4];
    float back = 1.f;  // undoes the scaling of fp32 queries
    {
      const Q* q0 = reinterpret_cast<const Q*>(smem + S::kRing + (segment & 1u) * S::kQueries) + g * HD + part * S::kWide + 2u * t4;
      float up = 1.f;
      if (sizeof(Q) == 4) {
        float big = 0.f;
#pragma unroll
        for (uint32_t x = 0; x < 2u * kSteps; ++x) {
          const float2 y = two(q0 + x * 8u);
          big = fmaxf(big, fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const uint32_t e = __float_as_uint(big) >> 23;  // 127 + floor(log2); 255: an infinity, left as it is
        const uint32_t f = e == 255u ? 127u : min(127u + 14u + 127u - e, 253u);
        up = __uint_as_float(f << 23);
        back = __uint_as_float((254u - f) << 23);
      }
#pragma unroll
      for (uint32_t kk = 0; kk < kSteps; ++kk)
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
          float2 x = two(q0 + kk * 16u + h * 8u);
          if (sizeof(Q) == 4) x = make_float2(x.x * up, x.y * up);
          qa[kk][2u * h] = N::pack(x.x, x.y);
          if (PAIR) {
            if (sizeof(Q) == 4) {
              const float2 hi = N::unpack(qa[kk][2u * h]);
              qa[kk][2u * h + 1u] = N::pack(x.x - hi.x, x.y - hi.y);
            } else {
              qa[kk][2u * h + 1u] = 0u;
            }
          } else {
            const float2 y = two(q0 + 8 * HD + kk * 16u + h * 8u);
            qa[kk][2u * h + 1u] = N::pack(y.x, y.y);
          }
        }
    }

    float o[S::kWide / 8][4];
#pragma unroll
    for (int j = 0; j < static_cast<int>(S::kWide / 8); ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    constexpr int kRows = PAIR ? 1 : 2;  // heads of this lane: g (and g + 8)
    float m[kRows], z[kRows], top[kRows];  // top: the largest score so far
#pragma unroll
    for (int r = 0; r < kRows; ++r) m[r] = top[r] = -INFINITY, z[r] = 0.f;

    for (uint32_t i = a + group; i < e; i += kGroups) {
      while (have && issued < consumed + STAGES) issue(more);
      if (issued == consumed + STAGES)
        cp_wait<STAGES - 1>();
      else
        cp_wait<0>();
      __syncwarp();
      const uint32_t st = ring + consumed % STAGES * S::kStage;
      // scores: two 8-position columns, even and odd dimension steps apart
      float sc[2][2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) sc[x][y][0] = sc[x][y][1] = sc[x][y][2] = sc[x][y][3] = 0.f;
#pragma unroll
      for (uint32_t kk = 0; kk < kSteps; ++kk) {
        uint32_t f[4];
        const uint32_t r = (lane & 7u) + ((lane >> 4) << 3), c = 2u * kk + ((lane >> 3) & 1u);
        ldsm4(st + r * S::kRow + ((c ^ (r & 7u)) << 4), f);
        N::mma(sc[kk & 1u][0], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], f[0], f[1]);
        N::mma(sc[kk & 1u][1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], f[2], f[3]);
      }
      // whole scores: both accumulators, the query's two halves, both parts
      float pr[kRows][2][2], rescale[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            pr[r][c][x] = sc[0][c][2 * r + x] + sc[1][c][2 * r + x];
            if (PAIR) pr[r][c][x] += sc[0][c][2 + x] + sc[1][c][2 + x];
            if (sizeof(Q) == 4) pr[r][c][x] *= back;
          }
      if (kParts == 2) {
        // two buffers taken in turn: the other warp has read one before this
        // warp, a barrier later, writes it again
        float* const swap = reinterpret_cast<float*>(smem + S::kRing + 2 * S::kQueries) +
                            (consumed & 1u) * (WARPS * S::kSwap * 32u) + lane * 4u;
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          store4(swap + (warp * kRows + r) * 128u, make_float4(pr[r][0][0], pr[r][0][1], pr[r][1][0], pr[r][1][1]));
        asm volatile("bar.sync %0, 64;" ::"r"(1u + group) : "memory");
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 y = *reinterpret_cast<const float4*>(swap + ((warp ^ 1u) * kRows + r) * 128u);
          pr[r][0][0] += y.x;
          pr[r][0][1] += y.y;
          pr[r][1][0] += y.z;
          pr[r][1][1] += y.w;
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float s = pr[r][c][x] * p.scale_log2;
            if (i * kTile + c * 8u + 2u * t4 + x >= u.seen) s = -INFINITY;
            pr[r][c][x] = s;
            mx = fmaxf(mx, s);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        float mn = fmaxf(m[r], mx);
        if (!N::kBf16) {
          top[r] = fmaxf(top[r], mx);
          if (mx < m[r] - N::kFar && mx > top[r] - N::kNothing) mn = mx;
        }
        const float base = mn == -INFINITY ? 0.f : mn;
        rescale[r] = m[r] == mn ? 1.f : exp2f(m[r] - base);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            pr[r][c][x] = exp2f(pr[r][c][x] - (base - N::kShift));
            sum += pr[r][c][x];
          }
        z[r] = z[r] * rescale[r] + sum;  // this lane's columns; the four lanes are added at the end
        m[r] = mn;
      }
      bool moved = rescale[0] != 1.f;
      if (!PAIR) moved |= rescale[kRows - 1] != 1.f;
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < static_cast<int>(S::kWide / 8); ++j) {
          o[j][0] *= rescale[0];
          o[j][1] *= rescale[0];
          o[j][2] *= rescale[kRows - 1];
          o[j][3] *= rescale[kRows - 1];
        }
      }
      // weights as 16-bit pairs: hi = T(w), lo = T(w - hi)
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        hi[2 * c] = N::pack(pr[0][c][0], pr[0][c][1]);
        const float2 h0 = N::unpack(hi[2 * c]);
        const uint32_t l0 = N::pack(pr[0][c][0] - h0.x, pr[0][c][1] - h0.y);
        if (PAIR) {
          hi[2 * c + 1] = l0;
        } else {
          lo[2 * c] = l0;
          hi[2 * c + 1] = N::pack(pr[kRows - 1][c][0], pr[kRows - 1][c][1]);
          const float2 h1 = N::unpack(hi[2 * c + 1]);
          lo[2 * c + 1] = N::pack(pr[kRows - 1][c][0] - h1.x, pr[kRows - 1][c][1] - h1.y);
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < S::kWide / 8u; j += 2u) {
        uint32_t f[4];
        const uint32_t r = (lane & 7u) + (((lane >> 3) & 1u) << 3), c = j + (lane >> 4);
        ldsm4_t(st + (kTile + r) * S::kRow + ((c ^ (r & 7u)) << 4), f);
        N::mma(o[j], hi[0], hi[1], hi[2], hi[3], f[0], f[1]);
        N::mma(o[j + 1], hi[0], hi[1], hi[2], hi[3], f[2], f[3]);
        if (!PAIR) {
          N::mma(o[j], lo[0], lo[1], lo[2], lo[3], f[0], f[1]);
          N::mma(o[j + 1], lo[0], lo[1], lo[2], lo[3], f[2], f[3]);
        }
      }
      __syncwarp();
      ++consumed;
    }

    // ---- add the warps of this CTA -----------------------------------------
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      z[r] += __shfl_xor_sync(0xffffffffu, z[r], 1);
      z[r] += __shfl_xor_sync(0xffffffffu, z[r], 2);
      if (t4 == 0u) {
        join_m[warp][g + 8 * r] = m[r];
        join_z[warp][g + 8 * r] = z[r];
      }
    }
    const bool whole = a == 0u && e == u.tiles;
    float* const rec = p.records + static_cast<size_t>(blockIdx.x * 2u + (segment ? 1u : 0u)) * record_floats(HD);
    float* const join = reinterpret_cast<float*>(smem + S::kRing + 2 * S::kQueries);  // [warp][head][dimensions of a pass]
    constexpr uint32_t kDims = S::kWide / S::kPasses;  // of each part
    cp_commit();
    cp_wait<0>();  // the next unit's queries, and its first tiles, are there
#pragma unroll
    for (uint32_t pass = 0; pass < S::kPasses; ++pass) {
      if (pass || kParts == 2) __syncthreads();  // the sums before, or the exchanges, have been read
#pragma unroll
      for (uint32_t j = 0; j < kDims / 8u; ++j) {
        const float(&x)[4] = o[pass * (kDims / 8u) + j];
        float* row = join + (warp * S::kHeads + g) * kDims + j * 8u + 2u * t4;
        if (PAIR) {
          *reinterpret_cast<float2*>(row) = make_float2(x[0] + x[2], x[1] + x[3]);
        } else {
          *reinterpret_cast<float2*>(row) = make_float2(x[0], x[1]);
          *reinterpret_cast<float2*>(row + 8u * kDims) = make_float2(x[2], x[3]);
        }
      }
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < kParts * heads * (kDims / 4u); i += kThreads) {
        const uint32_t hp = i / (kDims / 4u), h = hp / kParts, of = hp % kParts, dp = i % (kDims / 4u) * 4u;
        const uint32_t d = of * S::kWide + pass * kDims + dp;
        float mm = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < WARPS; w += kParts) mm = fmaxf(mm, join_m[w][h]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float zz = 0.f;
        float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t w = 0; w < WARPS; w += kParts) {
          const float f = exp2f(join_m[w][h] - base);
          const float4 x = *reinterpret_cast<const float4*>(join + ((w + of) * S::kHeads + h) * kDims + dp);
          zz += join_z[w][h] * f;
          oo.x += x.x * f;
          oo.y += x.y * f;
          oo.z += x.z * f;
          oo.w += x.w * f;
        }
        if (whole) {
          const float inv = 1.f / zz;
          const size_t row = static_cast<size_t>(u.b) * p.heads + head0 + h;
          store4(out + row * HD + d, make_float4(oo.x * inv, oo.y * inv, oo.z * inv, oo.w * inv));
          if (p.lse && d == 0u) p.lse[row] = (mm - N::kShift + log2f(zz)) * kLn2;
        } else {
          store4(rec + kRecHeader + h * HD + d, oo);
          if (d == 0u) {
            rec[h] = mm;
            rec[kHeadsMax + h] = zz;
          }
        }
      }
    }
    if (!whole && a == 0u && threadIdx.x == 0) {  // what the second launch has to know
      Cut& cut = cut_of(p, blockIdx.x);
      cut.parts = owner(cur.unit0 + entry + u.tiles - 1u) - blockIdx.x + 1u;
      cut.second = segment ? 1u : 0u;
      cut.b = u.b;
      cut.head0 = head0;
      cut.heads = heads;
    }
    if (!more) break;
    __syncthreads();  // join and its sums have been read; the next queries are seen by all
    cur = next;
    if (in_next)
      in_next = false;
    else
      tile = cur.a + group;
    more = follow(cur, next);
    if (!have) find(more);
  }
}

// Joins the records of a cut unit: blockIdx.x is the CTA in whose range it
// begins, blockIdx.y the head.  o = sum_j 2^(m_j - max m) o_j over
// sum_j 2^(m_j - max m) z_j.
template <typename T, typename Q, int HD>
__global__ void __launch_bounds__(256) decode_join_kernel(const AttendParams p) {
  using N = Num<T>;
  constexpr uint32_t kQuads = HD / 4, kGroups = 256 / kQuads;
  __shared__ float weight[kMaxDecodeCtas];
  __shared__ float4 sums[kGroups][kQuads];
  pdl_wait();
  pdl_launch_dependents();
  const Cut cut = cut_of(p, blockIdx.x);
  const uint32_t h = blockIdx.y;
  if (h >= cut.heads || cut.parts == 0u) return;
  const auto record = [&](uint32_t j) {
    return p.records + static_cast<size_t>((blockIdx.x + j) * 2u + (j == 0u ? cut.second : 0u)) * record_floats(HD);
  };
  const size_t row = static_cast<size_t>(cut.b) * p.heads + cut.head0 + h;
  if (threadIdx.x < 32u) {
    constexpr uint32_t kOwn = kMaxDecodeCtas / 32u;
    float m[kOwn], z[kOwn], mm = -INFINITY, zz = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < kOwn; ++k) {
      const uint32_t j = k * 32u + threadIdx.x;
      m[k] = j < cut.parts ? record(j)[h] : -INFINITY;
      z[k] = j < cut.parts ? record(j)[kHeadsMax + h] : 0.f;
    }
#pragma unroll
    for (uint32_t k = 0; k < kOwn; ++k) mm = fmaxf(mm, m[k]);
    mm = warp_max(mm);
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (uint32_t k = 0; k < kOwn; ++k) {
      m[k] = exp2f(m[k] - base);
      zz += m[k] * z[k];
    }
    zz = warp_sum(zz);
#pragma unroll
    for (uint32_t k = 0; k < kOwn; ++k) weight[k * 32u + threadIdx.x] = m[k] / zz;
    if (p.lse && threadIdx.x == 0u) p.lse[row] = (mm - N::kShift + log2f(zz)) * kLn2;
  }
  const uint32_t d = threadIdx.x % kQuads, group = threadIdx.x / kQuads;
  constexpr uint32_t kAhead = 8;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f), x[kAhead];
  const auto load = [&](uint32_t j0) {
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      const uint32_t j = j0 + k * kGroups;
      x[k] = j < cut.parts ? *reinterpret_cast<const float4*>(record(j) + kRecHeader + h * HD + d * 4u) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  load(group);
  __syncthreads();  // the weights are there
  for (uint32_t j0 = group; j0 < cut.parts; j0 += kGroups * kAhead) {
    if (j0 != group) load(j0);
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      const uint32_t j = j0 + k * kGroups;
      const float f = j < cut.parts ? weight[j] : 0.f;
      o.x += x[k].x * f;
      o.y += x[k].y * f;
      o.z += x[k].z * f;
      o.w += x[k].w * f;
    }
  }
  sums[group][d] = o;
  __syncthreads();
  if (group == 0u) {
#pragma unroll
    for (uint32_t k = 1; k < kGroups; ++k) {
      const float4 x = sums[k][d];
      o.x += x.x;
      o.y += x.y;
      o.z += x.z;
      o.w += x.w;
    }
    store4(static_cast<Q*>(p.out) + row * HD + d * 4u, o);
  }
}

template <typename T, typename Q, int HD, int WARPS, int STAGES, bool PAIR>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  constexpr uint32_t smem = Shape<T, Q, HD, WARPS, STAGES, PAIR>::kSmem;
  static std::atomic<int> sms_of[64];
  static std::mutex m;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  int sms = sms_of[dev].load(std::memory_order_acquire);
  if (sms <= 0) {
    std::lock_guard<std::mutex> lock(m);
    e = cudaFuncSetAttribute(decode_kernel<T, Q, HD, WARPS, STAGES, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem));
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (sms <= 0) return cudaErrorInvalidDevice;
    sms_of[dev].store(sms, std::memory_order_release);
  }
  const uint32_t most = static_cast<uint32_t>(sms) * Shape<T, Q, HD, WARPS, STAGES, PAIR>::kPerSm;
  const uint32_t ctas = most < kMaxDecodeCtas ? most : kMaxDecodeCtas;
  e = launch_early(decode_kernel<T, Q, HD, WARPS, STAGES, PAIR>, dim3(ctas), dim3(WARPS * 32), smem, s, p);
  if (e != cudaSuccess) return e;
  const uint32_t heads = Shape<T, Q, HD, WARPS, STAGES, PAIR>::kHeads;
  return launch_early(decode_join_kernel<T, Q, HD>, dim3(ctas, p.group < heads ? p.group : heads), dim3(256), 0, s, p);
}

// Two CTAs of four warps per SM where units are short or many for each SM: of 32
// / 8 heads x 128, 512 sequences of up to 300 positions take 86 us instead of
// 122, 100 of them 27 instead of 33, while 160 of up to 4000 take 233 instead of
// 223 and 100 windowed ones 248 instead of 240 (one CTA's rings are deeper).
// Lengths are device data: what the table and the window allow stands for them.
constexpr uint64_t kManyUnits = 8, kShort = 1024;
template <typename T, typename Q, bool PAIR>
cudaError_t by_dim(const AttendParams& p, cudaStream_t s) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  const uint32_t heads = PAIR ? 8u : 16u, blocks = (p.group + heads - 1u) / heads;
  const uint64_t units = static_cast<uint64_t>(p.c.batch) * p.c.kv_heads * blocks;
  uint64_t reach = static_cast<uint64_t>(p.c.width) * p.c.page_size;
  if (p.window && static_cast<uint64_t>(p.window) + p.sinks < reach) reach = static_cast<uint64_t>(p.window) + p.sinks;
  const bool many = units >= (reach <= kShort ? 1u : kManyUnits) * static_cast<uint64_t>(sms);
  switch (p.c.head_dim) {
    case 64: return many ? launch<T, Q, 64, 4, 6, PAIR>(p, s) : launch<T, Q, 64, 8, 6, PAIR>(p, s);
    case 128: return many ? launch<T, Q, 128, 4, 3, PAIR>(p, s) : launch<T, Q, 128, 8, 3, PAIR>(p, s);
    default: return launch<T, Q, 256, 8, 3, PAIR>(p, s);
  }
}

}  // namespace

size_t decode_record_bytes() { return static_cast<size_t>(kMaxDecodeCtas) * 2u * record_floats(256) * 4u; }

// Up to eight query heads per K/V head, and fp32 queries: paired rows.  More
// 16-bit heads: sixteen per unit (fewer passes over K and V).
cudaError_t launch_decode(const AttendParams& p, int fmt, int q, cudaStream_t s) {
  if (q == kF32) return by_dim<__half, float, true>(p, s);
  if (fmt == kF16)
    return p.group <= 8u ? by_dim<__half, __half, true>(p, s) : by_dim<__half, __half, false>(p, s);
  return p.group <= 8u ? by_dim<__nv_bfloat16, __nv_bfloat16, true>(p, s)
                       : by_dim<__nv_bfloat16, __nv_bfloat16, false>(p, s);
}

}  // namespace paged
}  // namespace rta
