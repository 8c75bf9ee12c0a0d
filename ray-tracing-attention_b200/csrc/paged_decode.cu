// paged_decode.cu -- attention of one new token per sequence over a paged K/V
// cache: o = sum_p softmax_p(scale q . k_p) v_p over the positions the token
// sees (all, or a window and the first tokens).
//
// One pass over K and V with a running maximum m and sum z per head: a tile of
// 16 positions gives scores s, m' = max(m, s), o' = o 2^(m - m') + sum
// 2^(s - m') v, z' likewise; partial results (m, z, o) of the same head add up
// the same way, so the positions are cut anywhere.
//
// Work: the tiles of all (sequence, K/V head, head block) units form one list;
// every CTA takes an equal contiguous range of it, whatever the lengths are
// (they are read on the device, so a step graph replays with them).  A unit
// that lies inside one range is written at once; one that is cut leaves a
// record per CTA, and the CTA that arrives last joins them in CTA order.
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

// PAIR: rows g and g + 8 of the MMA are the two 16-bit halves of head g's
// operand (x = T(x) + T(x - T(x))), so weights, and fp32 queries, enter with
// about twice the bits of T at no extra MMA; up to 8 heads per unit.
// Otherwise 16 heads per unit and the weights' lower half is a second MMA.
template <typename T, typename Q, int HD, int WARPS, int STAGES, bool PAIR>
struct Shape {
  static constexpr uint32_t kHeads = PAIR ? 8 : 16;
  static constexpr uint32_t kRow = HD * 2;             // bytes of one K or V row
  static constexpr uint32_t kChunks = kRow / 16;       // 16-byte chunks per row
  static constexpr uint32_t kStage = 2 * kTile * kRow; // K rows then V rows
  static constexpr uint32_t kRing = WARPS * STAGES * kStage;
  static constexpr uint32_t kJoin = WARPS * kHeads * (HD + 2) * 4;
  static constexpr uint32_t kSmem = (kRing > kJoin ? kRing : kJoin) > kMaxCtas * kHeadsMax * 4
                                        ? (kRing > kJoin ? kRing : kJoin)
                                        : kMaxCtas * kHeadsMax * 4;
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

template <typename Q>
__device__ __forceinline__ float load_q(const Q* q);
template <>
__device__ __forceinline__ float load_q<float>(const float* q) { return *q; }
template <>
__device__ __forceinline__ float load_q<__half>(const __half* q) { return __half2float(*q); }
template <>
__device__ __forceinline__ float load_q<__nv_bfloat16>(const __nv_bfloat16* q) { return __bfloat162float(*q); }

__device__ __forceinline__ void store4(float* dst, float4 v) { *reinterpret_cast<float4*>(dst) = v; }
__device__ __forceinline__ void store4(__half* dst, float4 v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(Num<__half>::pack(v.x, v.y), Num<__half>::pack(v.z, v.w));
}
__device__ __forceinline__ void store4(__nv_bfloat16* dst, float4 v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(Num<__nv_bfloat16>::pack(v.x, v.y), Num<__nv_bfloat16>::pack(v.z, v.w));
}

template <typename T, typename Q, int HD, int WARPS, int STAGES, bool PAIR>
__global__ void __launch_bounds__(WARPS * 32, 1) decode_kernel(const AttendParams p) {
  using S = Shape<T, Q, HD, WARPS, STAGES, PAIR>;
  using N = Num<T>;
  constexpr uint32_t kThreads = WARPS * 32, kSteps = HD / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t scan_part[WARPS];
  __shared__ uint32_t found_b;
  __shared__ uint64_t found_at;
  __shared__ float join_m[WARPS][S::kHeads], join_z[WARPS][S::kHeads];
  __shared__ uint32_t last_arrival;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t4 = lane & 3u;
  const uint32_t blocks = (p.group + S::kHeads - 1u) / S::kHeads;  // head blocks per K/V head
  const uint32_t per_seq = p.c.kv_heads * blocks;
  Q* const out = static_cast<Q*>(p.out);

  pdl_wait();
  pdl_launch_dependents();

  // ---- the list of tiles: its length, and this CTA's range -----------------
  uint64_t total = 0, own = 0, own_upto = 0;  // this thread's (last) sequence in the list
  for (uint32_t b0 = 0; b0 < p.c.batch; b0 += kThreads) {
    const uint32_t b = b0 + threadIdx.x;
    uint64_t mine = 0, sum;
    if (b < p.c.batch) {
      Unit u;
      visible(p, sequence(p.c, b, blockIdx.x == 0u ? p.err : nullptr), u);
      mine = static_cast<uint64_t>(u.tiles) * per_seq;
      if (u.seen == 0u && b % gridDim.x == blockIdx.x) {  // nothing to see: zeros
        for (uint32_t i = 0; i < p.heads * HD; i += 4u)
          store4(out + static_cast<size_t>(b) * p.heads * HD + i, make_float4(0.f, 0.f, 0.f, 0.f));
        if (p.lse)
          for (uint32_t h = 0; h < p.heads; ++h) p.lse[static_cast<size_t>(b) * p.heads + h] = -INFINITY;
      }
    }
    own = mine;
    own_upto = total + block_scan(mine, scan_part, sum);
    total += sum;
  }
  if (total == 0u) return;
  // at least a tile per warp for every CTA that takes part
  const uint64_t want = (total + WARPS - 1u) / WARPS;
  const uint64_t ctas = want < gridDim.x ? want : gridDim.x;
  if (blockIdx.x >= ctas) return;
  const uint64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1u) / ctas;
  const auto owner = [&](uint64_t t) { return static_cast<uint32_t>(((t + 1u) * ctas - 1u) / total); };

  // ---- the unit that holds the first tile ----------------------------------
  if (p.c.batch <= kThreads) {
    if (own && begin < own_upto && begin >= own_upto - own) {
      found_b = threadIdx.x;
      found_at = begin - (own_upto - own);
    }
    __syncthreads();
  } else {
    uint64_t base = 0;
    for (uint32_t b0 = 0; b0 < p.c.batch; b0 += kThreads) {
      const uint32_t b = b0 + threadIdx.x;
      uint64_t mine = 0, sum;
      if (b < p.c.batch) {
        Unit u;
        visible(p, sequence(p.c, b, nullptr), u);
        mine = static_cast<uint64_t>(u.tiles) * per_seq;
      }
      const uint64_t upto = base + block_scan(mine, scan_part, sum);
      if (mine && begin < upto && begin >= upto - mine) {
        found_b = b;
        found_at = begin - (upto - mine);
      }
      base += sum;
      if (begin < base) break;
    }
    __syncthreads();
  }
  Unit u;
  u.b = found_b;
  visible(p, sequence(p.c, u.b, nullptr), u);
  u.pr = static_cast<uint32_t>(found_at / u.tiles);
  uint32_t a = static_cast<uint32_t>(found_at % u.tiles);  // first tile of the segment in the unit

  const uint32_t ring = smem_u32(smem) + warp * STAGES * S::kStage;
  bool first_segment = true;
  for (uint64_t t = begin; t < end;) {
    const uint32_t e = static_cast<uint32_t>(min(static_cast<uint64_t>(u.tiles), a + (end - t)));
    const uint32_t kv = u.pr / blocks, head0 = kv * p.group + (u.pr % blocks) * S::kHeads;
    const uint32_t heads = min(S::kHeads, p.group - (u.pr % blocks) * S::kHeads);

    // One tile's rows: lane r < 16 looks position r up, then every lane copies
    // its 16-byte chunks; what lies past the visible positions becomes zeros.
    const auto issue = [&](uint32_t i, uint32_t stage) {
      uint64_t off = 0;
      uint32_t ok = 0;
      const uint32_t at = i * kTile + (lane & 15u);
      if (i < e && at < u.seen) {
        ok = locate(p.c, u.slot, at < u.first ? at : at + u.skip, off) ? 1u : 0u;
        if (!ok) atomicOr(p.err, RTA_DEVERR_PAGE);
        off += static_cast<uint64_t>(kv) * p.c.head_bytes;
      }
      if (i < e) {
        constexpr uint32_t kPer = 32 / S::kChunks;  // rows per warp instruction
        const uint32_t st = ring + stage * S::kStage;
#pragma unroll
        for (uint32_t r0 = 0; r0 < kTile; r0 += kPer) {
          const uint32_t r = r0 + lane / S::kChunks, c = lane % S::kChunks;
          const uint64_t o = __shfl_sync(0xffffffffu, off, r) + c * 16u;
          const bool real = __shfl_sync(0xffffffffu, ok, r) != 0u;
          const uint32_t dst = st + r * S::kRow + ((c ^ (r & 7u)) << 4);
          cp_async16(dst, p.c.k + o, real);
          cp_async16(dst + kTile * S::kRow, p.c.v + o, real);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (uint32_t s = 0; s + 1u < STAGES; ++s) issue(a + warp + s * WARPS, s);

    // Query fragments (A operand: rows are heads, k is the dimension).
    uint32_t qa[kSteps][4];
    {
      const Q* qb = static_cast<const Q*>(p.q) + static_cast<size_t>(u.b) * p.q_row + static_cast<size_t>(head0) * p.q_head;
      const Q* q0 = qb + static_cast<size_t>(g) * p.q_head;
      const Q* q1 = qb + static_cast<size_t>(g + 8u) * p.q_head;
      const bool on0 = g < heads, on1 = !PAIR && g + 8u < heads;
#pragma unroll
      for (uint32_t kk = 0; kk < kSteps; ++kk)
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
          const uint32_t d = kk * 16u + h * 8u + 2u * t4;
          const float x0 = on0 ? load_q<Q>(q0 + d) : 0.f, x1 = on0 ? load_q<Q>(q0 + d + 1u) : 0.f;
          qa[kk][2u * h] = N::pack(x0, x1);
          if (PAIR) {
            if (sizeof(Q) == 4) {
              const float2 hi = N::unpack(qa[kk][2u * h]);
              qa[kk][2u * h + 1u] = N::pack(x0 - hi.x, x1 - hi.y);
            } else {
              qa[kk][2u * h + 1u] = 0u;
            }
          } else {
            qa[kk][2u * h + 1u] = N::pack(on1 ? load_q<Q>(q1 + d) : 0.f, on1 ? load_q<Q>(q1 + d + 1u) : 0.f);
          }
        }
    }

    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    constexpr int kRows = PAIR ? 1 : 2;  // heads of this lane: g (and g + 8)
    float m[kRows], z[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) m[r] = -INFINITY, z[r] = 0.f;

    uint32_t stage = 0;
    for (uint32_t i = a + warp; i < e; i += WARPS) {
      issue(i + (STAGES - 1) * WARPS, stage == 0u ? STAGES - 1u : stage - 1u);
      cp_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t st = ring + stage * S::kStage;
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
      float pr[kRows][2][2], rescale[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float s = sc[0][c][2 * r + x] + sc[1][c][2 * r + x];
            if (PAIR) s += sc[0][c][2 + x] + sc[1][c][2 + x];  // the query's lower half
            s *= p.scale_log2;
            if (i * kTile + c * 8u + 2u * t4 + x >= u.seen) s = -INFINITY;
            pr[r][c][x] = s;
            mx = fmaxf(mx, s);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[r], mx);
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
        for (int j = 0; j < HD / 8; ++j) {
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
      for (uint32_t j = 0; j < HD / 8u; j += 2u) {
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
      stage = stage + 1u == STAGES ? 0u : stage + 1u;
    }
    cp_wait<0>();

    // ---- add the warps of this CTA -----------------------------------------
    __syncthreads();  // every warp is done with the ring
    float* const join = reinterpret_cast<float*>(smem);  // [warp][head][HD]
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      z[r] += __shfl_xor_sync(0xffffffffu, z[r], 1);
      z[r] += __shfl_xor_sync(0xffffffffu, z[r], 2);
      if (t4 == 0u) {
        join_m[warp][g + 8 * r] = m[r];
        join_z[warp][g + 8 * r] = z[r];
      }
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      float* row = join + (warp * S::kHeads + g) * HD + j * 8 + 2u * t4;
      if (PAIR) {
        *reinterpret_cast<float2*>(row) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
      } else {
        *reinterpret_cast<float2*>(row) = make_float2(o[j][0], o[j][1]);
        *reinterpret_cast<float2*>(row + 8 * HD) = make_float2(o[j][2], o[j][3]);
      }
    }
    __syncthreads();
    const uint64_t unit0 = t - a, unit1 = unit0 + u.tiles;  // the unit's tiles in the list
    const bool whole = a == 0u && e == u.tiles;
    float* const rec = p.records + static_cast<size_t>(blockIdx.x * 2u + (first_segment ? 0u : 1u)) * record_floats(HD);
    for (uint32_t i = threadIdx.x; i < heads * (HD / 4); i += kThreads) {
      const uint32_t h = i / (HD / 4), d = i % (HD / 4) * 4u;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, join_m[w][h]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float zz = 0.f;
      float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = exp2f(join_m[w][h] - base);
        const float4 x = *reinterpret_cast<const float4*>(join + (w * S::kHeads + h) * HD + d);
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
    if (!whole) {
      // ---- join the unit's records: the CTA that arrives last ----------------
      const uint32_t c0 = owner(unit0), c1 = owner(unit1 - 1u), parts = c1 - c0 + 1u;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        last_arrival = atomicAdd(&p.counters[c0], 1u) == parts - 1u ? 1u : 0u;
        if (last_arrival) p.counters[c0] = 0u;
      }
      __syncthreads();
      if (last_arrival) {
        __threadfence();
        // a CTA's record of this unit is its second one only when the unit
        // begins inside the CTA's range
        const auto record = [&](uint32_t c) {
          const bool second = c == c0 && total * c0 / ctas != unit0;
          return p.records + static_cast<size_t>(c * 2u + (second ? 1u : 0u)) * record_floats(HD);
        };
        float* const weight = reinterpret_cast<float*>(smem);  // [head][part]
        for (uint32_t h = warp; h < heads; h += WARPS) {
          float mm = -INFINITY, zz = 0.f;
          for (uint32_t j = lane; j < parts; j += 32u) mm = fmaxf(mm, __ldcg(record(c0 + j) + h));
          mm = warp_max(mm);
          const float base = mm == -INFINITY ? 0.f : mm;
          for (uint32_t j = lane; j < parts; j += 32u) {
            const float f = exp2f(__ldcg(record(c0 + j) + h) - base);
            zz += f * __ldcg(record(c0 + j) + kHeadsMax + h);
            weight[h * kMaxCtas + j] = f;
          }
          zz = warp_sum(zz);
          __syncwarp();
          for (uint32_t j = lane; j < parts; j += 32u) weight[h * kMaxCtas + j] /= zz;
          if (p.lse && lane == 0u)
            p.lse[static_cast<size_t>(u.b) * p.heads + head0 + h] = (mm - N::kShift + log2f(zz)) * kLn2;
        }
        // the records' O come through shared memory, as many at a time as fit:
        // all their 16-byte copies are in flight at once
        constexpr uint32_t kWeights = kMaxCtas * kHeadsMax * 4, kEach = (S::kHeads * (HD / 4) + kThreads - 1u) / kThreads;
        float* const stage = reinterpret_cast<float*>(smem + kWeights);
        const uint32_t quads = heads * (HD / 4), fit = min(parts, (S::kSmem - kWeights) / (quads * 16u));
        float4 oo[kEach];
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k) oo[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t j0 = 0; j0 < parts; j0 += fit) {
          const uint32_t n = min(fit, parts - j0);
          __syncthreads();  // the weights are there; the copies before have been used
          for (uint32_t j = 0; j < n; ++j) {
            const float* from = record(c0 + j0 + j) + kRecHeader;
            for (uint32_t i = threadIdx.x; i < quads; i += kThreads)
              cp_async16(smem_u32(stage + (j * quads + i) * 4u), from + i * 4u, true);
          }
          cp_commit();
          cp_wait<0>();
          __syncthreads();
#pragma unroll
          for (uint32_t k = 0; k < kEach; ++k) {
            const uint32_t i = k * kThreads + threadIdx.x;
            if (i < quads) {
              const uint32_t h = i / (HD / 4);
              for (uint32_t j = 0; j < n; ++j) {
                const float f = weight[h * kMaxCtas + j0 + j];
                const float4 x = *reinterpret_cast<const float4*>(stage + (j * quads + i) * 4u);
                oo[k].x += x.x * f;
                oo[k].y += x.y * f;
                oo[k].z += x.z * f;
                oo[k].w += x.w * f;
              }
            }
          }
        }
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k) {
          const uint32_t i = k * kThreads + threadIdx.x;
          if (i < quads)
            store4(out + (static_cast<size_t>(u.b) * p.heads + head0 + i / (HD / 4)) * HD + i % (HD / 4) * 4u, oo[k]);
        }
      }
    }
    __syncthreads();  // the ring is free again
    first_segment = false;
    t += e - a;
    a = 0;
    if (t < end && ++u.pr == per_seq) {
      u.pr = 0;
      do visible(p, sequence(p.c, ++u.b, nullptr), u);
      while (u.tiles == 0u);
    }
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
  const uint32_t ctas = static_cast<uint32_t>(sms) < kMaxCtas ? static_cast<uint32_t>(sms) : kMaxCtas;
  return launch_early(decode_kernel<T, Q, HD, WARPS, STAGES, PAIR>, dim3(ctas), dim3(WARPS * 32), smem, s, p);
}

template <typename T, typename Q, bool PAIR>
cudaError_t by_dim(const AttendParams& p, cudaStream_t s) {
  switch (p.c.head_dim) {
    case 64: return launch<T, Q, 64, 8, 6, PAIR>(p, s);
    case 128: return launch<T, Q, 128, 8, 3, PAIR>(p, s);
    default: return launch<T, Q, 256, 4, 3, PAIR>(p, s);
  }
}

}  // namespace

size_t decode_record_bytes() { return static_cast<size_t>(kMaxCtas) * 2u * record_floats(256) * 4u; }

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
