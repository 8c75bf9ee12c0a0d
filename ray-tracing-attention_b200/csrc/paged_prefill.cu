// paged_prefill.cu -- attention of many new tokens per sequence over a paged
// K/V cache, causal, with a window and first tokens that stay visible.
//
// The query heads that share a K/V head are rows of one matrix: row R of a
// sequence and K/V head is query R / group, head R % group, so a tile of rows
// reads the K/V head once for all of them.  The positions a tile needs are the
// first tokens, then a run of neighbours; they are numbered without the gap.
#include <atomic>
#include <mutex>

#include "paged_device.cuh"

namespace rta {
namespace paged {
namespace {

constexpr uint32_t kRows = 64;  // rows per CTA, sixteen per warp
constexpr uint32_t kKeys = 32;  // positions per step

template <typename T, int HD>
__global__ void __launch_bounds__(128, 1) prefill_kernel(const AttendParams p) {
  using N = Num<T>;
  constexpr uint32_t kRow = HD * 2, kChunks = kRow / 16, kSteps = HD / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t scan_part[4];
  __shared__ uint32_t found_b, found_tile;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t4 = lane & 3u;
  const uint32_t kv = blockIdx.y;
  if (threadIdx.x == 0) found_b = 0xffffffffu;
  uint64_t base = 0;
  for (uint32_t b0 = 0; b0 < p.c.batch; b0 += 128u) {
    const uint32_t b = b0 + threadIdx.x;
    uint64_t mine = 0, sum;
    uint32_t first;
    if (b < p.c.batch)
      mine = (static_cast<uint64_t>(new_rows(p, b, first, blockIdx.x + blockIdx.y == 0u ? p.err : nullptr)) * p.group + kRows - 1u) / kRows;
    const uint64_t upto = base + block_scan(mine, scan_part, sum);
    if (mine && blockIdx.x < upto && blockIdx.x >= upto - mine) {
      found_b = b;
      found_tile = static_cast<uint32_t>(blockIdx.x - (upto - mine));
    }
    base += sum;
  }
  __syncthreads();
  const uint32_t b = found_b;
  if (b == 0xffffffffu) return;
  uint32_t first_row;
  const uint32_t count = new_rows(p, b, first_row, nullptr);
  const Sequence seq = sequence(p.c, b, blockIdx.y == 0u ? p.err : nullptr);
  const int64_t past = static_cast<int64_t>(seq.length) - count;  // position of row 0 of the sequence
  const uint32_t R0 = found_tile * kRows, R1 = min(R0 + kRows, count * p.group);
  const int64_t t0 = past + R0 / p.group, t1 = past + (R1 - 1u) / p.group;  // positions of the tile's queries
  const uint32_t ta = t0 > 0 ? static_cast<uint32_t>(t0) : 0u;
  const uint32_t low = p.window && ta >= p.window ? ta - p.window + 1u : 0u;
  const uint32_t firsts = min(p.sinks, low), skip = low - firsts;
  const uint32_t seen = t1 < 0 ? 0u : static_cast<uint32_t>(t1) + 1u - skip;

  int64_t t_row[2];
  uint32_t at_row[2], head_row[2];
  bool real[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint32_t R = R0 + warp * 16u + g + 8u * r;
    real[r] = R < R1;
    t_row[r] = real[r] ? past + R / p.group : -1;
    at_row[r] = first_row + (real[r] ? R / p.group : 0u);
    head_row[r] = kv * p.group + R % p.group;
  }
  uint32_t qa[kSteps][4];
#pragma unroll
  for (uint32_t kk = 0; kk < kSteps; ++kk)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        qa[kk][2 * h + r] = real[r] ? *reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + at_row[r] * p.q_row + head_row[r] * p.q_head + kk * 16u + h * 8u + 2u * t4) : 0u;
  float o[HD / 8][4];
#pragma unroll
  for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, z[2] = {0.f, 0.f};
  const uint32_t ks = smem_u32(smem), vs = ks + kKeys * kRow;
  for (uint32_t u0 = 0; u0 < seen; u0 += kKeys) {
    for (uint32_t i = threadIdx.x; i < kKeys * kChunks; i += 128u) {
      const uint32_t r = i / kChunks, c = i % kChunks, u = u0 + r;
      uint64_t off = 0;
      bool ok = false;
      if (u < seen) {
        ok = locate(p.c, seq.slot, u < firsts ? u : u + skip, off);
        if (!ok) atomicOr(p.err, RTA_DEVERR_PAGE);
        off += kv * p.c.head_bytes + c * 16u;
      }
      const uint32_t dst = r * kRow + ((c ^ (r & 7u)) << 4);
      cp_async16(ks + dst, p.c.k + off, ok);
      cp_async16(vs + dst, p.c.v + off, ok);
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    float sc[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < static_cast<int>(kKeys / 8); ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
    for (uint32_t kk = 0; kk < kSteps; ++kk)
#pragma unroll
      for (uint32_t n = 0; n < kKeys / 16; ++n) {
        uint32_t f[4];
        const uint32_t r = n * 16u + (lane & 7u) + ((lane >> 4) << 3), c = 2u * kk + ((lane >> 3) & 1u);
        ldsm4(ks + r * kRow + ((c ^ (r & 7u)) << 4), f);
        N::mma(sc[2 * n], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], f[0], f[1]);
        N::mma(sc[2 * n + 1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], f[2], f[3]);
      }
    float scale[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < static_cast<int>(kKeys / 8); ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t u = u0 + n * 8u + 2u * t4 + x;
          const int64_t at = u < firsts ? u : static_cast<int64_t>(u) + skip;
          float& s = sc[n][2 * r + x];
          s *= p.scale_log2;
          const bool see = u < seen && at <= t_row[r] && (!p.window || at > t_row[r] - p.window || at < p.sinks);
          if (!see) s = -INFINITY;
          mx = fmaxf(mx, s);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[r], mx), bs = mn == -INFINITY ? 0.f : mn;
      scale[r] = m[r] == mn ? 1.f : exp2f(m[r] - bs);
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < static_cast<int>(kKeys / 8); ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) sum += sc[n][2 * r + x] = exp2f(sc[n][2 * r + x] - (bs - N::kShift));
      z[r] = z[r] * scale[r] + sum;
      m[r] = mn;
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      o[j][0] *= scale[0];
      o[j][1] *= scale[0];
      o[j][2] *= scale[1];
      o[j][3] *= scale[1];
    }
#pragma unroll
    for (uint32_t n = 0; n < kKeys / 16; ++n) {
      const uint32_t a0 = N::pack(sc[2 * n][0], sc[2 * n][1]), a1 = N::pack(sc[2 * n][2], sc[2 * n][3]);
      const uint32_t a2 = N::pack(sc[2 * n + 1][0], sc[2 * n + 1][1]), a3 = N::pack(sc[2 * n + 1][2], sc[2 * n + 1][3]);
#pragma unroll
      for (uint32_t j = 0; j < HD / 8u; j += 2u) {
        uint32_t f[4];
        const uint32_t r = n * 16u + (lane & 7u) + (((lane >> 3) & 1u) << 3), c = j + (lane >> 4);
        ldsm4_t(vs + r * kRow + ((c ^ (r & 7u)) << 4), f);
        N::mma(o[j], a0, a1, a2, a3, f[0], f[1]);
        N::mma(o[j + 1], a0, a1, a2, a3, f[2], f[3]);
      }
    }
    __syncthreads();
  }
  uint32_t again[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    z[r] += __shfl_xor_sync(0xffffffffu, z[r], 1);
    z[r] += __shfl_xor_sync(0xffffffffu, z[r], 2);
    const float inv = t_row[r] < 0 ? 0.f : 1.f / z[r];
    bool bad = false;
    const size_t at = static_cast<size_t>(at_row[r]) * p.heads + head_row[r];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      const float x = t_row[r] < 0 ? 0.f : o[j][2 * r] * inv, y = t_row[r] < 0 ? 0.f : o[j][2 * r + 1] * inv;
      bad |= !isfinite(x) || !isfinite(y);
      if (real[r]) *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + at * HD + j * 8 + 2u * t4) = N::pack(x, y);
    }
    if (real[r] && p.lse && t4 == 0u) p.lse[at] = t_row[r] < 0 ? -INFINITY : (m[r] - N::kShift + log2f(z[r])) * kLn2;
    again[r] = __ballot_sync(0xffffffffu, bad && real[r]);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r)
    for (uint32_t x = 0; x < 8u; ++x) {
      if (!(again[r] >> (4u * x) & 15u)) continue;
      const uint32_t R = R0 + warp * 16u + x + 8u * r;
      const uint32_t t = static_cast<uint32_t>(past + R / p.group);
      if (spoiled<T, HD>(p, seq.slot, kv, low, static_cast<uint32_t>(t1) + 1u, t))
        row_alone<T, HD>(p, seq.slot, kv, kv * p.group + R % p.group, first_row + R / p.group, t);
    }
}

template <typename T, int HD>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  constexpr uint32_t smem = 2 * kKeys * HD * 2;
  const uint64_t tiles = (static_cast<uint64_t>(p.rows) * p.group + kRows - 1u) / kRows + p.c.batch;
  prefill_kernel<T, HD><<<dim3(static_cast<uint32_t>(tiles), p.c.kv_heads), 128, smem, s>>>(p);
  return cudaGetLastError();
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

size_t prefill_record_bytes() { return static_cast<size_t>(kMaxCtas) * 2u * 256u * (128u + 2u) * 4u; }

cudaError_t launch_prefill(const AttendParams& p, int fmt, cudaStream_t s) {
  return fmt == kF16 ? by_dim<__half>(p, s) : by_dim<__nv_bfloat16>(p, s);
}

}  // namespace paged
}  // namespace rta
