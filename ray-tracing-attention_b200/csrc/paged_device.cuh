// paged_device.cuh -- device code shared by the paged K/V cache kernels:
// visibility, page lookup, 16-byte asynchronous copies and the fp16 / bf16
// tensor-core fragments.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace rta {
namespace paged {

constexpr float kLn2 = 0.6931471805599453f;

// Positions of one sequence: slot and length, checked against the map.
struct Sequence {
  uint32_t slot, length;
};
__device__ __forceinline__ Sequence sequence(const View& c, uint32_t b, uint32_t* err) {
  Sequence s;
  const int32_t slot = c.slots ? c.slots[b] : static_cast<int32_t>(b);
  s.slot = 0u;
  s.length = 0u;
  if (slot < 0 || static_cast<uint32_t>(slot) >= c.slot_count) {
    if (err) atomicOr(err, RTA_DEVERR_SLOT);
    return s;
  }
  s.slot = static_cast<uint32_t>(slot);
  const int32_t n = c.lengths[s.slot];
  const uint32_t room = c.width * c.page_size;  // < 2^31, checked on the host
  if (n < 0 || static_cast<uint32_t>(n) > room) {
    if (err) atomicOr(err, RTA_DEVERR_SLOT);
    return s;
  }
  s.length = static_cast<uint32_t>(n);
  return s;
}

__device__ __forceinline__ uint32_t page_of(const View& c, uint32_t p) {
  return (__umulhi(p, c.div_mul) + p) >> c.div_shift;
}

// Byte offset of (position, kv head 0) from k / v; false when the table entry
// is not a page of the pool.
__device__ __forceinline__ bool locate(const View& c, uint32_t slot, uint32_t p, uint64_t& offset) {
  const uint32_t j = page_of(c, p);
  const int32_t page = c.table[static_cast<size_t>(slot) * c.width + j];
  if (static_cast<uint32_t>(page) >= c.pages) return false;
  offset = static_cast<uint64_t>(static_cast<uint32_t>(page)) * c.page_bytes +
           static_cast<uint64_t>(p - j * c.page_size) * c.pos_bytes;
  return true;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  const uint32_t n = real ? 16u : 0u;  // 0: the 16 bytes become zeros, src is not read
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
struct Num;
template <>
struct Num<__half> {
  // The decode's weights are pairs (hi, lo) of exp2(score - reference) 2^kShift,
  // the sum carries the same factor: a pair is exact to 2^-22 from 2^-3 on and a
  // multiple of 2^-24 below, and ends at 2^16.  A tile whose largest score is more
  // than kFar below the reference takes its own as the new one, unless it is
  // kNothing below the largest of all (a part of 2^-56 or less, and o and z stay
  // within fp32 for 2^31 positions).  Behind a first token that scores 18 nats
  // above 120 others and holds zeros, fp32 results were 3.5e-4 off with shift 10
  // and no kFar, now 1e-5.
  static constexpr float kShift = 15.f, kFar = 12.f, kNothing = 56.f;
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Num<__nv_bfloat16> {
  // bf16 has fp32's exponents, and so have its values: weights of 2^-44 at most
  // leave room for the sum of 2^31 of the largest.
  static constexpr float kShift = -44.f, kFar = 0.f, kNothing = 0.f;
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Inclusive sum over the block's threads; `part` holds one word per warp.
// Every thread of the block calls it; total receives the block's sum.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= static_cast<uint32_t>(d)) v += o;
  }
  __syncthreads();  // part may still be read by the call before
  if (lane == 31u) part[warp] = v;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
  for (uint32_t w = 0; w < warps; ++w) {
    const uint64_t x = part[w];
    if (w < warp) before += x;
    total += x;
  }
  return v + before;
}

// Rows first .. of the call that belong to sequence b: starts[b], and how many.
// Offsets that do not ascend inside 0 .. rows are flagged and give no rows; rows
// that belong to no sequence are flagged.
__device__ __forceinline__ uint32_t new_rows(const AttendParams& p, uint32_t b, uint32_t& first, uint32_t* err) {
  const int32_t a = p.starts[b], e = p.starts[b + 1u];
  first = 0u;
  if (a < 0 || e < a || static_cast<uint32_t>(e) > p.rows) {
    if (err) atomicOr(err, RTA_DEVERR_SLOT);
    return 0u;
  }
  if (err && ((b == 0u && a != 0) || (b + 1u == p.c.batch && static_cast<uint32_t>(e) != p.rows)))
    atomicOr(err, RTA_DEVERR_SLOT);
  first = static_cast<uint32_t>(a);
  return static_cast<uint32_t>(e - a);
}

// ---- one row by itself ------------------------------------------------------
// A matrix product multiplies the values of masked positions by a weight of
// zero, and 0 * inf and 0 * NaN are NaN.  A row whose result is not finite is
// therefore looked at again: if a position that its tile read but the row does
// not see (of [sinks, firsts) and [low, high)) holds a non-finite value, the row
// is computed over its visible positions alone.  Both run on one full warp; a
// lane owns HD / 32 neighbouring dimensions.
template <typename T, int HD>
__device__ __forceinline__ void load_dims(const void* row, uint32_t lane, float (&x)[HD / 32]) {
  const T* r = static_cast<const T*>(row) + lane * (HD / 32);
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) x[i] = Num<T>::to(r[i]);
}

template <typename T, int HD>
__device__ bool spoiled(const AttendParams& p, uint32_t slot, uint32_t kv, uint32_t firsts, uint32_t low, uint32_t high,
                        uint32_t t) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t mine = p.window && t >= p.window ? t - p.window + 1u : 0u;  // the row's window: mine .. t
  bool bad = false;
  for (uint32_t x = p.sinks < firsts ? p.sinks : low; x < high; ++x) {
    if (x >= firsts && x < low) x = low;
    if (x <= t && (x >= mine || x < p.sinks)) {
      x = x < mine ? x : t;  // visible: go on behind it
      continue;
    }
    uint64_t off;
    if (!locate(p.c, slot, x, off)) continue;
    float v[HD / 32];
    load_dims<T, HD>(p.c.v + off + static_cast<uint64_t>(kv) * p.c.head_bytes, lane, v);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) bad |= !isfinite(v[i]);
  }
  return __any_sync(0xffffffffu, bad);
}

template <typename T, int HD>
__device__ void row_alone(const AttendParams& p, uint32_t slot, uint32_t kv, uint32_t head, uint32_t row, uint32_t t) {
  const uint32_t lane = threadIdx.x & 31u;
  constexpr int E = HD / 32;
  float q[E], k[E], v[E], o[E];
  load_dims<T, HD>(static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head, lane, q);
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  float m = -INFINITY, z = 0.f;
  const uint32_t mine = p.window && t >= p.window ? t - p.window + 1u : 0u;
  for (uint32_t x = 0; x <= t; ++x) {
    if (x < mine && x >= p.sinks) x = mine;
    uint64_t off;
    if (!locate(p.c, slot, x, off)) continue;
    off += static_cast<uint64_t>(kv) * p.c.head_bytes;
    load_dims<T, HD>(p.c.k + off, lane, k);
    load_dims<T, HD>(p.c.v + off, lane, v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += q[i] * k[i];
    s = warp_sum(s) * p.scale_log2;
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = m == mn ? 1.f : exp2f(m - base), w = exp2f(s - (base - Num<T>::kShift));
    z = z * f + w;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * f + w * v[i];
    m = mn;
  }
  const size_t at = static_cast<size_t>(row) * p.heads + head;
  T* out = static_cast<T*>(p.out) + at * HD + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) out[i] = Num<T>::from(o[i] / z);
  if (p.lse && lane == 0u) p.lse[at] = (m - Num<T>::kShift + log2f(z)) * kLn2;
}

}  // namespace paged
}  // namespace rta
