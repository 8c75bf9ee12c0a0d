// paged.h -- parameters of the paged K/V cache kernels (paged_decode.cu,
// paged_prefill.cu, pages.cu) and their workspace.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "rta_internal.h"

namespace rta {
namespace paged {

// A launch that may begin under the kernel before it: every kernel of the paged
// cache waits (griddepcontrol.wait) before it touches memory, so only the launch
// itself overlaps.
template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// CTAs of an attention launch at most (one per SM in the prefill, up to two in
// the decode): bounds the split records.
constexpr uint32_t kMaxCtas = 160, kMaxDecodeCtas = 320;

// Where position p of a sequence lives.  page_size is any number, so p /
// page_size is a multiply and a shift (exact for p < 2^31).
struct View {
  const uint8_t* k;  // base of the call's layer
  const uint8_t* v;
  uint64_t page_bytes, head_bytes, pos_bytes;  // strides in bytes
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* slots;  // null: 0 .. batch - 1
  uint32_t slot_count, width, pages, page_size, div_mul, div_shift;
  uint32_t batch, kv_heads, head_dim;
};

struct AttendParams {
  View c;
  const void* q;
  uint64_t q_row, q_head;  // strides in elements
  const int32_t* starts;   // prefill: batch + 1 row offsets
  uint32_t rows;           // prefill: rows of the call
  uint32_t heads, group;   // query heads, query heads per K/V head
  float scale_log2;        // scale * log2(e): the softmax runs in base 2
  uint32_t window, sinks;
  uint32_t align;  // prefill: reads begin at multiples of this many positions
  void* out;
  float* lse;
  uint32_t* err;
  void* cuts;  // [kMaxDecodeCtas, the larger of the two] what the second launch has to know, kCutBytes each
  float* records;
};
constexpr uint32_t kCutBytes = 64;

// q: the queries' format (kF32, kF16 or kBF16); fmt: the pool's.
cudaError_t launch_decode(const AttendParams& p, int fmt, int q, cudaStream_t s);
cudaError_t launch_prefill(const AttendParams& p, int fmt, cudaStream_t s);
size_t decode_record_bytes();
size_t prefill_record_bytes();

struct AppendParams {
  View c;
  const int32_t* starts;
  uint32_t rows;
  const void* k;
  const void* v;
  uint64_t row_stride, head_stride;  // elements
  uint32_t* err;
  uint32_t block_rows;  // set by the launch
};
cudaError_t launch_append(const AppendParams& p, int fmt, int in_fmt, cudaStream_t s);

struct MapArrays {
  int32_t* refs;
  int32_t* table;
  int32_t* lengths;
};
struct PagesParams {
  MapArrays map;   // updated in place
  MapArrays from;  // copied into it first, where refs is not null
  uint32_t slot_count, width, pages, page_size;
  uint8_t* k;
  uint8_t* v;
  uint64_t layer_bytes, page_bytes, head_bytes, pos_bytes;
  uint32_t layers, kv_heads, row_bytes;
  const int32_t* a;  // slots / src
  const int32_t* b;  // counts / dst
  uint32_t count;
  uint32_t* live;
  uint32_t* err;
  uint32_t* plan;  // scratch words: see pages.cu
};
size_t plan_bytes(uint32_t pages, uint32_t slots);
bool plan_copies(uint32_t pages, uint32_t slots, uint32_t width);  // whether a plan copies a map of this size itself
cudaError_t launch_map_copy(const MapArrays& from, const MapArrays& to, uint32_t pages, uint32_t slots,
                            uint32_t width, cudaStream_t s);
cudaError_t launch_reserve(const PagesParams& p, cudaStream_t s);
cudaError_t launch_fork(const PagesParams& p, cudaStream_t s);
cudaError_t launch_free(const PagesParams& p, cudaStream_t s);
cudaError_t launch_compact(const PagesParams& p, cudaStream_t s);
cudaError_t launch_copy(const PagesParams& p, cudaStream_t s);

}  // namespace paged
}  // namespace rta
