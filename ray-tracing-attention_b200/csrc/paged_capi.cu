// paged_capi.cu -- extern "C" entry points of the paged K/V cache (rta.h,
// section 1c): argument checks, the workspace's layout, status codes.
#include <cmath>
#include <string>

#include "../../include/rta.h"
#include "paged.h"

namespace {

using namespace rta;

rta_status refuse(const char* fn, const std::string& why) {
  set_last_error(std::string(fn) + ": " + why);
  return RTA_E_ARG;
}
rta_status status(cudaError_t e, const char* fn) {
  if (e == cudaSuccess) return RTA_OK;
  set_last_error(std::string(fn) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
  return RTA_E_CUDA;
}
bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

const char* bad_pool(const rta_page_pool* p) {
  if (!p || !p->k || !p->v) return "null pool";
  if (p->format != RTA_F16 && p->format != RTA_BF16) return "the pool's format is RTA_F16 or RTA_BF16";
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return "head_dim is 64, 128 or 256";
  if (!p->layers || !p->pages || p->pages > 0x7fffffffu || !p->kv_heads || p->kv_heads > 1024u || !p->page_size ||
      p->page_size > 65536u)
    return "layers >= 1, 1 <= pages < 2^31, 1 <= kv_heads <= 1024, 1 <= page_size <= 65536";
  if (p->layer_stride % 8 || p->page_stride % 8 || p->head_stride % 8 || p->position_stride % 8)
    return "the pool's strides are multiples of 8 elements";
  if (!aligned(p->k, 16) || !aligned(p->v, 16)) return "k and v must be 16-byte aligned";
  return nullptr;
}
const char* bad_batch(const rta_page_map* m, const int32_t* slots, uint32_t batch) {
  if (batch == 0 || batch > (slots ? 0x7fffffffu : m->slots))
    return "batch is at least 1, at most the slots without a slot list, and below 2^31";
  return nullptr;
}
const char* bad_map(const rta_page_pool* p, const rta_page_map* m) {
  if (!m || !m->refs || !m->table || !m->lengths) return "null map";
  if (!m->slots || m->slots > 0x7fffffffu || !m->width) return "slots and width are at least 1";
  if (static_cast<uint64_t>(m->width) * p->page_size >= (1ull << 31)) return "width * page_size must be below 2^31";
  return nullptr;
}

// Workspace: error word and padding, the descriptions of cut units, then either
// their records (an attention call) or the plan of a bookkeeping call.
constexpr size_t kErr = 256, kCuts = (paged::kMaxDecodeCtas * paged::kCutBytes + 255u) / 256u * 256u, kBody = kErr + kCuts;
size_t workspace_bytes_of(const rta_page_pool* p, const rta_page_map* m) {
  size_t body = paged::decode_record_bytes();
  if (paged::prefill_record_bytes() > body) body = paged::prefill_record_bytes();
  const size_t plan = paged::plan_bytes(p->pages, m->slots);
  return kBody + (plan > body ? plan : body);
}
const char* bad_workspace(const rta_page_pool* p, const rta_page_map* m, const void* ws, size_t bytes) {
  if (!ws || !aligned(ws, 16)) return "the workspace must be 16-byte aligned";
  if (bytes < workspace_bytes_of(p, m)) return "workspace too small";
  return nullptr;
}

size_t element(int format) { return format == RTA_F32 ? 4u : 2u; }

// x / d = (umulhi(x, mul) + x) >> shift for x < 2^31: mul = floor(2^32 (2^shift - d) / d) + 1, shift = ceil(log2 d)
void divide(uint32_t d, uint32_t& mul, uint32_t& shift) {
  shift = 0;
  while ((1u << shift) < d) ++shift;
  mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1u);
}

paged::View view(const rta_page_pool* p, const rta_page_map* m, uint32_t layer, const int32_t* slots, uint32_t batch) {
  paged::View v;
  v.k = static_cast<const uint8_t*>(p->k) + layer * p->layer_stride * 2u;
  v.v = static_cast<const uint8_t*>(p->v) + layer * p->layer_stride * 2u;
  v.page_bytes = p->page_stride * 2u;
  v.head_bytes = p->head_stride * 2u;
  v.pos_bytes = p->position_stride * 2u;
  v.table = m->table;
  v.lengths = m->lengths;
  v.slots = slots;
  v.slot_count = m->slots;
  v.width = m->width;
  v.pages = p->pages;
  v.page_size = p->page_size;
  divide(p->page_size, v.div_mul, v.div_shift);
  v.batch = batch;
  v.kv_heads = p->kv_heads;
  v.head_dim = p->head_dim;
  return v;
}

struct Workspace {
  uint32_t* err;
  void *cuts, *body;
  explicit Workspace(void* ws)
      : err(static_cast<uint32_t*>(ws)),
        cuts(static_cast<uint8_t*>(ws) + kErr),
        body(static_cast<uint8_t*>(ws) + kBody) {}
};

const char* attend_params(const rta_page_pool* pool, const rta_page_map* map, uint32_t layer, const int32_t* slots,
                          uint32_t batch, const void* q, int q_format, uint32_t heads, uint64_t q_row, uint64_t q_head,
                          float scale, uint32_t window, uint32_t sinks, void* out, float* lse, void* ws,
                          size_t ws_bytes, bool allow_f32, paged::AttendParams& p) {
  const char* why = bad_pool(pool);
  if (!why) why = bad_map(pool, map);
  if (!why) why = bad_workspace(pool, map, ws, ws_bytes);
  if (why) return why;
  if (layer >= pool->layers) return "no such layer";
  if (const char* bad = bad_batch(map, slots, batch)) return bad;
  if (!q || !out) return "null q or out";
  if (heads == 0 || heads % pool->kv_heads || heads / pool->kv_heads > 128u)
    return "heads is a multiple of kv_heads, at most 128 query heads per K/V head";
  if (q_format != pool->format && !(allow_f32 && q_format == RTA_F32 && pool->format == RTA_F16))
    return allow_f32 ? "q is in the pool's format, or fp32 with an fp16 pool" : "q is in the pool's format";
  const size_t unit = 16u / element(q_format);
  if (!aligned(q, 16) || q_row % unit || q_head % unit) return "q's rows must be 16-byte aligned";
  if (!aligned(out, 16)) return "out must be 16-byte aligned";
  if (lse && !aligned(lse, 4)) return "lse must be 4-byte aligned";
  if (!std::isfinite(scale * 1.4426950408889634f)) return "scale (and scale * log2 e) must be finite";
  const Workspace w(ws);
  p.c = view(pool, map, layer, slots, batch);
  p.q = q;
  p.q_row = q_row;
  p.q_head = q_head;
  p.heads = heads;
  p.group = heads / pool->kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.window = window;
  p.sinks = sinks;
  p.align = 1;
  p.out = out;
  p.lse = lse;
  p.err = w.err;
  p.cuts = w.cuts;
  p.records = static_cast<float*>(w.body);
  p.starts = nullptr;
  p.rows = batch;
  return nullptr;
}

bool same_map(const rta_page_map* a, const rta_page_map* b) {
  return a->refs == b->refs && a->table == b->table && a->lengths == b->lengths;
}

// Checks a bookkeeping call, fills its parameters, and has map copied to out when
// they are two maps: by a launch, by the call's plan where that can, or by the call.
enum Copies { kByLaunch, kByPlan, kByCall };
rta_status pages_params(const char* fn, Copies by, const rta_page_pool* pool, const rta_page_map* map, const rta_page_map* out,
                        uint32_t count, void* ws, size_t ws_bytes, cudaStream_t s, paged::PagesParams& p) {
  const char* why = bad_pool(pool);
  if (!why) why = bad_map(pool, map);
  if (!why) why = bad_map(pool, out);
  if (!why) why = bad_workspace(pool, map, ws, ws_bytes);
  if (!why && (out->slots != map->slots || out->width != map->width)) why = "map and out differ in slots or width";
  if (!why && !same_map(map, out) &&
      (map->refs == out->refs || map->table == out->table || map->lengths == out->lengths))
    why = "out is the map itself or has arrays of its own";
  if (!why && count > map->slots) why = "more sequences than slots";
  if (why) return refuse(fn, why);
  const Workspace w(ws);
  p.map = {out->refs, out->table, out->lengths};
  p.from = {nullptr, nullptr, nullptr};
  p.slot_count = map->slots;
  p.width = map->width;
  p.pages = pool->pages;
  p.page_size = pool->page_size;
  p.k = static_cast<uint8_t*>(pool->k);
  p.v = static_cast<uint8_t*>(pool->v);
  p.layer_bytes = pool->layer_stride * 2u;
  p.page_bytes = pool->page_stride * 2u;
  p.head_bytes = pool->head_stride * 2u;
  p.pos_bytes = pool->position_stride * 2u;
  p.layers = pool->layers;
  p.kv_heads = pool->kv_heads;
  p.row_bytes = pool->head_dim * 2u;
  p.a = p.b = nullptr;
  p.count = count;
  p.live = nullptr;
  p.err = w.err;
  p.plan = static_cast<uint32_t*>(w.body);
  if (same_map(map, out)) return RTA_OK;
  if (by == kByCall || (by == kByPlan && paged::plan_copies(pool->pages, map->slots, map->width))) {
    p.from = {map->refs, map->table, map->lengths};
    return RTA_OK;
  }
  return status(paged::launch_map_copy({map->refs, map->table, map->lengths}, p.map, pool->pages, map->slots,
                                       map->width, s),
                fn);
}

}  // namespace

extern "C" {

size_t rta_paged_workspace_bytes(const rta_page_pool* pool, const rta_page_map* map) {
  if (bad_pool(pool) || !map) return 0;
  return workspace_bytes_of(pool, map);
}

rta_status rta_paged_decode(const rta_page_pool* pool, const rta_page_map* map, uint32_t layer, const int32_t* slots,
                            uint32_t batch, const void* q, int q_format, uint32_t heads, uint64_t q_row_stride,
                            uint64_t q_head_stride, float scale, uint32_t window, uint32_t sinks, void* out, float* lse,
                            void* workspace, size_t workspace_bytes, void* stream) {
  paged::AttendParams p;
  const char* why = attend_params(pool, map, layer, slots, batch, q, q_format, heads, q_row_stride, q_head_stride,
                                  scale, window, sinks, out, lse, workspace, workspace_bytes, true, p);
  if (why) return refuse("rta_paged_decode", why);
  return status(paged::launch_decode(p, pool->format, q_format, static_cast<cudaStream_t>(stream)), "rta_paged_decode");
}

rta_status rta_paged_prefill(const rta_page_pool* pool, const rta_page_map* map, uint32_t layer, const int32_t* slots,
                             uint32_t batch, const int32_t* starts, uint32_t rows, const void* q, int q_format,
                             uint32_t heads, uint64_t q_row_stride, uint64_t q_head_stride, float scale,
                             uint32_t window, uint32_t sinks, void* out, float* lse, void* workspace,
                             size_t workspace_bytes, void* stream) {
  paged::AttendParams p;
  const char* why = attend_params(pool, map, layer, slots, batch, q, q_format, heads, q_row_stride, q_head_stride,
                                  scale, window, sinks, out, lse, workspace, workspace_bytes, false, p);
  if (!why && !starts) why = "null starts";
  if (!why && !aligned(out, 32)) why = "out must be 32-byte aligned";
  if (!why && (rows == 0 || static_cast<uint64_t>(rows) * heads >= (1ull << 31))) why = "rows is at least 1, rows * heads below 2^31";
  if (why) return refuse("rta_paged_prefill", why);
  p.starts = starts;
  p.rows = rows;
  return status(paged::launch_prefill(p, pool->format, static_cast<cudaStream_t>(stream)), "rta_paged_prefill");
}

rta_status rta_paged_append(const rta_page_pool* pool, const rta_page_map* map, uint32_t layer, const int32_t* slots,
                            uint32_t batch, const int32_t* starts, uint32_t rows, const void* k, const void* v,
                            int format, uint64_t row_stride, uint64_t head_stride, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* why = bad_pool(pool);
  if (!why) why = bad_map(pool, map);
  if (!why) why = bad_workspace(pool, map, workspace, workspace_bytes);
  if (!why && layer >= pool->layers) why = "no such layer";
  if (!why) why = bad_batch(map, slots, batch);
  if (!why && (!starts || !k || !v)) why = "null argument";
  if (!why && format != pool->format && format != RTA_F32) why = "the rows are fp32 or in the pool's format";
  if (!why) {
    const size_t unit = 16u / element(format);
    if (!aligned(k, 16) || !aligned(v, 16) || row_stride % unit || head_stride % unit)
      why = "k's and v's rows must be 16-byte aligned";
  }
  if (!why && rows > 0x7fffffffu) why = "rows is below 2^31";
  if (why) return refuse("rta_paged_append", why);
  paged::AppendParams p;
  p.c = view(pool, map, layer, slots, batch);
  p.starts = starts;
  p.rows = rows;
  p.k = k;
  p.v = v;
  p.row_stride = row_stride;
  p.head_stride = head_stride;
  p.err = Workspace(workspace).err;
  return status(paged::launch_append(p, pool->format, format, static_cast<cudaStream_t>(stream)), "rta_paged_append");
}

rta_status rta_pages_reserve(const rta_page_pool* pool, const rta_page_map* map, const rta_page_map* out,
                             const int32_t* slots, const int32_t* counts, uint32_t batch, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (!counts || !batch) return refuse("rta_pages_reserve", "null counts or an empty batch");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  paged::PagesParams p;
  const rta_status st = pages_params("rta_pages_reserve", kByPlan, pool, map, out, batch, workspace, workspace_bytes, s, p);
  if (st != RTA_OK) return st;
  p.a = slots;
  p.b = counts;
  return status(paged::launch_reserve(p, s), "rta_pages_reserve");
}

rta_status rta_pages_fork(const rta_page_pool* pool, const rta_page_map* map, const rta_page_map* out,
                          const int32_t* src, const int32_t* dst, uint32_t count, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!src || !dst || !count) return refuse("rta_pages_fork", "null src or dst, or nothing to fork");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  paged::PagesParams p;
  const rta_status st = pages_params("rta_pages_fork", kByPlan, pool, map, out, count, workspace, workspace_bytes, s, p);
  if (st != RTA_OK) return st;
  p.a = src;
  p.b = dst;
  return status(paged::launch_fork(p, s), "rta_pages_fork");
}

rta_status rta_pages_free(const rta_page_pool* pool, const rta_page_map* map, const rta_page_map* out,
                          const int32_t* slots, uint32_t count, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (!slots || !count) return refuse("rta_pages_free", "null slots or nothing to free");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  paged::PagesParams p;
  const rta_status st = pages_params("rta_pages_free", kByLaunch, pool, map, out, count, workspace, workspace_bytes, s, p);
  if (st != RTA_OK) return st;
  p.a = slots;
  return status(paged::launch_free(p, s), "rta_pages_free");
}

rta_status rta_pages_compact(const rta_page_pool* pool, const rta_page_map* map, const rta_page_map* out,
                             uint32_t* live, void* workspace, size_t workspace_bytes, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  paged::PagesParams p;
  const rta_status st = pages_params("rta_pages_compact", kByCall, pool, map, out, 0, workspace, workspace_bytes, s, p);
  if (st != RTA_OK) return st;
  p.live = live;
  return status(paged::launch_compact(p, s), "rta_pages_compact");
}

rta_status rta_pages_copy(const rta_page_pool* pool, const int32_t* src, const int32_t* dst, uint32_t count,
                          void* workspace, size_t workspace_bytes, void* stream) {
  const char* why = bad_pool(pool);
  if (!why && (!src || !dst || !count || count > pool->pages)) why = "null src or dst, or a count outside 1 .. pages";
  if (!why && (!workspace || !aligned(workspace, 16))) why = "the workspace must be 16-byte aligned";
  if (!why && workspace_bytes < kBody + paged::plan_bytes(pool->pages, 1)) why = "workspace too small";
  if (why) return refuse("rta_pages_copy", why);
  const Workspace w(workspace);
  paged::PagesParams p = {};
  p.slot_count = 1;
  p.pages = pool->pages;
  p.page_size = pool->page_size;
  p.k = static_cast<uint8_t*>(pool->k);
  p.v = static_cast<uint8_t*>(pool->v);
  p.layer_bytes = pool->layer_stride * 2u;
  p.page_bytes = pool->page_stride * 2u;
  p.head_bytes = pool->head_stride * 2u;
  p.pos_bytes = pool->position_stride * 2u;
  p.layers = pool->layers;
  p.kv_heads = pool->kv_heads;
  p.row_bytes = pool->head_dim * 2u;
  p.a = src;
  p.b = dst;
  p.count = count;
  p.err = w.err;
  p.plan = static_cast<uint32_t*>(w.body);
  return status(paged::launch_copy(p, static_cast<cudaStream_t>(stream)), "rta_pages_copy");
}

}  // extern "C"
