// The C ABI's ops over a step of many requests (include/frizzle_hip.h): their
// arguments checked, then enqueued on the device's stream with the handle's
// lock held. What lies in device memory (positions, tables, adapters) is
// checked by the kernels, which read and write nothing outside of what the
// arguments describe.

#include <cmath>
#include <string>

#include "backend.h"
#include "batch_rules.h"

namespace frz {
namespace {

constexpr size_t kStateFloats = (size_t)kMostStateValues * rules::kHeadBlock;
constexpr size_t kStatFloats = (size_t)kMostJoinedParts * rules::kHeadBlock * 2;
constexpr size_t kRecords = kMostJoinedParts / 2;
constexpr size_t kAttentionBytes =
    kStateFloats * 4 + kStatFloats * 4 + kRecords * sizeof(uint4) + 16;
constexpr size_t kAdapterBytes =
    (size_t)kMostAdapterSplits * rules::kMostRows * kMostAdapterRank * 4;
constexpr size_t kScratchBytes = kAttentionBytes > kAdapterBytes ? kAttentionBytes : kAdapterBytes;

constexpr int kMostHeads = 1024;
constexpr float kMostScale = 4096.0f;  // 2^13 in log2 units, as the kernel takes

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned_word(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// Enqueues one op with the lock held and the workspace there; nothing throws
// past it.
template <typename Launch>
int enqueue(frz_device* dev, const char* what, Launch launch) {
  try {
    OnDevice on(dev->ordinal);
    if (on.error() != hipSuccess) return check_hip(on.error(), what);
    std::lock_guard<std::mutex> lock(dev->ops);
    if (int rc = device_batch_scratch(dev)) return rc;
    return check_hip(launch(), what);
  } catch (const std::exception& e) {
    return fail(FRZ_ERR_DEVICE, std::string(what) + ": " + e.what());
  }
}

// The refusal's text, or null.
const char* refuse_pages(const frz_pages* c, int query_heads, uint32_t rows) {
  if (!c) return "null cache";
  if (!c->keys || !c->values || !c->table) return "null keys, values or table";
  if (!aligned(c->keys) || !aligned(c->values)) return "keys or values not at a multiple of 16 bytes";
  if (!aligned_word(c->table)) return "table not at a multiple of 4 bytes";
  if (c->format != FRZ_FORMAT_F16 && c->format != FRZ_FORMAT_BF16) return "cache format (F16 1 or BF16 30)";
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim (64, 128 or 256)";
  if (c->kv_heads < 1 || query_heads < 1 || query_heads > kMostHeads || query_heads % c->kv_heads)
    return "heads (query_heads a multiple of kv_heads, at most 1,024)";
  if (c->page_slots < 16 || c->page_slots % 16 || c->page_slots > rules::kMostKeys)
    return "page_slots (a multiple of 16)";
  if (c->sequences < 1 || c->pages < 1 || c->pages == FRZ_NO_PAGE) return "no sequences or pages";
  if (c->width < 1 || (uint64_t)c->width * c->page_slots > rules::kMostKeys)
    return "width (width * page_slots from 1 to 2^24 keys)";
  if (c->page_stride % 8 ||
      c->page_stride < (uint64_t)c->page_slots * c->kv_heads * c->head_dim)
    return "page_stride (a multiple of 8, at least a page)";
  // Their product is an offset in 64 bits.
  if (c->page_stride > (1ull << 48) / c->pages) return "page_stride (a pool of at most 2^48 values)";
  if (rows < 1 || rows > rules::kMostRows) return "rows (1 to 512)";
  return nullptr;
}

PagedCache cache_of(const frz_pages* c) {
  PagedCache p;
  p.keys = static_cast<uint16_t*>(c->keys);
  p.values = static_cast<uint16_t*>(c->values);
  p.bf16 = c->format == FRZ_FORMAT_BF16;
  p.kv_heads = (uint32_t)c->kv_heads;
  p.head_dim = (uint32_t)c->head_dim;
  p.page_slots = c->page_slots;
  p.pages = c->pages;
  p.page_stride = c->page_stride;
  p.table = c->table;
  p.sequences = c->sequences;
  p.width = c->width;
  return p;
}

int refuse(const char* what, const char* why) {
  return fail(FRZ_ERR_ARGUMENT, std::string(what) + ": " + why);
}

// Whether rows of `width` floats may be `stride` apart.
bool stride_ok(int stride, int64_t width) { return stride % 4 == 0 && stride >= width; }

}  // namespace

int device_batch_scratch(frz_device* dev) {
  if (dev->batch_scratch) return FRZ_OK;
  const int rc = check_hip(hipMalloc(&dev->batch_scratch, kScratchBytes), "hipMalloc(batch)");
  if (rc != FRZ_OK) dev->batch_scratch = nullptr;
  return rc;
}

}  // namespace frz

using namespace frz;

extern "C" {

int frz_op_rope_paged(frz_device* dev, const frz_pages* cache, const uint32_t* sequences,
                      const uint32_t* positions, const float* turns, const float* query_gain,
                      const float* key_gain, const float* query, const float* key,
                      const float* value, int q_stride, int kv_stride, float* roped,
                      int roped_stride, int query_heads, float epsilon, uint32_t rows) {
  const char* what = "frz_op_rope_paged";
  if (!dev) return refuse(what, "no device");
  if (const char* why = refuse_pages(cache, query_heads, rows)) return refuse(what, why);
  if (!positions || !turns || !query_gain || !key_gain || !query || !key || !value || !roped)
    return refuse(what, "null argument");
  if (!aligned(turns) || !aligned(query_gain) || !aligned(key_gain) || !aligned(query) ||
      !aligned(key) || !aligned(value) || !aligned(roped) || !aligned_word(positions) ||
      !aligned_word(sequences))
    return refuse(what, "a pointer not at a multiple of 16 bytes (positions and sequences: 4)");
  const int64_t q = (int64_t)query_heads * cache->head_dim;
  const int64_t kv = (int64_t)cache->kv_heads * cache->head_dim;
  if (!stride_ok(q_stride, q) || !stride_ok(kv_stride, kv) || !stride_ok(roped_stride, q))
    return refuse(what, "strides (multiples of 4, at least a row)");
  if (roped == key || roped == value) return refuse(what, "roped is key or value");
  if (roped == query && roped_stride != q_stride)
    return refuse(what, "roped in place with another stride");
  PagedRopeArgs a;
  a.cache = cache_of(cache);
  a.sequences = sequences;
  a.positions = positions;
  a.turns = turns;
  a.query_gain = query_gain;
  a.key_gain = key_gain;
  a.query = query;
  a.key = key;
  a.value = value;
  a.q_stride = (uint32_t)q_stride;
  a.kv_stride = (uint32_t)kv_stride;
  a.roped = roped;
  a.roped_stride = (uint32_t)roped_stride;
  a.query_heads = (uint32_t)query_heads;
  a.epsilon = epsilon;
  a.rows = rows;
  return enqueue(dev, what, [&] { return launch_paged_rope(dev->stream, a); });
}

int frz_op_attention_paged(frz_device* dev, const frz_pages* cache, const uint32_t* sequences,
                           const uint32_t* positions, const float* query, int q_stride,
                           float* out, int out_stride, int query_heads, uint32_t window,
                           float scale, uint32_t rows) {
  const char* what = "frz_op_attention_paged";
  if (!dev) return refuse(what, "no device");
  if (const char* why = refuse_pages(cache, query_heads, rows)) return refuse(what, why);
  if (!positions || !query || !out) return refuse(what, "null argument");
  if (!aligned(query) || !aligned(out) || !aligned_word(positions) || !aligned_word(sequences))
    return refuse(what, "a pointer not at a multiple of 16 bytes (positions and sequences: 4)");
  const int64_t q = (int64_t)query_heads * cache->head_dim;
  if (!stride_ok(q_stride, q) || !stride_ok(out_stride, q))
    return refuse(what, "strides (multiples of 4, at least a row)");
  if (out == query) return refuse(what, "out is query");
  if (window == 0) return refuse(what, "window 0");
  if (!(std::fabs(scale) <= kMostScale)) return refuse(what, "scale (a number of at most 4,096)");
  PagedAttentionArgs a;
  a.cache = cache_of(cache);
  a.sequences = sequences;
  a.positions = positions;
  a.query = query;
  a.q_stride = (uint32_t)q_stride;
  a.out = out;
  a.out_stride = (uint32_t)out_stride;
  a.query_heads = (uint32_t)query_heads;
  a.window = window;
  a.scale_log2e = (float)((double)scale * 1.4426950408889634);
  a.rows = rows;
  return enqueue(dev, what, [&] {
    float* at = static_cast<float*>(dev->batch_scratch);
    a.states = at;
    a.stats = at + kStateFloats;
    a.records = reinterpret_cast<uint4*>(at + kStateFloats + kStatFloats);
    a.record_count = reinterpret_cast<uint32_t*>(a.records + kRecords);
    return launch_paged_attention(dev->stream, a, dev->props.multiProcessorCount);
  });
}

int frz_op_adapters(frz_device* dev, const frz_adapters* adapters, const uint32_t* which,
                    const float* x, int x_stride, const float* base, int base_stride, float* y,
                    int y_stride, uint32_t tokens) {
  const char* what = "frz_op_adapters";
  if (!dev) return refuse(what, "no device");
  if (!adapters || !adapters->down || !adapters->up || !which || !x || !base || !y)
    return refuse(what, "null argument");
  const frz_adapters& p = *adapters;
  if (p.format != FRZ_FORMAT_F32 && p.format != FRZ_FORMAT_F16 && p.format != FRZ_FORMAT_BF16)
    return refuse(what, "format (F32 0, F16 1 or BF16 30)");
  if (p.count < 1 || p.count == FRZ_NO_ADAPTER) return refuse(what, "no adapters");
  if (p.rank < 8 || p.rank % 8 || p.rank > kMostAdapterRank)
    return refuse(what, "rank (a multiple of 8, at most 128)");
  if (p.cols < 8 || p.cols % 8 || p.rows < 1 || p.cols > (1 << 24) || p.rows > (1 << 24))
    return refuse(what, "shape (cols a multiple of 8, both at most 2^24)");
  if (tokens < 1 || tokens > rules::kMostRows) return refuse(what, "tokens (1 to 512)");
  if (!aligned(p.down) || !aligned(p.up) || !aligned(x) || !aligned(base) || !aligned(y) ||
      !aligned_word(which) || !aligned_word(p.ranks) || !aligned_word(p.scales))
    return refuse(what, "a pointer not at a multiple of 16 bytes (which, ranks and scales: 4)");
  if (!stride_ok(x_stride, p.cols) || !stride_ok(base_stride, p.rows) ||
      !stride_ok(y_stride, p.rows))
    return refuse(what, "strides (multiples of 4, at least a row)");
  if (x == y) return refuse(what, "y is x");
  if (base == y && base_stride != y_stride)
    return refuse(what, "y is base with another stride");
  AdapterArgs a;
  a.down = p.down;
  a.up = p.up;
  a.format = p.format;
  a.count = p.count;
  a.rank = p.rank;
  a.cols = p.cols;
  a.rows = p.rows;
  a.ranks = p.ranks;
  a.scales = p.scales;
  a.which = which;
  a.x = x;
  a.x_stride = x_stride;
  a.base = base;
  a.base_stride = base_stride;
  a.y = y;
  a.y_stride = y_stride;
  a.tokens = tokens;
  return enqueue(dev, what, [&] {
    a.low = static_cast<float*>(dev->batch_scratch);
    return launch_adapters(dev->stream, a);
  });
}

}  // extern "C"
