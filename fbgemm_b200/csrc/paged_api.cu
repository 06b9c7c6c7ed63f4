// The C ABI of the paged key-value cache: argument checks and launches (include/fbgemm_b200/embedding_c_api.h).
#include <atomic>

#include "context.h"
#include "paged_cache.h"

using namespace fbgemm_b200;

namespace {

constexpr int64_t kMostRows = 0x7fffff00LL;  // of a request, as far as its block table goes
constexpr int64_t kMostWait = 1000000000;
std::atomic<int64_t> g_copy_limit{kMostWait};

bool aligned(const void* p, uintptr_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0;
}

int refuse(const char* what) {
  set_error(what);
  return FBGEMM_B200_EINVAL;
}

int bits_of(const fbgemm_b200_paged_cache& c) {
  return c.in_dtype == FBGEMM_B200_IN_QUANTIZED ? c.bit_rate : 16;
}

int64_t row_bytes(const fbgemm_b200_paged_cache& c) {
  const int bits = bits_of(c);
  return (int64_t)c.head_dim * bits / 8 + (bits == 8 ? 8 : bits == 4 ? 4 : 0);
}

int shift_of(int32_t page_size) {
  int shift = 0;
  while ((1 << shift) < page_size) {
    ++shift;
  }
  return shift;
}

bool power_of_two(int32_t page_size) {
  return page_size >= 1 && page_size <= 65536 && (page_size & (page_size - 1)) == 0;
}

int check_cache(const fbgemm_b200_paged_cache* c) {
  if (!c) {
    return refuse("paged cache: null description");
  }
  if (c->in_dtype != FBGEMM_B200_IN_QUANTIZED && c->in_dtype != FBGEMM_B200_IN_F16 && c->in_dtype != FBGEMM_B200_IN_BF16) {
    return refuse("paged cache: rows are fp16, bf16 or quantized");
  }
  const int bits = bits_of(*c);
  if (bits != 16 && bits != 8 && bits != 4) {
    return refuse("paged cache: quantized rows have 8 or 4 bits");
  }
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % (bits == 4 ? 32 : 16) != 0) {
    return refuse("paged cache: head_dim is a multiple of 16 (4-bit rows: of 32), 256 at most");
  }
  if (!power_of_two(c->page_size)) {
    return refuse("paged cache: page_size is a power of two, 65536 at most");
  }
  if (c->num_pages < 1 || c->num_pages > 0x7fffffffLL || c->kv_heads < 1 || c->kv_heads > 4096) {
    return refuse("paged cache: 1 to 2^31 - 1 pages, 1 to 4096 heads");
  }
  const int align = bits == 16 ? 16 : 4;
  const int64_t bytes = row_bytes(*c);
  const int64_t strides[3] = {c->page_stride, c->slot_stride, c->head_stride};
  const int64_t counts[3] = {c->num_pages, c->page_size, c->kv_heads};
  for (int i = 0; i < 3; ++i) {
    if (strides[i] % align != 0 || strides[i] < 0 || (counts[i] > 1 && strides[i] < bytes)) {
      return refuse("paged cache: strides are multiples of 16 bytes (quantized rows: of 4) and at least a row");
    }
  }
  if (!c->k || !c->v || !aligned(c->k, align) || !aligned(c->v, align)) {
    return refuse("paged cache: null or unaligned rows");
  }
  return 0;
}

int check_call(const fbgemm_b200_ctx* ctx, int slot) {
  return ctx && slot >= 0 && slot < FBGEMM_B200_USER_SLOTS
      ? 0
      : refuse("bad context or status slot (callers own slots 0 .. FBGEMM_B200_USER_SLOTS - 1)");
}

// dtype of activations beside this cache.
int check_dtype(const fbgemm_b200_paged_cache& c, int32_t dtype) {
  if (dtype != FBGEMM_B200_OUT_F16 && dtype != FBGEMM_B200_OUT_BF16) {
    return refuse("activations beside a paged cache are fp16 or bf16");
  }
  if (c.in_dtype != FBGEMM_B200_IN_QUANTIZED && (c.in_dtype == FBGEMM_B200_IN_BF16) != (dtype == FBGEMM_B200_OUT_BF16)) {
    return refuse("activations beside a 16-bit paged cache have its type");
  }
  return 0;
}

bool good_rows(const void* p, int64_t token, int64_t head) {
  return p && aligned(p, 16) && token % 8 == 0 && head % 8 == 0;
}

// Whether [tokens, heads, dim] 16-bit values behind one another at `out` share memory with rows that strides (elements)
// place at p: what one block writes others may not have read yet.
bool overlaps(const void* out, const void* p, int64_t tokens, int64_t heads, int64_t dim, int64_t p_heads, int64_t token,
              int64_t head) {
  const int64_t t = (tokens - 1) * token, h = (p_heads - 1) * head;
  const intptr_t at = reinterpret_cast<intptr_t>(p), to = reinterpret_cast<intptr_t>(out);
  const intptr_t from = at + 2 * ((t < 0 ? t : 0) + (h < 0 ? h : 0));
  const intptr_t end = at + 2 * ((t > 0 ? t : 0) + (h > 0 ? h : 0) + dim);
  return from < to + 2 * tokens * heads * dim && to < end;
}

bool rows_aligned(const fbgemm_b200_paged_cache& c) {
  return aligned(c.k, 16) && aligned(c.v, 16) && (c.page_stride | c.slot_stride | c.head_stride) % 16 == 0;
}

PagedAttentionShape shape_of(const fbgemm_b200_paged_cache& c, int32_t q_heads, int32_t dtype) {
  PagedAttentionShape s;
  s.bits = bits_of(c);
  s.bf16 = dtype == FBGEMM_B200_OUT_BF16;
  s.dim = c.head_dim;
  s.group = q_heads / c.kv_heads;
  s.fast = c.page_size >= 16 && rows_aligned(c) && c.page_stride < (1LL << 39) && c.slot_stride < (1LL << 39) &&
      c.head_stride < (1LL << 39);
  return s;
}

int64_t workspace_bytes_of(const PagedAttentionPlan& plan) {
  return 2 * (int64_t)plan.workers * (2 * (int64_t)plan.part_floats * 4 + 16);  // (workers of either size)
}

// Rows that a request can have, as far as the host knows.
int64_t span_most(const fbgemm_b200_paged_cache& c, int32_t width, int32_t window) {
  const int64_t most = (int64_t)width * c.page_size;
  return window > 0 && window < most ? window : most;
}

int32_t cluster_of(const fbgemm_b200_paged_cache& c, const PagedAttentionPlan& plan, int64_t batch, int32_t width,
                   int32_t window) {
  return blocks_of_item(span_most(c, width, window), batch * c.kv_heads * plan.head_tiles, plan.blocks);
}

int check_heads(const fbgemm_b200_paged_cache& c, int32_t q_heads) {
  return q_heads >= 1 && q_heads <= 16384 && q_heads % c.kv_heads == 0
      ? 0
      : refuse("query heads are a multiple of the cached heads, 16384 at most");
}

}  // namespace

extern "C" {

int fbgemm_b200_paged_cache_check(const fbgemm_b200_paged_cache* cache) try {
  return check_cache(cache);
} catch (...) {
  return thrown();
}

int64_t fbgemm_b200_set_copy_limit(int64_t nanoseconds) try {
  if (nanoseconds < 0 || nanoseconds > kMostWait) {
    return refuse("a copy is waited for 0 to 1e9 nanoseconds");
  }
  return g_copy_limit.exchange(nanoseconds, std::memory_order_relaxed);
} catch (...) {
  return thrown();
}

int fbgemm_b200_paged_slots(
    fbgemm_b200_ctx* ctx,
    int32_t batch,
    const int32_t* lengths,
    const int32_t* new_tokens,
    int32_t* block_tables,
    int32_t width,
    int64_t table_stride,
    const int32_t* free_pages,
    int32_t free_capacity,
    const int32_t* num_free,
    int32_t page_size,
    int32_t capacity,
    int64_t* slots,
    int32_t* positions,
    int32_t* requests,
    int32_t* offsets,
    int32_t* lengths_out,
    int32_t* num_free_out,
    int slot,
    void* stream) try {
  if (int rc = check_call(ctx, slot)) {
    return rc;
  }
  if (batch < 1 || batch > FBGEMM_B200_PAGED_MAX_BATCH) {
    return refuse("paged_slots: 1 to 16384 requests");
  }
  if (!power_of_two(page_size) || width < 0 || (int64_t)width * page_size > kMostRows) {
    return refuse("paged_slots: page_size is a power of two, 65536 at most, and width * page_size <= 2^31 - 256");
  }
  if (capacity < 0 || free_capacity < 0 || table_stride < width) {
    return refuse("paged_slots: negative capacity, or table rows that overlap");
  }
  if (!lengths || !new_tokens || !num_free || !offsets || !lengths_out || !num_free_out || (width > 0 && !block_tables) ||
      (free_capacity > 0 && !free_pages) || (capacity > 0 && (!slots || !positions || !requests))) {
    return refuse("paged_slots: null pointer");
  }
  PagedSlotsParams p = {};
  p.lengths = lengths;
  p.fresh = new_tokens;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.free_pages = free_pages;
  p.num_free = num_free;
  p.slots = slots;
  p.positions = positions;
  p.requests = requests;
  p.offsets = offsets;
  p.lengths_out = lengths_out;
  p.num_free_out = num_free_out;
  p.status = ctx->status + 4 * slot;
  p.batch = batch;
  p.width = width;
  p.free_capacity = free_capacity;
  p.page_shift = shift_of(page_size);
  p.capacity = capacity;
  DeviceGuard guard(ctx->device);
  const cudaError_t e = launch_paged_slots(p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : fail_cuda(e, "paged_slots launch");
} catch (...) {
  return thrown();
}

int fbgemm_b200_rotary_append(
    fbgemm_b200_ctx* ctx,
    const fbgemm_b200_paged_cache* cache,
    int64_t tokens,
    int32_t q_heads,
    int32_t dtype,
    const void* q,
    int64_t q_token_stride,
    int64_t q_head_stride,
    const void* k,
    int64_t k_token_stride,
    int64_t k_head_stride,
    const void* v,
    int64_t v_token_stride,
    int64_t v_head_stride,
    void* q_out,
    const int64_t* slots,
    const int32_t* positions,
    int64_t positions_stride,
    const fbgemm_b200_rotary* rotary,
    int slot,
    void* stream) try {
  int rc = check_call(ctx, slot);
  rc = rc ? rc : check_cache(cache);
  rc = rc ? rc : check_dtype(*cache, dtype);
  if (rc) {
    return rc;
  }
  if (tokens < 0 || tokens > 0x7fffffffLL) {
    return refuse("rotary_append: 0 to 2^31 - 1 tokens");
  }
  if (tokens == 0) {
    return 0;
  }
  if (q_out && (q_heads < 1 || q_heads > 16384 || !good_rows(q, q_token_stride, q_head_stride) || !aligned(q_out, 16))) {
    return refuse("rotary_append: q is null or not aligned to 16 bytes, or has no heads");
  }
  if (!good_rows(k, k_token_stride, k_head_stride) || !good_rows(v, v_token_stride, v_head_stride) || !slots) {
    return refuse("rotary_append: k, v or slots is null or not aligned to 16 bytes");
  }
  if (cache->k == cache->v) {
    return refuse("rotary_append: keys and values in the same memory");
  }
  if (q_out) {
    const int64_t dim = cache->head_dim;
    const bool in_place = q_out == q && (tokens == 1 || q_token_stride == q_heads * dim) && (q_heads == 1 || q_head_stride == dim);
    if ((!in_place && overlaps(q_out, q, tokens, q_heads, dim, q_heads, q_token_stride, q_head_stride)) ||
        overlaps(q_out, k, tokens, q_heads, dim, cache->kv_heads, k_token_stride, k_head_stride) ||
        overlaps(q_out, v, tokens, q_heads, dim, cache->kv_heads, v_token_stride, v_head_stride)) {
      return refuse("rotary_append: q_out overlaps the memory of k, v or, unless it is q itself, q");
    }
  }
  RotaryAppendParams p = {};
  if (rotary) {
    const fbgemm_b200_rotary& r = *rotary;
    if (!r.cos_sin || !positions || r.max_pos < 1 || r.rot_dim < 16 || r.rot_dim % 16 != 0 || r.rot_dim > cache->head_dim ||
        r.axes < 1 || r.axes > 4 || !aligned(r.cos_sin, 4)) {
      return refuse("rotary_append: rot_dim is a multiple of 16 up to head_dim, with 1 to 4 axes and a table of angles");
    }
    for (int a = 0; a < 4; ++a) {
      p.section_end[a] = a < r.axes ? r.section_end[a] : r.rot_dim / 2;
      if (p.section_end[a] < (a ? p.section_end[a - 1] : 0)) {
        return refuse("rotary_append: sections do not follow one another");
      }
    }
    if (p.section_end[r.axes - 1] != r.rot_dim / 2) {
      return refuse("rotary_append: the sections add up to rot_dim / 2");
    }
    p.cos_sin = r.cos_sin;
    p.max_pos = r.max_pos;
    p.rot = r.rot_dim;
    p.axes = r.axes;
    p.interleaved = r.interleaved != 0;
    p.angles_aligned = aligned(r.cos_sin, 16);
    p.positions = positions;
    p.positions_stride = positions_stride;
  }
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_token = 2 * q_token_stride;
  p.q_head = 2 * q_head_stride;
  p.k_token = 2 * k_token_stride;
  p.k_head = 2 * k_head_stride;
  p.v_token = 2 * v_token_stride;
  p.v_head = 2 * v_head_stride;
  p.q_out = q_out;
  p.slots = slots;
  p.k_cache = static_cast<uint8_t*>(cache->k);
  p.v_cache = static_cast<uint8_t*>(cache->v);
  p.page_stride = cache->page_stride;
  p.slot_stride = cache->slot_stride;
  p.head_stride = cache->head_stride;
  p.page_shift = shift_of(cache->page_size);
  p.num_slots = cache->num_pages << p.page_shift;
  p.status = ctx->status + 4 * slot;
  p.tokens = tokens;
  p.heads = q_out ? q_heads : 0;
  p.kv_heads = cache->kv_heads;
  p.dim = cache->head_dim;
  p.bf16 = dtype == FBGEMM_B200_OUT_BF16;
  p.bits = bits_of(*cache);
  DeviceGuard guard(ctx->device);
  const cudaError_t e = launch_rotary_append(p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : fail_cuda(e, "rotary_append launch");
} catch (...) {
  return thrown();
}

int64_t fbgemm_b200_paged_attention_workspace(
    fbgemm_b200_ctx* ctx,
    const fbgemm_b200_paged_cache* cache,
    int32_t batch,
    int32_t q_heads,
    int32_t dtype,
    int32_t width,
    int32_t window) try {
  int rc = check_call(ctx, 0);
  rc = rc ? rc : check_cache(cache);
  rc = rc ? rc : check_dtype(*cache, dtype);
  rc = rc ? rc : check_heads(*cache, q_heads);
  if (rc) {
    return rc;
  }
  DeviceGuard guard(ctx->device);
  const PagedAttentionPlan plan = plan_paged_attention(shape_of(*cache, q_heads, dtype), sm_count());
  return cluster_of(*cache, plan, batch, width, window) ? 0 : workspace_bytes_of(plan);
} catch (...) {
  return thrown();
}

int fbgemm_b200_paged_attention(
    fbgemm_b200_ctx* ctx,
    const fbgemm_b200_paged_cache* cache,
    int32_t batch,
    int32_t q_heads,
    int32_t dtype,
    const void* q,
    int64_t q_token_stride,
    int64_t q_head_stride,
    const int32_t* block_tables,
    int32_t width,
    int64_t table_stride,
    const int32_t* lengths,
    float scale,
    int32_t window,
    void* out,
    float* lse,
    void* workspace,
    int64_t workspace_bytes,
    int slot,
    void* stream) try {
  int rc = check_call(ctx, slot);
  rc = rc ? rc : check_cache(cache);
  rc = rc ? rc : check_dtype(*cache, dtype);
  rc = rc ? rc : check_heads(*cache, q_heads);
  if (rc) {
    return rc;
  }
  if (batch < 0 || width < 0 || window < 0 || (int64_t)width * cache->page_size > kMostRows) {
    return refuse("paged_attention: negative size or window, or width * page_size > 2^31 - 256");
  }
  if (batch == 0) {
    return 0;
  }
  if (!good_rows(q, q_token_stride, q_head_stride) || !lengths || !out || !aligned(out, 16) ||
      (width > 0 && !block_tables)) {
    return refuse("paged_attention: q, block_tables, lengths or out is null, or q or out not aligned to 16 bytes");
  }
  if (overlaps(out, q, batch, q_heads, cache->head_dim, q_heads, q_token_stride, q_head_stride)) {
    return refuse("paged_attention: out overlaps the memory of q");
  }
  const PagedAttentionShape shape = shape_of(*cache, q_heads, dtype);
  DeviceGuard guard(ctx->device);
  const PagedAttentionPlan plan = plan_paged_attention(shape, sm_count());
  const int64_t items = (int64_t)batch * cache->kv_heads * plan.head_tiles;
  if (items > 0x7fffffffLL) {
    return refuse("paged_attention: 2^31 heads of all requests or more");
  }
  const int64_t most = (int64_t)width * cache->page_size;
  const int32_t cluster = cluster_of(*cache, plan, batch, width, window);
  const bool split = cluster == 0;
  if (split && (!workspace || !aligned(workspace, 16) || workspace_bytes < workspace_bytes_of(plan))) {
    return refuse("paged_attention: workspace missing, unaligned or too small (fbgemm_b200_paged_attention_workspace)");
  }
  PagedAttentionParams p = {};
  p.k = static_cast<const uint8_t*>(cache->k);
  p.v = static_cast<const uint8_t*>(cache->v);
  p.page_stride = cache->page_stride;
  p.slot_stride = cache->slot_stride;
  p.head_stride = cache->head_stride;
  p.q = static_cast<const uint8_t*>(q);
  p.q_token = 2 * q_token_stride;
  p.q_head = 2 * q_head_stride;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.lengths = lengths;
  p.out = out;
  p.lse = lse;
  if (split) {
    p.parts = static_cast<float*>(workspace);
    p.open = reinterpret_cast<int4*>(p.parts + 2 * plan.part_floats * 2 * plan.workers);
  }
  p.status = ctx->status + 4 * slot;
  p.copy_limit = (uint32_t)g_copy_limit.load(std::memory_order_relaxed);
  p.most_rows = most;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.num_pages = (int32_t)cache->num_pages;
  p.page_shift = shift_of(cache->page_size);
  p.batch = batch;
  p.kv_heads = cache->kv_heads;
  p.group = shape.group;
  p.head_tiles = plan.head_tiles;
  p.dim = cache->head_dim;
  p.window = window;
  p.workers = plan.workers;
  p.aligned = rows_aligned(*cache);
  p.tall = cache->page_size >= 32;
  p.cluster = cluster;
  p.two = split && two_sizes(shape.bits, plan.tile_heads, items, items * (span_most(*cache, width, window) / plan.unit + 1), plan.workers);
  const cudaError_t e = launch_paged_attention(shape, plan, p, split, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : fail_cuda(e, "paged_attention launch");
} catch (...) {
  return thrown();
}

}  // extern "C"
