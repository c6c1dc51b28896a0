// C ABI of the paged KV cache (include/bitgpu_attn.h): the pool's geometry over the caller's device
// memory, the batch (its checks, its plan, its upload and its workspace) and the two launches. Host code
// only; the kernels live in paged_prologue.hip and paged_attn.hip, the plan in bg_paged_plan.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>
#include <new>
#include <string>
#include <vector>

#include "../../include/bitgpu_attn.h"
#include "bg_api_util.h"
#include "bg_paged.h"

struct bg_paged_kv {
  int n_layers, kv_heads, D, dtype, page, shift, n_pages;
  char *k, *v;
  float *ks, *vs;
  int q8_row = 0;
  int device = 0, num_cus = 256;
};

namespace {

int32_t fail(int32_t code, const char* fmt, ...) {
  char buf[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return bg::api_fail(code, buf);
}

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

// the sections of a batch's device block and of each staging slot, in this order
enum { S_HDR, S_UNITS, S_TOKS, S_MERGES, S_PAGES, S_DST, S_POS, S_V_SINGLE, S_V_GROUP, N_SECTIONS };
constexpr int kSlots = 2;
constexpr int kMaxAxes = 4;

unsigned long long pool_values(int layers, int kv_heads, int D, int page, int n_pages) {
  return (unsigned long long)layers * n_pages * kv_heads * page * D;
}

int32_t check_pool(const char* who, int32_t n_layers, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t page_size,
                   int32_t n_pages) {
  if (n_layers < 1 || kv_heads < 1 || n_pages < 1)
    return fail(BG_E_INVALID, "%s: n_layers %d, kv_heads %d, n_pages %d must be >= 1", who, n_layers, kv_heads, n_pages);
  if (head_dim != 128 && head_dim != 256) return fail(BG_E_UNSUPPORTED, "%s: head_dim %d unsupported (128 or 256)", who, head_dim);
  if (dtype != BG_KV_F32 && dtype != BG_KV_F16 && dtype != BG_KV_Q8) return fail(BG_E_INVALID, "%s: unknown kv dtype %d", who, dtype);
  if (page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
    return fail(BG_E_UNSUPPORTED, "%s: page_size %d unsupported (32, 64, 128 or 256)", who, page_size);
  if ((long long)n_pages * page_size > INT_MAX)
    return fail(BG_E_UNSUPPORTED, "%s: %d pages of %d positions, beyond 2^31 - 1 positions", who, n_pages, page_size);
  if ((long long)n_layers * kv_heads > 1 << 22)  // with the line above: a region's bytes stay below 2^63
    return fail(BG_E_UNSUPPORTED, "%s: n_layers %d x kv_heads %d too large", who, n_layers, kv_heads);
  return BG_OK;
}

}  // namespace

struct bg_paged_batch {
  bg::PagedShape shape{};
  int H = 0, page_shift = 0, device = 0;
  char* dev = nullptr;               // the device block of all sections
  char* host[kSlots] = {};           // pinned staging, one block a slot
  hipEvent_t done[kSlots] = {};      // recorded behind the slot's upload
  bool pending[kSlots] = {};
  int slot = 0;
  size_t at[N_SECTIONS + 1] = {};
  float* ws = nullptr;
  size_t ws_bytes = 0;
  bg::PagedPlanner planner;
  bg::PagedPlan plan, next;
  int axes = 1, max_pos = -1;
  bool set = false;
  // The stream of the last call. A call on another one first waits there for what the batch has enqueued:
  // its launches read the arrays an upload writes, and share a workspace.
  hipStream_t last = nullptr;
  bool used = false;
  hipEvent_t moved = nullptr;
  // what launches under capture rely on and later sets have to keep
  int cap_tokens = INT_MAX, cap_rope = INT_MAX, cap_axes = 0;  // (cap_axes 0: nothing that rotates)
  bool cap_write = false;                                      // something that writes pages

  bg::PagedBatchView view(bool captured) const {
    bg::PagedBatchView b{};
    b.hdr = (const bg::PagedHeader*)(dev + at[S_HDR]);
    b.units = (const bg::PagedUnit*)(dev + at[S_UNITS]);
    b.toks = (const bg::PagedTok*)(dev + at[S_TOKS]);
    b.merges = (const bg::PagedMerge*)(dev + at[S_MERGES]);
    b.pages = (const int*)(dev + at[S_PAGES]);
    b.dst = (const int*)(dev + at[S_DST]);
    b.pos = (const int*)(dev + at[S_POS]);
    b.v_single = (const int*)(dev + at[S_V_SINGLE]);
    b.v_group = (const int*)(dev + at[S_V_GROUP]);
    b.pos_stride = shape.max_tokens;
    b.page_shift = page_shift;
    b.H = H;
    b.G = shape.G;
    b.captured = captured;
    if (!captured) {
      b.stream_few = plan.stream_few;
      b.n_units = (int)plan.units.size();
      b.n_many = plan.n_many;
      b.n_mid = plan.n_mid;
      b.n_merges = (int)plan.merges.size();
      b.n_merge_few = plan.n_merge_few;
      b.n_tokens = plan.n_tokens;
      b.n_v_single = (int)plan.v_single.size();
      b.n_v_group = (int)plan.v_group.size();
    }
    return b;
  }
};

namespace {

bg::LayerView layer_view(const bg_paged_kv* c, int layer) {
  bg::LayerView L{};
  const size_t rows = (size_t)layer * c->n_pages * c->kv_heads * c->page;
  L.k = c->k + rows * c->D * bg::kv_elem_bytes(c->dtype);
  L.v = c->v + rows * c->D * bg::kv_elem_bytes(c->dtype);
  L.ks = c->dtype == BG_KV_Q8 ? c->ks + rows * (c->D / 32) : nullptr;
  L.vs = c->dtype == BG_KV_Q8 ? c->vs + rows * (c->D / 32) : nullptr;
  L.cap = c->page;
  L.kv_heads = c->kv_heads;
  L.D = c->D;
  L.dtype = c->dtype;
  L.max_seq = c->page;
  L.q8_row = c->q8_row;
  return L;
}

// What every launch checks of its pool and batch.
int32_t check_pair(const char* who, const bg_paged_kv* c, const bg_paged_batch* b, int32_t layer) {
  if (!c || !b) return fail(BG_E_INVALID, "%s: NULL cache or batch", who);
  if (layer < 0 || layer >= c->n_layers) return fail(BG_E_INVALID, "%s: layer %d out of range", who, layer);
  const bg::PagedShape& s = b->shape;
  if (s.kv_heads != c->kv_heads || s.D != c->D || s.dtype != c->dtype || s.page != c->page || s.n_pages != c->n_pages)
    return fail(BG_E_INVALID, "%s: the batch was made for another cache", who);
  if (!b->set) return fail(BG_E_STATE, "%s: the batch has not been set", who);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != c->device || dev != b->device)
    return fail(BG_E_INVALID, "%s: the cache lives on device %d, the batch on %d, the current device is %d", who, c->device,
                b->device, dev);
  return BG_OK;
}

// Orders a call on `st` behind the batch's calls so far. (A launch under capture runs at replay: its order is
// the caller's.)
int32_t join_stream(const char* who, bg_paged_batch* b, hipStream_t st) {
  if (b->used && b->last != st) {
    if (bg::api_capturing(b->last))
      return fail(BG_E_STATE, "%s: the batch worked on a stream that is being captured now", who);
    hipError_t e = hipEventRecord(b->moved, b->last);
    if (e == hipSuccess) e = hipStreamWaitEvent(st, b->moved, 0);
    if (e != hipSuccess) return bg::api_hip_fail(e, "paged batch: the stream of its last call");
  }
  b->last = st;
  b->used = true;
  return BG_OK;
}

void free_batch(bg_paged_batch* b) {
  for (int i = 0; i < kSlots; i++) {
    if (b->host[i]) (void)hipHostFree(b->host[i]);
    if (b->done[i]) (void)hipEventDestroy(b->done[i]);
  }
  if (b->moved) (void)hipEventDestroy(b->moved);
  if (b->dev) (void)hipFree(b->dev);
  if (b->ws) (void)hipFree(b->ws);
  delete b;
}

}  // namespace

extern "C" {

int32_t bg_paged_region_bytes(int32_t n_layers, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t page_size,
                              int32_t n_pages, int32_t region, size_t* bytes) {
  if (!bytes) return fail(BG_E_INVALID, "bg_paged_region_bytes: bytes is NULL");
  const int32_t rc = check_pool("bg_paged_region_bytes", n_layers, kv_heads, head_dim, dtype, page_size, n_pages);
  if (rc != BG_OK) return rc;
  const unsigned long long n = pool_values(n_layers, kv_heads, head_dim, page_size, n_pages);
  if (region == BG_K || region == BG_V) {
    *bytes = (size_t)n * bg::kv_elem_bytes(dtype);
  } else if (region == BG_KSCALE || region == BG_VSCALE) {
    *bytes = dtype == BG_KV_Q8 ? (size_t)n / 32 * sizeof(float) : 0;
  } else {
    return fail(BG_E_INVALID, "bg_paged_region_bytes: unknown region %d", region);
  }
  return BG_OK;
}

int32_t bg_paged_create(int32_t n_layers, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t page_size,
                        int32_t n_pages, void* k, void* v, float* k_scale, float* v_scale, bg_paged_kv** out) {
  if (!out) return fail(BG_E_INVALID, "bg_paged_create: out is NULL");
  *out = nullptr;
  const int32_t rc = check_pool("bg_paged_create", n_layers, kv_heads, head_dim, dtype, page_size, n_pages);
  if (rc != BG_OK) return rc;
  if (!k || !v) return fail(BG_E_INVALID, "bg_paged_create: k or v is NULL");
  if ((dtype == BG_KV_Q8) != (k_scale != nullptr) || (dtype == BG_KV_Q8) != (v_scale != nullptr))
    return fail(BG_E_INVALID, "bg_paged_create: k_scale and v_scale belong to q8, and q8 needs both");
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15)
    return fail(BG_E_INVALID, "bg_paged_create: buffers must be 16-byte aligned");
  bg_paged_kv* c = new (std::nothrow) bg_paged_kv();
  if (!c) return fail(BG_E_OOM, "bg_paged_create: out of host memory");
  c->n_layers = n_layers;
  c->kv_heads = kv_heads;
  c->D = head_dim;
  c->dtype = dtype;
  c->page = page_size;
  c->shift = page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : 8;
  c->n_pages = n_pages;
  c->k = (char*)k;
  c->v = (char*)v;
  c->ks = k_scale;
  c->vs = v_scale;
  hipError_t e = hipGetDevice(&c->device);
  if (e != hipSuccess) {
    delete c;
    return bg::api_hip_fail(e, "bg_paged_create: current device");
  }
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, c->device) == hipSuccess && cus > 0) c->num_cus = cus;
  *out = c;
  return BG_OK;
}

int32_t bg_paged_destroy(bg_paged_kv* c) {
  delete c;  // the memory is the caller's
  return BG_OK;
}

int32_t bg_paged_set_q8_block(bg_paged_kv* c, int32_t block) {
  if (!c) return fail(BG_E_INVALID, "bg_paged_set_q8_block: NULL cache");
  if (c->dtype != BG_KV_Q8) return fail(BG_E_STATE, "bg_paged_set_q8_block: the cache is not q8");
  if (block != 32 && block != c->D) return fail(BG_E_INVALID, "bg_paged_set_q8_block: block %d (32 or head_dim %d)", block, c->D);
  c->q8_row = block == c->D;
  return BG_OK;
}

int32_t bg_paged_batch_create(const bg_paged_kv* c, int32_t H, int32_t max_seqs, int32_t max_tokens, int32_t max_pages,
                              bg_paged_batch** out) {
  if (!out) return fail(BG_E_INVALID, "bg_paged_batch_create: out is NULL");
  *out = nullptr;
  if (!c) return fail(BG_E_INVALID, "bg_paged_batch_create: NULL cache");
  if (H < c->kv_heads || H % c->kv_heads) return fail(BG_E_INVALID, "bg_paged_batch_create: heads %d must be a multiple of kv_heads %d", H, c->kv_heads);
  if (max_seqs < 1 || max_tokens < 1 || max_pages < 1)
    return fail(BG_E_INVALID, "bg_paged_batch_create: max_seqs %d, max_tokens %d, max_pages %d must be >= 1", max_seqs,
                max_tokens, max_pages);
  // row and unit numbers stay below 2^31
  if ((long long)max_tokens * (H + 2 * c->kv_heads) > INT_MAX / 16 || max_seqs > (1 << 20) || max_pages > (1 << 28))
    return fail(BG_E_UNSUPPORTED, "bg_paged_batch_create: max_tokens %d x heads %d, max_seqs %d or max_pages %d too large",
                max_tokens, H, max_seqs, max_pages);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != c->device)
    return fail(BG_E_INVALID, "bg_paged_batch_create: the cache lives on device %d, the current device is %d", c->device, dev);
  bg_paged_batch* b = new (std::nothrow) bg_paged_batch();
  if (!b) return fail(BG_E_OOM, "bg_paged_batch_create: out of host memory");
  b->shape = bg::PagedShape{c->kv_heads, H / c->kv_heads, c->D, c->dtype, c->page, c->n_pages, c->num_cus, max_seqs, max_tokens, max_pages};
  b->H = H;
  b->page_shift = c->shift;
  b->device = dev;
  const size_t bytes[N_SECTIONS] = {sizeof(bg::PagedHeader),
                                    (size_t)b->shape.max_units() * sizeof(bg::PagedUnit),
                                    (size_t)b->shape.max_toks() * sizeof(bg::PagedTok),
                                    (size_t)max_tokens * sizeof(bg::PagedMerge),
                                    (size_t)max_pages * 4,
                                    (size_t)max_tokens * 4,
                                    (size_t)max_tokens * 4 * kMaxAxes,
                                    (size_t)max_tokens * 4,
                                    (size_t)max_tokens * 4};
  for (int i = 0; i < N_SECTIONS; i++) b->at[i + 1] = b->at[i] + round256(bytes[i]);
  hipError_t e = hipMalloc((void**)&b->dev, b->at[N_SECTIONS]);
  if (e == hipSuccess) e = hipEventCreateWithFlags(&b->moved, hipEventDisableTiming);
  for (int i = 0; i < kSlots && e == hipSuccess; i++) {
    e = hipHostMalloc((void**)&b->host[i], b->at[N_SECTIONS], hipHostMallocMapped | hipHostMallocCoherent);
    if (e == hipSuccess) e = hipEventCreateWithFlags(&b->done[i], hipEventDisableTiming);
  }
  if (e != hipSuccess) {
    (void)hipGetLastError();
    free_batch(b);
    return bg::api_hip_fail(e, "paged batch allocation");
  }
  *out = b;
  return BG_OK;
}

int32_t bg_paged_batch_destroy(bg_paged_batch* b) {
  if (!b) return BG_OK;
  (void)hipDeviceSynchronize();
  free_batch(b);
  return BG_OK;
}

int32_t bg_paged_batch_set(bg_paged_batch* b, int32_t n_seqs, const int32_t* rows, const int32_t* lens, const int32_t* tables,
                           int32_t table_stride, const int32_t* positions, int32_t axes, void* stream) {
  if (!b) return fail(BG_E_INVALID, "bg_paged_batch_set: NULL batch");
  if (n_seqs < 0 || table_stride < 0 || (n_seqs > 0 && (!rows || !lens || (table_stride > 0 && !tables))))
    return fail(BG_E_INVALID, "bg_paged_batch_set: n_seqs %d, table_stride %d need rows, lens and tables", n_seqs, table_stride);
  if (positions && (axes < 1 || axes > kMaxAxes))
    return fail(BG_E_UNSUPPORTED, "bg_paged_batch_set: %d position axes (1 to %d)", axes, kMaxAxes);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != b->device)
    return fail(BG_E_INVALID, "bg_paged_batch_set: the batch lives on device %d, the current device is %d", b->device, dev);
  hipStream_t st = (hipStream_t)stream;
  if (bg::api_capturing(st))
    return fail(BG_E_STATE, "bg_paged_batch_set: a batch is set outside graph capture (its launches read it at replay)");
  try {
    const std::string wrong = b->planner.build(b->shape, n_seqs, rows, lens, tables, table_stride, b->next);
    if (!wrong.empty()) return fail(BG_E_INVALID, "bg_paged_batch_set: %s", wrong.c_str());
  } catch (const std::exception&) {  // the plan's arrays
    return fail(BG_E_OOM, "bg_paged_batch_set: out of host memory");
  }
  const bg::PagedPlan& p = b->next;
  const int T = p.n_tokens, n_axes = positions ? axes : 1;
  int max_pos = -1;
  if (positions) {
    for (long i = 0; i < (long)axes * T; i++) {
      if (positions[i] < 0) return fail(BG_E_INVALID, "bg_paged_batch_set: position %d of token %ld", positions[i], i % T);
      max_pos = std::max(max_pos, positions[i]);
    }
  } else {
    for (int s = 0; s < n_seqs; s++)
      if (rows[s]) max_pos = std::max(max_pos, lens[s] - 1);
  }
  if (T > b->cap_tokens)
    return fail(BG_E_STATE, "bg_paged_batch_set: %d new rows, but launches of this batch were captured with %d", T, b->cap_tokens);
  if (b->cap_axes && n_axes != b->cap_axes)
    return fail(BG_E_STATE, "bg_paged_batch_set: %d position axes, but a prologue of this batch was captured with %d", n_axes, b->cap_axes);
  if (T && max_pos >= b->cap_rope)
    return fail(BG_E_STATE, "bg_paged_batch_set: position %d outside the %d-row rope table of a captured prologue", max_pos, b->cap_rope);
  if (b->cap_write && p.write_page >= 0)
    return fail(BG_E_STATE, "bg_paged_batch_set: page %d is written and listed elsewhere, and a prologue of this batch was captured", p.write_page);
  const int32_t rc = join_stream("bg_paged_batch_set", b, st);
  if (rc != BG_OK) return rc;
  // the workspace of partials
  const size_t ml = round256((size_t)p.n_parts * b->H * sizeof(float2)), need = ml + (size_t)p.n_parts * b->H * b->shape.D * sizeof(float);
  const int slot = b->slot;
  if (b->pending[slot]) {
    const hipError_t e = hipEventSynchronize(b->done[slot]);
    if (e != hipSuccess) return bg::api_hip_fail(e, "paged batch staging");
    b->pending[slot] = false;
  }
  float* ws = b->ws;
  size_t ws_bytes = b->ws_bytes;
  if (need > ws_bytes) {
    ws_bytes = std::max(need, 2 * ws_bytes);  // at least twofold, where there is room: few are ever replaced
    hipError_t e = hipMalloc((void**)&ws, ws_bytes);
    if (e != hipSuccess && ws_bytes > need) {
      (void)hipGetLastError();
      e = hipMalloc((void**)&ws, ws_bytes = need);
    }
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return bg::api_hip_fail(e, "paged attention workspace allocation");
    }
  }
  char* h = b->host[slot];
  bg::PagedHeader hdr{};
  hdr.n_units = (int)p.units.size();
  hdr.n_many = p.n_many;
  hdr.n_mid = p.n_mid;
  hdr.n_merge_few = p.n_merge_few;
  hdr.n_merges = (int)p.merges.size();
  hdr.n_tokens = T;
  hdr.n_v_single = (int)p.v_single.size();
  hdr.n_v_group = (int)p.v_group.size();
  hdr.ws_ml = (float2*)ws;
  hdr.ws_o = ws ? (float*)((char*)ws + ml) : nullptr;
  bg::PagedUpload up{};
  auto put = [&](int section, size_t offset, const void* src, size_t bytes) {
    if (bytes) memcpy(h + b->at[section] + offset, src, bytes);
    const size_t end = offset + bytes;
    up.src[section] = h + b->at[section];
    up.dst[section] = b->dev + b->at[section];
    up.n16[section] = (unsigned)((end + 15) / 16);
  };
  put(S_HDR, 0, &hdr, sizeof(hdr));
  put(S_UNITS, 0, p.units.data(), p.units.size() * sizeof(bg::PagedUnit));
  put(S_TOKS, 0, p.toks.data(), p.toks.size() * sizeof(bg::PagedTok));
  put(S_MERGES, 0, p.merges.data(), p.merges.size() * sizeof(bg::PagedMerge));
  put(S_PAGES, 0, p.pages.data(), p.pages.size() * 4);
  put(S_DST, 0, p.dst.data(), p.dst.size() * 4);
  put(S_V_SINGLE, 0, p.v_single.data(), p.v_single.size() * 4);
  put(S_V_GROUP, 0, p.v_group.data(), p.v_group.size() * 4);
  if (positions) {
    for (int a = 0; a < axes; a++) put(S_POS, (size_t)a * b->shape.max_tokens * 4, positions + (size_t)a * T, (size_t)T * 4);
  } else {
    int* pos = (int*)(h + b->at[S_POS]);
    int t = 0;
    for (int s = 0; s < n_seqs; s++)
      for (int i = 0; i < rows[s]; i++) pos[t++] = lens[s] - rows[s] + i;
    up.src[S_POS] = pos;
    up.dst[S_POS] = b->dev + b->at[S_POS];
    up.n16[S_POS] = (unsigned)(((size_t)T * 4 + 15) / 16);
  }
  hipError_t e = bg::launch_paged_upload(up, st);
  if (e != hipSuccess) {
    if (ws != b->ws) (void)hipFree(ws);  // no launch knows it; those of before and captured ones keep the old
    b->set = false;
    return bg::api_hip_fail(e, "paged batch upload");
  }
  if (ws != b->ws) {
    std::swap(ws, b->ws);
    b->ws_bytes = ws_bytes;
    if (ws) {  // the old one: launches, and replays that began before the new header was there, are done with it
      (void)hipDeviceSynchronize();
      (void)hipFree(ws);
    }
  }
  e = hipEventRecord(b->done[slot], st);
  if (e != hipSuccess) {  // the arrays are another plan's than `plan`, and nothing says when the slot is free
    (void)hipDeviceSynchronize();
    b->set = false;
    return bg::api_hip_fail(e, "paged batch upload");
  }
  b->pending[slot] = true;
  b->slot = (slot + 1) % kSlots;
  std::swap(b->plan, b->next);
  b->axes = n_axes;
  b->max_pos = max_pos;
  b->set = true;
  return BG_OK;
}

int32_t bg_paged_batch_info(const bg_paged_batch* b, int64_t* out) {
  if (!b || !out) return fail(BG_E_INVALID, "bg_paged_batch_info: NULL argument");
  if (!b->set) return fail(BG_E_STATE, "bg_paged_batch_info: the batch has not been set");
  out[0] = b->plan.n_tokens;
  out[1] = (int64_t)b->plan.units.size() * b->shape.kv_heads;
  out[2] = b->plan.shared_segments;
  out[3] = b->plan.keys;
  out[4] = (int64_t)b->plan.merges.size();
  out[5] = b->plan.n_parts;
  return BG_OK;
}

int32_t bg_paged_batch_units(const bg_paged_batch* b, int64_t* out) {
  if (!b || !out) return fail(BG_E_INVALID, "bg_paged_batch_units: NULL argument");
  if (!b->set) return fail(BG_E_STATE, "bg_paged_batch_units: the batch has not been set");
  const bg::PagedPlan& p = b->plan;
  out[0] = (int64_t)p.n_many * b->shape.kv_heads;
  out[1] = (int64_t)p.n_mid * b->shape.kv_heads;
  out[2] = ((int64_t)p.units.size() - p.n_many - p.n_mid) * b->shape.kv_heads;
  out[3] = p.stream_few && bg::paged_has_stream(b->shape.D, b->shape.dtype);
  return BG_OK;
}

int32_t bg_paged_qkv_prologue(const bg_paged_kv* c, int32_t layer, bg_paged_batch* b, const float* q, int32_t q_stride,
                              const float* k, const float* v, const float* q_gamma, const float* k_gamma, float eps,
                              const float* cos_tab, const float* sin_tab, int32_t rope_positions, int32_t rot_dim,
                              const uint8_t* pair_axis, float* q_out, void* stream) {
  const int32_t rc = check_pair("bg_paged_qkv_prologue", c, b, layer);
  if (rc != BG_OK) return rc;
  if (q && (!q_out || !q_gamma)) return fail(BG_E_INVALID, "bg_paged_qkv_prologue: q needs q_out and q_gamma");
  if (q && q_stride < c->D) return fail(BG_E_INVALID, "bg_paged_qkv_prologue: q_stride %d < head_dim %d", q_stride, c->D);
  if (k && !k_gamma) return fail(BG_E_INVALID, "bg_paged_qkv_prologue: k needs k_gamma");
  bg::PagedAppendArgs a{};
  if (q || k) {
    if (!cos_tab || !sin_tab) return fail(BG_E_INVALID, "bg_paged_qkv_prologue: rope tables are NULL");
    if (rot_dim < 2 || (rot_dim & 1) || rot_dim > c->D) return fail(BG_E_INVALID, "bg_paged_qkv_prologue: bad rot_dim %d", rot_dim);
    if (b->max_pos >= rope_positions)
      return fail(BG_E_INVALID, "bg_paged_qkv_prologue: position %d outside the %d-row rope table", b->max_pos, rope_positions);
    if (b->axes > 1 && !pair_axis)
      return fail(BG_E_INVALID, "bg_paged_qkv_prologue: the batch has %d position axes and no pair_axis says which pair takes which", b->axes);
    for (int j = 0; pair_axis && j < rot_dim / 2; j++) {
      if (pair_axis[j] >= b->axes)
        return fail(BG_E_INVALID, "bg_paged_qkv_prologue: pair %d takes axis %d of %d", j, pair_axis[j], b->axes);
      a.pair_axis[j >> 4] |= (uint32_t)pair_axis[j] << (2 * (j & 15));
    }
  }
  const uintptr_t mis = ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)q_gamma |
                         (uintptr_t)k_gamma | (uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15;
  if (mis || (q && (q_stride & 3)))
    return fail(BG_E_INVALID, "bg_paged_qkv_prologue: buffers must be 16-byte aligned and q_stride a multiple of 4");
  if (q && b->plan.n_tokens) {  // q in place: its own rows, each read whole before it is written
    const size_t rows = (size_t)b->plan.n_tokens * b->H;
    const char *q0 = (const char*)q, *o0 = (const char*)q_out;
    const bool apart = q0 + ((rows - 1) * q_stride + c->D) * sizeof(float) <= o0 || o0 + rows * c->D * sizeof(float) <= q0;
    if (!apart && !(q == q_out && q_stride == c->D))
      return fail(BG_E_INVALID, "bg_paged_qkv_prologue: q_out overlaps q and is not q with q_stride head_dim");
  }
  if ((k || v) && b->plan.write_page >= 0)
    return fail(BG_E_INVALID, "bg_paged_qkv_prologue: page %d would be written by one sequence and is listed with these positions "
                              "by another (or twice): give the writer a page of its own", b->plan.write_page);
  hipStream_t st = (hipStream_t)stream;
  const bool captured = bg::api_capturing(st);
  if (!captured) {
    if (b->plan.n_tokens == 0) return BG_OK;
    const int32_t moved = join_stream("bg_paged_qkv_prologue", b, st);
    if (moved != BG_OK) return moved;
  }
  a.q = q;
  a.q_stride = q_stride;
  a.k = k;
  a.v = v;
  a.q_gamma = q_gamma;
  a.k_gamma = k_gamma;
  a.eps = eps;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.rot_dim = rot_dim;
  a.axes = pair_axis ? b->axes : 1;
  a.q_out = q_out;
  a.num_cus = c->num_cus;
  const hipError_t e = bg::launch_paged_prologue(layer_view(c, layer), b->view(captured), a, st);
  if (e != hipSuccess) return bg::api_hip_fail(e, "paged prologue launch");
  if (captured) {
    b->cap_tokens = std::min(b->cap_tokens, b->plan.n_tokens);
    if (q || k) {
      b->cap_rope = std::min(b->cap_rope, rope_positions);
      b->cap_axes = b->axes;
    }
    b->cap_write |= k || v;
  }
  return BG_OK;
}

int32_t bg_paged_attention(const bg_paged_kv* c, int32_t layer, bg_paged_batch* b, const float* q, float scale,
                           const float* gate, int32_t gate_stride, float* out, void* stream) {
  const int32_t rc = check_pair("bg_paged_attention", c, b, layer);
  if (rc != BG_OK) return rc;
  if (!(scale > 0.0f) || !(scale < 0x1p127f)) return fail(BG_E_INVALID, "bg_paged_attention: scale must be positive and below 2^127");
  if (gate && gate_stride < c->D) return fail(BG_E_INVALID, "bg_paged_attention: gate_stride %d < head_dim", gate_stride);
  hipStream_t st = (hipStream_t)stream;
  const bool captured = bg::api_capturing(st);
  if (!captured && b->plan.n_tokens == 0) return BG_OK;
  if (!q || !out) return fail(BG_E_INVALID, "bg_paged_attention: NULL argument");
  if (q == out) return fail(BG_E_INVALID, "bg_paged_attention: out is q");
  if (((uintptr_t)q | (uintptr_t)out) & 15) return fail(BG_E_INVALID, "bg_paged_attention: q and out must be 16-byte aligned");
  if (!captured) {
    const int32_t moved = join_stream("bg_paged_attention", b, st);
    if (moved != BG_OK) return moved;
  }
  bg::PagedAttnArgs a{};
  a.q = q;
  a.scale = scale;
  a.gate = gate;
  a.gate_stride = gate_stride;
  a.out = out;
  a.num_cus = c->num_cus;
  const hipError_t e = bg::launch_paged_attention(layer_view(c, layer), b->view(captured), a, st);
  if (e != hipSuccess) return bg::api_hip_fail(e, "paged attention launch");
  if (captured) b->cap_tokens = std::min(b->cap_tokens, b->plan.n_tokens);
  return BG_OK;
}

}  // extern "C"
