// C ABI of linear attention with a decay for each head (include/bitgpu_attn.h): the states' geometry over the
// caller's device memory, the batch (its checks and its upload) and the launches; and of the 4-bit
// projections. Host code only; the kernels live in linear_prologue.hip, linear_attn.hip, linear_chunk.hip and gemv4.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>
#include <new>
#include <vector>

#include "../../include/bitgpu_attn.h"
#include "bg_api_util.h"
#include "bg_linear.h"
#include "bg_paged.h"

struct bg_linear_cache {
  int n_layers, k_heads, v_heads, DK, DV, taps, n_slots, channels;
  float *state, *conv;
  int device = 0;
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

enum { S_HDR, S_SEQS, S_UNITS, N_SECTIONS };
constexpr int kSlots = 2;

struct Plan {
  std::vector<bg::LinSeq> seqs;    // those with new rows, the longest first
  std::vector<bg::LinUnit> units;
  int n_tokens = 0;
  int n_chunked = 0, n_chunk_units = 0;
};

// whether na f32 values at a and nb at b share memory
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const char *x = (const char*)a, *y = (const char*)b;
  return a && b && na && nb && x < y + nb * sizeof(float) && y < x + na * sizeof(float);
}

}  // namespace

struct bg_linear_batch {
  int k_heads, v_heads, DK, DV, n_slots, max_seqs, max_tokens, max_units, device;
  size_t unit_bytes;                // of a chunk in the workspace
  int window;                       // chunks of a pass, at most
  char* ws = nullptr;
  size_t ws_bytes = 0;
  char* dev = nullptr;              // the device block of all sections
  char* host[kSlots] = {};          // pinned staging, one block a slot
  hipEvent_t done[kSlots] = {};     // recorded behind the slot's upload
  bool pending[kSlots] = {};
  int slot = 0;
  size_t at[N_SECTIONS + 1] = {};
  Plan plan, next;
  std::vector<int> writer;          // by slot, while a set is checked
  bool set = false;
  // The stream of the last call: a call on another one first waits there for what the batch has enqueued (its
  // launches read the arrays an upload writes).
  hipStream_t last = nullptr;
  bool used = false;
  hipEvent_t moved = nullptr;
  int cap_tokens = INT_MAX;         // most new rows that launches under capture were made for

  bg::LinBatchView view(bool captured) const {
    bg::LinBatchView b{};
    b.hdr = (const bg::LinHeader*)(dev + at[S_HDR]);
    b.seqs = (const bg::LinSeq*)(dev + at[S_SEQS]);
    b.units = (const bg::LinUnit*)(dev + at[S_UNITS]);
    b.n_tokens = plan.n_tokens;
    b.n_seqs = captured ? std::min(max_seqs, plan.n_tokens) : (int)plan.seqs.size();
    b.n_units = captured ? b.n_seqs + plan.n_tokens / bg::kLinChunk : (int)plan.units.size();
    b.window = window;
    b.longest = plan.seqs.empty() ? 0 : plan.seqs[0].rows;
    if (captured) {
      b.most = std::min(plan.n_tokens, bg::kLinChunkFrom - 1);
      b.n_chunked = std::min(max_seqs, plan.n_tokens / bg::kLinChunkFrom);
      b.n_chunk_units = b.n_chunked ? b.n_chunked + plan.n_tokens / bg::kLinChunk : 0;
    } else {
      b.n_chunked = plan.n_chunked;
      b.n_chunk_units = plan.n_chunk_units;
      b.ws = ws;
      b.most = b.n_seqs > b.n_chunked ? plan.seqs[b.n_chunked].rows : 0;
    }
    return b;
  }
};

namespace {

bg::LinLayer layer_view(const bg_linear_cache* c, int layer) {
  bg::LinLayer L{};
  const size_t at = (size_t)layer * c->n_slots;
  L.state = c->state + at * c->v_heads * c->DV * c->DK;
  L.conv = c->taps ? c->conv + at * (c->taps - 1) * c->channels : nullptr;
  L.k_heads = c->k_heads;
  L.v_heads = c->v_heads;
  L.DK = c->DK;
  L.DV = c->DV;
  L.taps = c->taps;
  L.channels = c->channels;
  return L;
}

int32_t check_pair(const char* who, const bg_linear_cache* c, const bg_linear_batch* b, int32_t layer) {
  if (!c || !b) return fail(BG_E_INVALID, "%s: NULL cache or batch", who);
  if (layer < 0 || layer >= c->n_layers) return fail(BG_E_INVALID, "%s: layer %d out of range", who, layer);
  if (b->k_heads != c->k_heads || b->v_heads != c->v_heads || b->DK != c->DK || b->DV != c->DV || b->n_slots != c->n_slots)
    return fail(BG_E_INVALID, "%s: the batch was made for another cache", who);
  if (!b->set) return fail(BG_E_STATE, "%s: the batch has not been set", who);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != c->device || dev != b->device)
    return fail(BG_E_INVALID, "%s: the cache lives on device %d, the batch on %d, the current device is %d", who, c->device,
                b->device, dev);
  return BG_OK;
}

// Whether the scans of n chunked sequences are one launch: workgroups of 512 threads for 32 value dims of a head each,
// rounded up to eight key heads (linear_chunk.hip), and fewer than 2^32 threads on a grid's axis
bool one_launch(const bg_linear_batch* b, int n) {
  const long long groups = ((long long)n * b->k_heads + 7) / 8 * 8;
  return groups * (b->v_heads / b->k_heads) * (b->DV / 32) * 512 < 1ll << 32;
}

// Orders a call on `st` behind the batch's calls so far. (A launch under capture runs at replay: its order is
// the caller's.)
int32_t join_stream(const char* who, bg_linear_batch* b, hipStream_t st) {
  if (b->used && b->last != st) {
    if (bg::api_capturing(b->last))
      return fail(BG_E_STATE, "%s: the batch worked on a stream that is being captured now", who);
    hipError_t e = hipEventRecord(b->moved, b->last);
    if (e == hipSuccess) e = hipStreamWaitEvent(st, b->moved, 0);
    if (e != hipSuccess) return bg::api_hip_fail(e, "linear batch: the stream of its last call");
  }
  b->last = st;
  b->used = true;
  return BG_OK;
}

void free_batch(bg_linear_batch* b) {
  for (int i = 0; i < kSlots; i++) {
    if (b->host[i]) (void)hipHostFree(b->host[i]);
    if (b->done[i]) (void)hipEventDestroy(b->done[i]);
  }
  if (b->moved) (void)hipEventDestroy(b->moved);
  if (b->dev) (void)hipFree(b->dev);
  if (b->ws) (void)hipFree(b->ws);
  delete b;
}

// The plan of a set in b->next, or what is wrong with it.
int32_t make_plan(bg_linear_batch* b, int32_t n_seqs, const int32_t* rows, const int32_t* slots, const int32_t* sources) {
  Plan& p = b->next;
  p.seqs.clear();
  p.units.clear();
  p.n_chunked = p.n_chunk_units = 0;
  long long T = 0;
  b->writer.assign(b->n_slots, -1);
  for (int s = 0; s < n_seqs; s++) {
    const int src = sources ? sources[s] : slots[s];
    if (rows[s] < 0) return fail(BG_E_INVALID, "bg_linear_batch_set: sequence %d: %d new rows", s, rows[s]);
    if (slots[s] < 0 || slots[s] >= b->n_slots)
      return fail(BG_E_INVALID, "bg_linear_batch_set: sequence %d: slot %d of %d", s, slots[s], b->n_slots);
    if (src < -1 || src >= b->n_slots)
      return fail(BG_E_INVALID, "bg_linear_batch_set: sequence %d: source %d of %d slots", s, src, b->n_slots);
    if (rows[s] > 0) {
      if (b->writer[slots[s]] >= 0)
        return fail(BG_E_INVALID, "bg_linear_batch_set: slot %d is written by sequences %d and %d", slots[s], b->writer[slots[s]], s);
      b->writer[slots[s]] = s;
    }
    if (T + rows[s] > b->max_tokens)
      return fail(BG_E_INVALID, "bg_linear_batch_set: %lld new rows up to sequence %d, the batch holds %d", T + rows[s], s, b->max_tokens);
    if (rows[s] > 0) p.seqs.push_back(bg::LinSeq{(int)T, rows[s], src, slots[s], s, 0, {}});
    T += rows[s];
  }
  for (const bg::LinSeq& q : p.seqs)
    if (q.src >= 0 && b->writer[q.src] >= 0 && b->writer[q.src] != q.unit0)
      return fail(BG_E_INVALID, "bg_linear_batch_set: slot %d is read by sequence %d and written by sequence %d", q.src, q.unit0,
                  b->writer[q.src]);
  std::stable_sort(p.seqs.begin(), p.seqs.end(), [](const bg::LinSeq& x, const bg::LinSeq& y) { return x.rows > y.rows; });
  for (size_t i = 0; i < p.seqs.size(); i++) {
    bg::LinSeq& q = p.seqs[i];
    q.unit0 = (int)p.units.size();
    for (int r = 0; r < q.rows; r += bg::kLinChunk)
      p.units.push_back(bg::LinUnit{(int)i, q.row0 + r, std::min(bg::kLinChunk, q.rows - r), r / bg::kLinChunk});
    q.n_units = (int)p.units.size() - q.unit0;
    if (q.rows >= bg::kLinChunkFrom) {
      p.n_chunked = (int)i + 1;
      p.n_chunk_units = (int)p.units.size();
    }
  }
  p.n_tokens = (int)T;
  return BG_OK;
}

}  // namespace

extern "C" {

int32_t bg_linear_create(int32_t n_layers, int32_t k_heads, int32_t v_heads, int32_t k_dim, int32_t v_dim, int32_t conv_width,
                         int32_t n_slots, float* state, float* conv, bg_linear_cache** out) {
  if (!out) return fail(BG_E_INVALID, "bg_linear_create: out is NULL");
  *out = nullptr;
  if (n_layers < 1 || k_heads < 1 || v_heads < 1 || n_slots < 1)
    return fail(BG_E_INVALID, "bg_linear_create: n_layers %d, k_heads %d, v_heads %d, n_slots %d must be >= 1", n_layers, k_heads,
                v_heads, n_slots);
  if (v_heads % k_heads) return fail(BG_E_INVALID, "bg_linear_create: v_heads %d must be a multiple of k_heads %d", v_heads, k_heads);
  if ((k_dim != 64 && k_dim != 128) || (v_dim != 64 && v_dim != 128))
    return fail(BG_E_UNSUPPORTED, "bg_linear_create: k_dim %d, v_dim %d unsupported (64 or 128)", k_dim, v_dim);
  if (conv_width != 0 && (conv_width < 2 || conv_width > 4))
    return fail(BG_E_UNSUPPORTED, "bg_linear_create: conv_width %d unsupported (2 to 4, 0: no convolution)", conv_width);
  if (v_heads > 4096 || n_layers > (1 << 16) || n_slots > (1 << 24) ||  // a grid's heads; a state's bytes below 2^63
      (long double)n_layers * n_slots * v_heads * v_dim * k_dim * sizeof(float) >= 0x1p63L)
    return fail(BG_E_UNSUPPORTED, "bg_linear_create: v_heads %d, n_layers %d or n_slots %d too large", v_heads, n_layers, n_slots);
  if (!state || (conv_width != 0) != (conv != nullptr))
    return fail(BG_E_INVALID, "bg_linear_create: state is NULL, or conv and conv_width do not belong together");
  if (((uintptr_t)state | (uintptr_t)conv) & 15) return fail(BG_E_INVALID, "bg_linear_create: buffers must be 16-byte aligned");
  bg_linear_cache* c = new (std::nothrow) bg_linear_cache();
  if (!c) return fail(BG_E_OOM, "bg_linear_create: out of host memory");
  c->n_layers = n_layers;
  c->k_heads = k_heads;
  c->v_heads = v_heads;
  c->DK = k_dim;
  c->DV = v_dim;
  c->taps = conv_width;
  c->n_slots = n_slots;
  c->channels = 2 * k_heads * k_dim + v_heads * v_dim;
  c->state = state;
  c->conv = conv;
  const hipError_t e = hipGetDevice(&c->device);
  if (e != hipSuccess) {
    delete c;
    return bg::api_hip_fail(e, "bg_linear_create: current device");
  }
  *out = c;
  return BG_OK;
}

int32_t bg_linear_destroy(bg_linear_cache* c) {
  delete c;  // the memory is the caller's
  return BG_OK;
}

int32_t bg_linear_batch_create(const bg_linear_cache* c, int32_t max_seqs, int32_t max_tokens, bg_linear_batch** out) {
  if (!out) return fail(BG_E_INVALID, "bg_linear_batch_create: out is NULL");
  *out = nullptr;
  if (!c) return fail(BG_E_INVALID, "bg_linear_batch_create: NULL cache");
  if (max_seqs < 1 || max_tokens < 1)
    return fail(BG_E_INVALID, "bg_linear_batch_create: max_seqs %d, max_tokens %d must be >= 1", max_seqs, max_tokens);
  if (max_seqs > 65535 || max_tokens > (1 << 26))  // a grid's second axis; unit and row numbers
    return fail(BG_E_UNSUPPORTED, "bg_linear_batch_create: max_seqs %d or max_tokens %d too large", max_seqs, max_tokens);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != c->device)
    return fail(BG_E_INVALID, "bg_linear_batch_create: the cache lives on device %d, the current device is %d", c->device, dev);
  bg_linear_batch* b = new (std::nothrow) bg_linear_batch();
  if (!b) return fail(BG_E_OOM, "bg_linear_batch_create: out of host memory");
  b->k_heads = c->k_heads;
  b->v_heads = c->v_heads;
  b->DK = c->DK;
  b->DV = c->DV;
  b->n_slots = c->n_slots;
  b->max_seqs = max_seqs;
  b->max_tokens = max_tokens;
  b->max_units = std::min(max_seqs, max_tokens) + max_tokens / bg::kLinChunk;
  b->device = dev;
  b->unit_bytes = bg::linear_unit_bytes(c->DK, c->k_heads, c->v_heads);
  b->window = (int)std::max<size_t>(1, bg::kLinSpace / b->unit_bytes);
  const size_t bytes[N_SECTIONS] = {sizeof(bg::LinHeader), (size_t)std::min(max_seqs, max_tokens) * sizeof(bg::LinSeq),
                                    (size_t)b->max_units * sizeof(bg::LinUnit)};
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
    return bg::api_hip_fail(e, "linear batch allocation");
  }
  *out = b;
  return BG_OK;
}

int32_t bg_linear_batch_destroy(bg_linear_batch* b) {
  if (!b) return BG_OK;
  (void)hipDeviceSynchronize();
  free_batch(b);
  return BG_OK;
}

int32_t bg_linear_batch_set(bg_linear_batch* b, int32_t n_seqs, const int32_t* rows, const int32_t* slots, const int32_t* sources,
                            void* stream) {
  if (!b) return fail(BG_E_INVALID, "bg_linear_batch_set: NULL batch");
  if (n_seqs < 0 || (n_seqs > 0 && (!rows || !slots))) return fail(BG_E_INVALID, "bg_linear_batch_set: n_seqs %d need rows and slots", n_seqs);
  if (n_seqs > b->max_seqs) return fail(BG_E_INVALID, "bg_linear_batch_set: %d sequences, the batch holds %d", n_seqs, b->max_seqs);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != b->device)
    return fail(BG_E_INVALID, "bg_linear_batch_set: the batch lives on device %d, the current device is %d", b->device, dev);
  hipStream_t st = (hipStream_t)stream;
  if (bg::api_capturing(st))
    return fail(BG_E_STATE, "bg_linear_batch_set: a batch is set outside graph capture (its launches read it at replay)");
  try {
    const int32_t wrong = make_plan(b, n_seqs, rows, slots, sources);
    if (wrong != BG_OK) return wrong;
  } catch (const std::exception&) {  // the plan's arrays
    return fail(BG_E_OOM, "bg_linear_batch_set: out of host memory");
  }
  const Plan& p = b->next;
  if (p.n_tokens > b->cap_tokens)
    return fail(BG_E_STATE, "bg_linear_batch_set: %d new rows, but launches of this batch were captured with %d", p.n_tokens, b->cap_tokens);
  if (!one_launch(b, p.n_chunked))
    return fail(BG_E_UNSUPPORTED, "bg_linear_batch_set: %d sequences of at least %d new rows are too many at once for %d heads", p.n_chunked,
                bg::kLinChunkFrom, b->v_heads);
  const int32_t rc = join_stream("bg_linear_batch_set", b, st);
  if (rc != BG_OK) return rc;
  const int slot = b->slot;
  if (b->pending[slot]) {
    const hipError_t e = hipEventSynchronize(b->done[slot]);
    if (e != hipSuccess) return bg::api_hip_fail(e, "linear batch staging");
    b->pending[slot] = false;
  }
  const size_t need = std::min(p.n_chunk_units, b->window) * b->unit_bytes;
  char* ws = b->ws;
  size_t ws_bytes = b->ws_bytes;
  if (need > ws_bytes) {
    ws_bytes = std::min(std::max(need, 2 * ws_bytes), b->window * b->unit_bytes);  // at least twofold: few are ever replaced
    hipError_t e = hipMalloc((void**)&ws, ws_bytes);
    if (e != hipSuccess && ws_bytes > need) {
      (void)hipGetLastError();
      e = hipMalloc((void**)&ws, ws_bytes = need);
    }
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return bg::api_hip_fail(e, "linear attention workspace allocation");
    }
  }
  char* h = b->host[slot];
  bg::LinHeader hdr{(int)p.seqs.size(), p.n_tokens, (int)p.units.size(), p.n_chunked, p.n_chunk_units, 0, ws};
  bg::PagedUpload up{};
  auto put = [&](int section, const void* src, size_t bytes) {
    if (bytes) memcpy(h + b->at[section], src, bytes);
    up.src[section] = h + b->at[section];
    up.dst[section] = b->dev + b->at[section];
    up.n16[section] = (unsigned)((bytes + 15) / 16);
  };
  put(S_HDR, &hdr, sizeof(hdr));
  put(S_SEQS, p.seqs.data(), p.seqs.size() * sizeof(bg::LinSeq));
  put(S_UNITS, p.units.data(), p.units.size() * sizeof(bg::LinUnit));
  hipError_t e = bg::launch_paged_upload(up, st);
  if (e != hipSuccess) {
    if (ws != b->ws) (void)hipFree(ws);  // no launch knows it; those of before and captured ones keep the old
    b->set = false;
    return bg::api_hip_fail(e, "linear batch upload");
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
    return bg::api_hip_fail(e, "linear batch upload");
  }
  b->pending[slot] = true;
  b->slot = (slot + 1) % kSlots;
  std::swap(b->plan, b->next);
  b->set = true;
  return BG_OK;
}

int32_t bg_linear_prologue(const bg_linear_cache* c, int32_t layer, bg_linear_batch* b, const float* qkv, const float* conv_weight,
                           const float* a, const float* bb, int32_t ab_stride, const float* a_log, const float* dt_bias, float* q,
                           float* k, float* v, float* g, float* beta, void* stream) {
  const int32_t rc = check_pair("bg_linear_prologue", c, b, layer);
  if (rc != BG_OK) return rc;
  if (!c->taps) return fail(BG_E_STATE, "bg_linear_prologue: the cache has no convolution");
  hipStream_t st = (hipStream_t)stream;
  const bool captured = bg::api_capturing(st);
  const size_t T = b->plan.n_tokens;
  if (T == 0) {
    if (captured) b->cap_tokens = 0;
    return BG_OK;
  }
  if (!qkv || !conv_weight || !q || !k || !v) return fail(BG_E_INVALID, "bg_linear_prologue: NULL argument");
  if (g && (!a || !a_log || !dt_bias)) return fail(BG_E_INVALID, "bg_linear_prologue: g needs a, a_log and dt_bias");
  if (beta && !bb) return fail(BG_E_INVALID, "bg_linear_prologue: beta needs b");
  if ((g || beta) && ab_stride < c->v_heads) return fail(BG_E_INVALID, "bg_linear_prologue: ab_stride %d < v_heads %d", ab_stride, c->v_heads);
  if (((uintptr_t)qkv | (uintptr_t)conv_weight | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15)
    return fail(BG_E_INVALID, "bg_linear_prologue: buffers must be 16-byte aligned");
  const size_t nk = T * c->k_heads * c->DK, nv = T * c->v_heads * c->DV, ng = T * c->v_heads, na = (T - 1) * ab_stride + c->v_heads;
  const struct { const void* p; size_t n; } in[] = {{qkv, T * c->channels}, {conv_weight, (size_t)c->channels * c->taps},
                                                    {g ? a : nullptr, na}, {beta ? bb : nullptr, na},
                                                    {g ? a_log : nullptr, (size_t)c->v_heads}, {g ? dt_bias : nullptr, (size_t)c->v_heads}},
                                             o[] = {{q, nk}, {k, nk}, {v, nv}, {g, ng}, {beta, ng}};
  for (int i = 0; i < 5; i++) {
    for (const auto& x : in)
      if (overlap(o[i].p, o[i].n, x.p, x.n)) return fail(BG_E_INVALID, "bg_linear_prologue: an output overlaps an input");
    for (int j = 0; j < i; j++)
      if (overlap(o[i].p, o[i].n, o[j].p, o[j].n)) return fail(BG_E_INVALID, "bg_linear_prologue: two outputs overlap");
  }
  if (!captured) {
    const int32_t moved = join_stream("bg_linear_prologue", b, st);
    if (moved != BG_OK) return moved;
  }
  const bg::LinPrologueArgs args{qkv, conv_weight, a, bb, ab_stride, a_log, dt_bias, q, k, v, g, beta};
  const hipError_t e = bg::launch_linear_prologue(layer_view(c, layer), b->view(captured), args, st);
  if (e != hipSuccess) return bg::api_hip_fail(e, "linear prologue launch");
  if (captured) b->cap_tokens = std::min(b->cap_tokens, b->plan.n_tokens);
  return BG_OK;
}

int32_t bg_linear_attention(const bg_linear_cache* c, int32_t layer, bg_linear_batch* b, const float* q, const float* k,
                            const float* v, const float* g, int32_t g_stride, const float* beta, float scale, const float* gate,
                            const float* norm, float eps, float* out, void* stream) {
  const int32_t rc = check_pair("bg_linear_attention", c, b, layer);
  if (rc != BG_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  const bool captured = bg::api_capturing(st);
  const size_t T = b->plan.n_tokens;
  if (T == 0) {
    if (captured) b->cap_tokens = 0;
    return BG_OK;
  }
  if (!q || !k || !v || !g || !out) return fail(BG_E_INVALID, "bg_linear_attention: NULL argument");
  if (g_stride != 0 && g_stride < c->v_heads) return fail(BG_E_INVALID, "bg_linear_attention: g_stride %d < v_heads %d", g_stride, c->v_heads);
  if (!std::isfinite(scale)) return fail(BG_E_INVALID, "bg_linear_attention: scale is not finite");
  if (gate && !norm) return fail(BG_E_INVALID, "bg_linear_attention: gate needs norm");
  if (norm && !(eps >= 0.0f)) return fail(BG_E_INVALID, "bg_linear_attention: eps must not be negative");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)gate | (uintptr_t)norm | (uintptr_t)out) & 15)
    return fail(BG_E_INVALID, "bg_linear_attention: buffers must be 16-byte aligned");
  const size_t nk = T * c->k_heads * c->DK, nv = T * c->v_heads * c->DV, H = c->v_heads;
  const struct { const void* p; size_t n; } in[] = {{q, nk}, {k, nk}, {v, nv}, {g, g_stride ? (T - 1) * g_stride + H : H},
                                                    {beta, T * H}, {gate, nv}, {norm, (size_t)c->DV}};
  for (const auto& x : in)
    if (overlap(out, nv, x.p, x.n)) return fail(BG_E_INVALID, "bg_linear_attention: out overlaps an input");
  const bg::LinBatchView batch = b->view(captured);
  if (!one_launch(b, batch.n_chunked))
    return fail(BG_E_UNSUPPORTED, "bg_linear_attention: any batch of %d new rows, for a graph, may be too many sequences for %d heads",
                b->plan.n_tokens, c->v_heads);
  if (!captured) {
    const int32_t moved = join_stream("bg_linear_attention", b, st);
    if (moved != BG_OK) return moved;
  }
  const bg::LinAttnArgs args{q, k, v, g, g_stride, beta, scale, gate, norm, eps, out};
  const bg::LinLayer view = layer_view(c, layer);
  hipError_t e = hipSuccess;
  if (captured || batch.n_seqs > batch.n_chunked) e = bg::launch_linear_rows(view, batch, args, st);
  if (e == hipSuccess && batch.n_chunk_units) e = bg::launch_linear_chunks(view, batch, args, st);
  if (e != hipSuccess) return bg::api_hip_fail(e, "linear attention launch");
  if (captured) b->cap_tokens = std::min(b->cap_tokens, b->plan.n_tokens);
  return BG_OK;
}

static int32_t check_gemv4(const char* who, const bg::Gemv4Args& a, int32_t scale_type) {
  if (a.M < 0 || a.M > 16) return fail(BG_E_UNSUPPORTED, "%s: %d rows (at most 16)", who, a.M);
  if (a.K < 128 || a.K % 128) return fail(BG_E_INVALID, "%s: K %d must be a positive multiple of 128", who, a.K);
  if (a.K > (1 << 24)) return fail(BG_E_UNSUPPORTED, "%s: K %d too large", who, a.K);  // a workgroup's 128 rows in 32-bit offsets
  if (a.group != 32 && a.group != 64 && a.group != 128) return fail(BG_E_UNSUPPORTED, "%s: group %d unsupported (32, 64 or 128)", who, a.group);
  if (scale_type != BG_KV_F32 && scale_type != BG_KV_F16) return fail(BG_E_INVALID, "%s: unknown scale type %d", who, scale_type);
  if (a.N0 < 0 || a.N1 < 0 || a.N2 < 0 || (long long)a.N0 + a.N1 + a.N2 > INT_MAX / 16)
    return fail(BG_E_INVALID, "%s: output ranges %d/%d/%d", who, a.N0, a.N1, a.N2);
  if (a.M == 0 || a.N0 + a.N1 + a.N2 == 0) return BG_OK;
  if (!a.x || !a.codes || !a.scales) return fail(BG_E_INVALID, "%s: NULL argument", who);
  if ((a.N0 && !a.out0) || (a.N1 && !a.out1) || (a.N2 && !a.out2))
    return fail(BG_E_INVALID, "%s: output ranges %d/%d/%d need their buffers", who, a.N0, a.N1, a.N2);
  const size_t room = bg::gemv4_room(a.M, a.K) / 4;
  if (room && !a.room) return fail(BG_E_INVALID, "%s: %d rows need a workspace", who, a.M);
  if (((uintptr_t)a.x | (uintptr_t)a.codes | (uintptr_t)a.scales | (uintptr_t)a.mins | (uintptr_t)(room ? a.room : nullptr)) & 15)
    return fail(BG_E_INVALID, "%s: x, codes, scales, mins and the workspace must be 16-byte aligned", who);
  const size_t M = a.M, K = a.K, N = (size_t)a.N0 + a.N1 + a.N2;
  const struct { const void* p; size_t n; } o[] = {{a.out0, M * a.N0}, {a.out1, M * a.N1}, {a.out2, M * a.N2}, {a.room, room}};
  const size_t sc = (N * (K / a.group) * (a.scale_f16 ? 2 : 4) + 3) / 4;
  for (int i = 0; i < 4; i++) {
    if (overlap(o[i].p, o[i].n, a.x, M * K) || overlap(o[i].p, o[i].n, a.codes, N * K / 8) || overlap(o[i].p, o[i].n, a.scales, sc) ||
        overlap(o[i].p, o[i].n, a.mins, sc))
      return fail(BG_E_INVALID, "%s: an output or the workspace overlaps an input", who);
    for (int j = 0; j < i; j++)
      if (overlap(o[i].p, o[i].n, o[j].p, o[j].n)) return fail(BG_E_INVALID, "%s: two outputs, or one and the workspace, overlap", who);
  }
  if (overlap(a.room, room, a.resid, M * N)) return fail(BG_E_INVALID, "%s: the workspace overlaps resid", who);
  return BG_OK;
}

int64_t bg_gemv4_workspace(int32_t rows, int32_t K) { return rows > 16 || K < 1 ? 0 : (int64_t)bg::gemv4_room(rows, K); }

int32_t bg_gemv4_split(const float* x, int32_t rows, int32_t K, const uint32_t* codes, const void* scales, const void* mins,
                       int32_t scale_type, int32_t group, int32_t N0, int32_t N1, int32_t N2, float* out0, float* out1, float* out2,
                       void* workspace, void* stream) {
  const bg::Gemv4Args a{x, rows, K, codes, scales, mins, scale_type == BG_KV_F16, group, N0, N1, N2, out0, out1, out2, nullptr, (char*)workspace};
  const int32_t rc = check_gemv4("bg_gemv4_split", a, scale_type);
  if (rc != BG_OK) return rc;
  const hipError_t e = bg::launch_gemv4(a, (hipStream_t)stream);
  return e == hipSuccess ? BG_OK : bg::api_hip_fail(e, "gemv4 launch");
}

int32_t bg_gemv4_resid(const float* x, int32_t rows, int32_t K, const uint32_t* codes, const void* scales, const void* mins,
                       int32_t scale_type, int32_t group, int32_t N, const float* resid, float* y, void* workspace,
                       void* stream) {
  const bg::Gemv4Args a{x, rows, K, codes, scales, mins, scale_type == BG_KV_F16, group, N, 0, 0, y, nullptr, nullptr, resid, (char*)workspace};
  const int32_t rc = check_gemv4("bg_gemv4_resid", a, scale_type);
  if (rc != BG_OK) return rc;
  if (rows && N && !resid) return fail(BG_E_INVALID, "bg_gemv4_resid: resid is NULL");
  if (resid != y && overlap(y, (size_t)rows * N, resid, (size_t)rows * N))
    return fail(BG_E_INVALID, "bg_gemv4_resid: y overlaps resid and is not resid");
  const hipError_t e = bg::launch_gemv4(a, (hipStream_t)stream);
  return e == hipSuccess ? BG_OK : bg::api_hip_fail(e, "gemv4 launch");
}

}  // extern "C"
