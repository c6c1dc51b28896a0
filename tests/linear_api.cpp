// The C entries of linear attention and the 4-bit projections (linear_api.hip, host code) against a stand-in for the
// HIP runtime and the launches: what is refused, which call orders itself behind which, what an upload holds, what a
// launch is told, and how the workspace grows. Memory is the host's; every call that matters is written down.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "../bitgpu_amd/csrc/bg_api_util.h"
#include "../bitgpu_amd/csrc/bg_linear.h"
#include "../bitgpu_amd/csrc/bg_paged.h"
#include "../include/bitgpu_attn.h"

static std::vector<std::string> calls;
static std::set<hipStream_t> capturing_now;
static std::string message;
static int fail_record = 0, fail_upload = 0;
static size_t most_memory = ~(size_t)0;
static std::map<char*, size_t> blocks;
static uintptr_t events = 0;

static void note(const char* fmt, ...) {
  char b[200];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(b, sizeof(b), fmt, ap);
  va_end(ap);
  calls.push_back(b);
}
static int sid(hipStream_t s) { return (int)(uintptr_t)s; }
static hipStream_t stream(int i) { return (hipStream_t)(uintptr_t)i; }

// blocks with a guard behind them, checked when they go
static hipError_t take(void** p, size_t n) {
  char* b = (char*)malloc(n + 64);
  memset(b, 0xcd, n + 64);
  blocks[b] = n;
  *p = b;
  return hipSuccess;
}
static hipError_t give(void* p) {
  auto it = blocks.find((char*)p);
  if (it == blocks.end()) abort();
  for (int i = 0; i < 64; i++)
    if ((unsigned char)it->first[it->second + i] != 0xcd) abort();
  free(p);
  blocks.erase(it);
  return hipSuccess;
}
static bool inside(const void* p, size_t n) {
  auto it = blocks.upper_bound((char*)p);
  if (it == blocks.begin()) return false;
  --it;
  return (char*)p >= it->first && (char*)p + n <= it->first + it->second;
}

extern "C" {
hipError_t hipMalloc(void** p, size_t n) { return n > most_memory ? hipErrorOutOfMemory : take(p, n); }
hipError_t hipFree(void* p) { note("free"); return give(p); }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return take(p, n); }
hipError_t hipHostFree(void* p) { return give(p); }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { *v = 256; return hipSuccess; }
hipError_t hipDeviceSynchronize(void) { note("sync"); return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { *e = (hipEvent_t)++events; return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) {
  if (fail_record) return hipErrorInvalidHandle;
  note("record %d on %d", (int)(uintptr_t)e, sid(s));
  return hipSuccess;
}
hipError_t hipStreamWaitEvent(hipStream_t s, hipEvent_t e, unsigned) { note("%d waits for %d", sid(s), (int)(uintptr_t)e); return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t e) { note("host waits for %d", (int)(uintptr_t)e); return hipSuccess; }
}


namespace bg {
int32_t api_fail(int32_t code, const char* msg) { message = msg; return code; }
int32_t api_hip_fail(hipError_t e, const char* what) { message = what; return e == hipErrorOutOfMemory ? BG_E_OOM : BG_E_DEVICE; }
bool api_capturing(hipStream_t st) { return capturing_now.count(st) != 0; }
hipError_t launch_paged_upload(const PagedUpload& u, hipStream_t st) {
  if (fail_upload) return hipErrorUnknown;
  note("upload on %d", sid(st));
  for (int i = 0; i < 9; i++) {
    if (!u.n16[i]) continue;
    if (!inside(u.src[i], 16 * (size_t)u.n16[i]) || !inside(u.dst[i], 16 * (size_t)u.n16[i])) abort();
    memcpy(u.dst[i], u.src[i], 16 * (size_t)u.n16[i]);
  }
  return hipSuccess;
}
static LinBatchView seen;
static LinLayer layer;
static Gemv4Args product;
hipError_t launch_linear_prologue(const LinLayer& L, const LinBatchView& b, const LinPrologueArgs&, hipStream_t st) {
  seen = b;
  layer = L;
  note("prologue on %d", sid(st));
  return hipSuccess;
}
hipError_t launch_linear_rows(const LinLayer& L, const LinBatchView& b, const LinAttnArgs&, hipStream_t st) {
  seen = b;
  layer = L;
  note("rows on %d", sid(st));
  return hipSuccess;
}
hipError_t launch_linear_chunks(const LinLayer&, const LinBatchView& b, const LinAttnArgs&, hipStream_t st) {
  seen = b;
  note("chunks on %d", sid(st));
  return hipSuccess;
}
size_t linear_unit_bytes(int, int, int) { return bg::kLinSpace / 32; }
size_t gemv4_room(int M, int) { return M <= 4 ? 0 : 4096; }
hipError_t launch_gemv4(const Gemv4Args& a, hipStream_t st) {
  product = a;
  note("product on %d", sid(st));
  return hipSuccess;
}
}  // namespace bg

static int line_of_fault(int line, const char* what) {
  printf("line %d: %s\nmessage: %s\n", line, what, message.c_str());
  for (auto& c : calls) printf("  %s\n", c.c_str());
  exit(1);
}
#define CHECK(x) do { if (!(x)) line_of_fault(__LINE__, #x); } while (0)
static void expect(int line, std::vector<std::string> want) {
  if (calls != want) {
    for (auto& w : want) printf("wanted %s\n", w.c_str());
    line_of_fault(line, "calls");
  }
  calls.clear();
}
#define EXPECT(...) expect(__LINE__, std::vector<std::string>{__VA_ARGS__})


alignas(256) static float buf[1 << 20];
static float* at(size_t i) { return buf + i; }

// 1 key head, 2 value heads of 64 x 64: 64 | 64 | 128 channels
struct Batch {
  bg_linear_cache* c = nullptr;
  bg_linear_batch* b = nullptr;
  int moved, done0, done1;
  Batch(int max_seqs = 8, int max_tokens = 4096, int taps = 4) {
    CHECK(bg_linear_create(3, 1, 2, 64, 64, taps, 6, buf, taps ? buf : nullptr, &c) == BG_OK);
    moved = (int)events + 1;
    done0 = moved + 1;
    done1 = moved + 2;
    CHECK(bg_linear_batch_create(c, max_seqs, max_tokens, &b) == BG_OK);
    calls.clear();
  }
  ~Batch() {
    bg_linear_batch_destroy(b);
    bg_linear_destroy(c);
    calls.clear();
  }
  int32_t set(std::vector<int32_t> rows, std::vector<int32_t> slots, int st = 0, std::vector<int32_t> sources = {}) {
    return bg_linear_batch_set(b, (int)rows.size(), rows.data(), slots.data(), sources.empty() ? nullptr : sources.data(), stream(st));
  }
  int32_t attend(int st, int layer = 0) {
    return bg_linear_attention(c, layer, b, at(0), at(1 << 17), at(1 << 18), at(1 << 19), 2, nullptr, 1.0f, nullptr, nullptr, 1e-6f,
                               at(3 << 18), stream(st));
  }
  int32_t open(int st) {
    return bg_linear_prologue(c, 1, b, at(0), at(1 << 16), at(600000), at(600002), 4, at(700000), at(700008), at(1 << 17), at(3 << 16),
                              at(1 << 18), at(1 << 19), at(540000), stream(st));
  }
  std::string record(int e, int s) { return "record " + std::to_string(e) + " on " + std::to_string(s); }
  std::string wait(int s, int e) { return std::to_string(s) + " waits for " + std::to_string(e); }
};

static void caches() {
  bg_linear_cache* c = (bg_linear_cache*)buf;
  auto make = [&](int layers, int kh, int vh, int dk, int dv, int taps, int slots, float* state, float* conv) {
    const int32_t rc = bg_linear_create(layers, kh, vh, dk, dv, taps, slots, state, conv, &c);
    if (rc == BG_OK) bg_linear_destroy(c);
    else CHECK(!c);
    return rc;
  };
  CHECK(make(1, 2, 4, 128, 64, 4, 1, buf, buf) == BG_OK && make(1, 1, 1, 64, 64, 0, 1, buf, nullptr) == BG_OK);
  for (int i = 0; i < 5; i++) {
    int v[5] = {1, 1, 1, 4, 1};
    v[i] = i == 3 ? -1 : 0;
    CHECK(make(v[0], v[1], v[2], 64, 64, v[3], v[4], buf, buf) == (i == 3 ? BG_E_UNSUPPORTED : BG_E_INVALID));
  }
  CHECK(make(1, 2, 3, 64, 64, 4, 1, buf, buf) == BG_E_INVALID);                       // value heads of no key head
  CHECK(make(1, 1, 1, 96, 64, 4, 1, buf, buf) == BG_E_UNSUPPORTED && make(1, 1, 1, 64, 256, 4, 1, buf, buf) == BG_E_UNSUPPORTED);
  CHECK(make(1, 1, 1, 64, 64, 1, 1, buf, buf) == BG_E_UNSUPPORTED && make(1, 1, 1, 64, 64, 5, 1, buf, buf) == BG_E_UNSUPPORTED);
  CHECK(make(1, 1, 8192, 64, 64, 4, 1, buf, buf) == BG_E_UNSUPPORTED && make(1, 1, 1, 64, 64, 4, 1 << 25, buf, buf) == BG_E_UNSUPPORTED);
  CHECK(make(1, 1, 1, 64, 64, 4, 1, nullptr, buf) == BG_E_INVALID && make(1, 1, 1, 64, 64, 4, 1, buf, nullptr) == BG_E_INVALID);
  CHECK(make(1, 1, 1, 64, 64, 0, 1, buf, buf) == BG_E_INVALID && make(1, 1, 1, 64, 64, 4, 1, buf + 1, buf) == BG_E_INVALID);
  CHECK(bg_linear_create(1, 1, 1, 64, 64, 4, 1, buf, buf, nullptr) == BG_E_INVALID);
  bg_linear_batch* b = nullptr;
  CHECK(bg_linear_batch_create(nullptr, 1, 1, &b) == BG_E_INVALID && bg_linear_batch_set(nullptr, 0, nullptr, nullptr, nullptr, nullptr) == BG_E_INVALID);
  Batch x;
  CHECK(bg_linear_batch_create(x.c, 0, 1, &b) == BG_E_INVALID && bg_linear_batch_create(x.c, 1, 0, &b) == BG_E_INVALID);
  CHECK(bg_linear_batch_create(x.c, 1 << 16, 1, &b) == BG_E_UNSUPPORTED && bg_linear_batch_create(x.c, 1, (1 << 26) + 1, &b) == BG_E_UNSUPPORTED);
  CHECK(bg_linear_batch_create(x.c, 1, 1, nullptr) == BG_E_INVALID && !b);
  CHECK(bg_linear_destroy(nullptr) == BG_OK && bg_linear_batch_destroy(nullptr) == BG_OK);
}

static void sets() {
  Batch x(4, 300);
  CHECK(x.attend(0) == BG_E_STATE && x.open(0) == BG_E_STATE);                        // not set
  CHECK(x.set({1, 1}, {0, 0}) == BG_E_INVALID);                                       // one slot, two writers
  CHECK(x.set({1, -1}, {0, 1}) == BG_E_INVALID && x.set({1}, {6}) == BG_E_INVALID && x.set({1}, {-1}) == BG_E_INVALID);
  CHECK(x.set({1}, {0}, 0, {6}) == BG_E_INVALID && x.set({1}, {0}, 0, {-2}) == BG_E_INVALID);
  CHECK(x.set({1, 1}, {0, 1}, 0, {1, 1}) == BG_E_INVALID);                            // reads what another writes
  CHECK(x.set({301}, {0}) == BG_E_INVALID && x.set({200, 101}, {0, 1}) == BG_E_INVALID);
  CHECK(x.set({0x7fffffff, 0x7fffffff}, {0, 1}) == BG_E_INVALID);
  CHECK(x.set({1, 1, 1, 1, 1}, {0, 1, 2, 3, 4}) == BG_E_INVALID);
  CHECK(bg_linear_batch_set(x.b, -1, nullptr, nullptr, nullptr, nullptr) == BG_E_INVALID);
  CHECK(bg_linear_batch_set(x.b, 1, nullptr, nullptr, nullptr, nullptr) == BG_E_INVALID);
  EXPECT();
  CHECK(x.attend(0) == BG_E_STATE);
  CHECK(x.set({0, 1, 0}, {2, 2, 2}, 0, {2, -1, 2}) == BG_OK);                         // without rows a slot is not written
  CHECK(x.set({1, 1, 1}, {0, 1, 2}, 0, {5, 5, 2}) == BG_OK);                          // two forks of one state
  calls.clear();
  // longest first, units of 64 rows, slots and sources
  CHECK(x.set({3, 0, 150, 28}, {4, 0, 5, 1}, 0, {-1, 0, 3, 1}) == BG_OK && x.attend(0, 2) == BG_OK && x.open(0) == BG_OK);
  const bg::LinBatchView& v = bg::seen;
  CHECK(v.n_seqs == 3 && v.n_tokens == 181 && v.n_units == 5 && v.n_chunked == 2 && v.n_chunk_units == 4 && v.most == 3 && v.ws);
  CHECK(v.hdr->n_seqs == 3 && v.hdr->n_tokens == 181 && v.hdr->n_units == 5 && v.hdr->n_chunked == 2 && v.hdr->n_chunk_units == 4 && v.hdr->ws == v.ws);
  const int seqs[3][6] = {{3, 150, 3, 5, 0, 3}, {153, 28, 1, 1, 3, 1}, {0, 3, -1, 4, 4, 1}};
  for (int i = 0; i < 3; i++) CHECK(memcmp(&v.seqs[i], seqs[i], sizeof(seqs[i])) == 0);
  const int units[5][4] = {{0, 3, 64, 0}, {0, 67, 64, 1}, {0, 131, 22, 2}, {1, 153, 28, 0}, {2, 0, 3, 0}};
  CHECK(memcmp(v.units, units, sizeof(units)) == 0);
  CHECK(bg::layer.state == buf + (size_t)6 * 2 * 64 * 64 && bg::layer.conv == buf + (size_t)6 * 3 * 256);  // (the prologue's layer)
  EXPECT("host waits for " + std::to_string(x.done0), "upload on 0", x.record(x.done0, 0), "rows on 0", "chunks on 0", "prologue on 0");
  // only long ones, only short ones, none
  CHECK(x.set({28}, {0}) == BG_OK && x.attend(0) == BG_OK);
  CHECK(calls.back() == "chunks on 0" && std::count(calls.begin(), calls.end(), "rows on 0") == 0);
  CHECK(x.set({27}, {0}) == BG_OK);
  calls.clear();
  CHECK(x.attend(0) == BG_OK);
  EXPECT("rows on 0");
  CHECK(bg::seen.most == 27);
  CHECK(x.set({}, {}) == BG_OK && x.set({0}, {0}) == BG_OK);
  calls.clear();
  CHECK(x.attend(3) == BG_OK && x.open(3) == BG_OK);
  EXPECT();
}

static void arguments() {
  Batch x;
  CHECK(x.set({10}, {0}) == BG_OK);
  calls.clear();
  CHECK(x.attend(0, 3) == BG_E_INVALID && x.attend(0, -1) == BG_E_INVALID);
  float *q = at(0), *k = at(1 << 17), *v = at(1 << 18), *g = at(1 << 19), *o = at(3 << 18), *w = at(600000);
  auto attend = [&](float* q, float* k, float* v, float* g, int gs, float* beta, float scale, float* gate, float* norm, float eps, float* o) {
    return bg_linear_attention(x.c, 0, x.b, q, k, v, g, gs, beta, scale, gate, norm, eps, o, nullptr);
  };
  CHECK(attend(q, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o) == BG_OK && attend(q, k, v, g, 0, g, 1, v, w, 0, o) == BG_OK);
  calls.clear();
  CHECK(attend(nullptr, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID);
  CHECK(attend(q, nullptr, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID);
  CHECK(attend(q, k, nullptr, g, 2, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID);
  CHECK(attend(q, k, v, nullptr, 2, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID);
  CHECK(attend(q, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, nullptr) == BG_E_INVALID);
  CHECK(attend(q, k, v, g, 1, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID);          // rows of g overlap
  CHECK(attend(q, k, v, g, 2, nullptr, INFINITY, nullptr, nullptr, 0, o) == BG_E_INVALID);
  CHECK(attend(q, k, v, g, 2, nullptr, NAN, nullptr, nullptr, 0, o) == BG_E_INVALID);
  CHECK(attend(q, k, v, g, 2, nullptr, 1, v, nullptr, 0, o) == BG_E_INVALID);                // a gate without a norm
  CHECK(attend(q, k, v, g, 2, nullptr, 1, nullptr, w, -1, o) == BG_E_INVALID && attend(q, k, v, g, 2, nullptr, 1, nullptr, w, NAN, o) == BG_E_INVALID);
  CHECK(attend(q + 1, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID && attend(q, k, v, g, 2, nullptr, 1, nullptr, w + 2, 0, o) == BG_E_INVALID);
  for (float* in : {q, k, v, g, w})  // out over the last value of each
    for (int i = 0; i < 7; i++) {
      float* p[7] = {q, k, v, g, g, v, w};
      const size_t n[7] = {640, 640, 1280, 20, 20, 1280, 64};
      if (p[i] != in) continue;
      p[i] = o + 1280 - 4;
      CHECK(attend(p[0], p[1], p[2], p[3], 2, p[4], 1, p[5], p[6], 0, o) == BG_E_INVALID);
      p[i] = o + 1280;
      CHECK(attend(p[0], p[1], p[2], p[3], 2, p[4], 1, p[5], p[6], 0, o) == BG_OK);
      p[i] = o - (n[i] + 3) / 4 * 4;
      CHECK(attend(p[0], p[1], p[2], p[3], 2, p[4], 1, p[5], p[6], 0, o) == BG_OK);
    }
  CHECK(attend(q, k, v, o + 1278, 0, nullptr, 1, nullptr, nullptr, 0, o) == BG_E_INVALID);   // one decay a head
  CHECK(attend(q, k, v, o + 1280, 0, nullptr, 1, nullptr, nullptr, 0, o) == BG_OK);
  calls.clear();
  // the prologue: 10 rows of 256 channels
  float* p[11] = {at(0), at(1 << 16), at(100000), at(100002), at(110000), at(110008), at(1 << 17), at(3 << 16), at(1 << 18), at(1 << 19), at(540000)};
  auto open = [&](int stride = 4) {
    return bg_linear_prologue(x.c, 0, x.b, p[0], p[1], p[2], p[3], stride, p[4], p[5], p[6], p[7], p[8], p[9], p[10], nullptr);
  };
  CHECK(open() == BG_OK && open(1) == BG_E_INVALID);
  for (int i = 0; i < 11; i++) {
    float* was = p[i];
    p[i] = nullptr;
    CHECK(open() == (i == 9 || i == 10 ? BG_OK : BG_E_INVALID));  // (without g or beta: not asked for)
    p[i] = was;
    if (i < 2 || (i > 5 && i < 9)) {
      p[i] = was + 1;
      CHECK(open() == BG_E_INVALID);
      p[i] = was;
    }
  }
  float *a = p[2], *b = p[3];
  p[2] = p[9] = nullptr;
  CHECK(open() == BG_OK);
  p[3] = p[10] = nullptr;
  CHECK(open() == BG_OK);
  p[2] = a; p[3] = b; p[9] = at(1 << 19); p[10] = at(540000);
  const size_t in_n[6] = {2560, 1024, 38, 38, 2, 2}, out_n[5] = {640, 640, 1280, 20, 20};
  for (int o = 0; o < 5; o++)
    for (int i = 0; i < 11; i++) {
      if (i == 6 + o) continue;
      float* was = p[6 + o];
      const size_t n = i < 6 ? in_n[i] : out_n[i - 6];
      p[6 + o] = p[i] + (n - 1) / 4 * 4;
      CHECK(open() == BG_E_INVALID);
      p[6 + o] = p[i] - (out_n[o] - 4);
      CHECK(open() == BG_E_INVALID);
      p[6 + o] = was;
      CHECK(open() == BG_OK);
    }
  // caches and batches of other shapes; a cache without a convolution
  Batch y(8, 64, 0);
  CHECK(y.set({1}, {0}) == BG_OK && y.open(0) == BG_E_STATE && y.attend(0) == BG_OK);
  bg_linear_cache* c = nullptr;
  CHECK(bg_linear_create(3, 2, 2, 64, 64, 0, 6, buf, nullptr, &c) == BG_OK);
  CHECK(bg_linear_attention(c, 0, y.b, q, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o, nullptr) == BG_E_INVALID);
  bg_linear_destroy(c);
  CHECK(bg_linear_attention(nullptr, 0, y.b, q, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o, nullptr) == BG_E_INVALID);
  CHECK(bg_linear_attention(y.c, 0, nullptr, q, k, v, g, 2, nullptr, 1, nullptr, nullptr, 0, o, nullptr) == BG_E_INVALID);
}

static void streams() {
  Batch x;
  CHECK(x.set({1}, {0}) == BG_OK);
  EXPECT("upload on 0", x.record(x.done0, 0));
  CHECK(x.attend(7) == BG_OK);
  EXPECT(x.record(x.moved, 0), x.wait(7, x.moved), "rows on 7");
  CHECK(x.open(7) == BG_OK && x.open(9) == BG_OK);
  EXPECT("prologue on 7", x.record(x.moved, 7), x.wait(9, x.moved), "prologue on 9");
  CHECK(x.set({2}, {0}) == BG_OK);
  EXPECT(x.record(x.moved, 9), x.wait(0, x.moved), "upload on 0", x.record(x.done1, 0));
  CHECK(x.set({2}, {0}) == BG_OK);  // the staging's first block again
  EXPECT("host waits for " + std::to_string(x.done0), "upload on 0", x.record(x.done0, 0));
  fail_record = 1;
  CHECK(x.attend(4) == BG_E_DEVICE && x.open(4) == BG_E_DEVICE && x.set({1}, {0}, 4) == BG_E_DEVICE);
  fail_record = 0;
  EXPECT();
  fail_upload = 1;
  CHECK(x.set({1}, {0}) == BG_E_DEVICE && x.attend(0) == BG_E_STATE);
  fail_upload = 0;
  CHECK(x.set({1}, {0}) == BG_OK && x.attend(0) == BG_OK);
}

static void capture() {
  Batch x;
  CHECK(x.set({30, 20}, {0, 1}) == BG_OK);
  calls.clear();
  capturing_now.insert(stream(6));
  CHECK(x.set({1}, {0}, 6) == BG_E_STATE);
  CHECK(x.attend(6) == BG_OK);
  EXPECT("rows on 6", "chunks on 6");  // any batch of 50 rows
  CHECK(!bg::seen.ws && bg::seen.n_seqs == 8 && bg::seen.n_chunked == 1 && bg::seen.n_chunk_units == 1 && bg::seen.most == 27 && bg::seen.n_units == 8);
  CHECK(x.open(6) == BG_OK && x.attend(0) == BG_OK);
  CHECK(bg::seen.ws && bg::seen.n_seqs == 2 && bg::seen.most == 20);
  capturing_now.clear();
  CHECK(x.set({51}, {0}) == BG_E_STATE && x.set({25, 26}, {0, 1}) == BG_E_STATE && x.set({50}, {0}) == BG_OK);
  // fewer rows captured later bind as well, and none at all
  CHECK(x.set({3}, {0}) == BG_OK);
  capturing_now.insert(stream(6));
  CHECK(x.attend(6) == BG_OK && bg::seen.n_seqs == 3 && bg::seen.n_chunked == 0);
  capturing_now.clear();
  CHECK(x.set({4}, {0}) == BG_E_STATE && x.set({0}, {0}) == BG_OK);
  capturing_now.insert(stream(6));
  CHECK(x.attend(6) == BG_OK);
  capturing_now.clear();
  CHECK(x.set({1}, {0}) == BG_E_STATE && x.set({0}, {0}) == BG_OK);
  // a stream that is being captured cannot be left with an event
  Batch y;
  CHECK(y.set({1}, {0}, 6) == BG_OK);
  capturing_now.insert(stream(6));
  CHECK(y.attend(0) == BG_E_STATE && y.set({1}, {0}, 0) == BG_E_STATE && y.attend(6) == BG_OK);
  capturing_now.clear();
  CHECK(y.attend(0) == BG_OK);
}

// 32 units to a pass
static void workspace() {
  Batch x(4, 1 << 16);
  CHECK(x.set({27}, {0}) == BG_OK && x.attend(0) == BG_OK && !bg::seen.ws);
  auto size = [&]() { return blocks.at(bg::seen.ws) / (bg::kLinSpace / 32); };
  CHECK(x.set({64}, {0}) == BG_OK && x.attend(0) == BG_OK && size() == 1 && bg::seen.window == 32);
  calls.clear();
  char* was = bg::seen.ws;
  CHECK(x.set({64, 100}, {0, 1}) == BG_OK);           // the old one is freed once the device is done with it
  EXPECT("host waits for " + std::to_string(x.done0), "upload on 0", "sync", "free", x.record(x.done0, 0));
  CHECK(x.attend(0) == BG_OK && size() == 3 && bg::seen.ws != was && bg::seen.hdr->ws == bg::seen.ws);
  CHECK(x.set({256}, {0}) == BG_OK && x.attend(0) == BG_OK && size() == 6);     // twofold
  CHECK(x.set({2049}, {0}) == BG_OK && x.attend(0) == BG_OK && size() == 32);  // a pass
  calls.clear();
  CHECK(x.set({30}, {0}) == BG_OK && x.attend(0) == BG_OK && size() == 32);
  CHECK(std::count(calls.begin(), calls.end(), "free") == 0);
  // no memory: the batch before stays
  Batch y;
  CHECK(y.set({64, 64}, {0, 1}) == BG_OK && y.attend(0) == BG_OK);
  was = bg::seen.ws;
  most_memory = bg::kLinSpace / 32 * 5 / 2;
  CHECK(y.set({64, 65}, {0, 1}) == BG_E_OOM);
  most_memory = bg::kLinSpace / 32 * 3;                     // not twofold, but what is needed
  CHECK(y.attend(0) == BG_OK && bg::seen.ws == was && bg::seen.hdr->n_tokens == 128 && bg::seen.n_tokens == 128);
  CHECK(y.set({64, 65}, {0, 1}) == BG_OK && y.attend(0) == BG_OK && size() == 3);
  most_memory = ~(size_t)0;
  fail_upload = 1;                                    // the new one goes with a failed upload
  const size_t n = blocks.size();
  CHECK(y.set({640}, {0}) == BG_E_DEVICE && blocks.size() == n && y.attend(0) == BG_E_STATE);
  fail_upload = 0;
  CHECK(y.set({640}, {0}) == BG_OK && y.attend(0) == BG_OK && size() == 10);
}

static void products() {
  float *x = at(0), *y = at(1 << 17), *z = at(1 << 18), *r = at(1 << 19), *h = at(3 << 18), *ws = at(900000);
  uint32_t* codes = (uint32_t*)at(200000);
  float *sc = at(300000), *mn = at(310000);
  auto split = [&](int rows, int K, int group, int type, int N0, int N1, int N2, float* y, float* z, float* r, float* ws) {
    return bg_gemv4_split(x, rows, K, codes, sc, mn, type, group, N0, N1, N2, y, z, r, ws, stream(2));
  };
  calls.clear();
  CHECK(split(2, 256, 64, BG_KV_F16, 10, 20, 0, y, z, nullptr, nullptr) == BG_OK && bg::product.scale_f16 && bg::product.N1 == 20);
  CHECK(split(16, 256, 64, BG_KV_F32, 10, 0, 5, y, nullptr, r, ws) == BG_OK && !bg::product.scale_f16 && bg::product.room == (char*)ws);
  EXPECT("product on 2", "product on 2");
  CHECK(split(17, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_E_UNSUPPORTED && split(-1, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_E_UNSUPPORTED);
  CHECK(split(1, 0, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_E_INVALID && split(1, 192, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_E_INVALID);
  CHECK(split(1, (1 << 24) + 128, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_E_UNSUPPORTED);
  CHECK(split(1, 256, 16, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_E_UNSUPPORTED && split(1, 256, 64, BG_KV_Q8, 10, 0, 0, y, z, r, ws) == BG_E_INVALID);
  CHECK(split(1, 256, 64, BG_KV_F16, -1, 2, 0, y, z, r, ws) == BG_E_INVALID && split(1, 256, 64, BG_KV_F16, 0x7fffffff, 0x7fffffff, 2, y, z, r, ws) == BG_E_INVALID);
  CHECK(split(1, 256, 64, BG_KV_F16, 10, 1, 0, y, nullptr, r, ws) == BG_E_INVALID && split(1, 256, 64, BG_KV_F16, 10, 1, 1, y, z, nullptr, ws) == BG_E_INVALID);
  CHECK(split(5, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, nullptr) == BG_E_INVALID && split(5, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws + 1) == BG_E_INVALID);
  CHECK(split(5, 256, 64, BG_KV_F16, 10, 0, 0, ws + 1023, z, r, ws) == BG_E_INVALID && split(4, 256, 64, BG_KV_F16, 10, 0, 0, ws + 1023, z, r, ws) == BG_OK);
  CHECK(split(5, 256, 64, BG_KV_F16, 10, 0, 0, ws + 1024, z, r, ws) == BG_OK && split(5, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, x + 1276) == BG_E_INVALID);
  CHECK(split(5, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, x + 1280) == BG_OK);
  calls.clear();
  CHECK(split(0, 256, 64, BG_KV_F16, 10, 0, 0, y, z, r, ws) == BG_OK && split(3, 256, 64, BG_KV_F16, 0, 0, 0, nullptr, nullptr, nullptr, nullptr) == BG_OK);
  // outputs over inputs: 2 rows of x, 10 rows of 32 words, of 4 scales of 2 bytes
  for (float* over : {x + 511, (float*)codes + 319, sc + 19, mn + 19}) {
    CHECK(split(2, 256, 64, BG_KV_F16, 10, 0, 0, over, z, r, nullptr) == BG_E_INVALID);
    CHECK(split(2, 256, 64, BG_KV_F16, 10, 0, 0, over + 1, z, r, nullptr) == BG_OK);
  }
  CHECK(split(2, 256, 64, BG_KV_F16, 5, 5, 0, y, y + 9, r, nullptr) == BG_E_INVALID && split(2, 256, 64, BG_KV_F16, 5, 5, 0, y, y + 10, r, nullptr) == BG_OK);
  calls.clear();
  auto add = [&](int rows, float* h, float* y, float* ws) { return bg_gemv4_resid(x, rows, 256, codes, sc, mn, BG_KV_F16, 64, 10, h, y, ws, stream(2)); };
  CHECK(add(2, h, y, nullptr) == BG_OK && bg::product.resid == h && bg::product.out0 == y && add(2, y, y, nullptr) == BG_OK && add(8, y, y, ws) == BG_OK);
  CHECK(add(2, nullptr, y, nullptr) == BG_E_INVALID && add(2, y + 1, y, nullptr) == BG_E_INVALID && add(8, ws + 1020, y, ws) == BG_E_INVALID);
  CHECK(add(8, h, y, nullptr) == BG_E_INVALID && add(0, nullptr, nullptr, nullptr) == BG_OK);
  CHECK(bg_gemv4_workspace(4, 256) == 0 && bg_gemv4_workspace(5, 256) == 4096 && bg_gemv4_workspace(17, 256) == 0 && bg_gemv4_workspace(5, 0) == 0);
}

int main() {
  caches();
  sets();
  arguments();
  streams();
  capture();
  workspace();
  products();
  if (!blocks.empty()) line_of_fault(__LINE__, "blocks left");
  printf("ok\n");
}
