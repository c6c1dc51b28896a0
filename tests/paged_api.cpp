// The paged cache's C entries (paged_api.hip, host code) against a stand-in for the HIP runtime and the
// launches: which call orders itself behind which, what an upload holds and where it goes, and what a
// capture keeps later sets to. Memory is the host's; every call that matters is written down.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "../bitgpu_amd/csrc/bg_api_util.h"
#include "../bitgpu_amd/csrc/bg_paged.h"
#include "../include/bitgpu_attn.h"

static std::vector<std::string> calls;
static std::set<hipStream_t> capturing_now;
static std::string message;
static int fail_record = 0, fail_upload = 0;
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
hipError_t hipMalloc(void** p, size_t n) { return take(p, n); }
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
int32_t api_hip_fail(hipError_t, const char* what) { message = what; return BG_E_DEVICE; }
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
static PagedBatchView seen;
hipError_t launch_paged_prologue(const LayerView&, const PagedBatchView& b, const PagedAppendArgs&, hipStream_t st) {
  seen = b;
  note("prologue on %d%s", sid(st), b.captured ? " captured" : "");
  return hipSuccess;
}
hipError_t launch_paged_attention(const LayerView&, const PagedBatchView& b, const PagedAttnArgs&, hipStream_t st) {
  seen = b;
  note("attention on %d%s", sid(st), b.captured ? " captured" : "");
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

alignas(256) static float buf[4096];

struct Batch {
  bg_paged_kv* kv = nullptr;
  bg_paged_batch* b = nullptr;
  int moved, done0, done1;
  Batch(int max_tokens = 64, int H = 8) {
    CHECK(bg_paged_create(2, 2, 128, BG_KV_F16, 32, 4096, buf, buf, nullptr, nullptr, &kv) == BG_OK);
    moved = (int)events + 1;
    done0 = moved + 1;
    done1 = moved + 2;
    CHECK(bg_paged_batch_create(kv, H, 8, max_tokens, 4096, &b) == BG_OK);
    calls.clear();
  }
  ~Batch() {
    bg_paged_batch_destroy(b);
    bg_paged_destroy(kv);
    calls.clear();
  }
  int32_t set(std::vector<int32_t> rows, std::vector<int32_t> lens, std::vector<std::vector<int32_t>> tables, int st,
              const int32_t* positions = nullptr, int axes = 1) {
    size_t w = 1;
    for (auto& t : tables) w = std::max(w, t.size());
    std::vector<int32_t> flat(w * tables.size());
    for (size_t i = 0; i < tables.size(); i++) std::copy(tables[i].begin(), tables[i].end(), flat.begin() + i * w);
    return bg_paged_batch_set(b, (int)rows.size(), rows.data(), lens.data(), flat.data(), (int)w, positions, axes, stream(st));
  }
  int32_t attend(int st) { return bg_paged_attention(kv, 0, b, buf, 1.0f, nullptr, 0, buf + 2048, stream(st)); }
  int32_t append(int st, int rope = 4096, const uint8_t* axis = nullptr) {
    return bg_paged_qkv_prologue(kv, 0, b, buf, 128, buf, buf, buf, buf, 1e-6f, buf, buf, rope, 128, axis, buf, stream(st));
  }
  std::string record(int e, int s) { return "record " + std::to_string(e) + " on " + std::to_string(s); }
  std::string wait(int s, int e) { return std::to_string(s) + " waits for " + std::to_string(e); }
};

static std::vector<int32_t> range(int a, int n) {
  std::vector<int32_t> r(n);
  for (int i = 0; i < n; i++) r[i] = a + i;
  return r;
}

// the usual: every call on one stream, no waits
static void one_stream() {
  for (int st : {0, 5}) {
    Batch x;
    for (int i = 0; i < 4; i++) {
      CHECK(x.set({1, 2}, {40, 70}, {{0, 1}, {2, 3, 4}}, st) == BG_OK);
      std::vector<std::string> w;
      if (i >= 2) w.push_back("host waits for " + std::to_string(i % 2 ? x.done1 : x.done0));
      w.push_back("upload on " + std::to_string(st));
      w.push_back(x.record(i % 2 ? x.done1 : x.done0, st));
      CHECK(calls == w);
      calls.clear();
      CHECK(x.append(st) == BG_OK && x.attend(st) == BG_OK);
      EXPECT("prologue on " + std::to_string(st), "attention on " + std::to_string(st));
    }
  }
}

// a call on another stream waits for the last one's
static void streams() {
  Batch x;
  CHECK(x.set({1}, {40}, {{0, 1}}, 0) == BG_OK);
  EXPECT("upload on 0", x.record(x.done0, 0));
  CHECK(x.attend(7) == BG_OK);  // its units are what the upload on stream 0 writes
  EXPECT(x.record(x.moved, 0), x.wait(7, x.moved), "attention on 7");
  CHECK(x.append(7) == BG_OK);
  EXPECT("prologue on 7");
  CHECK(x.append(9) == BG_OK);
  EXPECT(x.record(x.moved, 7), x.wait(9, x.moved), "prologue on 9");
  CHECK(x.set({1}, {41}, {{0, 1}}, 0) == BG_OK);  // the upload waits for who reads what it overwrites
  EXPECT(x.record(x.moved, 9), x.wait(0, x.moved), "upload on 0", x.record(x.done1, 0));
  // what is refused enqueues nothing and moves nothing
  CHECK(x.set({1}, {41}, {{0}}, 7) == BG_E_INVALID);
  CHECK(bg_paged_attention(x.kv, 0, x.b, buf, 0.0f, nullptr, 0, buf + 2048, stream(7)) == BG_E_INVALID);
  CHECK(bg_paged_attention(x.kv, 0, x.b, buf, 1.0f, nullptr, 0, buf, stream(7)) == BG_E_INVALID);
  CHECK(bg_paged_attention(x.kv, 2, x.b, buf, 1.0f, nullptr, 0, buf + 2048, stream(7)) == BG_E_INVALID);
  EXPECT();
  CHECK(x.attend(0) == BG_OK);
  EXPECT("attention on 0");
  // an empty batch's calls enqueue nothing
  CHECK(x.set({}, {}, {}, 0) == BG_OK);
  calls.clear();
  CHECK(x.attend(3) == BG_OK && x.append(3) == BG_OK);
  EXPECT();
}

static void failures() {
  Batch x;
  CHECK(x.attend(0) == BG_E_STATE && x.append(0) == BG_E_STATE);  // not set
  CHECK(x.set({1}, {40}, {{0, 1}}, 0) == BG_OK);
  calls.clear();
  fail_record = 1;
  CHECK(x.attend(4) == BG_E_DEVICE && x.append(4) == BG_E_DEVICE && x.set({1}, {40}, {{0, 1}}, 4) == BG_E_DEVICE);
  fail_record = 0;
  EXPECT();
  CHECK(x.attend(4) == BG_OK);
  EXPECT(x.record(x.moved, 0), x.wait(4, x.moved), "attention on 4");
  // an upload that fails after the workspace moved: the batch has to be set again
  fail_upload = 1;
  CHECK(x.set({4}, {60000}, {range(0, 1875)}, 4) == BG_E_DEVICE);
  fail_upload = 0;
  calls.clear();
  CHECK(x.set({1}, {3000}, {range(0, 94)}, 4) == BG_OK && x.attend(4) == BG_OK);
  fail_upload = 1;
  CHECK(x.set({64}, {60000}, {range(0, 1875)}, 4) == BG_E_DEVICE);
  fail_upload = 0;
  CHECK(x.attend(4) == BG_E_STATE);
  CHECK(x.set({1}, {3000}, {range(0, 94)}, 4) == BG_OK && x.attend(4) == BG_OK);
}

static void capture() {
  Batch x;
  CHECK(x.set({1, 2}, {40, 70}, {{0, 1}, {2, 3, 4}}, 0) == BG_OK);
  calls.clear();
  capturing_now.insert(stream(6));
  CHECK(x.set({1}, {40}, {{0, 1}}, 6) == BG_E_STATE);
  CHECK(x.append(6, 100) == BG_OK && x.attend(6) == BG_OK);
  EXPECT("prologue on 6 captured", "attention on 6 captured");
  CHECK(bg::seen.captured && bg::seen.n_units == 0 && bg::seen.n_tokens == 0);
  CHECK(x.attend(0) == BG_OK);  // eager beside it, on the stream of the set: no event, none into the capture
  EXPECT("attention on 0");
  capturing_now.clear();
  // what the graph relies on
  CHECK(x.set({2, 2}, {40, 70}, {{0, 1}, {2, 3, 4}}, 0) == BG_E_STATE);     // a row more
  CHECK(x.set({1}, {101}, {{0, 1, 2, 3}}, 0) == BG_E_STATE);                // past the captured table
  CHECK(x.set({1, 1}, {40, 40}, {{0, 1}, {2, 1}}, 0) == BG_E_STATE);        // writes a page that is read
  const int32_t pos[6] = {1, 2, 3, 4, 5, 6};
  CHECK(x.set({3}, {40}, {{0, 1}}, 0, pos, 2) == BG_E_STATE);               // other axes
  EXPECT();
  CHECK(x.set({3}, {100}, {{0, 1, 2, 3}}, 0) == BG_OK);
  calls.clear();
  // a batch that worked on a stream now being captured cannot leave it: an event would enter the capture
  CHECK(x.attend(6) == BG_OK);
  capturing_now.insert(stream(6));
  calls.clear();
  CHECK(x.attend(0) == BG_E_STATE && x.append(0) == BG_E_STATE && x.set({1}, {40}, {{0, 1}}, 0) == BG_E_STATE);
  EXPECT();
  CHECK(x.attend(6) == BG_OK);
  EXPECT("attention on 6 captured");
  capturing_now.clear();
  CHECK(x.attend(0) == BG_OK);
}

// what an upload brings: the arrays as the plan has them, positions by axis or from the lengths
static void contents() {
  Batch x;
  const int32_t pos[3 * 5] = {7, 8, 9, 10, 11, 20, 21, 22, 23, 24, 3, 3, 3, 4, 4};
  CHECK(x.set({2, 0, 3}, {33, 64, 70}, {{9, 8}, {7, 6}, {1, 2, 3}}, 0, pos, 3) == BG_OK);
  uint8_t axis[64];
  for (int i = 0; i < 64; i++) axis[i] = i % 3;
  CHECK(x.append(0, 25, axis) == BG_OK);
  const bg::PagedBatchView& v = bg::seen;
  CHECK(v.n_tokens == 5 && v.hdr->n_tokens == 5 && v.pos_stride == 64);
  for (int a = 0; a < 3; a++)
    for (int t = 0; t < 5; t++) CHECK(v.pos[a * v.pos_stride + t] == pos[5 * a + t]);
  const int dst[5] = {9 * 32 + 31, 8 * 32, 3 * 32 + 3, 3 * 32 + 4, 3 * 32 + 5};
  for (int t = 0; t < 5; t++) CHECK(v.dst[t] == dst[t]);
  const int pages[7] = {9, 8, 7, 6, 1, 2, 3};
  for (int i = 0; i < 7; i++) CHECK(v.pages[i] == pages[i]);
  CHECK(v.n_units == v.hdr->n_units && v.n_units > 0);
  CHECK(x.append(0, 24, axis) == BG_E_INVALID);       // position 24 needs 25 rows
  axis[5] = 3;
  CHECK(x.append(0, 25, axis) == BG_E_INVALID);       // an axis the batch does not have
  CHECK(x.append(0, 25, nullptr) == BG_E_INVALID);
  CHECK(x.set({2, 3}, {33, 70}, {{9, 8}, {1, 2, 3}}, 0) == BG_OK && x.append(0, 70) == BG_OK);
  const int own[5] = {31, 32, 67, 68, 69};
  for (int t = 0; t < 5; t++) CHECK(bg::seen.pos[t] == own[t]);
  CHECK(x.append(0, 69) == BG_E_INVALID);
  // rows of q8 and other caches' batches are told apart
  bg_paged_kv* other = nullptr;
  CHECK(bg_paged_create(2, 2, 128, BG_KV_F32, 32, 4096, buf, buf, nullptr, nullptr, &other) == BG_OK);
  CHECK(bg_paged_attention(other, 0, x.b, buf, 1.0f, nullptr, 0, buf + 2048, nullptr) == BG_E_INVALID);
  CHECK(bg_paged_set_q8_block(other, 32) == BG_E_STATE);
  bg_paged_destroy(other);
  // misaligned and missing buffers
  CHECK(bg_paged_attention(x.kv, 0, x.b, buf + 1, 1.0f, nullptr, 0, buf + 2048, nullptr) == BG_E_INVALID);
  CHECK(bg_paged_attention(x.kv, 0, x.b, nullptr, 1.0f, nullptr, 0, buf + 2048, nullptr) == BG_E_INVALID);
  CHECK(bg_paged_attention(x.kv, 0, x.b, buf, 1.0f, buf, 64, buf + 2048, nullptr) == BG_E_INVALID);
}

// full arrays: the guards behind every block stand when it is freed
static void full() {
  Batch x(64, 64);
  std::vector<int32_t> pos(4 * 64);
  for (int i = 0; i < 256; i++) pos[i] = i;
  CHECK(x.set({64}, {131072}, {range(0, 4096)}, 0, pos.data(), 4) == BG_OK && x.attend(0) == BG_OK);
  CHECK(x.set(std::vector<int32_t>(8, 8), std::vector<int32_t>(8, 16384), {range(0, 512), range(512, 512), range(1024, 512),
              range(1536, 512), range(2048, 512), range(2560, 512), range(3071, 512), range(3583, 512)}, 0) == BG_OK);
  CHECK(x.set(std::vector<int32_t>(9, 1), std::vector<int32_t>(9, 1), std::vector<std::vector<int32_t>>(9, {0}), 0) == BG_E_INVALID);
  CHECK(x.set({65}, {65}, {{0, 1, 2}}, 0) == BG_E_INVALID);
}

int main() {
  one_stream();
  streams();
  failures();
  capture();
  contents();
  full();
  if (!blocks.empty()) line_of_fault(__LINE__, "blocks left");
  printf("ok\n");
}
