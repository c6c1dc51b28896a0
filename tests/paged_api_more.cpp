// More of the paged cache's C entries against the stand-in runtime of paged_api.cpp: what a batch does when
// the device has no memory or an event fails, what each kind of captured launch binds later sets to, and
// which choices of a plan a captured launch may not keep.
#include <hip/hip_runtime.h>

#define main paged_api_main
#define hipMalloc plain_malloc
#include "paged_api.cpp"
#undef hipMalloc
#undef main

static size_t room = ~(size_t)0;  // the largest block that the device has
extern "C" hipError_t hipMalloc(void** p, size_t n) {
  if (n > room) return hipErrorOutOfMemory;
  note("malloc %zu", n);
  return plain_malloc(p, n);
}

// f16 pages past 64 MB a layer that one row each reads: nontemporal, but not in a graph, whose batch changes
static void cache_policy_under_capture() {
  bg_paged_kv* kv = nullptr;
  bg_paged_batch* b = nullptr;
  CHECK(bg_paged_create(1, 8, 128, BG_KV_F16, 64, 1024, buf, buf, nullptr, nullptr, &kv) == BG_OK);
  CHECK(bg_paged_batch_create(kv, 32, 9, 9, 1024, &b) == BG_OK);
  std::vector<int32_t> rows(9, 1), lens(9, 2100), tables;
  for (int i = 0; i < 9 * 33; i++) tables.push_back(i);
  CHECK(bg_paged_batch_set(b, 9, rows.data(), lens.data(), tables.data(), 33, nullptr, 1, stream(0)) == BG_OK);
  CHECK(bg_paged_attention(kv, 0, b, buf, 1.0f, nullptr, 0, buf + 2048, stream(0)) == BG_OK);
  CHECK(!bg::seen.captured && bg::seen.stream_few == 1);
  capturing_now.insert(stream(3));
  CHECK(bg_paged_attention(kv, 0, b, buf, 1.0f, nullptr, 0, buf + 2048, stream(3)) == BG_OK);
  capturing_now.clear();
  CHECK(bg::seen.captured && bg::seen.stream_few == 0);
  bg_paged_batch_destroy(b);
  bg_paged_destroy(kv);
  calls.clear();
}

// the workspace of partials, as the uploaded header (which captured launches read) has it
static bool workspace_stands(size_t bytes = 4) { return inside(bg::seen.hdr->ws_o, bytes); }

static void workspace_growth() {
  Batch x;
  CHECK(x.set({4}, {8000}, {range(0, 250)}, 0) == BG_OK && x.attend(0) == BG_OK);
  CHECK(bg::seen.n_merges > 0 && workspace_stands());
  size_t first = 0;
  for (auto& c : calls)
    if (sscanf(c.c_str(), "malloc %zu", &first) == 1) break;
  const float* old = bg::seen.hdr->ws_o;
  // an upload that fails: what the header names is still there
  fail_upload = 1;
  CHECK(x.set({64}, {60000}, {range(0, 1875)}, 0) == BG_E_DEVICE);
  fail_upload = 0;
  CHECK(bg::seen.hdr->ws_o == old && workspace_stands());
  CHECK(x.attend(0) == BG_E_STATE);
  // no room at all: the batch before stays set
  CHECK(x.set({4}, {8000}, {range(0, 250)}, 0) == BG_OK);
  calls.clear();
  room = 1;
  CHECK(x.set({64}, {60000}, {range(0, 1875)}, 0) != BG_OK);
  calls.clear();
  room = first;
  CHECK(x.attend(0) == BG_OK && bg::seen.hdr->ws_o == old && workspace_stands());
  EXPECT("attention on 0");
  // room for what is needed, not for twice the old one
  int len = 8000;
  size_t bytes = 0;
  room = 2 * first - 1;
  while (len < 60000 && !bytes) {
    len += 32;
    calls.clear();
    CHECK(x.set({4}, {len}, {range(0, (len + 31) / 32)}, 0) == BG_OK);
    for (auto& c : calls) sscanf(c.c_str(), "malloc %zu", &bytes);
  }
  CHECK(bytes > first && bytes < 2 * first);
  CHECK(x.attend(0) == BG_OK && workspace_stands());
  // the old block goes behind the upload that replaces it
  room = ~(size_t)0;
  CHECK(x.set({1}, {40}, {{0, 1}}, 0) == BG_OK);
  calls.clear();
  CHECK(x.set({64}, {60000}, {range(0, 1875)}, 0) == BG_OK);
  std::vector<std::string> order;
  for (auto& c : calls)
    if (c[0] == 'u' || c == "sync" || c == "free") order.push_back(c);
  CHECK((order == std::vector<std::string>{"upload on 0", "sync", "free"}));
  CHECK(x.attend(0) == BG_OK && workspace_stands());
}

// an event that fails behind an upload: the arrays are no longer those of the plan that was set
static void failed_event() {
  Batch x;
  CHECK(x.set({1, 1, 1}, {40, 40, 40}, {{0, 1}, {2, 3}, {4, 5}}, 0) == BG_OK && x.attend(0) == BG_OK);
  calls.clear();
  fail_record = 1;
  CHECK(x.set({1}, {40}, {{0, 1}}, 0) == BG_E_DEVICE);
  fail_record = 0;
  EXPECT("upload on 0", "sync");
  CHECK(x.attend(0) == BG_E_STATE && x.append(0) == BG_E_STATE);
  CHECK(x.set({1}, {40}, {{0, 1}}, 0) == BG_OK && x.attend(0) == BG_OK);
  CHECK(bg::seen.n_tokens == 1 && bg::seen.hdr->n_tokens == 1);
}

// what a captured launch keeps later sets to is what that launch uses
static void captured_parts() {
  const int32_t pos[2] = {300, 300};
  auto shared = [](Batch& x) { return x.set({1, 1}, {40, 40}, {{0, 1}, {2, 1}}, 0); };  // page 1 written by both
  auto far = [](Batch& x) { return x.set({1}, {301}, {range(0, 10)}, 0); };
  auto two = [&](Batch& x) { return x.set({1}, {40}, {{0, 1}}, 0, pos, 2); };
  auto many = [](Batch& x) { return x.set({4}, {40}, {{0, 1}}, 0); };
  struct { bool q, k, v; int32_t shared, far, two; } cases[] = {
      {true, false, false, BG_OK, BG_E_STATE, BG_E_STATE}, {false, true, false, BG_E_STATE, BG_E_STATE, BG_E_STATE},
      {false, false, true, BG_E_STATE, BG_OK, BG_OK}, {true, false, true, BG_E_STATE, BG_E_STATE, BG_E_STATE}};
  for (auto& c : cases) {
    Batch x;
    CHECK(x.set({2}, {40}, {{0, 1}}, 0) == BG_OK);
    capturing_now.insert(stream(6));
    CHECK(bg_paged_qkv_prologue(x.kv, 0, x.b, c.q ? buf : nullptr, 128, c.k ? buf : nullptr, c.v ? buf : nullptr, buf, buf, 1e-6f, buf,
                                buf, 100, 128, nullptr, buf, stream(6)) == BG_OK);
    capturing_now.clear();
    CHECK(shared(x) == c.shared && far(x) == c.far && two(x) == c.two && many(x) == BG_E_STATE);
  }
  {  // attention reads what it is given; a launch that was refused binds nothing
    Batch x;
    CHECK(x.set({2}, {40}, {{0, 1}}, 0) == BG_OK);
    capturing_now.insert(stream(6));
    CHECK(x.attend(6) == BG_OK && x.append(6, 39) == BG_E_INVALID);
    capturing_now.clear();
    CHECK(shared(x) == BG_OK && far(x) == BG_OK && two(x) == BG_OK && many(x) == BG_E_STATE);
  }
  calls.clear();
}

// q_out over q: in place, or not at all
static void overlaps() {
  Batch x;  // 8 heads
  CHECK(x.set({2}, {40}, {{0, 1}}, 0) == BG_OK);
  static float mem[2 * 8 * 256 * 3];
  float* m = (float*)(((uintptr_t)mem + 63) & ~(uintptr_t)63);
  auto call = [&](const float* q, int stride, float* out) {
    return bg_paged_qkv_prologue(x.kv, 0, x.b, q, stride, nullptr, nullptr, buf, nullptr, 1e-6f, buf, buf, 4096, 128, nullptr, out, stream(0));
  };
  const int dense = 2 * 8 * 128, wide = 15 * 256 + 128;
  CHECK(call(m, 128, m) == BG_OK && call(m, 128, m + dense) == BG_OK && call(m + dense, 128, m) == BG_OK);
  CHECK(call(m, 256, m + wide) == BG_OK && call(m + dense, 256, m) == BG_OK);
  CHECK(call(m, 256, m) == BG_E_INVALID);                  // a head's row is written before the next is read
  CHECK(call(m, 128, m + 128) == BG_E_INVALID && call(m + 128, 128, m) == BG_E_INVALID);
  CHECK(call(m, 128, m + dense - 4) == BG_E_INVALID && call(m + dense - 4, 128, m) == BG_E_INVALID);
  CHECK(call(m, 256, m + wide - 4) == BG_E_INVALID && call(m, 256, m + 128) == BG_E_INVALID);
}

int main() {
  overlaps();
  captured_parts();
  failed_event();
  workspace_growth();
  cache_policy_under_capture();
  if (!blocks.empty()) line_of_fault(__LINE__, "blocks left");
  printf("ok\n");
}
