// More of the paged cache's C entries against the stand-in runtime of paged_api.cpp: what a batch does when
// the device has no memory or an event fails, what each kind of captured launch binds later sets to, and
// which choices of a plan a captured launch may not keep.
#include <hip/hip_runtime.h>

#define main paged_api_main
#include "paged_api.cpp"
#undef main

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

int main() {
  cache_policy_under_capture();
  if (!blocks.empty()) line_of_fault(__LINE__, "blocks left");
  printf("ok\n");
}
