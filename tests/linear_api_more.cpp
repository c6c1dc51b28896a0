// More of the linear C entries against the stand-in runtime of linear_api.cpp: sizes past what addresses and launches
// hold.
#define main linear_api_main
#include "linear_api.cpp"
#undef main

// a state's bytes, 4 layers slots v_heads v_dim k_dim, stay below 2^63
static void sizes_of_caches() {
  bg_linear_cache* c = nullptr;
  auto make = [&](int layers, int vh, int dk, int dv, int slots, int taps) {
    const int32_t rc = bg_linear_create(layers, 1, vh, dk, dv, taps, slots, buf, taps ? buf : nullptr, &c);
    if (rc == BG_OK) bg_linear_destroy(c);
    return rc;
  };
  CHECK(make(1 << 16, 4096, 128, 128, 1 << 24, 0) == BG_E_UNSUPPORTED);  // 2^68
  CHECK(make(1 << 15, 4096, 64, 64, 1 << 22, 0) == BG_E_UNSUPPORTED);    // 2^63
  CHECK(make(1 << 15, 2048, 64, 64, 1 << 22, 4) == BG_OK);
  CHECK(make((1 << 15) - 1, 4096, 64, 64, 1 << 22, 0) == BG_OK);
}

// A scan has v_heads v_dim / 32 workgroups of 512 threads for each sequence of 28 rows and more, and a grid's axis fewer
// than 2^32 threads: 4096 heads of 64, 1022 sequences (of four key heads: 4092 would be rounded up to 4096).
static void many_scans() {
  bg_linear_cache* c = nullptr;
  bg_linear_batch* b = nullptr;
  CHECK(bg_linear_create(1, 4, 4096, 64, 64, 0, 2048, buf, nullptr, &c) == BG_OK);
  CHECK(bg_linear_batch_create(c, 2048, 1 << 16, &b) == BG_OK);
  std::vector<int32_t> rows(1024, 28), slots(1024);
  for (int i = 0; i < 1024; i++) slots[i] = i;
  calls.clear();
  CHECK(bg_linear_batch_set(b, 1024, rows.data(), slots.data(), nullptr, stream(0)) == BG_E_UNSUPPORTED);
  EXPECT();
  rows[5] = 27;
  CHECK(bg_linear_batch_set(b, 1024, rows.data(), slots.data(), nullptr, stream(0)) == BG_E_UNSUPPORTED);
  CHECK(bg_linear_batch_set(b, 1023, rows.data(), slots.data(), nullptr, stream(0)) == BG_OK);
  calls.clear();
  auto attend = [&](int st) {
    return bg_linear_attention(c, 0, b, at(0), (float*)(1ull << 44), (float*)(1ull << 45), at(1 << 19), 0, nullptr, 1.0f, nullptr, nullptr,
                               1e-6f, (float*)(1ull << 46), stream(st));
  };
  CHECK(attend(0) == BG_OK);
  EXPECT("rows on 0", "chunks on 0");
  capturing_now.insert(stream(6));  // a captured launch is for any batch of as many rows: 28,643, at most 1022 times 28
  CHECK(attend(6) == BG_OK);
  capturing_now.clear();
  rows.assign(1, 28672);
  CHECK(bg_linear_batch_set(b, 1, rows.data(), slots.data(), nullptr, stream(0)) == BG_E_STATE);
  bg_linear_batch_destroy(b);
  CHECK(bg_linear_batch_create(c, 2048, 1 << 16, &b) == BG_OK);
  CHECK(bg_linear_batch_set(b, 1, rows.data(), slots.data(), nullptr, stream(0)) == BG_OK);
  calls.clear();
  CHECK(attend(0) == BG_OK);
  EXPECT("chunks on 0");
  capturing_now.insert(stream(6));
  CHECK(attend(6) == BG_E_UNSUPPORTED);
  capturing_now.clear();
  EXPECT();
  rows[0]++;  // and binds nothing
  CHECK(bg_linear_batch_set(b, 1, rows.data(), slots.data(), nullptr, stream(0)) == BG_OK);
  bg_linear_batch_destroy(b);
  bg_linear_destroy(c);
}

int main() {
  sizes_of_caches();
  many_scans();
  if (!blocks.empty()) line_of_fault(__LINE__, "blocks left");
  printf("ok\n");
}
