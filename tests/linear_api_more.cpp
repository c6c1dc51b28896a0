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

int main() {
  sizes_of_caches();
  if (!blocks.empty()) line_of_fault(__LINE__, "blocks left");
  printf("ok\n");
}
