// Prints the plan of a paged batch (bg_paged_plan.h) read from stdin, for tests/test_paged_plan.py.
//   in : kv_heads G D dtype page n_pages cus max_seqs max_tokens max_pages repeat n_seqs stride, rows, lens, tables
//   out: "error <text>" or counts and arrays, one line each
#include <cstdio>
#include <cstdlib>

#include "../bitgpu_amd/csrc/bg_paged_plan.h"

static int next_int() {
  int x = 0;
  if (scanf("%d", &x) != 1) exit(2);
  return x;
}

template <class T>
static void line(const char* name, const std::vector<T>& v) {
  printf("%s", name);
  for (const T& x : v)
    for (size_t i = 0; i < sizeof(T) / 4; i++) printf(" %d", ((const int*)&x)[i]);
  printf("\n");
}

int main() {
  bg::PagedShape s{};
  s.kv_heads = next_int();
  s.G = next_int();
  s.D = next_int();
  s.dtype = next_int();
  s.page = next_int();
  s.n_pages = next_int();
  s.cus = next_int();
  s.max_seqs = next_int();
  s.max_tokens = next_int();
  s.max_pages = next_int();
  const int repeat = next_int(), n = next_int(), stride = next_int();
  std::vector<int> rows(n), lens(n), table((size_t)n * stride);
  for (int& x : rows) x = next_int();
  for (int& x : lens) x = next_int();
  for (int& x : table) x = next_int();
  bg::PagedPlanner planner;
  bg::PagedPlan p;
  for (int i = 0; i < repeat; i++) {  // a planner keeps nothing from one batch to the next
    const std::string wrong = planner.build(s, n, rows.data(), lens.data(), table.data(), stride, p);
    if (!wrong.empty()) {
      printf("error %s\n", wrong.c_str());
      return 0;
    }
  }
  printf("counts %d %d %d %d %ld %d\n", p.n_tokens, p.n_parts, p.shared_segments, p.write_page, s.max_units(), s.max_toks());
  line("units", p.units);
  line("toks", p.toks);
  line("merges", p.merges);
  line("pages", p.pages);
  line("dst", p.dst);
  line("v_single", p.v_single);
  line("v_group", p.v_group);
  return 0;
}
