// Host-only check of the rule that says which shared prefixes pay: times measured on a B200 near the rule's border, us per call
// with and without the prefix pass (rows with suffixes of up to 64 tokens), and the side that the planner takes.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "csrc/kv_host.hpp"

using namespace yahkv;

int main() {
  struct Point {
    int fmt, rows, pages;
    double with, without;
  };
  const std::vector<Point> points = {
      {YAHKV_FMT_F16, 4, 64, 13.9, 21.1},
      {YAHKV_FMT_F16, 5, 2, 9.5, 8.2},
      {YAHKV_FMT_F16, 5, 64, 14.2, 23.0},
      {YAHKV_FMT_F16, 6, 2, 9.8, 8.4},
      {YAHKV_FMT_F16, 6, 64, 14.5, 23.5},
      {YAHKV_FMT_F16, 8, 2, 10.1, 8.6},
      {YAHKV_FMT_F16, 8, 8, 10.8, 13.1},
      {YAHKV_FMT_F16, 10, 4, 10.5, 9.1},
      {YAHKV_FMT_F16, 10, 6, 10.8, 12.9},
      {YAHKV_FMT_F16, 12, 4, 11.1, 9.3},
      {YAHKV_FMT_F16, 12, 8, 11.5, 14.2},
      {YAHKV_FMT_F16, 16, 1, 11.6, 9.0},
      {YAHKV_FMT_F16, 16, 8, 12.0, 15.1},
      {YAHKV_FMT_F16, 20, 2, 13.4, 10.5},
      {YAHKV_FMT_F16, 20, 6, 12.6, 16.6},
      {YAHKV_FMT_F16, 24, 2, 12.5, 10.5},
      {YAHKV_FMT_F16, 24, 6, 13.1, 17.1},
      {YAHKV_FMT_F16, 32, 3, 12.9, 11.3},
      {YAHKV_FMT_F16, 32, 6, 13.2, 17.7},
      {YAHKV_FMT_F16, 43, 2, 14.7, 16.7},
      {YAHKV_FMT_F16, 48, 2, 14.7, 16.9},
      {YAHKV_FMT_F16, 64, 2, 14.8, 18.5},
      {YAHKV_FMT_F16, 80, 1, 16.4, 20.7},
      {YAHKV_FMT_F16, 96, 1, 17.5, 21.3},
      {YAHKV_FMT_Q8_0, 2, 4, 10.2, 8.6},
      {YAHKV_FMT_Q8_0, 3, 1, 10.2, 8.3},
      {YAHKV_FMT_Q8_0, 3, 32, 13.5, 16.0},
      {YAHKV_FMT_Q8_0, 4, 2, 10.5, 9.2},
      {YAHKV_FMT_Q8_0, 4, 32, 13.8, 16.6},
      {YAHKV_FMT_Q8_0, 5, 1, 10.5, 8.9},
      {YAHKV_FMT_Q8_0, 5, 32, 14.2, 16.1},
      {YAHKV_FMT_Q8_0, 6, 32, 14.5, 17.1},
      {YAHKV_FMT_Q8_0, 8, 8, 11.7, 13.8},
      {YAHKV_FMT_Q8_0, 10, 4, 11.5, 14.2},
      {YAHKV_FMT_Q8_0, 12, 4, 11.9, 15.1},
      {YAHKV_FMT_Q8_0, 16, 4, 13.0, 15.3},
      {YAHKV_FMT_Q8_0, 20, 1, 14.3, 11.6},
      {YAHKV_FMT_Q8_0, 20, 4, 13.5, 15.5},
      {YAHKV_FMT_Q8_0, 24, 1, 13.4, 11.5},
      {YAHKV_FMT_Q8_0, 24, 6, 13.9, 17.8},
      {YAHKV_FMT_Q8_0, 32, 1, 13.4, 11.5},
      {YAHKV_FMT_Q8_0, 32, 6, 14.1, 17.9},
      {YAHKV_FMT_Q8_0, 43, 2, 15.6, 13.3},
      {YAHKV_FMT_Q8_0, 43, 8, 16.9, 20.5},
      {YAHKV_FMT_Q8_0, 48, 2, 15.6, 13.4},
      {YAHKV_FMT_Q8_0, 48, 16, 18.3, 30.1},
      {YAHKV_FMT_Q8_0, 64, 4, 21.0, 17.4},
      {YAHKV_FMT_Q8_0, 64, 16, 21.0, 31.8},
      {YAHKV_FMT_Q8_0, 80, 6, 21.4, 27.9},
      {YAHKV_FMT_Q8_0, 96, 4, 21.7, 24.8},
      {YAHKV_FMT_Q4_0, 2, 2, 9.4, 8.1},
      {YAHKV_FMT_Q4_0, 2, 64, 14.6, 19.2},
      {YAHKV_FMT_Q4_0, 3, 1, 9.6, 8.1},
      {YAHKV_FMT_Q4_0, 3, 32, 13.0, 15.2},
      {YAHKV_FMT_Q4_0, 4, 2, 10.0, 8.7},
      {YAHKV_FMT_Q4_0, 4, 16, 12.8, 15.0},
      {YAHKV_FMT_Q4_0, 5, 2, 10.4, 9.0},
      {YAHKV_FMT_Q4_0, 5, 16, 13.0, 16.0},
      {YAHKV_FMT_Q4_0, 6, 1, 10.3, 8.8},
      {YAHKV_FMT_Q4_0, 6, 16, 13.1, 15.3},
      {YAHKV_FMT_Q4_0, 8, 8, 11.4, 13.5},
      {YAHKV_FMT_Q4_0, 10, 4, 11.2, 12.8},
      {YAHKV_FMT_Q4_0, 12, 8, 12.0, 13.7},
      {YAHKV_FMT_Q4_0, 16, 1, 12.1, 10.4},
      {YAHKV_FMT_Q4_0, 16, 16, 15.3, 18.4},
      {YAHKV_FMT_Q4_0, 20, 6, 13.5, 17.0},
      {YAHKV_FMT_Q4_0, 24, 6, 13.7, 17.9},
      {YAHKV_FMT_Q4_0, 32, 2, 13.3, 15.1},
      {YAHKV_FMT_Q4_0, 43, 2, 13.9, 15.9},
      {YAHKV_FMT_Q4_0, 48, 2, 13.9, 15.8},
      {YAHKV_FMT_Q4_0, 64, 4, 15.8, 19.2},
      {YAHKV_FMT_Q4_0, 80, 3, 16.0, 19.9},
      {YAHKV_FMT_Q4_0, 96, 4, 16.8, 22.4}};
  int bad = 0, taken = 0;
  for (const Point& p : points) {
    yahkv_config c{};
    c.n_layers = 1, c.num_pages = 400, c.fmt = p.fmt, c.max_seqs = 100, c.max_pages_per_seq = 130, c.max_batch_tokens = 64, c.max_splits = 64;
    KvHost host(c);
    std::int32_t root = -1, src, dst;
    host.SeqCreate(&root), host.SeqReserve(root, p.pages * 64), host.SeqSetLen(root, -1, p.pages * 64);
    std::vector<std::int32_t> ids;
    std::vector<std::int64_t> lens;
    for (int i = 0; i < p.rows; ++i) {
      std::int32_t s = -1;
      if (host.SeqFork(root, p.pages * 64, &s, &src, &dst).code != YAHKV_OK) return 2;
      host.SeqReserve(s, p.pages * 64 + 1), host.SeqSetLen(s, -1, p.pages * 64 + 1);
      ids.push_back(s), lens.push_back(p.pages * 64 + 1);
    }
    const auto groups = host.FindPrefixes(p.rows, ids.data(), lens.data());
    const bool take = groups.size() == 1 && static_cast<int>(groups[0].rows.size()) == p.rows && groups[0].pages == p.pages;
    if (!take && !groups.empty()) return 3;
    taken += take ? 1 : 0;
    if (take != (p.with < p.without)) {
      std::printf("format %d, %d rows x %d pages: %.1f us with the pass, %.1f without, taken: %d\n", p.fmt, p.rows, p.pages, p.with, p.without, take);
      ++bad;
    }
  }
  if (bad > 0 || taken == 0 || taken == static_cast<int>(points.size())) return 1;
  std::printf("prefix_rule_test: ok\n");
  return 0;
}
