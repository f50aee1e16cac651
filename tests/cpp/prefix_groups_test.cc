// Host-only checks of KvHost::FindPrefixes on trees of forks: the groups are disjoint, their rows agree in the group's pages
// and fill them, and together they save as many page reads as the best assignment found by trying all of them.
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "csrc/kv_host.hpp"

#define EXPECT(c)                                                         \
  do {                                                                    \
    if (!(c)) {                                                           \
      std::fprintf(stderr, "%s:%d: EXPECT(%s) failed\n", __FILE__, __LINE__, #c); \
      std::exit(1);                                                       \
    }                                                                     \
  } while (0)

using namespace yahkv;

static yahkv_config Config(int max_seqs, int max_pages, int num_pages, int fmt = YAHKV_FMT_Q8_0) {
  yahkv_config c{};
  c.n_layers = 1, c.num_pages = num_pages, c.fmt = fmt, c.max_seqs = max_seqs, c.max_pages_per_seq = max_pages;
  c.max_batch_tokens = 8192, c.max_splits = 64;
  return c;
}
static std::int32_t Grow(KvHost& host, std::int32_t s, std::int64_t len) {
  if (s < 0) EXPECT(host.SeqCreate(&s).code == YAHKV_OK);
  EXPECT(host.SeqReserve(s, len).code == YAHKV_OK && host.SeqSetLen(s, -1, len).code == YAHKV_OK);
  return s;
}
static std::int32_t Fork(KvHost& host, std::int32_t from, std::int64_t n, std::int64_t len) {
  std::int32_t s = -1, src, dst;
  EXPECT(host.SeqFork(from, n, &s, &src, &dst).code == YAHKV_OK);
  return Grow(host, s, len);
}
static int Common(const KvHost& host, int x, int y) {
  const int n = static_cast<int>(std::min(host.len(x, 0), host.len(y, 0)) / kPageTokens);
  int i = 0;
  while (i < n && host.table_row(x)[i] == host.table_row(y)[i]) ++i;
  return i;
}
// Pages of the group every row is in (0: none), after checking the groups; *saved: the page reads they save.
static std::vector<int> Groups(const KvHost& host, const std::vector<std::int32_t>& ids, std::int64_t* saved) {
  std::vector<std::int64_t> lens;
  for (int s : ids) lens.push_back(host.len(s, 0));
  std::vector<int> pages(ids.size(), 0);
  *saved = 0;
  for (const auto& g : host.FindPrefixes(static_cast<int>(ids.size()), ids.data(), lens.data())) {
    EXPECT(g.rows.size() >= 2 && g.pages >= 1);
    for (std::int32_t b : g.rows) {
      EXPECT(pages[static_cast<std::size_t>(b)] == 0);
      pages[static_cast<std::size_t>(b)] = g.pages;
      EXPECT(Common(host, ids[static_cast<std::size_t>(g.rows[0])], ids[static_cast<std::size_t>(b)]) >= g.pages);
      EXPECT(lens[static_cast<std::size_t>(b)] >= static_cast<std::int64_t>(g.pages) * kPageTokens);
    }
    *saved += static_cast<std::int64_t>(g.rows.size() - 1) * g.pages;
  }
  return pages;
}

// A long conversation behind the same prompt does not take the prompt from the other rows.
static void CheckLeftRows() {
  KvHost host(Config(20, 300, 2000));
  const std::int32_t prompt = Grow(host, -1, 20 * 64);
  std::vector<std::int32_t> ids;
  for (int i = 0; i < 8; ++i) ids.push_back(Fork(host, prompt, 20 * 64, 20 * 64 + 30 + i));
  const std::int32_t conv = Fork(host, prompt, 20 * 64, 200 * 64);
  for (int i = 0; i < 2; ++i) ids.push_back(Fork(host, conv, 200 * 64, 200 * 64 + 5 + i));
  std::int64_t saved;
  const auto pages = Groups(host, ids, &saved);
  for (int i = 0; i < 10; ++i) EXPECT(pages[static_cast<std::size_t>(i)] == (i < 8 ? 20 : 200));
  EXPECT(saved == 7 * 20 + 200);
  // three levels: a tool prompt of 10 pages, two system prompts of 60 behind it, a conversation of 160 behind one of them
  KvHost deep(Config(64, 300, 6000));
  const std::int32_t tool = Grow(deep, -1, 10 * 64);
  ids.clear();
  for (int i = 0; i < 9; ++i) ids.push_back(Fork(deep, tool, 10 * 64, 10 * 64 + i));        // 0 .. 8
  for (int c = 0; c < 2; ++c) {
    const std::int32_t sys = Fork(deep, tool, 10 * 64, 60 * 64);
    for (int i = 0; i < 4; ++i) ids.push_back(Fork(deep, sys, 60 * 64, 60 * 64 + i));       // 9 .. 12, 13 .. 16
    if (c == 0) {
      const std::int32_t talk = Fork(deep, sys, 60 * 64, 160 * 64);
      for (int i = 0; i < 3; ++i) ids.push_back(Fork(deep, talk, 160 * 64, 160 * 64 + i));  // 17 .. 19, sorted below
    }
  }
  const auto deep_pages = Groups(deep, ids, &saved);
  EXPECT(saved == 8 * 10 + 3 * 60 * 2 + 2 * 160);
  std::map<int, int> sizes;
  for (int p : deep_pages) ++sizes[p];
  EXPECT(sizes[10] == 9 && sizes[60] == 8 && sizes[160] == 3 && sizes[0] == 0);
}

// Random small trees against all assignments of the rows to prefixes. Page counts are large enough that no rest of rows is
// too small for a group of its own.
static void CheckAgainstAll(unsigned seed) {
  std::mt19937 rng(seed);
  KvHost host(Config(24, 2000, 24 * 2000));
  host.SetSharedMinSaved(1);
  std::vector<std::int32_t> all{Grow(host, -1, 64 * (64 + static_cast<int>(rng() % 200)))};
  const int n = 3 + static_cast<int>(rng() % 5);
  for (int i = 1; i < n; ++i) {
    const std::int32_t from = all[rng() % all.size()];
    const std::int64_t have = host.len(from, 0) / 64, at = rng() % 3 == 0 ? have : 64 + static_cast<std::int64_t>(rng() % (have - 63));
    all.push_back(Fork(host, from, at * 64, (at + (rng() % 2 ? static_cast<std::int64_t>(rng() % 200) : 0)) * 64));
  }
  std::int64_t saved;
  Groups(host, all, &saved);
  // best over all partitions of the rows: a part of k rows saves (k - 1) x (the pages all of it have in common)
  std::vector<std::vector<int>> parts;
  std::int64_t best = 0;
  std::function<void(std::size_t)> place = [&](std::size_t i) {
    if (i == all.size()) {
      std::int64_t total = 0;
      for (const auto& p : parts) {
        int common = 1 << 30;
        for (std::size_t a = 1; a < p.size(); ++a) common = std::min(common, Common(host, p[0], p[a]));
        if (p.size() > 1) total += static_cast<std::int64_t>(p.size() - 1) * common;
      }
      best = std::max(best, total);
      return;
    }
    for (std::size_t g = 0; g <= parts.size(); ++g) {
      if (g == parts.size()) parts.push_back({all[i]});
      else parts[g].push_back(all[i]);
      place(i + 1);
      if (parts[g].size() == 1) parts.pop_back();
      else parts[g].pop_back();
      if (g == parts.size()) break;
    }
  };
  place(0);
  EXPECT(saved == best);
}

int main() {
  CheckLeftRows();
  for (unsigned s = 0; s < 300; ++s) CheckAgainstAll(s);
  std::printf("prefix_groups_test: ok\n");
  return 0;
}
