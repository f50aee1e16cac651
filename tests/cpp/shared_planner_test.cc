// Host-only checks of the shared-prefix planner and of the eviction's page plan in csrc/kv_host.hpp.
//   PlanDecodeShared: for every (batch row, kv head) the prefix parts and the suffix units cover every page of the row
//   exactly once, in order; prefix pages are full for every row of the group; a CTA pair's two tiles have the same pages
//   and kv head; no two CTAs write the same workspace row and none lies outside the workspace; the combine's item finds
//   exactly the rows the tiles write.
//   PlanEvict / CommitEvict: shared pages are replaced by pages nobody holds, also when all their holders are cut at once.
#include <cstdio>
#include <cstdlib>
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

static yahkv_config Config(int max_seqs, int max_pages, int num_pages, int n_layers = 1) {
  yahkv_config c{};
  c.n_layers = n_layers;
  c.num_pages = num_pages;
  c.fmt = YAHKV_FMT_Q8_0;
  c.max_seqs = max_seqs;
  c.max_pages_per_seq = max_pages;
  c.max_batch_tokens = 8192;
  c.max_splits = 64;
  return c;
}

static std::int32_t Grow(KvHost& host, std::int32_t s, std::int64_t len) {
  if (s < 0) EXPECT(host.SeqCreate(&s).code == YAHKV_OK);
  EXPECT(host.SeqReserve(s, len).code == YAHKV_OK);
  EXPECT(host.SeqSetLen(s, -1, len).code == YAHKV_OK);
  return s;
}

// groups: (prefix tokens, rows); every row of a group is a fork at the prefix with a suffix of its own
static void CheckShared(const std::vector<std::pair<int, int>>& groups, int singles, int n_splits, int n_pairs, unsigned seed, int min_saved = 1) {
  std::mt19937 rng(seed);
  int n_rows = singles;
  for (auto& g : groups) n_rows += g.second;
  const int cap = n_rows + static_cast<int>(groups.size());
  KvHost host(Config(cap, 2048, cap * 2048));
  host.SetSharedMinSaved(min_saved);
  std::vector<std::int32_t> ids;
  std::vector<int> group_of;
  for (std::size_t gi = 0; gi < groups.size(); ++gi) {
    const std::int32_t root = Grow(host, -1, groups[gi].first);
    for (int r = 0; r < groups[gi].second; ++r) {
      std::int32_t child = -1, src = -1, dst = -1;
      EXPECT(host.SeqFork(root, groups[gi].first, &child, &src, &dst).code == YAHKV_OK);
      EXPECT((src >= 0) == (groups[gi].first % kPageTokens != 0) && (src >= 0) == (dst >= 0) && (src < 0 || src != dst));
      Grow(host, child, groups[gi].first + static_cast<int>(rng() % 700));
      ids.push_back(child);
      group_of.push_back(static_cast<int>(gi));
    }
  }
  for (int i = 0; i < singles; ++i) ids.push_back(Grow(host, -1, 1 + static_cast<int>(rng() % 3000))), group_of.push_back(-1);
  for (std::size_t i = ids.size(); i > 1; --i) {   // any order
    const std::size_t j = rng() % i;
    std::swap(ids[i - 1], ids[j]), std::swap(group_of[i - 1], group_of[j]);
  }
  const int n = static_cast<int>(ids.size());
  const std::int64_t max_rows = std::max<std::int64_t>(cap * kQHeads, 4LL * kPrefillTileRows * n_pairs);
  bool changed = false;
  EXPECT(host.PlanDecodeShared(0, n, ids.data(), n_splits, 64, cap * kKvHeads * 64, n_pairs, max_rows, &changed).code == YAHKV_OK);
  EXPECT(changed);
  const auto& p = host.shared_plan();
  EXPECT(p.tiles.size() % 2 == 0 && static_cast<int>(p.items.size()) == n * kKvHeads && static_cast<int>(p.prefix_items.size()) == n * kKvHeads);
  const int combos = kKvHeads * (cap / 2 + cap * kGroup / (2 * kPrefillTileRows) + 1);
  EXPECT(static_cast<int>(p.tiles.size()) <= 2 * std::max(4 * n_pairs, combos));
  // who writes which workspace row: (batch row, kvh, query head) and pages
  struct Written {
    int b, h, j, lo, hi;
  };
  std::map<std::int64_t, Written> written;
  for (std::size_t i = 0; i < p.tiles.size(); ++i) {
    const PrefixTile& t = p.tiles[i];
    const PrefixTile& other = p.tiles[i ^ 1];
    EXPECT(t.kvh == other.kvh && t.page_begin == other.page_begin && t.page_end == other.page_end && t.seq == other.seq);
    EXPECT(t.page_end > t.page_begin && t.n_rows >= 0 && t.n_rows <= kPrefillTileRows && t.row0 % kPrefillTileRows == 0);
    if (i % 2 == 0) EXPECT(t.n_rows > 0 && other.row0 == t.row0 + kPrefillTileRows);
    for (int r = 0; r < t.n_rows; ++r) {
      const int gr = t.row0 + r;
      EXPECT(t.row_list + gr / kGroup < static_cast<int>(p.rows.size()));
      const std::int64_t at = static_cast<std::int64_t>(t.part_row0) + r;
      EXPECT(at >= 0 && at < max_rows);
      EXPECT(written.emplace(at, Written{p.rows[static_cast<std::size_t>(t.row_list + gr / kGroup)], t.kvh, gr % kGroup, t.page_begin, t.page_end}).second);
    }
    // the pages the CTA reads are the row's own
    for (int r = 0; r < t.n_rows; r += kGroup) {
      const int b = p.rows[static_cast<std::size_t>(t.row_list + (t.row0 + r) / kGroup)];
      for (int k = t.page_begin; k < t.page_end; ++k) EXPECT(host.table_row(ids[static_cast<std::size_t>(b)])[k] == host.table_row(t.seq)[k]);
    }
  }
  std::size_t found = 0;
  for (int b = 0; b < n; ++b) {
    const int s = ids[static_cast<std::size_t>(b)];
    const std::int64_t len = host.len(s, 0);
    const int pages = static_cast<int>((len + kPageTokens - 1) / kPageTokens);
    const int g = group_of[static_cast<std::size_t>(b)];
    int shared = g >= 0 ? groups[static_cast<std::size_t>(g)].first / kPageTokens : 0;
    if (g >= 0 && (groups[static_cast<std::size_t>(g)].second - 1) * shared < min_saved) shared = 0;
    EXPECT(p.first_page[static_cast<std::size_t>(b)] == shared);
    EXPECT(static_cast<std::int64_t>(shared) * kPageTokens <= len);
    for (int h = 0; h < kKvHeads; ++h) {
      const PrefixItem pi = p.prefix_items[static_cast<std::size_t>(b) * kKvHeads + h];
      for (int j = 0; j < kGroup; ++j) {
        int at = 0;
        for (int k = 0; k < pi.n_parts; ++k) {
          const auto it = written.find(static_cast<std::int64_t>(pi.first) + static_cast<std::int64_t>(k) * pi.stride + j);
          EXPECT(it != written.end());
          EXPECT(it->second.b == b && it->second.h == h && it->second.j == j && it->second.lo == at);
          at = it->second.hi;
          ++found;
        }
        EXPECT(at == shared);
      }
      const CombineItem ci = p.items[static_cast<std::size_t>(b) * kKvHeads + h];
      std::map<int, DecodeUnit> mine;
      for (const DecodeUnit& u : p.units)
        if (u.batch == b && u.kvh == h) EXPECT(mine.emplace(u.partial, u).second && u.seq == s && u.n_keys == len);
      EXPECT(static_cast<int>(mine.size()) == ci.n_partials);
      int at = shared, k = ci.first_partial;
      for (auto& e : mine) {
        EXPECT(e.first == k++ && e.second.page_begin == at && e.second.page_end > at);
        at = e.second.page_end;
      }
      EXPECT(at == pages);
    }
  }
  EXPECT(found == written.size());
  EXPECT(host.PlanDecodeShared(0, n, ids.data(), n_splits, 64, cap * kKvHeads * 64, n_pairs, max_rows, &changed).code == YAHKV_OK && !changed);
  EXPECT(host.SeqReserve(ids[0], host.len(ids[0], 0) + 200).code == YAHKV_OK);   // a changed table is a changed plan
  EXPECT(host.PlanDecodeShared(0, n, ids.data(), n_splits, 64, cap * kKvHeads * 64, n_pairs, max_rows, &changed).code == YAHKV_OK && changed);
}

// Forks of forks: the grouping that saves the most page reads.
static void CheckNested() {
  KvHost host(Config(40, 512, 4096));
  host.SetSharedMinSaved(1);
  std::int32_t src, dst;
  auto fork = [&](std::int32_t from, std::int64_t n, std::int64_t len) {
    std::int32_t s = -1;
    EXPECT(host.SeqFork(from, n, &s, &src, &dst).code == YAHKV_OK);
    return Grow(host, s, len);
  };
  const std::int32_t root = Grow(host, -1, 100 * 64);
  std::vector<std::int32_t> ids;
  for (int i = 0; i < 8; ++i) ids.push_back(fork(root, 100 * 64, 100 * 64 + 10));
  ids.push_back(fork(root, 64, 70));   // a short row: one page in common with all
  auto pages = [&] {
    std::vector<std::int64_t> lens;
    for (int s : ids) lens.push_back(host.len(s, 0));
    std::vector<int> first(ids.size(), 0);
    std::set<std::int32_t> seen;
    for (const auto& g : host.FindPrefixes(static_cast<int>(ids.size()), ids.data(), lens.data()))
      for (std::int32_t b : g.rows) {
        EXPECT(seen.insert(b).second);
        first[static_cast<std::size_t>(b)] = g.pages;
      }
    return first;
  };
  auto first = pages();
  for (int i = 0; i < 8; ++i) EXPECT(first[static_cast<std::size_t>(i)] == 100);
  EXPECT(first[8] == 0);
  // two conversations behind one system prompt: 20 pages for all six rows save 100, 20 + 100 pages for 3 + 3 save 2 x 2 x 120
  ids.clear();
  const std::int32_t sys = Grow(host, -1, 20 * 64);
  for (int c = 0; c < 2; ++c) {
    const std::int32_t conv = fork(sys, 20 * 64, 120 * 64);
    for (int i = 0; i < 3; ++i) ids.push_back(fork(conv, 120 * 64, 120 * 64 + 1 + i));
  }
  for (int p : pages()) EXPECT(p == 120);
  // the same with conversations of two pages each: the system prompt saves more
  ids.clear();
  for (int c = 0; c < 2; ++c) {
    const std::int32_t conv = fork(sys, 20 * 64, 22 * 64);
    for (int i = 0; i < 3; ++i) ids.push_back(fork(conv, 22 * 64, 22 * 64 + 1 + i));
  }
  for (int p : pages()) EXPECT(p == 20);
  // a chain of forks, each one page further
  ids.clear();
  std::int32_t last = Grow(host, -1, 64);
  for (int i = 0; i < 12; ++i) ids.push_back(last = fork(last, (i + 1) * 64, (i + 2) * 64));
  std::int64_t saved = 0;
  std::map<int, int> sizes;
  for (int p : pages()) ++sizes[p];
  for (auto& e : sizes)
    if (e.first > 0) saved += static_cast<std::int64_t>(e.first) * (e.second - 1);
  // row k holds k + 2 pages and shares them with every later row: rows k .. 11 save (11 - k)(k + 2), 42 at most (k = 4, 5)
  EXPECT(sizes.size() <= 2 && saved == 42);
  // below the threshold nothing is grouped
  host.SetSharedMinSaved(43);
  for (int p : pages()) EXPECT(p == 0);
}

static void CheckEvict() {
  KvHost host(Config(6, 8, 24, 2));
  std::int32_t a = Grow(host, -1, 400), b = -1, c = -1, src, dst;   // 7 pages
  EXPECT(host.SeqFork(a, 384, &b, &src, &dst).code == YAHKV_OK && host.SeqFork(a, 384, &c, &src, &dst).code == YAHKV_OK);
  EXPECT(host.SeqFree(a).code == YAHKV_OK);   // b and c share six pages, page 7 is free again
  const std::vector<std::int32_t> before(host.table_row(b), host.table_row(b) + 6);
  const std::int32_t ids[2] = {b, c};
  std::vector<EvictSeq> seqs;
  std::vector<std::int32_t> dsts;
  bool any = false;
  EXPECT(host.PlanEvict(2, ids, 130, &seqs, &dsts, &any).code == YAHKV_OK && any && dsts.size() == 6);
  std::set<std::int32_t> fresh(dsts.begin(), dsts.end());
  EXPECT(fresh.size() == 6);
  for (std::int32_t p : before) EXPECT(fresh.count(p) == 0);   // both still read the shared pages while they move
  EXPECT(host.pages_free() == 18);
  host.CommitEvict(130, seqs, dsts);
  EXPECT(host.pages_free() == 18);   // six taken, six let go of
  for (int i = 0; i < 3; ++i) EXPECT(host.table_row(b)[i] == dsts[static_cast<std::size_t>(i)] && host.table_row(c)[i] == dsts[static_cast<std::size_t>(3 + i)]);
  EXPECT(host.n_pages(b) == 3 && host.len(b, 0) == 130 && host.len(b, 1) == 130 && host.evicted(b));
  // alone in its pages: they stay, and what is behind them is let go of
  const std::vector<std::int32_t> own(host.table_row(b), host.table_row(b) + 3);
  EXPECT(host.PlanEvict(1, &b, 64, &seqs, &dsts, &any).code == YAHKV_OK && any && dsts == std::vector<std::int32_t>{own[0]});
  host.CommitEvict(64, seqs, dsts);
  EXPECT(host.n_pages(b) == 1 && host.table_row(b)[0] == own[0] && host.pages_free() == 20);
  // nothing longer than n_keep: nothing happens
  EXPECT(host.PlanEvict(1, &b, 64, &seqs, &dsts, &any).code == YAHKV_OK && !any && dsts.empty());
  const std::int32_t twice[2] = {b, b};
  EXPECT(host.PlanEvict(2, twice, 10, &seqs, &dsts, &any).code == YAHKV_ERR_INVALID);
  // a fork inherits that slots are not positions; starting over ends it
  std::int32_t d = -1;
  EXPECT(host.SeqFork(b, 64, &d, &src, &dst).code == YAHKV_OK && host.evicted(d));
  EXPECT(host.SeqSetLen(d, -1, 0).code == YAHKV_OK && !host.evicted(d));
  std::int32_t none = -1;   // a fork that holds nothing has no such slots
  EXPECT(host.SeqFork(b, 0, &none, &src, &dst).code == YAHKV_OK && !host.evicted(none) && host.SeqFree(none).code == YAHKV_OK);
  // appending into a page that is shared is refused, and nothing changes
  std::int64_t slot = -1;
  const std::int64_t pos = 0;
  for (int l = 0; l < 2; ++l) EXPECT(host.PlanAppend(l, 1, &d, &pos, &slot).code == YAHKV_ERR_INVALID && host.len(d, l) == 0);
  // no free page left to replace a shared one
  KvHost full(Config(3, 4, 3));
  std::int32_t x = Grow(full, -1, 192), y = -1;
  EXPECT(full.SeqFork(x, 192, &y, &src, &dst).code == YAHKV_OK);
  EXPECT(full.PlanEvict(1, &y, 100, &seqs, &dsts, &any).code == YAHKV_ERR_NO_PAGES && full.n_pages(y) == 3);
}

int main() {
  CheckShared({}, 5, 0, 74, 1);
  CheckShared({{64, 2}}, 0, 0, 74, 2);
  CheckShared({{63, 4}}, 2, 0, 74, 3);
  CheckShared({{8192, 32}}, 0, 0, 74, 4);
  CheckShared({{65536, 16}}, 1, 0, 74, 5);
  CheckShared({{16421, 96}}, 0, 3, 74, 6);
  CheckShared({{640, 43}, {100, 2}, {4000, 1}, {5000, 22}}, 7, 0, 74, 7);
  CheckShared({{2000, 300}}, 3, 64, 74, 8);
  for (unsigned s = 0; s < 30; ++s) {
    std::mt19937 rng(100 + s);
    std::vector<std::pair<int, int>> groups;
    for (unsigned g = 0; g < rng() % 40; ++g) groups.push_back({1 + static_cast<int>(rng() % 3000), 1 + static_cast<int>(rng() % 5)});
    CheckShared(groups, static_cast<int>(rng() % 5) + 1, static_cast<int>(rng() % 9), s % 2 ? 74 : 3, s);
  }
  CheckShared({{640, 8}, {128, 2}, {64 * 64, 2}, {64 * 64 - 1, 2}}, 2, 0, 74, 77, 64);
  CheckNested();
  CheckEvict();
  std::printf("shared_planner_test: ok\n");
  return 0;
}
