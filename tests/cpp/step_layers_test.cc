// Host-only check of when a plan is made: once per step for all layers of it, again when a layer comes again, and with lists
// that do not depend on what was planned before.
#include <cstdio>
#include <cstdlib>
#include <cstring>
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

template <class T>
static bool Same(const std::vector<T>& a, const std::vector<T>& b) {
  return a.size() == b.size() && (a.empty() || std::memcmp(a.data(), b.data(), a.size() * sizeof(T)) == 0);
}

int main() {
  yahkv_config c{};
  c.n_layers = 3, c.num_pages = 2000, c.fmt = YAHKV_FMT_Q8_0, c.max_seqs = 12, c.max_pages_per_seq = 300, c.max_batch_tokens = 64, c.max_splits = 64;
  KvHost host(c);
  std::int32_t root = -1, src, dst;
  EXPECT(host.SeqCreate(&root).code == YAHKV_OK && host.SeqReserve(root, 100 * 64).code == YAHKV_OK && host.SeqSetLen(root, -1, 100 * 64).code == YAHKV_OK);
  std::vector<std::int32_t> ids;
  for (int i = 0; i < 9; ++i) {
    std::int32_t s = -1;
    EXPECT(host.SeqFork(root, 100 * 64, &s, &src, &dst).code == YAHKV_OK && host.SeqReserve(s, 150 * 64).code == YAHKV_OK);
    EXPECT(host.SeqSetLen(s, -1, 100 * 64 + 300 * i).code == YAHKV_OK);
    ids.push_back(s);
  }
  const int n = static_cast<int>(ids.size());
  StepLayers layers;
  int plans = 0;
  auto call = [&](int layer) {   // as the entry point does
    bool changed = false;
    if (layers.Comes(layer)) host.InvalidateSharedPlan();
    EXPECT(host.PlanDecodeShared(layer, n, ids.data(), 0, 64, 12 * 256, 74, 40000, &changed).code == YAHKV_OK);
    layers.Serve(layer, c.n_layers, changed);
    plans += changed ? 1 : 0;
  };
  EXPECT(!layers.Comes(-1) && !layers.Comes(0) && !layers.Comes(99));
  for (int l = 0; l < 3; ++l) call(l);
  EXPECT(plans == 1);
  const KvHost::SharedPlan first = host.shared_plan();
  for (int l = 0; l < 3; ++l) call(l);   // the next step, nothing has changed
  EXPECT(plans == 2);
  call(0), call(0), call(0);             // one layer only: every call plans
  EXPECT(plans == 5);
  call(1), call(2), call(2);
  EXPECT(plans == 6);
  const KvHost::SharedPlan again = host.shared_plan();
  EXPECT(Same(first.tiles, again.tiles) && Same(first.rows, again.rows) && Same(first.prefix_items, again.prefix_items) &&
         Same(first.units, again.units) && Same(first.items, again.items) && first.first_page == again.first_page);
  for (std::int32_t s : ids) EXPECT(host.SeqSetLen(s, 1, 50 * 64 + s).code == YAHKV_OK);   // another length in one layer
  call(1), call(0);
  EXPECT(plans == 8);
  // units, longest first and equal ones in order, whatever was planned before; partials and score slots in the order they were cut
  bool changed = false;
  for (std::int32_t s : ids) EXPECT(host.SeqSetLen(s, -1, 100 * 64 + 7 * s).code == YAHKV_OK);
  EXPECT(host.PlanDecode(0, n, ids.data(), 5, 64, 12 * 256, &changed).code == YAHKV_OK && changed);
  const auto units = host.units();
  const auto items = host.items();
  EXPECT(host.PlanDecode(0, 2, ids.data(), 0, 64, 12 * 256, &changed).code == YAHKV_OK && changed);
  EXPECT(host.PlanDecode(0, n, ids.data(), 5, 64, 12 * 256, &changed).code == YAHKV_OK && changed);
  EXPECT(Same(units, host.units()) && Same(items, host.items()));
  std::vector<int> slot_of(units.size(), -1), pages_of(units.size(), 0);
  for (std::size_t i = 0; i < units.size(); ++i) {
    const int len = units[i].page_end - units[i].page_begin;
    if (i > 0) {
      const int before = units[i - 1].page_end - units[i - 1].page_begin;
      EXPECT(len < before || (len == before && units[i].partial > units[i - 1].partial));
    }
    EXPECT(slot_of[static_cast<std::size_t>(units[i].partial)] < 0);
    slot_of[static_cast<std::size_t>(units[i].partial)] = units[i].pad, pages_of[static_cast<std::size_t>(units[i].partial)] = len;
  }
  int slot = 0;
  for (std::size_t i = 0; i < units.size(); ++i) {
    EXPECT(slot_of[i] == slot);
    slot += pages_of[i];
  }
  EXPECT(slot == host.unit_pages());
  std::printf("step_layers_test: ok\n");
  return 0;
}
