// Host-only check that the second half of an eviction, which follows the kernels, cannot fail: with every allocation refused
// after PlanEvict, CommitEvict still moves the tables over. And that decode plans made before it are dropped.
#include <cstdio>
#include <cstdlib>
#include <new>

#include "csrc/kv_host.hpp"

static bool g_refuse = false;
void* operator new(std::size_t n) {
  void* p = g_refuse ? nullptr : std::malloc(n);
  if (p == nullptr) throw std::bad_alloc();
  return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

#define EXPECT(c)                                                         \
  do {                                                                    \
    if (!(c)) {                                                           \
      std::fprintf(stderr, "%s:%d: EXPECT(%s) failed\n", __FILE__, __LINE__, #c); \
      std::exit(1);                                                       \
    }                                                                     \
  } while (0)

using namespace yahkv;

int main() {
  yahkv_config c{};
  c.n_layers = 2, c.num_pages = 64, c.fmt = YAHKV_FMT_Q8_0, c.max_seqs = 8, c.max_pages_per_seq = 16, c.max_batch_tokens = 64;
  c.max_splits = 64;
  KvHost host(c);
  std::int32_t ids[3] = {-1, -1, -1}, src, dst;
  EXPECT(host.SeqCreate(&ids[0]).code == YAHKV_OK && host.SeqReserve(ids[0], 900).code == YAHKV_OK && host.SeqSetLen(ids[0], -1, 900).code == YAHKV_OK);
  for (int i = 1; i < 3; ++i) EXPECT(host.SeqFork(ids[0], 896, &ids[i], &src, &dst).code == YAHKV_OK);
  host.ForEachDirty([](int, int, int) {});
  std::vector<EvictSeq> seqs;
  std::vector<std::int32_t> pages;
  bool any = false;
  EXPECT(host.PlanEvict(3, ids, 130, &seqs, &pages, &any).code == YAHKV_OK && any);
  const int free_before = host.pages_free();
  bool threw = false;
  g_refuse = true;
  try {
    host.CommitEvict(130, seqs, pages);
  } catch (...) {
    threw = true;
  }
  g_refuse = false;
  EXPECT(!threw);
  int held = 0;
  for (std::int32_t s : ids) {
    EXPECT(host.len(s, 0) == 130 && host.len(s, 1) == 130 && host.n_pages(s) == 3);
    for (int i = 0; i < 3; ++i, ++held) EXPECT(host.page_refs(host.table_row(s)[i]) == 1);
  }
  EXPECT(held == 9 && host.pages_free() == 64 - held && host.pages_free() > free_before);
  int dirty = 0;
  host.ForEachDirty([&](int, int lo, int hi) { dirty += hi - lo; });
  EXPECT(dirty == 9);
  // the lists of a decode call are made anew, also where id and length come again
  bool changed = false;
  EXPECT(host.PlanDecode(0, 1, &ids[1], 0, 64, 256, &changed).code == YAHKV_OK && changed);
  EXPECT(host.PlanDecode(0, 1, &ids[1], 0, 64, 256, &changed).code == YAHKV_OK && !changed);
  EXPECT(host.PlanDecodeShared(0, 1, &ids[1], 0, 64, 256, 74, 40000, &changed).code == YAHKV_OK && changed);
  const std::int32_t id = ids[1];
  EXPECT(host.SeqFree(ids[1]).code == YAHKV_OK && host.SeqCreate(&ids[1]).code == YAHKV_OK && ids[1] == id);
  EXPECT(host.SeqReserve(id, 900).code == YAHKV_OK && host.SeqSetLen(id, -1, 900).code == YAHKV_OK);
  EXPECT(host.PlanEvict(1, &id, 130, &seqs, &pages, &any).code == YAHKV_OK && any);
  host.CommitEvict(130, seqs, pages);
  EXPECT(host.PlanDecode(0, 1, &id, 0, 64, 256, &changed).code == YAHKV_OK && changed);
  EXPECT(host.PlanDecodeShared(0, 1, &id, 0, 64, 256, 74, 40000, &changed).code == YAHKV_OK && changed);
  std::printf("evict_commit_test: ok\n");
  return 0;
}
