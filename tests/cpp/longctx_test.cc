// The adapter's long-context calls on a host-only context: forks share pages, and what needs a GPU throws KvError.
#include <cstdio>
#include <cstdlib>

#include "engine/model/kv_cache.hpp"

using yah::model::KvCache;
using yah::model::KvError;

#define EXPECT(c)                                                         \
  do {                                                                    \
    if (!(c)) {                                                           \
      std::fprintf(stderr, "%s:%d: EXPECT(%s) failed\n", __FILE__, __LINE__, #c); \
      std::exit(1);                                                       \
    }                                                                     \
  } while (0)

template <class F>
static int CodeOf(F&& f) {
  try {
    f();
  } catch (const KvError& e) {
    return e.code();
  }
  return YAHKV_OK;
}

int main() {
  KvCache kv = KvCache::OwnState(KvCache::Config(/*device=*/-1, /*n_layers=*/2, /*num_pages=*/8, /*max_seqs=*/3, /*max_pages_per_seq=*/4));
  const std::int32_t a = kv.NewSequence();
  kv.Reserve(a, 200);
  kv.SetLength(a, 200);
  const std::int32_t b = kv.Fork(a, 128);
  EXPECT(kv.Length(b, 1) == 128 && kv.Table(b).size() == 2 && kv.Table(b)[1] == kv.Table(a)[1] && kv.PagesFree() == 4);
  EXPECT(CodeOf([&] { (void)kv.Fork(a, 201); }) == YAHKV_ERR_ORDER);
  EXPECT(CodeOf([&] { (void)kv.Fork(a, 100); }) == YAHKV_ERR_NO_DEVICE);
  EXPECT(CodeOf([&] { kv.AttendDecodeShared(0, {a, b}, nullptr, nullptr, nullptr); }) == YAHKV_ERR_NO_DEVICE);
  EXPECT(CodeOf([&] { kv.AttendDecodeWeights(0, {a}, nullptr, nullptr, nullptr, nullptr, 256); }) == YAHKV_ERR_NO_DEVICE);
  EXPECT(CodeOf([&] { kv.Evict({a}, 64, 0, 0, nullptr, 256, 0, nullptr); }) == YAHKV_ERR_NO_DEVICE);
  yahkv_rope_config rc{};
  rc.rotary_dim = 64, rc.theta = 1e7, rc.max_positions = 1024;
  EXPECT(CodeOf([&] { KvCache::Rope rope(kv, rc); }) == YAHKV_ERR_NO_DEVICE);
  kv.FreeSequence(a);
  EXPECT(kv.PagesFree() == 6);
  kv.FreeSequence(b);
  EXPECT(kv.PagesFree() == 8);
  std::puts("longctx_test: ok");
  return 0;
}
