"""A sequence whose table was set to fewer pages than its length needs: what lies behind the table is not the sequence's, so it
can be neither forked nor cut until its length fits."""
import os
import subprocess

import pytest

import yahkv
from test_longctx_cpu import code, grown, host_ctx
from test_planner_cpu import PKG, ROOT, _cuda_include


def test_no_page_behind_the_table_is_shared():
    c = host_ctx()
    a = grown(c, 256)
    pages = c.seq_table(a).tolist()
    c.seq_set_table(a, pages[:1])                            # three pages go back to the pool, the length stays
    assert code(c.seq_fork, a, 128) == yahkv.ERR_ORDER
    assert c.pages_free() == 9
    b = c.seq_fork(a, 64)
    assert c.seq_table(b).tolist() == pages[:1]
    c.seq_set_len(a, 64)
    d = c.seq_fork(a, 64)
    others = [grown(c, 64 * 6), grown(c, 64 * 3)]            # every free page, once each
    held = [p for s in others for p in c.seq_table(s).tolist()]
    assert len(set(held)) == 9 and pages[0] not in held
    for s in (a, b, d, *others):
        c.seq_free(s)
    assert c.pages_free() == 10


def test_no_page_behind_the_table_is_cut(tmp_path):
    inc = _cuda_include()
    if inc is None:
        pytest.skip("no CUDA include directory found")
    src = tmp_path / "short_table.cc"
    src.write_text(r'''
#include <cstdio>
#include "csrc/kv_host.hpp"
using namespace yahkv;
int main() {
  yahkv_config c{};
  c.n_layers = 1, c.num_pages = 16, c.fmt = YAHKV_FMT_Q8_0, c.max_seqs = 4, c.max_pages_per_seq = 8, c.max_batch_tokens = 64, c.max_splits = 64;
  KvHost host(c);
  std::int32_t s = -1, first = 0;
  host.SeqCreate(&s), host.SeqReserve(s, 400), host.SeqSetLen(s, -1, 400);
  first = host.table_row(s)[0];
  host.SeqSetTable(s, &first, 1);
  std::vector<EvictSeq> seqs;
  std::vector<std::int32_t> pages;
  bool any = false;
  if (host.PlanEvict(1, &s, 130, &seqs, &pages, &any).code != YAHKV_ERR_ORDER || host.pages_free() != 15) return 1;
  host.SeqReserve(s, 400);                       // pages for the length again: other ones, but its own
  if (host.PlanEvict(1, &s, 130, &seqs, &pages, &any).code != YAHKV_OK || !any || pages.size() != 3) return 2;
  for (int i = 0; i < 3; ++i) if (pages[i] != host.table_row(s)[i]) return 3;
  host.CommitEvict(130, seqs, pages);
  if (host.pages_free() != 13 || host.n_pages(s) != 3) return 4;
  std::puts("ok");
  return 0;
}
''')
    exe = tmp_path / "short_table"
    cmd = ["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", PKG, "-I", inc, str(src), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "ok" in r.stdout, (r.returncode, r.stdout, r.stderr)
