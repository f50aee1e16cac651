"""Forked sequences on a host-only context: shared pages are counted, never handed out twice and never written; the calls
that need a GPU refuse to run; the host-only planner test of shared prefixes."""
import os
import subprocess

import numpy as np
import pytest

import yahkv
from test_planner_cpu import PKG, ROOT, _cuda_include


def host_ctx(**kw):
    args = dict(device=-1, n_layers=2, num_pages=10, max_seqs=6, max_pages_per_seq=6)
    args.update(kw)
    return yahkv.KvCache(**args)


def code(call, *a, **k):
    with pytest.raises(yahkv.YahkvError) as e:
        call(*a, **k)
    return e.value.code


def grown(c, n):
    s = c.seq_create()
    c.seq_reserve(s, n)
    c.seq_set_len(s, n)
    return s


def test_fork_shares_whole_pages_and_counts_them():
    c = host_ctx()
    a = grown(c, 200)                                        # pages 0 .. 3
    free = c.pages_free()
    b = c.seq_fork(a, 128)
    assert c.seq_table(b).tolist() == c.seq_table(a).tolist()[:2] and c.pages_free() == free
    assert c.seq_len(b, 0) == c.seq_len(b, 1) == 128
    d = c.seq_fork(b, 64)                                    # a fork of a fork
    assert c.seq_table(d).tolist() == [0]
    e = c.seq_fork(a, 0)
    assert c.seq_table(e).size == 0 and c.seq_len(e, 0) == 0
    c.seq_free(a)                                            # pages 0, 1 stay with b and d
    assert c.pages_free() == free + 2
    c.seq_reserve(e, 64 * 6)
    assert not set(c.seq_table(e).tolist()) & {0, 1}
    c.seq_free(b)
    assert c.seq_table(d).tolist() == [0]
    c.seq_free(e)
    c.seq_free(d)
    assert c.pages_free() == 10
    every = [grown(c, 64) for _ in range(6)]                 # every page is handed out once
    assert len({int(c.seq_table(s)[0]) for s in every}) == 6


def test_fork_refusals_leave_everything_as_it_was():
    c = host_ctx(num_pages=3, max_seqs=2)
    a = grown(c, 150)
    c.seq_set_len(a, 100, layer=1)
    assert code(c.seq_fork, a, 128) == yahkv.ERR_ORDER       # layer 1 holds 100
    assert code(c.seq_fork, a, -1) == yahkv.ERR_INVALID
    assert code(c.seq_fork, 1, 0) == yahkv.ERR_INVALID       # not live
    assert code(c.seq_fork, a, 70) == yahkv.ERR_NO_DEVICE    # a copy of a page needs the GPU
    b = c.seq_fork(a, 64)
    assert code(c.seq_fork, a, 64) == yahkv.ERR_CAPACITY     # max_seqs
    c.seq_free(b)
    assert c.pages_free() == 0 and c.seq_table(a).size == 3
    t = host_ctx(fmt=yahkv.FMT_KV8A16)
    s = t.seq_create()
    assert code(t.seq_fork, s, 0) == yahkv.ERR_INVALID


def test_shared_pages_cannot_be_claimed_by_a_table():
    c = host_ctx()
    a = grown(c, 192)
    b = c.seq_fork(a, 128)
    p = c.seq_table(a).tolist()
    assert code(c.seq_set_table, b, [p[0], p[1]]) == yahkv.ERR_INVALID   # held by a as well
    assert code(c.seq_set_table, a, p) == yahkv.ERR_INVALID              # held by b as well
    assert code(c.seq_set_table, b, [p[2]]) == yahkv.ERR_INVALID         # a's own
    assert c.seq_table(b).tolist() == p[:2]
    c.seq_free(a)
    c.seq_set_table(b, [p[1], 9])                                        # now b's own, and a free one
    assert c.seq_table(b).tolist() == [p[1], 9] and c.pages_free() == 8


def test_gpu_calls_refuse_a_host_only_context():
    c = host_ctx()
    s = grown(c, 64)
    x = np.zeros(8)
    assert code(c.attend_decode_shared, 0, [s], x, x) == yahkv.ERR_NO_DEVICE
    assert yahkv.lib.yahkv_attend_decode_weights(c._h, 0, 0, None, None, None, None, 0, 0, None, 0, None) == yahkv.ERR_NO_DEVICE
    assert yahkv.lib.yahkv_evict(c._h, 0, None, 1, 0, 0, None, 0, 0, None, None) == yahkv.ERR_NO_DEVICE
    assert code(yahkv.Rope, c) == yahkv.ERR_NO_DEVICE
    with pytest.raises(ValueError):
        yahkv.Rope(c, layout="diagonal")


def test_shared_prefix_planner_on_the_host(tmp_path):
    inc = _cuda_include()
    if inc is None:
        pytest.skip("no CUDA include directory found")
    exe = tmp_path / "shared_planner_test"
    cmd = ["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", PKG, "-I", inc,
           os.path.join(ROOT, "tests", "cpp", "shared_planner_test.cc"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "shared_planner_test: ok" in r.stdout, r.stdout + r.stderr


def test_cpp_adapter_calls_on_a_host_only_context(tmp_path):
    exe = tmp_path / "longctx_test"
    cmd = ["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", PKG,
           os.path.join(ROOT, "tests", "cpp", "longctx_test.cc"), yahkv.LIB_PATH, "-Wl,-rpath," + PKG, "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "longctx_test: ok" in r.stdout, r.stdout + r.stderr


def test_tables_of_shared_pages_cannot_be_set_by_hand():
    cache = yahkv.KvCache(device=-1, num_pages=8, max_seqs=3, max_pages_per_seq=8)
    a = cache.seq_create()
    cache.seq_reserve(a, 256)
    cache.seq_set_len(a, 256)
    table = cache.seq_table(a)
    cache.seq_set_table(a, table[::-1].copy())                 # its own pages, in another order
    cache.seq_set_table(a, table)
    cache.seq_set_len(a, 256)
    b = cache.seq_fork(a, 128)
    for s, pages in ((a, table), (b, table[:2]), (b, table[2:3])):
        with pytest.raises(yahkv.YahkvError) as e:
            cache.seq_set_table(s, pages)
        assert e.value.code == yahkv.ERR_INVALID
    assert list(cache.seq_table(a)) == list(table) and list(cache.seq_table(b)) == list(table[:2])
    cache.seq_set_table(a, table[2:])                          # what only it holds
    assert cache.pages_free() == 4
    cache.seq_set_table(b, table[:2])                          # alone in them now
    cache.seq_free(b)
    cache.seq_free(a)
    assert cache.pages_free() == 8


def test_sequence_ids_of_any_kind():
    for ids in ([3, 0, 7], (3, 0, 7), np.array([3, 0, 7]), np.array([3, 0, 7], np.int64), [3.0, 0.0, 7.0], np.array([[3], [0], [7]])):
        keep, address, n = yahkv._ids(ids)
        assert n == 3 and list(keep) == [3, 0, 7] and address == keep.buffer_info()[0]
    assert yahkv._ids([])[1:] == (None, 0)
