"""Accumulated attention weights and eviction by them, against the definitions in float64 over the bytes the cache holds.

Tolerances. A weight is exp of a score over a row sum. A score is the sum of exact products in fp32 (eight partial sums of 32
products each: 8 x 2^-24 of sum|q k| / 16 < 16) of the query, which the quantized formats hold in steps of amax / 524287: half
a step of amax < 5 on each of 256 elements against |k| < 5 is below 5e-6 x 256 x 5 / 16 x 0.5 = 2e-4 if all went one way and
sqrt(256) instead of 256 of it, 1.3e-5, as they do. Once more for the row sum: the bar is 3e-5 of the largest weight. What eviction moves and selects is compared exactly."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from longctx_util import attend64, rows64, select
from test_shared_gpu import FMTS, check, grow, normal

pytestmark = pytest.mark.gpu


def code(f, *args, **kw):
    with pytest.raises(yahkv.YahkvError) as e:
        f(*args, **kw)
    return e.value.code


@pytest.mark.parametrize("fmt", FMTS)
def test_weights_add_up(fmt):
    rng = np.random.default_rng(21)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 130, 1000, 2500]
    cache = yahkv.KvCache(num_pages=sum((n + 64) // 64 + 1 for n in lens), fmt=fmt, max_seqs=len(lens) + 1, max_pages_per_seq=41)
    unused = cache.seq_create()
    seqs = [cache.seq_create() for _ in lens]
    for s, n in zip(seqs, lens):
        grow(cache, rng, s, n)
    order = rng.permutation(len(lens))
    keys = 2503                                            # odd: rows are not 8-byte aligned
    w0 = rng.random((len(lens) + 1, 4, keys), dtype=np.float32) / 64
    w = dev(w0)
    want = w0.astype(np.float64)
    for n_splits in (0, 1, 7):
        q = normal(rng, len(lens), 24, 256)
        rows = [seqs[i] for i in order]
        out, ref = torch.empty(len(lens), 24, 256, device="cuda"), torch.empty(len(lens), 24, 256, device="cuda")
        gate = rng.standard_normal((len(lens), 24, 256)).astype(np.float32)
        cache.attend_decode_weights(0, rows, dev(q), out, w, gate=dev(gate), out_dtype=yahkv.OUT_F32, n_splits=n_splits)
        cache.attend_decode(0, rows, dev(q), ref, gate=dev(gate), out_dtype=yahkv.OUT_F32, n_splits=n_splits)
        cache.sync()
        if fmt == yahkv.FMT_F16:                           # the attention itself is attend_decode's
            assert torch.equal(out, ref)
        else:                                              # whose query is off by up to amax / 64000 per element
            assert (out - ref).abs().max() <= 1e-4 * ref.abs().max()
        top = 0.0
        for b, s in enumerate(rows):
            n = lens[seqs.index(s)]
            p = attend64(q[b], *rows64(cache, 0, s, n))[1].reshape(4, 6, n).sum(1)
            want[s, :, :n] += p
            got = w[s, :, :n].double().cpu().numpy()
            assert np.abs(got - want[s, :, :n]).max() <= 3e-5 * p.max() + 2.0 ** -22 * want[s].max(), (n, n_splits)
            want[s, :, :n] = got                           # the next step is judged by itself
    got = w.cpu().numpy()
    assert np.array_equal(got[unused], w0[unused])
    for s, n in zip(seqs, lens):
        assert np.array_equal(got[s, :, n:], w0[s, :, n:])  # nothing behind the last key
    # the same call again gives the same bits
    a, b = dev(w0), dev(w0)
    for acc in (a, b):
        cache.attend_decode_weights(0, seqs, dev(q), out, acc, out_dtype=yahkv.OUT_F32)
    cache.sync()
    assert torch.equal(a, b)


def weights_of(kind, rng, shape):
    if kind == "heavy":
        return np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 3, shape).astype(np.float32)
    if kind == "zero":
        return np.zeros(shape, np.float32)
    w = rng.standard_normal(shape).astype(np.float32)       # signs, infinities, NaN, both zeros, subnormals
    special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42, -1e-42, 3e38], np.float32)
    hit = rng.random(shape) < 0.4
    return np.where(hit, special[rng.integers(0, len(special), shape)], w).astype(np.float32)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", ["heavy", "ties", "zero", "special"])
@pytest.mark.parametrize("forked", [False, True])
def test_evict_keeps_moves_and_releases(fmt, kind, forked):
    rng = np.random.default_rng(31)
    layers, keys = 2, 2600
    for keep, sink, recent in ((1, 0, 0), (1, 1, 0), (64, 4, 16), (100, 0, 100), (129, 129, 0), (500, 3, 77), (1024, 1, 1)):
        lens = [keep, keep + 1, max(keep - 5, 1), keep + 64, keep + 700, 2 * keep + 1]
        cache = yahkv.KvCache(n_layers=layers, num_pages=sum((n + 63) // 64 for n in lens) * 2 + 8, fmt=fmt, max_seqs=2 * len(lens),
                              max_pages_per_seq=42)
        seqs = [cache.seq_create() for _ in lens]
        for s, n in zip(seqs, lens):
            grow(cache, rng, s, n, range(layers))
        origin, before = list(seqs), {}
        if forked:                                          # shared pages stay with the origin
            seqs = [cache.seq_fork(s, n) for s, n in zip(seqs, lens)]
        for layer in range(layers):
            for i, s in enumerate(origin):
                before[layer, i] = rows64(cache, layer, s, lens[i])
        w0 = weights_of(kind, rng, (layers, 2 * len(lens), 4, keys))
        w, kept = dev(w0), torch.full((layers, len(seqs), 4, keep), -7, device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        free, tables = cache.pages_free(), [cache.seq_table(s) for s in seqs]
        cache.evict(seqs, keep, w, kept, n_sink=sink, n_recent=recent)
        cache.sync()
        got_w, got = w.cpu().numpy(), kept.cpu().numpy()
        for i, (s, n) in enumerate(zip(seqs, lens)):
            np_keep = (keep + 63) // 64
            for layer in range(layers):
                m = min(n, keep)
                assert cache.seq_len(s, layer) == m
                k, v = rows64(cache, layer, s, m)
                for h in range(4):
                    want = select(w0[layer, s, h], n, keep, sink, recent)
                    assert got[layer, i, h].tolist() == want, (keep, n, layer, h)
                    idx = want[:m]
                    assert np.array_equal(k[:, h], before[layer, i][0][idx, h]) and np.array_equal(v[:, h], before[layer, i][1][idx, h])
                    row = w0[layer, s, h].copy()
                    if n > keep:
                        row[:keep], row[keep:n] = w0[layer, s, h][idx], 0.0
                    assert np.array_equal(got_w[layer, s, h], row, equal_nan=True)
                if forked:
                    now = rows64(cache, layer, origin[i], n)
                    assert all(np.array_equal(now[side], before[layer, i][side]) for side in (0, 1))
            if n > keep:
                assert len(cache.seq_table(s)) == np_keep
                if not forked:
                    assert cache.seq_table(s).tolist() == tables[i][:np_keep].tolist()
            else:
                assert cache.seq_table(s).tolist() == tables[i].tolist()
        live = sum(len(set(cache.seq_table(s).tolist())) for s in seqs)
        if not forked:
            assert cache.pages_free() == free + sum(len(t) for t in tables) - live
        # attention over what is left, and the next token
        q = normal(rng, len(seqs), 24, 256)
        out = torch.empty(len(seqs), 24, 256, device="cuda")
        for s in seqs:
            grow(cache, rng, s, 1, range(layers))
        cache.attend_decode(1, seqs, dev(q), out, out_dtype=yahkv.OUT_F32)
        cache.sync()
        check(cache, 1, seqs, q, out.double().cpu().numpy())
        cache.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_branches_of_one_prefix_cut_in_one_call(fmt):
    """Two holders of the same pages, nobody else: both are cut at once, each by its own weights, in a full pool."""
    rng = np.random.default_rng(41)
    cache = yahkv.KvCache(num_pages=16, fmt=fmt, max_seqs=3, max_pages_per_seq=10)
    root = cache.seq_create()
    grow(cache, rng, root, 640)
    a, b = cache.seq_fork(root, 640), cache.seq_fork(root, 640)
    before = rows64(cache, 0, a, 640)
    cache.seq_free(root)
    w0 = weights_of("heavy", rng, (1, 3, 4, 640))
    kept = torch.empty(1, 2, 4, 150, device="cuda", dtype=torch.int32)
    assert cache.pages_free() == 6
    cache.evict([a, b], 150, dev(w0), kept, n_recent=30)
    cache.sync()
    assert cache.pages_free() == 10
    for i, s in enumerate((a, b)):
        k, v = rows64(cache, 0, s, 150)
        for h in range(4):
            want = select(w0[0, s, h], 640, 150, 0, 30)
            assert kept[0, i, h].tolist() == want
            assert np.array_equal(k[:, h], before[0][want, h]) and np.array_equal(v[:, h], before[1][want, h])


def test_a_long_row():
    """More keys than a CTA takes in one turn, many of them tied at the border."""
    rng = np.random.default_rng(43)
    n, keep = 40000, 9001
    cache = yahkv.KvCache(num_pages=626, fmt=yahkv.FMT_Q4_0, max_seqs=1, max_pages_per_seq=626)
    s = cache.seq_create()
    grow(cache, rng, s, n)
    before = rows64(cache, 0, s, n)
    w0 = np.floor(8 * rng.random((1, 1, 4, n))).astype(np.float32)
    kept = torch.empty(1, 1, 4, keep, device="cuda", dtype=torch.int32)
    cache.evict([s], keep, dev(w0), kept, n_sink=5, n_recent=1000)
    cache.sync()
    k, v = rows64(cache, 0, s, keep)
    for h in range(4):
        want = select(w0[0, 0, h], n, keep, 5, 1000)
        assert kept[0, 0, h].tolist() == want
        assert np.array_equal(k[:, h], before[0][want, h]) and np.array_equal(v[:, h], before[1][want, h])


def test_head_sharded_contexts_cut_their_own_heads():
    rng = np.random.default_rng(47)
    cache = yahkv.KvCache(num_pages=20, fmt=yahkv.FMT_Q8_0, max_seqs=1, max_pages_per_seq=10, kv_head_begin=2, kv_head_count=1)
    s = cache.seq_create()
    grow(cache, rng, s, 300)
    before = rows64(cache, 0, s, 300)
    w0 = weights_of("heavy", rng, (1, 1, 4, 300))
    w, kept = dev(w0), torch.full((1, 1, 4, 70), -7, device="cuda", dtype=torch.int32)
    q, out = normal(rng, 1, 24, 256), torch.zeros(1, 24, 256, device="cuda")
    cache.attend_decode_weights(0, [s], dev(q), out, w[0], out_dtype=yahkv.OUT_F32)
    cache.sync()
    now = w.cpu().numpy()
    assert np.array_equal(now[:, :, [0, 1, 3]], w0[:, :, [0, 1, 3]]) and not np.array_equal(now[:, :, 2], w0[:, :, 2])
    cache.evict([s], 70, w, kept)
    cache.sync()
    want = select(now[0, 0, 2], 300, 70, 0, 0)
    assert kept[0, 0, 2].tolist() == want and (kept[0, 0, [0, 1, 3]] == -7).all()
    assert np.array_equal(rows64(cache, 0, s, 70)[0][:, 2], before[0][want, 2])


def test_refusals_and_positions_after_an_eviction(tmp_path):
    rng = np.random.default_rng(51)
    cache = yahkv.KvCache(n_layers=2, num_pages=16, fmt=yahkv.FMT_Q8_0, max_seqs=3, max_pages_per_seq=6)
    a, b = cache.seq_create(), cache.seq_create()
    grow(cache, rng, a, 200, (0, 1))
    grow(cache, rng, b, 100, (0, 1))
    w = torch.rand(2, 3, 4, 200, device="cuda")
    kept = torch.empty(2, 1, 4, 50, device="cuda", dtype=torch.int32)
    q, out = dev(normal(rng, 1, 24, 256)), torch.zeros(1, 24, 256, device="cuda")
    aw = cache.attend_decode_weights
    two = torch.empty(2, 2, 4, 50, device="cuda", dtype=torch.int32)
    assert code(aw, 0, [a, a], q, out, w[0]) == yahkv.ERR_INVALID
    assert code(aw, 0, [2], q, out, w[0]) == yahkv.ERR_INVALID
    assert code(aw, 2, [a], q, out, w[0]) == yahkv.ERR_INVALID
    assert code(aw, 0, [a], q.flatten()[1:], out, w[0]) == yahkv.ERR_INVALID
    assert code(aw, 0, [a], q, out, w[0, :, :, :199].contiguous()) == yahkv.ERR_CAPACITY
    with pytest.raises(ValueError):
        aw(0, [a], q, out, w[0, :2])
    with pytest.raises(ValueError):
        aw(0, [a], q, out, w[0].double())
    with pytest.raises(ValueError):
        aw(0, [a], q, out, w[0].cpu())
    ev = cache.evict
    for n_keep, sink, recent in ((50, -1, 0), (50, 0, -1), (50, 51, 0), (50, 30, 21)):
        assert code(ev, [a], n_keep, w, kept, n_sink=sink, n_recent=recent) == yahkv.ERR_INVALID
    assert code(ev, [a], 0, w, kept[..., :0].contiguous()) == yahkv.ERR_INVALID
    raw = yahkv.lib.yahkv_evict
    assert raw(cache._h, 1, yahkv._ptr(yahkv._i32([a])), 50, 0, 0, w.data_ptr() + 2, 200, 2400, yahkv._ptr(kept), None) == yahkv.ERR_INVALID
    assert raw(cache._h, 1, yahkv._ptr(yahkv._i32([a])), 50, 0, 0, yahkv._ptr(w), 200, 2400, kept.data_ptr() + 2, None) == yahkv.ERR_INVALID
    assert code(ev, [a, a], 50, w, two) == yahkv.ERR_INVALID
    assert code(ev, [2], 50, w, kept) == yahkv.ERR_INVALID
    assert yahkv.lib.yahkv_evict(cache._h, 1, yahkv._ptr(yahkv._i32([a])), 50, 0, 0, yahkv._ptr(w), 200, 100, yahkv._ptr(kept), None) == yahkv.ERR_INVALID
    assert yahkv.lib.yahkv_evict(cache._h, 1, yahkv._ptr(yahkv._i32([a])), 50, 0, 0, yahkv._ptr(w), 200, 2400, None, None) == yahkv.ERR_INVALID
    assert yahkv.lib.yahkv_evict(cache._h, 1, yahkv._ptr(yahkv._i32([a])), 50, 0, 0, None, 200, 2400, yahkv._ptr(kept), None) == yahkv.ERR_INVALID
    with pytest.raises(ValueError):
        ev([a], 51, w, kept)
    cache.seq_set_len(b, 90, layer=1)
    assert code(ev, [b], 50, w, kept) == yahkv.ERR_ORDER                # unequal layers
    assert cache.seq_len(a, 0) == 200 and cache.seq_len(b, 0) == 100    # nothing happened
    ev([], 50, w, torch.empty(2, 0, 4, 50, device="cuda", dtype=torch.int32))
    # host tables change or host lists are read: not inside a capture
    graph, spare = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        spare += 1
        sp = torch.cuda.current_stream().cuda_stream
        assert code(ev, [a], 50, w, kept, stream=sp) == yahkv.ERR_ORDER
        assert code(cache.seq_fork, a, 70, stream=sp) == yahkv.ERR_ORDER
        assert code(aw, 0, [a], q, out, w[0], stream=sp) == yahkv.ERR_ORDER
        assert code(cache.attend_decode_shared, 0, [a], q, out, stream=sp) == yahkv.ERR_ORDER
    assert cache.seq_len(a, 0) == 200 and cache.pages_free() == 10
    ev([a], 50, w, kept)
    # slots are not positions any more: the calls that would take them for positions refuse, for forks as well
    f32 = [dev(rng.standard_normal((1, n, 256)).astype(np.float32)) for n in (24, 4, 4)]
    ones = torch.ones(256, device="cuda")
    fork = cache.seq_fork(a, 40)
    for s, n in ((a, 50), (fork, 40)):
        assert code(cache.rope_append, 0, [s], [n], *f32, ones, ones, 1e-6, None) == yahkv.ERR_ORDER
        assert code(cache.attend_decode_qraw, 0, [s], f32[0], ones, 1e-6, out, out_dtype=yahkv.OUT_F32) == yahkv.ERR_ORDER
        assert code(cache.attend_prefill_qraw, 0, [s], [1], f32[0], ones, 1e-6, out, out_dtype=yahkv.OUT_F32) == yahkv.ERR_ORDER
    batch = yahkv.DecodeBatch(cache, [a])
    batch.prepare(2)
    batch.plan()
    assert code(batch.decode_layer_raw, 0, *f32, ones, ones, 1e-6, out, out_dtype=yahkv.OUT_F32) == yahkv.ERR_ORDER
    # a batch's lengths are on the device: its sequences are not cut under it
    few = torch.empty(2, 1, 4, 20, device="cuda", dtype=torch.int32)
    n = cache.seq_len(a, 0)
    second = yahkv.DecodeBatch(cache, [a])
    assert n > 20 and code(ev, [a], 20, w, few) == yahkv.ERR_ORDER
    batch.close()
    assert code(ev, [a], 20, w, few) == yahkv.ERR_ORDER and cache.seq_len(a, 0) == n
    second.close()
    # a snapshot keeps the mark
    cache.snapshot_save([b], tmp_path / "plain")
    cache.snapshot_save([a, b], tmp_path / "marked")
    assert open(tmp_path / "plain", "rb").read(8) == b"YAHKVSN1" and open(tmp_path / "marked", "rb").read(8) == b"YAHKVSN2"
    cache.seq_free(fork)
    other = yahkv.KvCache(n_layers=2, num_pages=16, fmt=yahkv.FMT_Q8_0, max_seqs=3, max_pages_per_seq=6)
    x, y = other.snapshot_load(tmp_path / "marked")
    assert code(other.rope_append, 0, [x], [50], *f32, ones, ones, 1e-6, None) == yahkv.ERR_ORDER
    for side in (0, 1):
        assert np.array_equal(rows64(other, 1, x, 50)[side], rows64(cache, 1, a, 50)[side])
    other.seq_reserve(y, 101)
    other.rope_append(0, [y], [100], *f32, ones, ones, 1e-6, None)
    cache.seq_set_len(a, 0)                                             # starts over
    cache.rope_append(0, [a], [0], *f32, ones, ones, 1e-6, None)
    cache.sync()
    other.sync()
    tile = yahkv.KvCache(num_pages=2, fmt=yahkv.FMT_KV4A16, max_seqs=1, max_pages_per_seq=2)
    s = tile.seq_create()
    tw = torch.zeros(1, 1, 4, 128, device="cuda")
    assert code(tile.evict, [s], 10, tw, torch.empty(1, 1, 4, 10, device="cuda", dtype=torch.int32)) == yahkv.ERR_INVALID
    assert code(tile.attend_decode_weights, 0, [s], q, out, tw[0]) == yahkv.ERR_INVALID
