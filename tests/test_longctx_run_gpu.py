"""The long-context calls together, as a batch server uses them, and shared prefixes in device-resident decode batches (eager and
replayed), against float64 attention over the bytes the caches hold (tolerances: test_shared_gpu.py)."""
import math

import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from longctx_util import attend64, rows64, select
from test_rope_rows_gpu import freqs, rotate64
from test_shared_gpu import FMTS, check, extend, grow, normal, shared, small_cache

pytestmark = pytest.mark.gpu
EPS = 1e-6


def forked_batch(fmt, rng, layers=2, extra=8, prefix=200, max_seqs=8):
    """Two groups of forks and a lone row: (cache, sequences)."""
    cache = small_cache(n_layers=layers, num_pages=80, fmt=fmt, max_seqs=max_seqs, max_pages_per_seq=30)
    seqs = []
    for n, rows in ((prefix, 3), (700, 2)):
        root = cache.seq_create()
        grow(cache, rng, root, n, range(layers))
        kids = [cache.seq_fork(root, n) for _ in range(rows)]
        cache.seq_free(root)
        for i, s in enumerate(kids):
            if i:
                grow(cache, rng, s, 61 * i, range(layers))
        seqs += kids
    lone = cache.seq_create()
    grow(cache, rng, lone, 100, range(layers))
    return cache, [seqs[3], seqs[0], lone, seqs[1], seqs[4], seqs[2]]


@pytest.mark.parametrize("fmt", FMTS)
def test_batch_steps_eager(fmt):
    rng = np.random.default_rng(71)
    cache, seqs = forked_batch(fmt, rng)
    n = len(seqs)
    batch = yahkv.DecodeBatch(cache, seqs)
    batch.set_shared()
    assert batch.prepare(70) is True               # crosses a page boundary in every row
    for step in range(66):
        k, v, q = normal(rng, 2, n, 4, 256), normal(rng, 2, n, 4, 256), normal(rng, 2, n, 24, 256)
        gate = rng.standard_normal((n, 24, 256)).astype(np.float32)
        batch.plan()
        outs = []
        for layer in range(2):
            out = torch.zeros(n, 24, 256, device="cuda")
            torch.cuda.synchronize()
            batch.decode_layer(layer, dev(k[layer]), dev(v[layer]), dev(q[layer]), out, gate=dev(gate), out_dtype=yahkv.OUT_F32)
            outs.append(out)
        batch.advance()
        batch.commit(1)
        cache.sync()
        if step in (0, 1, 62, 63, 64, 65):
            for layer in range(2):
                check(cache, layer, seqs, q[layer], outs[layer].double().cpu().numpy(), gate)
    batch.set_shared(False)                        # from the next prepare on
    assert batch.prepare(2) is True
    batch.plan()
    out = torch.zeros(n, 24, 256, device="cuda")
    torch.cuda.synchronize()
    for layer in range(2):
        batch.decode_layer(layer, dev(k[layer]), dev(v[layer]), dev(q[layer]), out, out_dtype=yahkv.OUT_F32)
    batch.advance()
    batch.commit(1)
    cache.sync()
    check(cache, 1, seqs, q[1], out.double().cpu().numpy())
    batch.close()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("raw", [False, True])
def test_batch_steps_replayed(fmt, raw):
    rng = np.random.default_rng(73)
    cache, seqs = forked_batch(fmt, rng)
    n, kind = len(seqs), torch.float32 if raw else torch.float16
    batch = yahkv.DecodeBatch(cache, seqs)
    batch.set_shared()
    batch.prepare(40)
    k, v = torch.zeros(2, n, 4, 256, device="cuda", dtype=kind), torch.zeros(2, n, 4, 256, device="cuda", dtype=kind)
    q, out = torch.zeros(2, n, 24, 256, device="cuda", dtype=kind), torch.zeros(2, n, 24, 256, device="cuda")
    ones = torch.ones(256, device="cuda")

    def step(stream=None):
        batch.plan(stream=stream)
        for layer in range(2):
            if raw:
                batch.decode_layer_raw(layer, q[layer], k[layer], v[layer], ones, ones, EPS, out[layer], out_dtype=yahkv.OUT_F32, stream=stream)
            else:
                batch.decode_layer(layer, k[layer], v[layer], q[layer], out[layer], out_dtype=yahkv.OUT_F32, stream=stream)
        batch.advance(stream=stream)

    def fill():
        for t in (k, v, q):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float32)))

    def queries(lens):
        """The fp16 queries the attention works on."""
        x = q.cpu().numpy()
        if not raw:
            return x
        f, m = freqs(64, 1e7, "none", 1, 0, 0, 0, 0)
        return np.stack([rotate64(x[layer], np.array(lens) - 1, "half", 64, f, m, np.ones(256, np.float32))[1] for layer in range(2)]).astype(np.float16)

    torch.cuda.synchronize()
    fill()
    step()                                          # eagerly first: the raw path builds its table
    batch.commit(1)
    cache.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(30):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        batch.commit(1)
        if i in (0, 7, 29):
            lens = [cache.seq_len(s, 0) for s in seqs]
            for layer in range(2):
                got = out[layer].double().cpu().numpy()
                want_q = queries(lens)[layer]
                if raw:
                    # q is rounded to fp16 a step apart at most: its share of a score is 2^-10 sum|q k| / 16, the roundings' of test_shared_gpu twice
                    err = ref = 0.0
                    for b, s in enumerate(seqs):
                        w = attend64(want_q[b], *rows64(cache, layer, s, lens[b]))[0]
                        err, ref = err + ((got[b] - w) ** 2).sum(), ref + (w ** 2).sum()
                    assert math.sqrt(err / ref) <= 4e-3
                else:
                    check(cache, layer, seqs, want_q, got)
    cache.sync()
    batch.close()


def test_two_captured_batches_of_one_cache():
    """Two graphs share the context's workspaces; replayed in turn on one stream they do not disturb each other."""
    rng = np.random.default_rng(79)
    cache, seqs = forked_batch(yahkv.FMT_Q8_0, rng, layers=1)
    parts = [seqs[1:4], [seqs[0], seqs[4], seqs[5]]]
    batches, graphs, bufs = [], [], []
    side = torch.cuda.Stream()
    for ids in parts:
        b = yahkv.DecodeBatch(cache, ids)
        b.set_shared()
        b.prepare(8)
        n = len(ids)
        t = dict(k=torch.zeros(n, 4, 256, device="cuda", dtype=torch.float16), v=torch.zeros(n, 4, 256, device="cuda", dtype=torch.float16),
                 q=torch.zeros(n, 24, 256, device="cuda", dtype=torch.float16), out=torch.zeros(n, 24, 256, device="cuda"))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            sp = torch.cuda.current_stream().cuda_stream
            b.plan(stream=sp)
            b.decode_layer(0, t["k"], t["v"], t["q"], t["out"], out_dtype=yahkv.OUT_F32, stream=sp)
            b.advance(stream=sp)
        batches.append(b), graphs.append(g), bufs.append(t)
    for _ in range(3):
        for t in bufs:
            for x in ("k", "v", "q"):
                t[x].copy_(torch.from_numpy(normal(rng, *t[x].shape)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for b, ids, t in zip(batches, parts, bufs):
            b.commit(1)
            check(cache, 0, ids, t["q"].cpu().numpy(), t["out"].double().cpu().numpy())
    for b in batches:
        b.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_a_prompt_forked_decoded_cut_and_continued(fmt):
    """A prompt rotated for a long context and appended once; three branches decode over it together, one of them with its keys
    watched; that branch is cut, its slots stop being positions, and it goes on at its true positions."""
    rng = np.random.default_rng(83)
    prompt, steps, keep = 450, 6, 150
    cache = small_cache(num_pages=60, fmt=fmt, max_seqs=5, max_pages_per_seq=12)
    rope = yahkv.Rope(cache, layout="interleaved", rotary_dim=128, theta=1e6, scaling="yarn", factor=8.0, original_len=4096.0,
                      max_positions=40000)
    f, m = freqs(128, 1e6, "yarn", 8.0, 4096.0, 32.0, 1.0, 0.0)
    base = 30000                                                        # the prompt sits far inside a context

    def rotate(x, pos):
        out = torch.empty(x.shape, device="cuda", dtype=torch.float16)
        torch.cuda.synchronize()
        rope.rows(dev(x), dev(np.asarray(pos, np.int64)), out)
        cache.sync()
        _, want = rotate64(x, np.asarray(pos), "interleaved", 128, f, m, None)
        # half an fp16 step of the value and fp32 roundings of a row's largest value (below 16)
        assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -24 * 400).all()
        return out

    root = cache.seq_create()
    cache.seq_reserve(root, prompt)
    k, v = rng.standard_normal((prompt, 4, 256)).astype(np.float32), normal(rng, prompt, 4, 256)
    cache.append(0, [root] * prompt, np.arange(prompt), rotate(k, base + np.arange(prompt)), dev(v))
    rows = [cache.seq_fork(root, prompt) for _ in range(3)]
    watched = rows[1]
    acc = torch.zeros(1, 5, 4, 768, device="cuda")
    want_acc = np.zeros((4, prompt + steps))
    out = torch.empty(3, 24, 256, device="cuda")
    for i in range(steps):
        for s in rows:
            cache.seq_reserve(s, prompt + i + 1)
        kk = rotate(rng.standard_normal((3, 4, 256)).astype(np.float32), [base + prompt + i] * 3)
        cache.append(0, rows, [prompt + i] * 3, kk, dev(normal(rng, 3, 4, 256)))
        q = rotate(rng.standard_normal((3, 24, 256)).astype(np.float32), [base + prompt + i] * 3)
        cache.attend_decode_shared(0, rows, q, out, out_dtype=yahkv.OUT_F32)
        cache.sync()
        qh = q.cpu().numpy()
        check(cache, 0, rows, qh, out.double().cpu().numpy())
        cache.attend_decode_weights(0, [watched], q[1:2], out[1:2], acc[0], out_dtype=yahkv.OUT_F32)
        cache.sync()
        n = prompt + i + 1
        ko, vo = rows64(cache, 0, watched, n)
        o, p = attend64(qh[1], ko, vo)
        assert np.abs(out[1].double().cpu().numpy() - o).max() <= 2e-3
        want_acc[:, :n] += p.reshape(4, 6, n).sum(1)
    got_acc = acc[0, watched, :, :prompt + steps].double().cpu().numpy()
    assert np.abs(got_acc - want_acc).max() <= 1e-3 * want_acc.max()
    n = prompt + steps
    ko, vo = rows64(cache, 0, watched, n)
    w = acc[0, watched].cpu().numpy()
    kept = torch.empty(1, 1, 4, keep, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    cache.evict([watched], keep, acc, kept, n_sink=4, n_recent=40)
    cache.sync()
    for h in range(4):
        want = select(w[h], n, keep, 4, 40)
        assert kept[0, 0, h].tolist() == want
        now = rows64(cache, 0, watched, keep)
        assert np.array_equal(now[0][:, h], ko[want, h]) and np.array_equal(now[1][:, h], vo[want, h])
    other = rows64(cache, 0, rows[0], prompt)                           # the branches beside it keep the prompt
    assert np.array_equal(other[0], rows64(cache, 0, root, prompt)[0])
    # the cut branch goes on: slot `keep`, position base + n; the others still share the prompt
    for s in rows:
        cache.seq_reserve(s, cache.seq_len(s, 0) + 1)
    kk = rotate(rng.standard_normal((3, 4, 256)).astype(np.float32), [base + n] * 3)
    cache.append(0, rows, [cache.seq_len(s, 0) for s in rows], kk, dev(normal(rng, 3, 4, 256)))
    assert cache.seq_len(watched, 0) == keep + 1
    q = rotate(rng.standard_normal((3, 24, 256)).astype(np.float32), [base + n] * 3).cpu().numpy()
    check(cache, 0, rows, q, shared(cache, 0, rows, q))


def test_contexts_on_their_own_streams_at_once():
    """Three contexts, a stream each, calls queued in turn without waiting: the bits of the same calls made one at a time."""
    rng = np.random.default_rng(83)
    jobs = []
    for fmt in FMTS:
        cache, seqs = forked_batch(fmt, rng, layers=1)
        n = len(seqs)
        q = [dev(normal(rng, n, 24, 256)) for _ in range(6)]
        x = dev(rng.standard_normal((40, 24, 256)).astype(np.float32))
        jobs.append((cache, seqs, q, x, yahkv.Rope(cache, rotary_dim=128, max_positions=4096), dev(rng.integers(0, 4096, 40))))

    def call(job, i, outs, stream=None):
        cache, seqs, q, x, rope, pos = job
        shared_out, plain_out, w, turned = outs
        cache.attend_decode_shared(0, seqs, q[i], shared_out[i], out_dtype=yahkv.OUT_F32, stream=stream)
        cache.attend_decode_weights(0, seqs, q[i], plain_out[i], w, out_dtype=yahkv.OUT_F32, stream=stream)
        rope.rows(x, pos, turned[i], stream=stream)

    def buffers(job):
        n = len(job[1])
        return (torch.zeros(6, n, 24, 256, device="cuda"), torch.zeros(6, n, 24, 256, device="cuda"),
                torch.zeros(job[0].cfg.max_seqs, 4, 900, device="cuda"), torch.zeros(6, 40, 24, 256, device="cuda"))
    alone = [buffers(j) for j in jobs]
    torch.cuda.synchronize()
    for job, outs in zip(jobs, alone):
        for i in range(6):
            call(job, i, outs)
            job[0].sync()
    together = [buffers(j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for i in range(6):
        for job, outs, st in zip(jobs, together, streams):
            call(job, i, outs, st.cuda_stream)
    torch.cuda.synchronize()
    for job, a, b in zip(jobs, alone, together):
        job[0].sync()
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_evict_and_fork_in_a_loop_reuse_pages():
    """Cut, forked, appended and freed again and again with no page to spare: what a sequence holds stays its own."""
    rng = np.random.default_rng(89)
    cache = small_cache(num_pages=13, fmt=yahkv.FMT_Q8_0, max_seqs=3, max_pages_per_seq=6)
    a = cache.seq_create()
    grow(cache, rng, a, 150)
    w = torch.rand(1, 3, 4, 400, device="cuda")
    for turn in range(12):
        n = cache.seq_len(a)
        b = cache.seq_fork(a, n - turn % 3)
        grow(cache, rng, b, 90)
        w.uniform_()
        w0 = w.double().cpu().numpy()
        before = {s: rows64(cache, 0, s, cache.seq_len(s)) for s in (a, b)}
        kept = torch.empty(1, 2, 4, 100, device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        cache.evict([b, a], 100, w, kept, n_sink=2, n_recent=5)
        cache.sync()
        for r, s in enumerate((b, a)):
            assert cache.seq_len(s) == 100
            now = rows64(cache, 0, s, 100)
            for h in range(4):
                want = select(w0[0, s, h], len(before[s][0]), 100, 2, 5)
                assert kept[0, r, h].tolist() == want
                for side in (0, 1):
                    assert np.array_equal(now[side][:, h], before[s][side][want, h])
        q = normal(rng, 2, 24, 256)
        check(cache, 0, [a, b], q, shared(cache, 0, [a, b], q))
        cache.seq_free(a)
        a = b
        grow(cache, rng, a, 50)
    cache.seq_free(a)
    assert cache.pages_free() == 13


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sharded", [True, False])
def test_forks_of_a_cut_sequence(fmt, sharded):
    """Forks of a sequence that was cut: eager calls of a context of kv heads 1 and 2 (which makes no batches), and a
    batch with a fixed number of units per row."""
    rng = np.random.default_rng(97)
    heads = slice(6, 18) if sharded else slice(0, 24)
    cache = small_cache(num_pages=40, fmt=fmt, max_seqs=4, max_pages_per_seq=12, **(dict(kv_head_begin=1, kv_head_count=2) if sharded else {}))
    root = cache.seq_create()
    grow(cache, rng, root, 500)
    kept = torch.full((1, 1, 4, 330), -7, device="cuda", dtype=torch.int32)
    w = torch.rand(1, 4, 4, 500, device="cuda")
    torch.cuda.synchronize()
    cache.evict([root], 330, w, kept)
    cache.sync()
    assert (kept[0, 0, [1, 2]] >= 0).all() and (kept[0, 0, [0, 3]] == -7).all().item() == sharded   # other heads are left alone
    seqs = [cache.seq_fork(root, 330) for _ in range(3)]
    batch = None
    if not sharded:
        batch = yahkv.DecodeBatch(cache, seqs)
        batch.set_splits(3)
        batch.set_shared()
        batch.prepare(4)
    for _ in range(3):
        k, v, q = normal(rng, 3, 4, 256), normal(rng, 3, 4, 256), normal(rng, 3, 24, 256)
        out = torch.full((3, 24, 256), float("nan"), device="cuda")
        if sharded:
            for i, s in enumerate(seqs):
                extend(cache, 0, s, k[i:i + 1], v[i:i + 1])
            got = shared(cache, 0, seqs, q, n_splits=3)
            assert np.isnan(got[:, :6]).all() and np.isnan(got[:, 18:]).all()
        else:
            batch.plan()
            torch.cuda.synchronize()
            batch.decode_layer(0, dev(k), dev(v), dev(q), out, out_dtype=yahkv.OUT_F32)
            batch.advance()
            batch.commit(1)
            cache.sync()
            got = out.double().cpu().numpy()
        check(cache, 0, seqs, q, got, heads=heads)
    if batch is not None:
        with pytest.raises(yahkv.YahkvError) as e:      # positions are not slots
            x = [torch.zeros(3, h, 256, device="cuda") for h in (24, 4, 4)]
            one = torch.ones(256, device="cuda")
            batch.decode_layer_raw(0, *x, one, one, EPS, torch.zeros(3, 24, 256, device="cuda"))
        assert e.value.code == yahkv.ERR_ORDER
        batch.close()
