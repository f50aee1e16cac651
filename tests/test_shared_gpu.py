"""Forked sequences and decode attention over shared prefixes on the GPU, against float64 attention over the bytes the cache
holds.

Tolerance. Against exact softmax attention over the cached values the prefix pass rounds the softmax weights and, for
quantized pages, K and V to fp16: half a step is 2^-11 of a value. A weight's rounding and V's move an output by at
most 2^-11 max|v| each; K's moves a score by at most 2^-11 sum|q k| / 16, which for N(0, 1) data is below 6e-3 for a
single key and averages out over keys; an fp16 output adds 2^-11 |out|. The bar is the library's bar for the prefill
kernel, which has the same roundings (2e-3), plus the worst case of the two that do not average out, 2 x 2^-11 max|v|,
where few keys carry the output. In the 2-norm four independent roundings of at most 2^-11 each stay below
4 x 2^-11 = 2e-3."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from longctx_util import attend64, rows64

pytestmark = pytest.mark.gpu
FMTS = [yahkv.FMT_F16, yahkv.FMT_Q8_0, yahkv.FMT_Q4_0]


def normal(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32).astype(np.float16)


def small_cache(**kw):
    """A cache that computes every shared prefix once, however little it saves, so that small tests reach that path."""
    cache = yahkv.KvCache(**kw)
    cache.debug_set_shared_min(1)
    return cache


def extend(cache, layer, seq, k, v):
    n0 = cache.seq_len(seq, layer)
    cache.seq_reserve(seq, n0 + len(k))
    for a in range(0, len(k), 4096):
        e = min(len(k), a + 4096)
        cache.append(layer, [seq] * (e - a), np.arange(n0 + a, n0 + e), dev(k[a:e]), dev(v[a:e]))


def grow(cache, rng, seq, n, layers=(0,)):
    for layer in layers:
        extend(cache, layer, seq, normal(rng, n, 4, 256), normal(rng, n, 4, 256))


def shared(cache, layer, seqs, q, gate=None, out_dtype=yahkv.OUT_F32, n_splits=0, stream=None):
    out = torch.full((len(seqs), 24, 256), float("nan"), device="cuda",
                     dtype=torch.float32 if out_dtype == yahkv.OUT_F32 else torch.float16)
    qd, gd = dev(q), None if gate is None else dev(gate)
    cache.attend_decode_shared(layer, seqs, qd, out, gate=gd, out_dtype=out_dtype, n_splits=n_splits, stream=stream)
    cache.sync()
    return out.double().cpu().numpy()


def check(cache, layer, seqs, q, got, gate=None, heads=slice(0, 24)):
    err2 = ref2 = 0.0
    for b, s in enumerate(seqs):
        k, v = rows64(cache, layer, s, cache.seq_len(s, layer))
        want = attend64(q[b], k, v, None if gate is None else gate[b])[0][heads]
        tol = 2e-3 + 2.0 ** -10 * np.abs(v).max() + 2.0 ** -11 * np.abs(want).max()
        err = np.abs(got[b][heads] - want)
        assert err.max() <= tol, (b, err.max(), tol, np.unravel_index(err.argmax(), err.shape))
        err2, ref2 = err2 + (err ** 2).sum(), ref2 + (want ** 2).sum()
    assert np.sqrt(err2 / ref2) <= 2e-3, np.sqrt(err2 / ref2)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,prefix,suffix", [(2, 64, 1), (2, 128, 3), (3, 65, 40), (5, 640, 0), (21, 200, 70), (22, 333, 17),
                                                (43, 129, 100), (64, 1000, 5), (4, 5000, 200)])
def test_one_group(fmt, rows, prefix, suffix):
    rng = np.random.default_rng(rows * 1000 + prefix)
    cache = small_cache(num_pages=(prefix + 63) // 64 + rows * ((suffix + 127) // 64 + 1), fmt=fmt, max_seqs=rows + 1,
                          max_pages_per_seq=(prefix + suffix + 127) // 64)
    root = cache.seq_create()
    grow(cache, rng, root, prefix)
    seqs = [cache.seq_fork(root, prefix) for _ in range(rows)]
    for i, s in enumerate(seqs):
        grow(cache, rng, s, min(suffix, 1 + i * 13 % max(suffix, 1)))     # every suffix another length, at least one of them whole
    q = normal(rng, rows, 24, 256)
    check(cache, 0, seqs, q, shared(cache, 0, seqs, q))


@pytest.mark.parametrize("fmt", FMTS)
def test_groups_single_rows_and_repeats_in_any_order(fmt):
    rng = np.random.default_rng(7)
    cache = small_cache(n_layers=2, num_pages=150, fmt=fmt, max_seqs=24, max_pages_per_seq=40)
    seqs = []
    for prefix, rows in ((300, 5), (64, 2), (1500, 3)):
        root = cache.seq_create()
        grow(cache, rng, root, prefix, (0, 1))
        kids = [cache.seq_fork(root, prefix) for _ in range(rows)]
        for i, s in enumerate(kids):
            grow(cache, rng, s, 1 + 50 * i, (0, 1))
        seqs += kids + [root]                      # the root itself is a row of its group
    lone = cache.seq_create()
    grow(cache, rng, lone, 500, (0, 1))
    short = cache.seq_create()
    grow(cache, rng, short, 1, (0, 1))
    seqs += [lone, short, seqs[0]]                 # one sequence asked twice, with two queries
    order = rng.permutation(len(seqs))
    seqs = [seqs[i] for i in order]
    for layer in (0, 1):
        for n_splits in (0, 1, 5):
            q = normal(rng, len(seqs), 24, 256)
            gate = rng.standard_normal((len(seqs), 24, 256)).astype(np.float32)
            check(cache, layer, seqs, q, shared(cache, layer, seqs, q, gate, n_splits=n_splits), gate)
    q = normal(rng, len(seqs), 24, 256)
    check(cache, 0, seqs, q, shared(cache, 0, seqs, q, out_dtype=yahkv.OUT_F16))
    got = shared(cache, 0, [lone], q[:1])          # nobody shares anything
    check(cache, 0, [lone], q[:1], got)


@pytest.mark.parametrize("fmt", FMTS)
def test_steps_interleaved_with_plain_decode(fmt):
    """The two calls keep plans of their own; tables and lengths change between the steps."""
    rng = np.random.default_rng(11)
    cache = small_cache(num_pages=60, fmt=fmt, max_seqs=5, max_pages_per_seq=20)
    root = cache.seq_create()
    grow(cache, rng, root, 250)
    seqs = [cache.seq_fork(root, 250) for _ in range(4)]
    side = torch.cuda.Stream()
    for step in range(8):
        for s in seqs:
            grow(cache, rng, s, 1)
        q = normal(rng, 4, 24, 256)
        st = side.cuda_stream if step % 2 else None
        torch.cuda.synchronize()
        got = shared(cache, 0, seqs, q, stream=st)
        plain = torch.empty(4, 24, 256, device="cuda")
        cache.attend_decode(0, seqs, dev(q), plain, out_dtype=yahkv.OUT_F32, stream=st)
        cache.sync()
        check(cache, 0, seqs, q, got)
        check(cache, 0, seqs, q, plain.double().cpu().numpy())
        if step == 4:                              # a member leaves, another one joins
            cache.seq_free(seqs[1])
            seqs[1] = cache.seq_fork(root, 192)


@pytest.mark.parametrize("fmt", FMTS)
def test_a_fork_and_its_origin_grow_apart(fmt):
    rng = np.random.default_rng(5)
    cache = small_cache(n_layers=3, num_pages=12, fmt=fmt, max_seqs=3, max_pages_per_seq=6)
    a = cache.seq_create()
    grow(cache, rng, a, 100, (0, 1, 2))
    before = [rows64(cache, l, a, 100) for l in range(3)]
    b = cache.seq_fork(a, 90)                       # ends inside the second page: copied
    assert cache.seq_table(b)[0] == cache.seq_table(a)[0] and cache.seq_table(b)[1] != cache.seq_table(a)[1]
    grow(cache, rng, b, 40, (0, 1, 2))
    grow(cache, rng, a, 40, (0, 1, 2))
    for l in range(3):
        for side in (0, 1):
            assert np.array_equal(rows64(cache, l, a, 100)[side], before[l][side])
            assert np.array_equal(rows64(cache, l, b, 90)[side], before[l][side][:90])
    cache.seq_free(a)
    q = normal(rng, 1, 24, 256)
    check(cache, 1, [b], q, shared(cache, 1, [b], q))


def test_long_groups_short_rows_and_forks_of_forks_at_the_default_threshold():
    """Groups that save too little, a short row among long ones, two conversations behind one prompt."""
    rng = np.random.default_rng(17)
    cache = yahkv.KvCache(num_pages=160, fmt=yahkv.FMT_Q8_0, max_seqs=24, max_pages_per_seq=40)
    root = cache.seq_create()
    grow(cache, rng, root, 1100)
    seqs = [cache.seq_fork(root, 1100) for _ in range(6)] + [cache.seq_fork(root, 100)]       # 17 pages x 5, one row of 1
    for _ in range(2):
        conv = cache.seq_fork(root, 640)
        grow(cache, rng, conv, 900)
        seqs += [cache.seq_fork(conv, 1540) for _ in range(4)]                                  # 24 pages x 3 behind 10
    lone = cache.seq_create()
    grow(cache, rng, lone, 64)
    seqs += [lone, cache.seq_fork(lone, 64)]                                                    # saves one page
    for i, s in enumerate(seqs):
        grow(cache, rng, s, 1 + 7 * i)
    seqs = [seqs[i] for i in rng.permutation(len(seqs))]
    q = normal(rng, len(seqs), 24, 256)
    before = cache.launch_count()
    got = shared(cache, 0, seqs, q)
    assert cache.launch_count() - before >= 3      # a prefix pass ran
    check(cache, 0, seqs, q, got)
    few = [seqs.index(s) for s in seqs[:2]]
    check(cache, 0, [seqs[i] for i in few], q[few], shared(cache, 0, [seqs[i] for i in few], q[few]))


@pytest.mark.parametrize("fmt", FMTS)
def test_values_at_the_end_of_fp16(fmt):
    """Blocks whose largest value is fp16's largest: q8_0 stores it as 127 x 516 = 65532, which as fp16 would be infinite; the
    pass takes 65504, off by less than half a step (28 of 65532 < 2^-11). A block whose scale is infinite stays that."""
    rng = np.random.default_rng(23)
    cache = small_cache(num_pages=8, fmt=fmt, max_seqs=3, max_pages_per_seq=3)
    root = cache.seq_create()
    k, v = normal(rng, 128, 4, 256), (normal(rng, 128, 4, 256) * np.float16(1000)).astype(np.float16)
    v[..., ::32] = 65504
    v[::2, :, 3::32] = -65504
    extend(cache, 0, root, k, v)
    seqs = [cache.seq_fork(root, 128) for _ in range(2)]
    q = normal(rng, 2, 24, 256)
    check(cache, 0, seqs, q, shared(cache, 0, seqs, q))
    if fmt != yahkv.FMT_F16:
        page = int(cache.seq_table(root)[0])
        codes, scales = cache.read_page(0, yahkv.SIDE_V, page)
        scales = scales.copy()
        scales.view(np.float16)[0, 5, 1] = np.inf           # kv head 0, token 5, dims 32 .. 63
        cache.write_page(0, yahkv.SIDE_V, page, codes, scales)
        got = shared(cache, 0, seqs, q)
        assert not np.isfinite(got[:, :6, 32:64]).any()
        assert np.isfinite(got[:, 6:]).all() and np.isfinite(got[:, :6, :32]).all() and np.isfinite(got[:, :6, 64:]).all()


def test_a_head_sharded_context_writes_its_own_heads_only():
    rng = np.random.default_rng(3)
    for fmt in (yahkv.FMT_F16, yahkv.FMT_Q8_0):
        cache = small_cache(num_pages=30, fmt=fmt, max_seqs=4, max_pages_per_seq=10, kv_head_begin=1, kv_head_count=2)
        root = cache.seq_create()
        grow(cache, rng, root, 320)
        seqs = [cache.seq_fork(root, 320) for _ in range(3)]
        for s in seqs:
            grow(cache, rng, s, 9)
        q = normal(rng, 3, 24, 256)
        got = shared(cache, 0, seqs, q)
        check(cache, 0, seqs, q, got, heads=slice(6, 18))
        assert np.isnan(got[:, :6]).all() and np.isnan(got[:, 18:]).all()


def test_refusals():
    rng = np.random.default_rng(1)
    cache = small_cache(num_pages=8, max_seqs=3, max_pages_per_seq=4)
    a = cache.seq_create()
    grow(cache, rng, a, 128)
    b = cache.seq_fork(a, 128)
    q, out = dev(normal(rng, 4, 24, 256)), torch.zeros(4, 24, 256, device="cuda")

    def code(f, *args, **kw):
        with pytest.raises(yahkv.YahkvError) as e:
            f(*args, **kw)
        return e.value.code
    call = cache.attend_decode_shared
    assert code(call, 1, [a, b], q, out) == yahkv.ERR_INVALID
    assert code(call, 0, [a, 2], q, out) == yahkv.ERR_INVALID
    assert code(call, 0, [a, b], None, out) == yahkv.ERR_INVALID
    assert code(call, 0, [a, b], q, None) == yahkv.ERR_INVALID
    assert code(call, 0, [a, b], q.flatten()[1:], out) == yahkv.ERR_INVALID
    assert code(call, 0, [a, b], q, out, out_dtype=2) == yahkv.ERR_INVALID
    assert code(call, 0, [a, b], q, out, n_splits=-1) == yahkv.ERR_INVALID
    assert code(call, 0, [a, b], q, out, n_splits=65) == yahkv.ERR_CAPACITY
    assert code(call, 0, [a, b, a, b], q, out) == yahkv.ERR_CAPACITY
    empty = cache.seq_create()
    assert code(call, 0, [a, empty], q, out) == yahkv.ERR_ORDER
    call(0, [], q, out)
    # a sequence rolled back below its fork may not write into the shared page
    cache.seq_set_len(b, 100)
    x = dev(normal(rng, 1, 4, 256))
    assert code(cache.append, 0, [b], [100], x, x) == yahkv.ERR_INVALID
    batch = yahkv.DecodeBatch(cache, [b])
    assert code(batch.prepare, 4) == yahkv.ERR_INVALID
    batch.close()
    cache.seq_free(a)
    cache.append(0, [b], [100], x, x)               # its own page now
    cache.sync()
    assert code(cache.debug_set_shared_min, 0) == yahkv.ERR_INVALID
    tile = small_cache(num_pages=2, fmt=yahkv.FMT_KV8A16, max_seqs=1, max_pages_per_seq=2)
    s = tile.seq_create()
    assert code(tile.attend_decode_shared, 0, [s], q, out) == yahkv.ERR_INVALID
