"""Whatever the rows behind a sequence's last key hold (inf or no number left there by a page's former owner, by a cut or by
the source of a fork), decode attention gives the bits that it gives with zeros there."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from test_shared_gpu import FMTS, extend, normal, small_cache

pytestmark = pytest.mark.gpu
LENS = [1, 63, 64, 65, 70, 130, 200]
BAD = np.array([0x7C00, 0x7E00, 0xFC00, 0xFE00], np.uint16)     # inf, NaN, -inf, -NaN


def spoil(cache, layer, seq, n, bad=True):
    """Rows n .. of the sequence's pages become inf and NaN (bad) or zero, in K and V."""
    table = cache.seq_table(seq)
    for p in range(n // 64, len(table)):
        first = max(n - 64 * p, 0)
        for side in (yahkv.SIDE_K, yahkv.SIDE_V):
            codes, scales = cache.read_page(layer, side, int(table[p]))
            rows = codes.view(np.uint16) if cache.fmt == yahkv.FMT_F16 else scales
            rows[:, first:] = np.resize(BAD, rows[:, first:].shape) if bad else 0
            cache.write_page(layer, side, int(table[p]), codes, scales)


def filled(fmt, bad):
    rng = np.random.default_rng(41)
    cache = small_cache(num_pages=40, fmt=fmt, max_seqs=16, max_pages_per_seq=6)
    seqs = []
    for n in LENS:
        s = cache.seq_create()
        extend(cache, 0, s, normal(rng, n, 4, 256), normal(rng, n, 4, 256))
        cache.seq_reserve(s, n + 64)
        spoil(cache, 0, s, n, bad)
        seqs.append(s)
    return cache, seqs, rng


def both(call):
    """The results of call(bad) with the rows spoilt and with zeros there: equal to the bit, and numbers."""
    got, want = call(True), call(False)
    for g, w in zip(got, want):
        assert torch.isfinite(w).all()
        assert torch.equal(g, w), (g - w).abs().max()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n_splits", [0, 2])
def test_decode(fmt, n_splits):
    def call(bad):
        cache, seqs, rng = filled(fmt, bad)
        q, out = dev(normal(rng, len(seqs), 24, 256)), torch.zeros(len(seqs), 24, 256, device="cuda")
        raw = torch.zeros_like(out)
        ones = torch.ones(256, device="cuda")
        torch.cuda.synchronize()
        cache.attend_decode(0, seqs, q, out, out_dtype=yahkv.OUT_F32, n_splits=n_splits)
        cache.attend_decode_qraw(0, seqs, q.float(), ones, 1e-6, raw, out_dtype=yahkv.OUT_F32, n_splits=n_splits)
        cache.sync()
        return out, raw
    both(call)


@pytest.mark.parametrize("fmt", FMTS)
def test_weights(fmt):
    def call(bad):
        cache, seqs, rng = filled(fmt, bad)
        q, out = dev(normal(rng, len(seqs), 24, 256)), torch.zeros(len(seqs), 24, 256, device="cuda")
        w = torch.zeros(16, 4, 256, device="cuda")
        torch.cuda.synchronize()
        cache.attend_decode_weights(0, seqs, q, out, w, out_dtype=yahkv.OUT_F32)
        cache.sync()
        return out, w
    both(call)


@pytest.mark.parametrize("fmt", FMTS)
def test_shared_prefix(fmt):
    def call(bad):
        rng = np.random.default_rng(43)
        cache = small_cache(num_pages=40, fmt=fmt, max_seqs=16, max_pages_per_seq=6)
        root = cache.seq_create()
        extend(cache, 0, root, normal(rng, 200, 4, 256), normal(rng, 200, 4, 256))
        seqs = [cache.seq_fork(root, n) for n in (200, 192, 150, 200)]
        for s, n in zip(seqs, (3, 1, 60, 100)):
            extend(cache, 0, s, normal(rng, n, 4, 256), normal(rng, n, 4, 256))
            spoil(cache, 0, s, cache.seq_len(s, 0), bad)
        q, out = dev(normal(rng, len(seqs), 24, 256)), torch.zeros(len(seqs), 24, 256, device="cuda")
        torch.cuda.synchronize()
        cache.attend_decode_shared(0, seqs, q, out, out_dtype=yahkv.OUT_F32)
        cache.sync()
        return (out,)
    both(call)


@pytest.mark.parametrize("fmt", FMTS)
def test_batch_steps(fmt):
    def call(bad):
        cache, seqs, rng = filled(fmt, bad)
        batch = yahkv.DecodeBatch(cache, seqs)
        batch.prepare(3)
        outs = []
        for _ in range(3):
            k, v, q = dev(normal(rng, len(seqs), 4, 256)), dev(normal(rng, len(seqs), 4, 256)), dev(normal(rng, len(seqs), 24, 256))
            out = torch.zeros(len(seqs), 24, 256, device="cuda")
            torch.cuda.synchronize()
            batch.plan()
            batch.decode_layer(0, k, v, q, out, out_dtype=yahkv.OUT_F32)
            batch.advance()
            batch.commit(1)
            cache.sync()
            outs.append(out)
        batch.close()
        return outs
    both(call)


def attend(cache, seq, q):
    out = torch.zeros(1, 24, 256, device="cuda")
    torch.cuda.synchronize()
    cache.attend_decode(0, [seq], q, out, out_dtype=yahkv.OUT_F32)
    cache.sync()
    return out


@pytest.mark.parametrize("fmt", FMTS)
def test_fork_below_a_row_that_overflowed(fmt):
    def call(bad):
        rng = np.random.default_rng(47)
        cache = yahkv.KvCache(num_pages=8, fmt=fmt, max_seqs=2, max_pages_per_seq=4)
        root = cache.seq_create()
        k, v = normal(rng, 130, 4, 256), normal(rng, 130, 4, 256)
        if bad:
            v[100] = np.inf
        extend(cache, 0, root, k, v)
        fork = cache.seq_fork(root, 70)              # its second page is a copy of 64 tokens, the 36th of it that row
        extend(cache, 0, fork, normal(rng, 3, 4, 256), normal(rng, 3, 4, 256))
        return (attend(cache, fork, dev(normal(rng, 1, 24, 256))),)
    both(call)


@pytest.mark.parametrize("fmt", FMTS)
def test_cut_of_rows_that_overflowed(fmt):
    def call(bad):
        rng = np.random.default_rng(53)
        cache = yahkv.KvCache(num_pages=8, fmt=fmt, max_seqs=1, max_pages_per_seq=4)
        seq = cache.seq_create()
        k, v = normal(rng, 200, 4, 256), normal(rng, 200, 4, 256)
        if bad:
            v[100:] = np.inf
        extend(cache, 0, seq, k, v)
        w = torch.zeros(1, 1, 4, 256, device="cuda")
        w[..., :100] = 1.0
        kept = torch.zeros(1, 1, 4, 100, device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        cache.evict([seq], 100, w, kept)             # slots 100 .. 127 keep what they held
        return (attend(cache, seq, dev(normal(rng, 1, 24, 256))),)
    both(call)


@pytest.mark.parametrize("fmt", FMTS)
def test_pages_of_a_freed_sequence(fmt):
    def call(bad):
        rng = np.random.default_rng(59)
        cache = yahkv.KvCache(num_pages=2, fmt=fmt, max_seqs=1, max_pages_per_seq=2)
        seq = cache.seq_create()
        extend(cache, 0, seq, normal(rng, 128, 4, 256), np.full((128, 4, 256), np.inf if bad else 0.0, np.float16))
        cache.seq_free(seq)
        seq = cache.seq_create()
        extend(cache, 0, seq, normal(rng, 70, 4, 256), normal(rng, 70, 4, 256))
        return (attend(cache, seq, dev(normal(rng, 1, 24, 256))),)
    both(call)
