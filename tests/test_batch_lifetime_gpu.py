"""What a decode batch holds is its sequences, not their ids, and it may outlive its cache."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from test_shared_gpu import grow, normal

pytestmark = pytest.mark.gpu


def code(call, *a, **k):
    with pytest.raises(yahkv.YahkvError) as e:
        call(*a, **k)
    return e.value.code


def made(n, **kw):
    cache = yahkv.KvCache(num_pages=16, max_seqs=3, max_pages_per_seq=6, **kw)
    rng = np.random.default_rng(83)
    seqs = []
    for _ in range(n):
        s = cache.seq_create()
        grow(cache, rng, s, 100)
        seqs.append(s)
    return cache, seqs, rng


def cut(cache, seq):
    w = torch.zeros(1, 3, 4, 384, device="cuda")
    kept = torch.zeros(1, 1, 4, 50, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    cache.evict([seq], 50, w, kept)
    cache.sync()
    assert cache.seq_len(seq, 0) == 50 and kept[0, 0, 0].tolist() == list(range(50))


def test_a_sequence_that_takes_the_id_of_a_freed_one_can_be_cut():
    cache, (a, b), rng = made(2)
    batch = yahkv.DecodeBatch(cache, [a, b])
    cache.seq_free(a)
    c = cache.seq_create()
    assert c == a
    grow(cache, rng, c, 100)
    cut(cache, c)                                            # the batch holds the freed one
    w = torch.zeros(1, 3, 4, 384, device="cuda")
    kept = torch.zeros(1, 1, 4, 50, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    assert code(cache.evict, [b], 50, w, kept) == yahkv.ERR_ORDER
    batch.close()
    cut(cache, b)


def test_a_batch_does_not_take_a_new_sequence_for_a_freed_one():
    cache, (a, b), rng = made(2)
    batch = yahkv.DecodeBatch(cache, [a, b])
    batch.prepare(4)
    cache.seq_free(a)
    c = cache.seq_create()
    assert c == a
    grow(cache, rng, c, 100)                                 # of the same length, even
    assert code(batch.commit, 1) == yahkv.ERR_ORDER
    assert cache.seq_len(c, 0) == 100 and cache.seq_len(b, 0) == 100
    assert code(batch.prepare, 4) == yahkv.ERR_ORDER
    batch.close()
    batch = yahkv.DecodeBatch(cache, [c, b])
    batch.prepare(1)
    batch.plan()
    out = torch.zeros(2, 24, 256, device="cuda")
    torch.cuda.synchronize()
    batch.decode_layer(0, dev(normal(rng, 2, 4, 256)), dev(normal(rng, 2, 4, 256)), dev(normal(rng, 2, 24, 256)), out, out_dtype=yahkv.OUT_F32)
    batch.advance()
    batch.commit(1)
    cache.sync()
    assert cache.seq_len(c, 0) == 101 and torch.isfinite(out).all()
    batch.close()


def test_a_batch_outlives_its_cache():
    cache, seqs, _ = made(2)
    batch = yahkv.DecodeBatch(cache, seqs)
    batch.set_shared()
    batch.prepare(2)
    cache.close()
    for call in (lambda: batch.prepare(1), batch.plan, batch.advance, lambda: batch.commit(1), lambda: batch.set_splits(1),
                 batch.set_shared):
        assert code(call) == yahkv.ERR_INVALID
    batch.close()
    cache, seqs, _ = made(2)                                 # the device is as it was
    cut(cache, seqs[0])
