"""Rows of one call in groups at several levels of the tree of forks: a long conversation and the rows beside it, which share the
prompt among themselves; in single calls and in a decode batch."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from test_shared_gpu import FMTS, check, grow, normal, shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
def test_a_conversation_and_the_rows_beside_it(fmt):
    rng = np.random.default_rng(97)
    cache = yahkv.KvCache(num_pages=160, fmt=fmt, max_seqs=16, max_pages_per_seq=80)
    prompt = cache.seq_create()
    grow(cache, rng, prompt, 20 * 64)
    seqs = [cache.seq_fork(prompt, 20 * 64) for _ in range(8)]
    talk = cache.seq_fork(prompt, 20 * 64)
    grow(cache, rng, talk, 52 * 64 + 9)
    seqs += [cache.seq_fork(talk, 72 * 64 + 9) for _ in range(3)]
    for i, s in enumerate(seqs):
        grow(cache, rng, s, 1 + 29 * i)
    seqs = [seqs[i] for i in rng.permutation(len(seqs))]
    n = len(seqs)
    q = normal(rng, n, 24, 256)
    check(cache, 0, seqs, q, shared(cache, 0, seqs, q))
    batch = yahkv.DecodeBatch(cache, seqs)
    batch.set_shared()
    batch.prepare(3)
    for _ in range(3):
        k, v, q, out = dev(normal(rng, n, 4, 256)), dev(normal(rng, n, 4, 256)), normal(rng, n, 24, 256), torch.zeros(n, 24, 256, device="cuda")
        qd = dev(q)
        batch.plan()
        batch.decode_layer(0, k, v, qd, out, out_dtype=yahkv.OUT_F32)
        batch.advance()
        batch.commit(1)
        cache.sync()
        check(cache, 0, seqs, q, out.double().cpu().numpy())
    batch.close()
