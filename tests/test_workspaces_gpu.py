"""What the calls work in exists before the first of them: a context holds as much device memory after them as at its creation."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from test_shared_gpu import FMTS, grow, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("max_seqs,max_pages", [(1, 1), (3, 40), (40, 30)])
def test_first_calls_allocate_nothing(fmt, max_seqs, max_pages):
    rng = np.random.default_rng(91)
    cache = yahkv.KvCache(num_pages=max_seqs * max_pages, fmt=fmt, max_seqs=max_seqs, max_pages_per_seq=max_pages)
    held = cache.device_bytes()
    n = min(max_pages * 64 - 1, 1000)
    root = cache.seq_create()
    grow(cache, rng, root, n)
    seqs = [root] + [cache.seq_fork(root, n) for _ in range(max_seqs - 1)]
    q, out = dev(normal(rng, len(seqs), 24, 256)), torch.zeros(len(seqs), 24, 256, device="cuda", dtype=torch.float16)
    w = torch.zeros(1, max_seqs, 4, max_pages * 64, device="cuda")
    kept = torch.zeros(1, len(seqs), 4, n // 2, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    cache.attend_decode_shared(0, seqs, q, out)
    cache.attend_decode_weights(0, seqs, q, out, w[0])
    cache.evict(seqs, n // 2, w, kept)
    cache.attend_decode_shared(0, seqs, q, out)
    cache.sync()
    assert cache.device_bytes() == held and torch.isfinite(out).all()


def test_scores_of_forks_beyond_the_workspace():
    # 180 forks of 10,000 tokens: 1.8 million keys in one call, where the workspace holds 1.4 million
    rng = np.random.default_rng(93)
    rows, n = 180, 10000
    cache = yahkv.KvCache(num_pages=157 + rows, fmt=yahkv.FMT_Q4_0, max_seqs=rows + 1, max_pages_per_seq=157)
    held = cache.device_bytes()
    root = cache.seq_create()
    grow(cache, rng, root, n)
    seqs = [cache.seq_fork(root, n) for _ in range(rows)]
    row = normal(rng, 1, 24, 256)
    q = dev(np.repeat(row, rows, 0))
    out, few = torch.zeros(rows, 24, 256, device="cuda"), torch.zeros(2, 24, 256, device="cuda")
    w, wf = torch.zeros(rows + 1, 4, n, device="cuda"), torch.zeros(rows + 1, 4, n, device="cuda")
    torch.cuda.synchronize()
    cache.attend_decode_weights(0, seqs[:2], q[:2], few, wf, out_dtype=yahkv.OUT_F32, n_splits=8)
    assert cache.device_bytes() == held
    for _ in range(2):
        cache.attend_decode_weights(0, seqs, q, out, w, out_dtype=yahkv.OUT_F32, n_splits=8)
    cache.sync()
    assert cache.device_bytes() > held
    # the same cut for every row: the same bits in every row, and the weights of two calls are twice those of one
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(out[:2], few)
    assert torch.equal(w[seqs[5]], 2 * wf[seqs[0]]) and torch.equal(w[seqs[-1]], w[seqs[0]])
