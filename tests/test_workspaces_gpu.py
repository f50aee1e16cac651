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


def test_a_context_on_a_full_device_does_without_them():
    rng = np.random.default_rng(95)
    kw = dict(num_pages=64, fmt=yahkv.FMT_Q8_0, max_seqs=24, max_pages_per_seq=60)
    torch.cuda.empty_cache()
    torch.cuda.synchronize()
    free0 = torch.cuda.mem_get_info()[0]
    cache = yahkv.KvCache(**kw)
    whole = free0 - torch.cuda.mem_get_info()[0]               # 38 MB of it shared prefixes, 8.8 the scores
    cache.close()
    filler = torch.empty(torch.cuda.mem_get_info()[0] - whole + (24 << 20), dtype=torch.uint8, device="cuda")
    try:
        cache = yahkv.KvCache(**kw)                            # without them it fits
        seq = cache.seq_create()
        k, v = normal(rng, 200, 4, 256), normal(rng, 200, 4, 256)
        cache.seq_reserve(seq, 200)
        tensors = [torch.from_numpy(x).pin_memory() for x in (k, v, normal(rng, 1, 24, 256))]
        out = torch.zeros(1, 24, 256).pin_memory()             # page-locked: the device has no room for tensors either
        cache.append(0, [seq] * 200, np.arange(200), tensors[0], tensors[1])
        cache.attend_decode(0, [seq], tensors[2], out, out_dtype=yahkv.OUT_F32)
        cache.sync()
        want = out.clone()
        assert torch.isfinite(want).all() and want.abs().max() > 0
        with pytest.raises(yahkv.YahkvError) as e:
            cache.attend_decode_shared(0, [seq], tensors[2], out, out_dtype=yahkv.OUT_F32)
        assert e.value.code == yahkv.ERR_CUDA and "memory" in e.value.message
    finally:
        del filler
        torch.cuda.empty_cache()
    out.zero_()
    cache.attend_decode_shared(0, [seq], tensors[2], out, out_dtype=yahkv.OUT_F32)
    cache.sync()
    # the same scores and products, cut into units and joined in another order: a few roundings of f32 apart
    assert (out - want).abs().max() <= 1e-5 * want.abs().max()
