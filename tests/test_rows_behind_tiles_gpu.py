"""The tile formats: a sequence in the pages and the open tile of one whose values overflowed fp16 attends as in a cache of
its own."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from test_shared_gpu import extend, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [yahkv.FMT_KV8A16, yahkv.FMT_KV4A16])
@pytest.mark.parametrize("reset", [False, True])
@pytest.mark.parametrize("n", [1, 5, 16, 17, 70])
def test_open_tiles_and_pages_used_again(fmt, reset, n):
    def call(bad):
        rng = np.random.default_rng(61)
        cache = yahkv.KvCache(num_pages=2, fmt=fmt, max_seqs=1, max_pages_per_seq=2)
        seq = cache.seq_create()
        extend(cache, 0, seq, normal(rng, 127, 4, 256), np.full((127, 4, 256), np.inf if bad else 0.0, np.float16))
        if reset:
            cache.seq_set_len(seq, 0)
        else:
            cache.seq_free(seq)
            seq = cache.seq_create()
        extend(cache, 0, seq, normal(rng, n, 4, 256), normal(rng, n, 4, 256))
        q = dev(normal(rng, n, 24, 256))
        out, pre = torch.zeros(1, 24, 256, device="cuda"), torch.zeros(n, 24, 256, device="cuda")
        torch.cuda.synchronize()
        cache.attend_decode(0, [seq], q[-1:], out, out_dtype=yahkv.OUT_F32)
        cache.attend_prefill(0, [seq], [n], q, pre, out_dtype=yahkv.OUT_F32)
        cache.sync()
        return out, pre
    got, want = call(True), call(False)
    for g, w in zip(got, want):
        assert torch.isfinite(w).all()
        assert torch.equal(g, w)
