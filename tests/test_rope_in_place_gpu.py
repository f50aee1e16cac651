"""A rotation in place needs equal types and strides: the call refuses what would overwrite rows before they are read."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev

pytestmark = pytest.mark.gpu


def test_in_place():
    cache = yahkv.KvCache(num_pages=1, max_seqs=1, max_pages_per_seq=1)
    rope = yahkv.Rope(cache, rotary_dim=128, max_positions=4096)
    rng = np.random.default_rng(3)
    x = dev(rng.standard_normal((40, 6, 256)).astype(np.float32))
    pos = dev(np.arange(100, 140))
    want = torch.empty_like(x)
    torch.cuda.synchronize()
    rope.rows(x, pos, want)
    wide = x.clone()
    half = x.half()
    torch.cuda.synchronize()
    for bad_x, bad_out in ((wide, wide.view(torch.float16).flatten()[:40 * 6 * 256].view(40, 6, 256)),      # f32 onto fp16
                           (wide[:20], wide.as_strided((20, 6, 256), (2 * 6 * 256, 256, 1)))):               # another stride
        with pytest.raises(yahkv.YahkvError) as e:
            rope.rows(bad_x, pos[:bad_x.shape[0]], bad_out)
        assert e.value.code == yahkv.ERR_INVALID
    rope.rows(wide, pos, wide)
    one = x[:1].clone()
    torch.cuda.synchronize()
    rope.rows(one, pos[:1], one)                                 # a single token has no stride
    out16 = torch.empty_like(half)
    torch.cuda.synchronize()
    rope.rows(half, pos, out16)
    rope.rows(half, pos, half)
    cache.sync()
    assert torch.equal(wide, want) and torch.equal(one, want[:1]) and torch.equal(half, out16)
