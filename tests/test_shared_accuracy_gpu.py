"""How near decode attention over shared prefixes comes to float64 attention on average: groups of more than 64 rows (three CTA
pairs and more per kv head), long prefixes and more groups than the device runs pairs at once.

Bar. The pass rounds the softmax weights to fp16 and, for quantized pages, K and V (products of codes and scales). A rounding
is off by at most 2^-11 of the value, and by 2^-11 / sqrt(3) at most in the root mean square, evenly spread over the step. With q, K
and V of unit normal entries each of them moves an output by its own relative size: V's and the weights' directly, since the
output is a sum of such products with independent errors; K's through the score, whose error sum_d q_d k_d e_d / 16 has the
root mean square |q| / 16 = 1 times the entries'. Independent errors add in squares: 2^-11 / sqrt(3) for fp16 pages, sqrt(3) times
that, 2^-11, for quantized ones. Outputs are f32. The largest error is held to the bar of test_shared_gpu.py."""
import math

import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from longctx_util import rows64
from test_shared_gpu import FMTS, grow, normal, shared, small_cache

pytestmark = pytest.mark.gpu


def compare(cache, seqs, q, got):
    err2 = ref2 = 0.0
    for b, s in enumerate(seqs):
        k, v = (torch.from_numpy(x).cuda() for x in rows64(cache, 0, s, cache.seq_len(s, 0)))
        qb = torch.from_numpy(q[b].astype(np.float64)).cuda().view(4, 6, 256)
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", qb, k) / 16.0, -1)
        want = torch.einsum("hgn,nhd->hgd", p, v).reshape(24, 256).cpu().numpy()
        err = np.abs(got[b] - want)
        assert err.max() <= 2e-3 + 2.0 ** -10 * float(v.abs().max()), (b, err.max())
        err2, ref2 = err2 + (err ** 2).sum(), ref2 + (want ** 2).sum()
    bar = 2.0 ** -11 / (math.sqrt(3.0) if cache.fmt == yahkv.FMT_F16 else 1.0)
    assert math.sqrt(err2 / ref2) <= bar, (math.sqrt(err2 / ref2), bar)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("groups", [[(96, 640, 70)], [(131, 200, 3)], [(65, 1300, 64)], [(3, 20000, 30)], [(2, 40000, 1)],
                                    [(2, 700, 9)] * 30, [(70, 400, 5), (44, 3000, 20), (2, 9000, 100)]])
def test_mean_error(fmt, groups):
    rng = np.random.default_rng(sum(r * p for r, p, _ in groups))
    pages = sum((p + 63) // 64 + r * ((s + 127) // 64 + 1) for r, p, s in groups)
    cache = small_cache(num_pages=pages, fmt=fmt, max_seqs=sum(r + 1 for r, _, _ in groups),
                        max_pages_per_seq=max((p + s + 127) // 64 for _, p, s in groups))
    seqs = []
    for rows, prefix, suffix in groups:
        root = cache.seq_create()
        grow(cache, rng, root, prefix)
        kids = [cache.seq_fork(root, prefix) for _ in range(rows)]
        for i, s in enumerate(kids):
            grow(cache, rng, s, 1 + i * 13 % suffix)
        cache.seq_free(root)
        seqs += kids
    seqs = [seqs[i] for i in rng.permutation(len(seqs))]
    q = normal(rng, len(seqs), 24, 256)
    compare(cache, seqs, q, shared(cache, 0, seqs, q))
