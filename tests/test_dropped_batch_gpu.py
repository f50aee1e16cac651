"""A decode batch that is dropped without being closed keeps its device memory for captured graphs, and gives way when one of
its sequences is cut."""
import gc

import pytest
import torch

import yahkv
from gpu_util import dev
from test_batch_lifetime_gpu import cut, made
from test_shared_gpu import normal

pytestmark = pytest.mark.gpu


def test_a_dropped_batch_gives_way():
    cache, (a, b, c), _ = made(3)
    kept = yahkv.DecodeBatch(cache, [c])
    batch = yahkv.DecodeBatch(cache, [a, b])
    batch.prepare(2)
    del batch
    gc.collect()
    cut(cache, a)
    cut(cache, b)
    w = torch.zeros(1, 3, 4, 384, device="cuda")
    rows = torch.zeros(1, 1, 4, 50, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    with pytest.raises(yahkv.YahkvError) as e:
        cache.evict([c], 50, w, rows)                        # in a batch that is still there
    assert e.value.code == yahkv.ERR_ORDER
    kept.close()
    cut(cache, c)


def test_the_graph_of_a_dropped_batch_replays():
    outs = []
    for drop in (False, True):
        cache, (a, b), rng = made(2)
        k, v, q = dev(normal(rng, 2, 4, 256)), dev(normal(rng, 2, 4, 256)), dev(normal(rng, 2, 24, 256))
        out = torch.zeros(2, 24, 256, device="cuda")
        batch = yahkv.DecodeBatch(cache, [a, b])
        batch.prepare(8)
        cache.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st = torch.cuda.current_stream().cuda_stream
            batch.plan(stream=st)
            batch.decode_layer(0, k, v, q, out, out_dtype=yahkv.OUT_F32, stream=st)
            batch.advance(stream=st)
        if drop:
            del batch
            gc.collect()
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        outs.append(out.clone())
        del graph
        cache.close()
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])
