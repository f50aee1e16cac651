"""Prefill attention gives the same bits whatever the rows behind a sequence's last key hold (see test_rows_behind_gpu.py)."""
import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev
from test_rows_behind_gpu import LENS, both, filled
from test_shared_gpu import FMTS, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
def test_prefill(fmt):
    def call(bad):
        cache, seqs, rng = filled(fmt, bad)
        chunks = [min(n, c) for n, c in zip(LENS, (1, 63, 10, 65, 5, 130, 129))]
        q = dev(normal(rng, sum(chunks), 24, 256))
        out, raw = torch.zeros(sum(chunks), 24, 256, device="cuda"), torch.zeros(sum(chunks), 24, 256, device="cuda")
        ones = torch.ones(256, device="cuda")
        torch.cuda.synchronize()
        cache.attend_prefill(0, seqs, chunks, q, out, out_dtype=yahkv.OUT_F32)
        cache.attend_prefill_qraw(0, seqs, chunks, q.float(), ones, 1e-6, raw, out_dtype=yahkv.OUT_F32)
        cache.sync()
        return out, raw
    both(call)
