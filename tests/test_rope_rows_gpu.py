"""yahkv_rope_rows against rotation in float64.

Tolerance. Relative to a row's largest |x| = X (after the norm) and magnitude m: cos and sin are the product of two
fp32-rounded pairs (each entry off by 2^-24 of at most 1, the two-term product by 4 x 2^-24 + two roundings of 2^-24),
the turn is two products and a sum (3 x 2^-24 of at most 2 X m): below 2 X m x 10 x 2^-24. The norm adds a sum of 256 squares
(256 x 2^-24 in the worst order, halved by the root), a root, a division and two products: 132 x 2^-24 of the value.
An fp16 output adds half a step, 2^-11 of the value, or 2^-25 below the normal range."""
import math

import numpy as np
import pytest
import torch

import yahkv
from gpu_util import dev

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def cache():
    return yahkv.KvCache(num_pages=2, max_seqs=1, max_pages_per_seq=2)


def freqs(r, theta, scaling, factor, original, fast, slow, magnitude):
    p = np.arange(r // 2, dtype=np.float64)
    m = magnitude or 1.0
    if scaling == "ntk":
        theta = theta * factor ** (r / (r - 2.0))
    f = theta ** (-2.0 * p / r)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        k = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        f = (1 - k) * f / factor + k * f
        m = magnitude or 0.1 * math.log(factor) + 1.0
    return f, m


def rotate64(x, pos, layout, r, f, m, weight):
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + EPS) * weight.astype(np.float64)
    a = pos[:, None, None].astype(np.float64) * f
    c, s = m * np.cos(a), m * np.sin(a)
    y = x.copy()
    i = np.arange(r // 2)
    i, j = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return x, y


def bound(x, want, m, normed, out16):
    top = np.abs(x).max(-1, keepdims=True)
    tol = 20 * 2.0 ** -24 * top * m + (132 * 2.0 ** -24 * 2 * top * m if normed else 0)
    return tol + (np.maximum(2.0 ** -11 * np.abs(want), 2.0 ** -25) if out16 else 0)


CASES = [(layout, r, scaling) for layout in ("half", "interleaved")
         for r, scaling in ((64, "none"), (256, "yarn"), (2, "linear"), (4, "ntk"), (108, "yarn"), (30, "none"), (128, "linear"), (254, "ntk"))]


@pytest.mark.parametrize("layout,r,scaling", CASES)
def test_rows(cache, layout, r, scaling):
    rng = np.random.default_rng(r)
    top = 1 << 20
    kw = dict(factor=7.5, original_len=4096.0, beta_fast=24.0, beta_slow=2.0)
    magnitude = 1.25 if r == 128 else 0.0
    rope = yahkv.Rope(cache, layout=layout, rotary_dim=r, theta=1e6, scaling=scaling, max_positions=top, magnitude=magnitude, **kw)
    f, m = freqs(r, 1e6, scaling, 7.5, 4096.0, 24.0, 2.0, magnitude)
    for tokens, heads, x32, out32, normed in ((1, 1, True, False, True), (3, 24, False, False, False), (33, 4, True, True, True),
                                              (257, 28, False, True, False), (700, 24, True, False, False)):
        x = rng.standard_normal((tokens, heads + 2, 256)).astype(np.float32 if x32 else np.float16)
        pos = rng.integers(0, top, tokens)
        pos[0] = top - 1
        pos[-1] = 0 if tokens > 1 else top - 1
        weight = (1 + 0.2 * rng.standard_normal(256)).astype(np.float32) if normed else None
        xd = dev(x)
        out = torch.full((tokens, heads + 1, 256), float("nan"), device="cuda", dtype=torch.float32 if out32 else torch.float16)
        torch.cuda.synchronize()
        rope.rows(xd[:, 1:1 + heads], dev(pos), out[:, :heads], weight=None if weight is None else dev(weight), eps=EPS)
        cache.sync()
        base, want = rotate64(x[:, 1:1 + heads], pos, layout, r, f, m, weight)
        got = out[:, :heads].double().cpu().numpy()
        tol = bound(base, want, max(m, 1.0), normed, not out32)
        assert (np.abs(got - want) <= tol).all(), (tokens, (np.abs(got - want) / tol).max())
        assert torch.isnan(out[:, heads:]).all()                      # nothing outside the rows
        if not normed and not x32 and not out32:                      # what is not rotated passes through
            assert np.array_equal(out[:, :heads].cpu().numpy()[..., r:], x[:, 1:1 + heads, r:])


def test_agrees_with_rope_append():
    """The fused call's rotation (half layout, 64 of 256, theta 1e7) is a case of this one."""
    rng = np.random.default_rng(9)
    n = 70
    c = yahkv.KvCache(num_pages=4, max_seqs=1, max_pages_per_seq=4)
    s = c.seq_create()
    c.seq_reserve(s, n)
    q, k, v = (dev(rng.standard_normal((n, h, 256)).astype(np.float32)) for h in (24, 4, 4))
    w = dev((1 + 0.1 * rng.standard_normal(256)).astype(np.float32))
    a, b = torch.empty(n, 24, 256, device="cuda", dtype=torch.float16), torch.empty(n, 24, 256, device="cuda", dtype=torch.float16)
    c.rope_append(0, [s] * n, np.arange(n), q, k, v, w, w, EPS, a)
    yahkv.Rope(c, max_positions=256).rows(q, torch.arange(n, device="cuda"), b, weight=w, eps=EPS)
    c.sync()
    # both within half a step of the exact value and a few fp32 roundings: at most one step apart
    step = 2.0 ** -10 * torch.maximum(a.double().abs(), torch.tensor(2.0 ** -14, device="cuda"))
    assert ((a.double() - b.double()).abs() <= step).all()


def test_in_place_on_a_stream_and_replayed(cache):
    rng = np.random.default_rng(12)
    rope = yahkv.Rope(cache, rotary_dim=128, layout="interleaved", max_positions=5000)
    f, m = freqs(128, 1e7, "none", 1, 0, 0, 0, 0)
    x = rng.standard_normal((40, 24, 256)).astype(np.float16)
    pos = rng.integers(0, 5000, 40)
    t, p = dev(x), dev(pos)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    rope.rows(t, p, t, stream=side.cuda_stream)
    cache.sync()
    base, want = rotate64(x, pos, "interleaved", 128, f, m, None)
    assert (np.abs(t.double().cpu().numpy() - want) <= bound(base, want, 1.0, False, True)).all()
    src, out = dev(x), torch.empty(40, 24, 256, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.rows(src, p, out, stream=torch.cuda.current_stream().cuda_stream)
    pos2 = rng.integers(0, 5000, 40)
    p.copy_(torch.from_numpy(pos2))
    graph.replay()
    torch.cuda.synchronize()
    base, want = rotate64(x, pos2, "interleaved", 128, f, m, None)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound(base, want, 1.0, False, False)).all()


def test_a_position_out_of_range_is_reported(cache):
    rope = yahkv.Rope(cache, max_positions=100)
    x = torch.ones(3, 4, 256, device="cuda")
    for bad in (100, -1, 1 << 40):
        pos = torch.tensor([5, bad, 7], device="cuda")
        torch.cuda.synchronize()
        out = torch.empty_like(x)
        rope.rows(x, pos, out)
        with pytest.raises(yahkv.YahkvError) as e:
            cache.sync()
        assert e.value.code == yahkv.ERR_CUDA and "position" in e.value.message
        cache.sync()                                                   # cleared
        good = torch.empty(2, 4, 256, device="cuda")
        rope.rows(x[:2], torch.tensor([5, 7], device="cuda"), good)
        cache.sync()
        assert torch.equal(out[[0, 2]], good)                          # the other rows are right


def test_refusals(cache):
    def code(f, *a, **k):
        with pytest.raises(yahkv.YahkvError) as e:
            f(*a, **k)
        return e.value.code
    for bad in (dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=258), dict(theta=1.0), dict(theta=float("nan")),
                dict(scaling="linear", factor=0.5), dict(scaling="ntk", rotary_dim=2, factor=2.0), dict(max_positions=0),
                dict(scaling="yarn", factor=2.0), dict(scaling="yarn", factor=2.0, original_len=10.0, beta_fast=1.0, beta_slow=1.0),
                dict(magnitude=-1.0), dict(max_positions=1 << 32)):
        assert code(yahkv.Rope, cache, **bad) == yahkv.ERR_INVALID, bad
    rope = yahkv.Rope(cache, max_positions=64)
    x, p = torch.ones(2, 4, 256, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int64)
    h, ptr = rope._h, yahkv._ptr
    call = yahkv.lib.yahkv_rope_rows
    assert call(h, -1, 4, ptr(p), ptr(x), 1, 1024, None, 0.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    assert call(h, 2, 4, None, ptr(x), 1, 1024, None, 0.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    assert call(h, 2, 4, ptr(p), ptr(x), 2, 1024, None, 0.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    assert call(h, 2, 4, ptr(p), ptr(x), 1, 1020, None, 0.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    assert call(h, 2, 4, ptr(p), ptr(x), 1, 1024, None, 0.0, ptr(x), 1, 1016, None) == yahkv.ERR_INVALID
    assert call(h, 2, 4, ptr(p), ptr(x.flatten()[1:]), 1, 1024, None, 0.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    assert call(h, 2, 4, ptr(p), ptr(x), 1, 1024, ptr(x), -1.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    assert call(h, 0, 4, ptr(p), ptr(x), 1, 1024, None, 0.0, ptr(x), 1, 1024, None) == yahkv.OK
    assert call(None, 0, 4, ptr(p), ptr(x), 1, 1024, None, 0.0, ptr(x), 1, 1024, None) == yahkv.ERR_INVALID
    with pytest.raises(ValueError):
        rope.rows(x[:, :, :128], p, x)
    with pytest.raises(ValueError):
        rope.rows(x, p.cpu(), x)
    with pytest.raises(ValueError):
        rope.rows(x.cpu(), p, x)
    other = yahkv.KvCache(num_pages=1, max_seqs=1, max_pages_per_seq=1)
    left = yahkv.Rope(other, max_positions=64)
    other.close()                                   # out of order: nothing of the cache is touched any more
    with pytest.raises(ValueError):
        left.rows(x, p, x)
    left.close()
    with pytest.raises(ValueError):
        rope.rows(x, p.int(), x)
    with pytest.raises(ValueError):
        rope.rows(x, p, x.transpose(0, 1).contiguous().transpose(0, 1))
