"""What is measured of the long-context serving operators: decode attention over a prefix that a batch shares, decode
attention that also accumulates every key's attention weight, the eviction of keys by that weight, and the rotation of
head rows at given positions.

`own` false: the operators in elementary torch operations on plain tensors. `own` true: the calls that a user of the
library makes. Geometry as everywhere in the library: 24 query heads, 4 KV heads, head_dim 256, 64-token pages.
"""
import math
import os
import sys

import torch

own = False

QH, KVH, GROUP, DIM, PAGE = 24, 4, 6, 256, 64
SCALE = 1.0 / 16.0
TOKEN_BYTES = {"f16": 4096, "q8_0": 2176, "q4_0": 1152}     # K and V of one token in one layer
EPS = 1e-6


def listed():
    return [
        # two answers sampled from one short prompt: what a call costs when there is next to nothing to read
        dict(name="shared f16 2 x 128", op="shared", fmt="f16", rows=2, prefix=128, suffix=3),
        # a serving batch behind one system prompt with documents
        dict(name="shared q8_0 32 x 8192", op="shared", fmt="q8_0", rows=32, prefix=8192, suffix=700),
        # sixteen questions about one long document, in the smallest cache format
        dict(name="shared q4_0 16 x 65536", op="shared", fmt="q4_0", rows=16, prefix=65536, suffix=1000),
        # a wide sampling batch; the prefix ends inside a page
        dict(name="shared f16 96 x 16421", op="shared", fmt="f16", rows=96, prefix=16421, suffix=512),
        # one conversation whose cache is watched for eviction
        dict(name="weights q8_0 1 x 777", op="weights", fmt="q8_0", rows=1, lo=777, hi=777),
        # a batch of contexts of all lengths
        dict(name="weights q8_0 32 x 16384", op="weights", fmt="q8_0", rows=32, lo=1024, hi=16384),
        # a few long contexts, unquantized
        dict(name="weights f16 5 x 30001", op="weights", fmt="f16", rows=5, lo=29000, hi=30001),
        # one short conversation cut to a quarter, one layer
        dict(name="evict q8_0 1 x 1000", op="evict", fmt="q8_0", layers=1, rows=1, lo=1000, hi=1000, keep=250),
        # a batch of long contexts cut in all of its layers at once
        dict(name="evict q8_0 4 x 8 x 16384", op="evict", fmt="q8_0", layers=4, rows=8, lo=12000, hi=16384, keep=4096),
        # the queries of a decode batch: norm and a quarter of the head rotated, straight from the projection
        dict(name="rope 32 x 24 half 64", op="rope", tokens=32, heads=24, layout="half", rotary=64, scaling="none",
             factor=1.0, x="f32", out="f16", norm=True, span=32768),
        # a prefill chunk's queries and keys in the middle of a very long context, whole heads, neighbouring pairs
        dict(name="rope 8192 x 28 interleaved", op="rope", tokens=8192, heads=28, layout="interleaved", rotary=256,
             scaling="yarn", factor=32.0, x="f32", out="f16", norm=True, span=1000000),
        # keys turned without a norm, an odd count of tokens, a rotated part that is no multiple of eight
        dict(name="rope 1999 x 4 half 108", op="rope", tokens=1999, heads=4, layout="half", rotary=108, scaling="ntk",
             factor=4.0, x="f16", out="f32", norm=False, span=131072),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "weights", "evict", "rope"])
    fmt = rng.choice(["f16", "q8_0", "q4_0"])
    if op == "shared":
        rows = _log_int(rng, 2, 96)
        return dict(op=op, fmt=fmt, rows=rows, prefix=_log_int(rng, 65, min(65536, 96 * 16384 // rows)),
                    suffix=_log_int(rng, 1, min(1000, 49152 // rows)))
    if op == "weights":
        rows = _log_int(rng, 1, 32)
        hi = _log_int(rng, 1, 150000 // rows)
        return dict(op=op, fmt=fmt, rows=rows, lo=max(1, hi // rng.randint(1, 16)), hi=hi)
    if op == "evict":
        rows, layers = _log_int(rng, 1, 8), rng.randint(1, 4)
        hi = _log_int(rng, 100, 16384)
        lo = hi - hi // rng.randint(4, 9)
        return dict(op=op, fmt=fmt, layers=layers, rows=rows, lo=lo, hi=hi, keep=rng.randint(20, max(21, lo // 2)))
    rotary = 2 * rng.randint(2, 128)
    return dict(op=op, tokens=_log_int(rng, 1, 8000), heads=rng.choice([1, 4, 24, 28]),
                layout=rng.choice(["half", "interleaved"]), rotary=rotary,
                scaling=rng.choice(["none", "linear", "ntk", "yarn"]), factor=rng.choice([2.0, 4.0, 7.5, 32.0]),
                x=rng.choice(["f16", "f32"]), out=rng.choice(["f16", "f32"]), norm=rng.choice([True, False]),
                span=_log_int(rng, 4096, 1000000))


# ---- sizes that follow from a case alone ----

def _spread(lo, hi, n):
    """n lengths between lo and hi, the largest among them, in no order."""
    return [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _sink_recent(keep):
    return min(4, keep // 4), keep // 4


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * DIM
        b = n * ((4 if case["x"] == "f32" else 2) + (4 if case["out"] == "f32" else 2)) + 8 * case["tokens"]
        return dict(bytes=b, flops=n * (4 if case["norm"] else 0) + 3 * case["tokens"] * case["heads"] * case["rotary"])
    tb, rows = TOKEN_BYTES[case["fmt"]], case["rows"]
    if op == "shared":
        suffix = sum(_spread(1, case["suffix"], rows))
        return dict(bytes=tb * (case["prefix"] + suffix) + rows * QH * DIM * 4,
                    flops=4 * QH * DIM * (rows * case["prefix"] + suffix))
    lens = _spread(case["lo"], case["hi"], rows)
    if op == "weights":
        return dict(bytes=sum(lens) * (tb + KVH * 8) + rows * QH * DIM * 4, flops=4 * QH * DIM * sum(lens))
    layers, keep = case["layers"], case["keep"]
    kept = layers * rows * keep
    return dict(bytes=layers * sum(lens) * KVH * 4 + kept * (KVH * 8 + 3 * tb) + layers * rows * QH * DIM * 4,
                flops=4 * QH * DIM * kept)


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFF)


def _rows(g, shape):
    """K or V rows: channels of unequal size, a few of them large, as projections give them."""
    size = torch.exp(0.3 * torch.randn(KVH, DIM, generator=g, device="cuda"))
    size[:, ::61] *= 3.0
    x = torch.randn(*shape, KVH, DIM, generator=g, device="cuda", dtype=torch.float16)
    return x.mul_(size.half())


def _quantize(x, fmt):
    """fp16 rows -> what a cache of this format holds of them: the rows, or (codes, fp16 block scales)."""
    if fmt == "f16":
        return (x,)
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1] + (DIM // 32,), dtype=torch.float16, device=x.device)
    flat, cf, sf = x.view(-1, DIM), codes.view(-1, DIM), scales.view(-1, DIM // 32)
    for at in range(0, flat.shape[0], 1 << 18):
        b = flat[at:at + (1 << 18)].float().view(-1, DIM // 32, 32)
        mag = b.abs()
        top = mag.amax(-1, keepdim=True)
        if fmt == "q8_0":
            d = top / 127.0
            y = b * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
            c = torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y))
        else:
            index = torch.arange(32, device=x.device)
            first = torch.where(mag == top, index, 32).amin(-1, keepdim=True)
            d = b.gather(-1, first) / -8.0
            y = b * torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
            c = torch.clamp(torch.trunc(y + 8.5), max=15.0) - 8.0
        cf[at:at + (1 << 18)] = c.view(-1, DIM).to(torch.int8)
        sf[at:at + (1 << 18)] = d.view(-1, DIM // 32).half()
    return codes, scales


def _inputs(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "rope":
        n, span = case["tokens"], case["span"]
        kind = torch.float32 if case["x"] == "f32" else torch.float16
        # rows are a slice of a wider projection output, as a fused q/k/v product leaves them
        wide = torch.randn(n, (case["heads"] + 4) * DIM, generator=g, device="cuda").to(kind)
        if n < 256:     # a decode batch: every row its own sequence
            pos = torch.randint(0, span, (n,), generator=g, device="cuda")
        else:           # a chunk of one sequence, up to the end of the span
            pos = torch.arange(max(span - n, 0), max(span - n, 0) + n, device="cuda")
        return dict(wide=wide, pos=pos, weight=1.0 + 0.1 * torch.randn(DIM, generator=g, device="cuda"))
    rows, fmt = case["rows"], case["fmt"]
    s = {}
    if op == "shared":
        lens = _spread(1, case["suffix"], rows)
        s["kp16"], s["vp16"] = _rows(g, (case["prefix"],)), _rows(g, (case["prefix"],))
        s["ks16"], s["vs16"] = _rows(g, (rows, max(lens))), _rows(g, (rows, max(lens)))
        s["q"] = torch.randn(rows, QH, DIM, generator=g, device="cuda", dtype=torch.float16)
    else:
        layers = case.get("layers", 1)
        lens = _spread(case["lo"], case["hi"], rows)
        s["k16"], s["v16"] = _rows(g, (layers, rows, max(lens))), _rows(g, (layers, rows, max(lens)))
        s["q"] = torch.randn(layers, rows, QH, DIM, generator=g, device="cuda", dtype=torch.float16)
        # weights collected by the steps before: most keys near nothing, a few of them heavy, some never looked at
        w = torch.randn(layers, rows, KVH, max(lens), generator=g, device="cuda")
        w = torch.exp(2.0 * w - 6.0)
        w = torch.where(w < 2e-4, torch.zeros_like(w), w)
        s["w"] = w * (2 * GROUP / w.sum(-1, keepdim=True))      # what two steps add up to
    s["lens_host"] = lens
    s["lens"] = torch.tensor(lens, device="cuda")
    for name in [n for n in s if n.endswith("16")]:
        s[name[:-2]] = _quantize(s[name], fmt)
    return s


# ---- the plain forms ----

def _value(held):
    """The f32 values of what the cache holds."""
    if len(held) == 1:
        return held[0].float()
    codes, scales = held
    return (codes.float().unflatten(-1, (DIM // 32, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _plain_shared(s):
    q = s["q"].float().unflatten(1, (KVH, GROUP))                                     # [b, h, g, d]
    sp = torch.einsum("bhgd,phd->bhgp", q, _value(s["kp"])) * SCALE
    ss = torch.einsum("bhgd,bshd->bhgs", q, _value(s["ks"])) * SCALE
    seen = torch.arange(ss.shape[-1], device="cuda") < s["lens"][:, None]
    ss = torch.where(seen[:, None, None, :], ss, -torch.inf)
    top = torch.maximum(sp.amax(-1, keepdim=True), ss.amax(-1, keepdim=True))
    ep, es = torch.exp(sp - top), torch.exp(ss - top)
    total = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    o = torch.einsum("bhgp,phd->bhgd", ep, _value(s["vp"])) + torch.einsum("bhgs,bshd->bhgd", es, _value(s["vs"]))
    return (o / total).flatten(1, 2).half()


def _plain_weights(s):
    q = s["q"][0].float().unflatten(1, (KVH, GROUP))
    z = torch.einsum("bhgd,bshd->bhgs", q, _value([t[0] for t in s["k"]])) * SCALE
    seen = torch.arange(z.shape[-1], device="cuda") < s["lens"][:, None]
    z = torch.where(seen[:, None, None, :], z, -torch.inf)
    e = torch.exp(z - z.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    s["acc"] += p.sum(2)
    o = torch.einsum("bhgs,bshd->bhgd", p, _value([t[0] for t in s["v"]]))
    return dict(out=o.flatten(1, 2).half(), weights=s["acc"])


def _plain_evict(s):
    keep = s["keep"]
    sink, recent = _sink_recent(keep)
    w, lens = s["w"], s["lens"][None, :, None, None]
    index = torch.arange(w.shape[-1], device="cuda")
    rank = torch.where((index < sink) | (index >= lens - recent), torch.inf, w)
    rank = torch.where(index < lens, rank, -torch.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kept = torch.sort(order[..., :keep], dim=-1).values                               # [l, b, h, keep]
    rows = kept.movedim(2, 3)                                                         # [l, b, keep, h]
    take = lambda held: [t.gather(2, rows.unsqueeze(-1).expand(*rows.shape, t.shape[-1])) for t in held]  # noqa: E731
    q = s["q"].float().unflatten(2, (KVH, GROUP))
    z = torch.einsum("lbhgd,lbshd->lbhgs", q, _value(take(s["k"]))) * SCALE
    e = torch.exp(z - z.amax(-1, keepdim=True))
    o = torch.einsum("lbhgs,lbshd->lbhgd", e, _value(take(s["v"]))) / e.sum(-1, keepdim=True)
    return dict(kept=kept.int(), weights=w.gather(-1, kept), out=o.flatten(2, 3).half())


def _yarn(case):
    return dict(original=case["span"] / case["factor"], fast=32.0, slow=1.0)


def _plain_rope(s):
    case, half = s["case"], s["case"]["rotary"] // 2
    x = s["x"].float()
    if case["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"]
    pair = torch.arange(half, device="cuda", dtype=torch.float64)
    theta, factor = 1e7, case["factor"]
    if case["scaling"] == "ntk":
        theta = theta * factor ** (case["rotary"] / (case["rotary"] - 2))
    freq = theta ** (-pair / half)
    size = 1.0
    if case["scaling"] == "linear":
        freq = freq / factor
    if case["scaling"] == "yarn":
        y = _yarn(case)
        turns = y["original"] * freq / (2 * math.pi)
        ramp = ((turns - y["slow"]) / (y["fast"] - y["slow"])).clamp(0, 1)
        freq = freq / factor * (1 - ramp) + freq * ramp
        size = 0.1 * math.log(factor) + 1.0
    angle = s["pos"].double()[:, None, None] * freq                                   # far positions: 64 bits
    cos, sin = (torch.cos(angle) * size).float(), (torch.sin(angle) * size).float()
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["layout"] == "half":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(torch.float32 if case["out"] == "f32" else torch.float16)


# ---- the library's side ----

def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "yet-another-halo-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import yahkv
    return yahkv


def _fill(cache, layer, seqs, starts, lens, k16, v16, k, v):
    """Appends rows [i, :lens[i]] of k16, v16 to sequence seqs[i] behind its first starts[i] tokens. q8_0: the cache is
    then given the very codes that k, v hold of them; a value that lies between two codes may be rounded to either side
    by two quantizers whose block maxima are divided in different ways."""
    chunk = 8192
    for i, seq in enumerate(seqs):
        cache.seq_reserve(seq, starts[i] + lens[i])
        for a in range(0, lens[i], chunk):
            n = min(chunk, lens[i] - a)
            cache.append(layer, [seq] * n, list(range(starts[i] + a, starts[i] + a + n)), k16[i, a:a + n], v16[i, a:a + n])
    if cache.fmt != _library().FMT_Q8_0:
        return
    for i, seq in enumerate(seqs):
        first, shift = starts[i] // PAGE, starts[i] % PAGE
        pages = cache.seq_table(seq)[first:(starts[i] + lens[i] + PAGE - 1) // PAGE]
        for side, held in enumerate((k, v)):
            as_pages = []
            for t in held:
                x = torch.zeros(len(pages) * PAGE, KVH, t.shape[-1], dtype=t.dtype, device="cuda")
                x[shift:shift + lens[i]] = t[i, :lens[i]]
                as_pages.append(x.unflatten(0, (-1, PAGE)).transpose(1, 2).contiguous().cpu().numpy())
            codes, scales = as_pages[0].view("uint8"), as_pages[1].view("uint16")
            for n, page in enumerate(pages):
                if n == 0 and shift:
                    old = cache.read_page(layer, side, int(page))
                    codes[0, :, :shift], scales[0, :, :shift] = old[0][:, :shift], old[1][:, :shift]
                cache.write_page(layer, side, int(page), codes[n], scales[n])


def _handle(case, s):
    """What the user's program keeps beside its tensors: the cache with the sequences in it, or the rotation."""
    yahkv = _library()
    if case["op"] == "rope":
        y = _yarn(case)
        cache = yahkv.KvCache(num_pages=1, max_seqs=1, max_pages_per_seq=1, max_batch_tokens=64)
        s["rope"] = yahkv.Rope(cache, layout=case["layout"], rotary_dim=case["rotary"], theta=1e7, scaling=case["scaling"],
                               factor=case["factor"], original_len=y["original"], beta_fast=y["fast"],
                               beta_slow=y["slow"], max_positions=max(case["span"], case["tokens"]))
        s["out"] = torch.empty(s["x"].shape, device="cuda", dtype=torch.float32 if case["out"] == "f32" else torch.float16)
        s["cache"] = cache
        return
    fmt = dict(f16=yahkv.FMT_F16, q8_0=yahkv.FMT_Q8_0, q4_0=yahkv.FMT_Q4_0)[case["fmt"]]
    pages = lambda n: (n + PAGE - 1) // PAGE  # noqa: E731
    rows, lens = case["rows"], s["lens_host"]
    if case["op"] == "shared":
        longest = case["prefix"] + max(lens)
        cache = yahkv.KvCache(num_pages=pages(case["prefix"]) + rows * (pages(max(lens)) + 2), fmt=fmt, max_seqs=rows + 1,
                              max_pages_per_seq=pages(longest) + 1)
        root = cache.seq_create()
        _fill(cache, 0, [root], [0], [case["prefix"]], s["kp16"][None], s["vp16"][None],
              [t[None] for t in s["kp"]], [t[None] for t in s["vp"]])
        s["seqs"] = [cache.seq_fork(root, case["prefix"]) for _ in range(rows)]
        _fill(cache, 0, s["seqs"], [case["prefix"]] * rows, lens, s["ks16"], s["vs16"], s["ks"], s["vs"])
        s["out"] = torch.empty(rows, QH, DIM, device="cuda", dtype=torch.float16)
    else:
        layers = case.get("layers", 1)
        extra = case["op"] == "evict"
        cache = yahkv.KvCache(n_layers=layers, fmt=fmt, max_seqs=rows * (2 if extra else 1), max_pages_per_seq=pages(max(lens)),
                              num_pages=sum(pages(n) for n in lens) + (rows * (pages(case["keep"]) + 1) if extra else 0))
        s["seqs"] = [cache.seq_create() for _ in range(rows)]
        for layer in range(layers):
            _fill(cache, layer, s["seqs"], [0] * rows, lens, s["k16"][layer], s["v16"][layer],
                  [t[layer] for t in s["k"]], [t[layer] for t in s["v"]])
        s["out"] = torch.empty(layers, rows, QH, DIM, device="cuda", dtype=torch.float16)
        if extra:
            s["branch_w"] = torch.zeros(layers, 2 * rows, KVH, max(lens), device="cuda")
            s["kept"] = torch.empty(layers, rows, KVH, case["keep"], device="cuda", dtype=torch.int32)
    cache.sync()
    s["cache"] = cache


def _own_shared(s):
    s["cache"].attend_decode_shared(0, s["seqs"], s["q"], s["out"])
    return s["out"]


def _own_weights(s):
    s["cache"].attend_decode_weights(0, s["seqs"], s["q"][0], s["out"][0], s["acc"])
    return dict(out=s["out"][0], weights=s["acc"])


def _own_evict(s):
    # a branch of every sequence is cut, the sequence itself stays whole
    cache, keep, rows = s["cache"], s["keep"], len(s["seqs"])
    sink, recent = _sink_recent(keep)
    branch = [cache.seq_fork(seq, n) for seq, n in zip(s["seqs"], s["lens_host"])]
    s["branch_w"][:, rows:] = s["w"]        # a branch takes the sequence slots behind the whole ones
    cache.evict(branch, keep, s["branch_w"], s["kept"], n_sink=sink, n_recent=recent)
    for layer in range(s["q"].shape[0]):
        cache.attend_decode(layer, branch, s["q"][layer], s["out"][layer])
    for seq in reversed(branch):
        cache.seq_free(seq)
    return dict(kept=s["kept"], weights=s["branch_w"][:, rows:, :, :keep], out=s["out"])


def _own_rope(s):
    s["rope"].rows(s["x"], s["pos"], s["out"], weight=s["weight"] if s["case"]["norm"] else None, eps=EPS)
    return s["out"]


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rope":
        s["case"] = case
        s["x"] = s.pop("wide")[:, :case["heads"] * DIM].unflatten(-1, (case["heads"], DIM))
    if case["op"] == "weights":
        s["acc"] = s.pop("w")[0].clone()
    if case["op"] == "evict":
        s["keep"] = case["keep"]
    if own:
        _handle(case, s)
        torch.cuda.synchronize()
    for name in [n for n in s if n.endswith("16")]:
        del s[name]
    if own:     # the cache holds them
        for name in ("kp", "vp", "ks", "vs", "k", "v"):
            s.pop(name, None)
    s["op"] = case["op"]
    return s


def run(state):
    if own:
        return dict(shared=_own_shared, weights=_own_weights, evict=_own_evict, rope=_own_rope)[state["op"]](state)
    return dict(shared=_plain_shared, weights=_plain_weights, evict=_plain_evict, rope=_plain_rope)[state["op"]](state)


# ---- the definitions in 64 bits ----

def _value64(held, at=...):
    if len(held) == 1:
        return held[0][at].double()
    c, d = held[0][at].double(), held[1][at].double()
    return c * d.repeat_interleave(32, dim=-1)


def _attend64(q, k, v):
    """q [24, 256], k, v [n, 4, 256] -> out [24, 256] and the weights [24, n], all in 64 bits."""
    out = torch.empty(QH, DIM, device="cuda", dtype=torch.float64)
    p = torch.empty(QH, k.shape[0], device="cuda", dtype=torch.float64)
    for h in range(KVH):
        z = (q[GROUP * h:GROUP * (h + 1)].double() @ k[:, h].T) / 16.0
        p[GROUP * h:GROUP * (h + 1)] = torch.softmax(z, dim=-1)
        out[GROUP * h:GROUP * (h + 1)] = p[GROUP * h:GROUP * (h + 1)] @ v[:, h]
    return out, p


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    lens, rows = s["lens_host"], case["rows"]
    if case["op"] == "shared":
        out = torch.empty(rows, QH, DIM, device="cuda", dtype=torch.float64)
        kp, vp = _value64(s["kp"]), _value64(s["vp"])
        for b in range(rows):
            k = torch.cat([kp, _value64(s["ks"], (b, slice(0, lens[b])))])
            v = torch.cat([vp, _value64(s["vs"], (b, slice(0, lens[b])))])
            out[b] = _attend64(s["q"][b], k, v)[0]
        return out
    if case["op"] == "weights":
        out = torch.empty(rows, QH, DIM, device="cuda", dtype=torch.float64)
        acc = s["w"][0].double()
        for b, n in enumerate(lens):
            at = (0, b, slice(0, n))
            out[b], p = _attend64(s["q"][0, b], _value64(s["k"], at), _value64(s["v"], at))
            acc[b, :, :n] += p.view(KVH, GROUP, n).sum(1)
        return dict(out=out, weights=acc)
    layers, keep = case["layers"], case["keep"]
    sink, recent = _sink_recent(keep)
    out = torch.empty(layers, rows, QH, DIM, device="cuda", dtype=torch.float64)
    kept = torch.empty(layers, rows, KVH, keep, device="cuda", dtype=torch.int32)
    weights = torch.empty(layers, rows, KVH, keep, device="cuda", dtype=torch.float64)
    for layer in range(layers):
        for b, n in enumerate(lens):
            for h in range(KVH):
                w = s["w"][layer, b, h, :n].double().cpu().numpy()
                middle = sorted(range(sink, n - recent), key=lambda i, w=w: (-w[i], i))[:keep - sink - recent]
                chosen = list(range(sink)) + sorted(middle) + list(range(n - recent, n))
                kept[layer, b, h] = torch.tensor(chosen, dtype=torch.int32)
                weights[layer, b, h] = s["w"][layer, b, h, chosen].double()
                rows_at = (layer, b, torch.tensor(chosen, device="cuda"), h)
                k, v = _value64(s["k"], rows_at), _value64(s["v"], rows_at)
                q = s["q"][layer, b, GROUP * h:GROUP * (h + 1)].double()
                out[layer, b, GROUP * h:GROUP * (h + 1)] = torch.softmax(q @ k.T / 16.0, dim=-1) @ v
    return dict(kept=kept, weights=weights, out=out)


def _exact_rope(case, s):
    heads, r = case["heads"], case["rotary"]
    x = s["wide"][:, :heads * DIM].double().view(-1, heads, DIM)
    if case["norm"]:
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / DIM + EPS) * s["weight"].double()
    theta, f = 1e7, case["factor"]
    if case["scaling"] == "ntk":
        theta *= f ** (r / (r - 2.0))
    out = x.clone()
    for p in range(r // 2):
        w, m = theta ** (-2.0 * p / r), 1.0
        if case["scaling"] == "linear":
            w /= f
        if case["scaling"] == "yarn":
            y = _yarn(case)
            g = min(1.0, max(0.0, (y["original"] * w / (2 * math.pi) - y["slow"]) / (y["fast"] - y["slow"])))
            w, m = (1 - g) * w / f + g * w, 0.1 * math.log(f) + 1.0
        c, d = m * torch.cos(s["pos"].double() * w)[:, None], m * torch.sin(s["pos"].double() * w)[:, None]
        i, j = (p, p + r // 2) if case["layout"] == "half" else (2 * p, 2 * p + 1)
        out[..., i] = x[..., i] * c - x[..., j] * d
        out[..., j] = x[..., i] * d + x[..., j] * c
    return out
