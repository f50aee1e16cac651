"""Float64 models of the long-context operators over what a cache holds (read back through the C ABI)."""
import numpy as np

import yahkv


def rows64(cache, layer, seq, n):
    """K and V of the first n tokens of a sequence as the cache holds them: two [n][4][256] float64 arrays."""
    table = cache.seq_table(seq)
    out = []
    for side in (yahkv.SIDE_K, yahkv.SIDE_V):
        pages = [page64(cache, layer, side, int(p)) for p in table[:(n + 63) // 64]]
        out.append(np.concatenate(pages)[:n] if pages else np.zeros((0, 4, 256)))
    return out


def page64(cache, layer, side, page):
    """[64][4][256] float64 values of one page."""
    codes, scales = cache.read_page(layer, side, page)
    if cache.fmt == yahkv.FMT_F16:
        x = codes.view(np.float16).astype(np.float64)                                        # [4][64][256]
    else:
        if cache.fmt == yahkv.FMT_Q8_0:
            c = codes.view(np.int8).astype(np.float64).reshape(4, 64, 8, 32)
        else:
            b = codes.reshape(4, 64, 8, 16)
            c = np.concatenate([b & 15, b >> 4], -1).astype(np.float64) - 8.0
        x = (c * scales.view(np.float16).astype(np.float64)[..., None]).reshape(4, 64, 256)
    return x.transpose(1, 0, 2)


def attend64(q, k, v, gate=None, scale=1.0 / 16.0):
    """q [24][256], k, v [n][4][256] -> out [24][256], weights [24][n], in float64."""
    out, p = np.zeros((24, 256)), np.zeros((24, k.shape[0]))
    q = np.asarray(q, np.float64)
    for h in range(24):
        s = k[:, h // 6] @ q[h] * scale
        e = np.exp(s - s.max())
        p[h] = e / e.sum()
        out[h] = p[h] @ v[:, h // 6]
    if gate is not None:
        out = out / (1.0 + np.exp(-np.asarray(gate, np.float64)))
    return out, p


def select(w, n, n_keep, n_sink, n_recent):
    """Kept slots of one kv head by the definition: sinks, recent ones, of the rest the largest (lowest slot on ties)."""
    if n <= n_keep:
        return list(range(n)) + [-1] * (n_keep - n)
    middle = list(range(n_sink, n - n_recent))
    value = {i: -np.inf if np.isnan(w[i]) else float(w[i]) for i in middle}
    nan = {i: bool(np.isnan(w[i])) for i in middle}
    middle.sort(key=lambda i: (nan[i], -value[i], i))
    return sorted(list(range(n_sink)) + middle[:n_keep - n_sink - n_recent] + list(range(n - n_recent, n)))
