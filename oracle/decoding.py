"""The operators of a decoding step over a paged cache, from their definitions, in 64 bits: test infrastructure only.
Inputs are NumPy arrays of values (bf16 as the float values), results are float64."""
import numpy as np


def rope(x, positions, inv_freq, interleaved=False, amplitude=1.0):
    x = np.asarray(x, np.float64)
    half = len(inv_freq)
    y = x.copy()
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)[None, :]
    c, s = amplitude * np.cos(angle)[:, None, :], amplitude * np.sin(angle)[:, None, :]
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def sequences(query_start, context_len, tokens, max_keys):
    """(first token, tokens, keys) of every sequence, with out-of-range values clamped as the kernels clamp them."""
    out = []
    for b in range(len(context_len)):
        start = int(np.clip(query_start[b], 0, tokens))
        end = int(np.clip(query_start[b + 1], start, tokens))
        out.append((start, end - start, int(np.clip(context_len[b], 0, max_keys))))
    return out


def kv_append(k, v, k_cache, v_cache, page_table, query_start, context_len, inv_freq=None, interleaved=False, amplitude=1.0):
    kc, vc = np.array(k_cache, np.float64), np.array(v_cache, np.float64)
    pages, page = kc.shape[:2]
    for b, (start, n, ctx) in enumerate(sequences(query_start, context_len, k.shape[0], page_table.shape[1] * page)):
        for i in range(n):
            p = ctx - n + i
            if p < 0 or not 0 <= page_table[b, p // page] < pages:
                continue
            row = np.asarray(k[start + i], np.float64)
            if inv_freq is not None:
                row = rope(row[None], [p], inv_freq, interleaved, amplitude)[0]
            kc[page_table[b, p // page], p % page] = row
            vc[page_table[b, p // page], p % page] = v[start + i]
    return kc, vc


def paged_attention(q, k_cache, v_cache, page_table, query_start, context_len, scale, window=0, magnitudes=None):
    """`magnitudes`, a dict, receives what error bounds need: per output element sum of weight * |v| ("weighted") and of
    |v| over the keys seen ("plain"), per row the largest sum of |q k| * scale ("scores")."""
    q = np.asarray(q, np.float64)
    T, H, D = q.shape
    pages, page, HKV = k_cache.shape[:3]
    out = np.zeros((T, H, D))
    weighted, plain, scores = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H))
    for b, (start, n, ctx) in enumerate(sequences(query_start, context_len, T, page_table.shape[1] * page)):
        if n == 0 or ctx == 0:
            continue
        where = np.clip(page_table[b, np.arange(ctx) // page], 0, pages - 1), np.arange(ctx) % page
        k, v = np.asarray(k_cache[where], np.float64), np.asarray(v_cache[where], np.float64)
        for i in range(n):
            p = ctx - n + i
            lo = max(0, p - window + 1) if window else 0
            if p < lo:
                continue
            for h in range(H):
                g = h * HKV // H
                s = (k[lo:p + 1, g] @ q[start + i, h]) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[start + i, h] = w @ v[lo:p + 1, g]
                if magnitudes is not None:
                    weighted[start + i, h] = w @ np.abs(v[lo:p + 1, g])
                    plain[start + i, h] = np.abs(v[lo:p + 1, g]).sum(0)
                    scores[start + i, h] = (np.abs(k[lo:p + 1, g]) @ np.abs(q[start + i, h])).max() * abs(scale)
    if magnitudes is not None:
        magnitudes.update(weighted=weighted, plain=plain, scores=scores)
    return out


def matvec_w4(x, weight, scales, zeros=None, magnitudes=None):
    """`magnitudes` receives sum of |scale * x| * (|value - zero|, 1) per result as ("products", "ones")."""
    x, scales = np.asarray(x, np.float64), np.asarray(scales, np.float64)
    N, K = weight.shape[0], 2 * weight.shape[1]
    value = np.stack((weight & 15, weight >> 4), axis=-1).reshape(N, K).astype(np.float64)
    group = K // scales.shape[1]
    zero = np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64)
    s, d = np.repeat(scales, group, axis=1), value - np.repeat(zero, group, axis=1)
    if magnitudes is not None:
        magnitudes.update(products=np.abs(x) @ np.abs(d * s).T, ones=np.abs(x) @ np.abs(s).T)
    return x @ (d * s).T
