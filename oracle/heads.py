"""The operators on heads and paged caches in float64 numpy: rotary positions, RMS
norm of each head with the rotation, appending to a paged cache, attention from new
tokens to it.  Pinned by ``tests/test_heads_oracle.py`` against torch's autograd and
against the definitions written out in loops."""
from __future__ import annotations

import numpy as np


def f64(x):
    return np.asarray(x, dtype=np.float64)


def rope(x, positions, inv_freq, layout="half", magnitude=1.0, transposed=False):
    """x [tokens, heads, dim]: its first 2 len(inv_freq) elements turned."""
    x = f64(x)
    y = x.copy()
    n = len(inv_freq)
    if n == 0:
        return y
    angle = f64(positions)[:, None, None] * f64(inv_freq) * (-1.0 if transposed else 1.0)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
    ia, ib = ((slice(0, n), slice(n, 2 * n)) if layout == "half"
              else (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def head_rstd(x, eps):
    x = f64(x)
    return 1.0 / np.sqrt((x * x).mean(-1) + eps)


def norm_rope(x, weight, positions, inv_freq, layout="half", magnitude=1.0, eps=1e-6):
    """One of the two tensors' way: (output, rstd [tokens, heads])."""
    r = head_rstd(x, eps)
    return rope(f64(x) * r[..., None] * f64(weight), positions, inv_freq, layout, magnitude), r


def norm_rope_bwd(x, weight, rstd, dy, positions, inv_freq, layout="half", magnitude=1.0):
    """(dx, dweight) from the forward's input and rstd."""
    d = rope(dy, positions, inv_freq, layout, magnitude, transposed=True)
    r = f64(rstd)[..., None]
    n = f64(x) * r
    u = d * f64(weight)
    return r * (u - n * (u * n).mean(-1, keepdims=True)), (d * n).sum((0, 1))


def append(cache, new, slots):
    """The cache [pages, page size, heads, dim] with new[t] at slot slots[t]."""
    out = f64(cache).copy()
    pages, size = out.shape[:2]
    for t, slot in enumerate(slots):
        if 0 <= slot < pages * size:
            out[slot // size, slot % size] = new[t]
    return out


def paged_attention(q, k_cache, v_cache, pages, q_start, kv_len, scale, window=0):
    """(out, lse): attention of the tokens of each sequence, the last of its
    kv_len positions, to the positions up to their own (the last `window` of them);
    rows that see nothing 0 and -inf, those behind the last sequence NaN (not
    written), those that see a page outside the cache NaN."""
    q, k_cache, v_cache = f64(q), f64(k_cache), f64(v_cache)
    tokens, heads, dim = q.shape
    n_pages, size, kv_heads = k_cache.shape[:3]
    out, lse = np.full(q.shape, np.nan), np.full((tokens, heads), np.nan)
    for b, kv in enumerate(kv_len):
        new = q_start[b + 1] - q_start[b]
        for i in range(new):
            t, last = q_start[b] + i, kv - new + i
            at = np.arange(max(0, last - window + 1) if window else 0, max(0, last + 1))
            page = np.asarray(pages[b])[at // size] if len(at) else at
            missing = ((page < 0) | (page >= n_pages)).any()
            page = np.clip(page, 0, max(0, n_pages - 1))
            for h in range(heads):
                g = h // (heads // kv_heads)
                if len(at) == 0:
                    out[t, h], lse[t, h] = 0.0, -np.inf
                    continue
                if missing:
                    continue
                with np.errstate(all="ignore"):
                    x = scale * (k_cache[page, at % size, g] @ q[t, h])
                    m = x.max()
                    if m == -np.inf:
                        out[t, h], lse[t, h] = 0.0, -np.inf
                        continue
                    p = np.exp(x - m)
                    out[t, h] = (p[:, None] * v_cache[page, at % size, g]).sum(0) / p.sum()
                    lse[t, h] = m + np.log(p.sum())
    return out, lse
