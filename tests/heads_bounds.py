"""Error bounds of the operators on heads, element by element, counted from the
kernels' roundings.  E = 2^-24, half a step of fp32."""
import numpy as np
import torch

from oracle import heads as ref

E = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def angle_error(positions, inv_freq) -> np.ndarray:
    """Absolute error of a sine or cosine [tokens, pairs].  What is left of the
    angle, at most pi/4, has three roundings (to fp32, of 2 pi, their product): at
    most 2.4 E.  The polynomials: their last addition, products before it of at
    most 2 E together, the remainder of the series (2e-9, 0.04 E).  The turns, in
    64 bits: two roundings, 2^-52 of them, times 2 pi: |angle| 2^-52."""
    turned = np.abs(np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64))
    return (2.4 + 1 + 2 + 0.1) * E + turned * 2.0 ** -52


def rotated(x, err, positions, inv_freq, layout, magnitude, transposed=False):
    """Bound of rope(x) in fp32 where x is off by err: magnitude times each element
    of its pair times the angle's error and the magnitude's rounding; the products'
    rounding and the sum's."""
    x = np.abs(np.asarray(x, np.float64))
    err = np.broadcast_to(err, x.shape)
    n = len(inv_freq)
    out = err.copy()
    if n == 0:
        return out
    ia, ib = ((slice(0, n), slice(n, 2 * n)) if layout == "half"
              else (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    both = x[..., ia] + x[..., ib]
    both_err = err[..., ia] + err[..., ib]
    a = angle_error(positions, inv_freq)[:, None]
    pair = abs(magnitude) * (both * (a + 3 * E) * (1 + E) + both_err * (1 + a))
    out[..., ia] = pair
    out[..., ib] = pair
    return out


def rounded(bound, want, dtype):
    """The bound with the rounding to the output's type of a value off by it."""
    if dtype == "f32":
        return bound + 1e-38
    return bound + (np.abs(want) + bound) * torch.finfo(DTYPES[dtype]).eps / 2 + 1e-38


def chain(dim: int) -> float:
    """Roundings of a sum over a head's elements: at most 16 in a lane (two units
    of 8, or four pairs) and 6 between lanes."""
    return min(dim, 16) + 6


def rstd_error(dim: int) -> float:
    """Relative error of (mean x^2 + eps)^(-1/2): the sum's (a term's product is
    fused with its addition), the division by dim, the addition of eps: half of
    them; the square root's and the reciprocal's own (one each)."""
    return ((chain(dim) + 2) / 2 + 2) * E


def norm_rope(x, weight, positions, inv_freq, layout, magnitude, eps):
    x, w = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    n = x * ref.head_rstd(x, eps)[..., None] * w
    return rotated(n, np.abs(n) * (rstd_error(x.shape[-1]) + 2 * E), positions, inv_freq, layout,
                   magnitude)


def norm_rope_bwd(x, weight, rstd, dy, positions, inv_freq, layout, magnitude):
    """(bound of dx, of dweight) in fp32.  n = x r: one rounding; u = d w another
    beside d's own error; the mean: its terms' errors, the chain and two roundings;
    dx: the product with the mean (fused) and with r.  dweight: as many additions
    as there are tokens and heads at most, each fused with its product."""
    x, w, r = (np.asarray(t, np.float64) for t in (x, weight, rstd))
    r = r[..., None]
    dim = x.shape[-1]
    d = ref.rope(dy, positions, inv_freq, layout, magnitude, transposed=True)
    d_err = rotated(dy, 0.0, positions, inv_freq, layout, magnitude)
    n = np.abs(x * r)
    u, u_err = np.abs(d * w), d_err * np.abs(w) + np.abs(d * w) * E
    un = u * n
    mean = un.mean(-1, keepdims=True)
    mean_err = (u_err * n + un * E).mean(-1, keepdims=True) + mean * (chain(dim) + 2) * E
    dx = r * (u_err + n * mean_err + (u + 3 * n * mean) * E) * (1 + 2 * E) \
        + r * (u + n * mean) * E
    dn = np.abs(d) * n
    dw = (d_err * n + dn * E).sum((0, 1)) + (x.shape[0] * x.shape[1] + 2) * E * dn.sum((0, 1))
    return dx, dw


RAISES = 16  # times that a row's maximum is raised, waves and parts joined


def attention(q, k_cache, v_cache, pages, q_start, kv_len, scale, window=0):
    """(bound of out in fp32 before its rounding, of lse).  A score: dim products,
    exact in fp32, each addition off by at most a step (2 E).  A weight: the score's
    error; the exponent's factor, base, and their fused product, each E of it; the
    exponential, 2 E; the same for each time that it is rescaled; its rounding to
    bf16, 2^-8.  Sums over the positions: a step (2 E) each.  Weights below the
    smallest normal number count as 0."""
    q, k_cache, v_cache = (np.asarray(t, np.float64) for t in (q, k_cache, v_cache))
    tokens, heads, dim = q.shape
    size, kv_heads = k_cache.shape[1:3]
    out, lse = np.zeros(q.shape), np.zeros((tokens, heads))
    for b, kv in enumerate(kv_len):
        new = q_start[b + 1] - q_start[b]
        for i in range(new):
            t, last = q_start[b] + i, kv - new + i
            at = np.arange(max(0, last - window + 1) if window else 0, max(0, last + 1))
            if len(at) == 0:
                continue
            page = np.asarray(pages[b])[at // size]
            if (page < 0).any() or (page >= k_cache.shape[0]).any():
                continue
            for h in range(heads):
                g = h // (heads // kv_heads)
                k, v = k_cache[page, at % size, g], np.abs(v_cache[page, at % size, g])
                with np.errstate(all="ignore"):
                    x = scale * (k @ q[t, h])
                # A score of -inf makes a weight of exactly 0, which adds nothing
                # and no error; a row of nothing else is written as it is, and one
                # of +inf or NaN is NaN: no bound is asked for.
                live = x > -np.inf
                k, v, x = k[live], v[live], x[live]
                if not live.any() or not np.isfinite(x).all():
                    continue
                w = np.exp(x - x.max())
                total = w.sum()
                w /= total
                big = np.abs(x).max()
                d = (scale * 2 * dim * E * (np.abs(k) @ np.abs(q[t, h]))
                     + 4 * E * (np.abs(x) + big) + 2 * E + RAISES * (4 + 2 * big) * E)
                wd, n = (w * d).sum(), 2 * (len(at) + RAISES) * E
                out[t, h] = ((w * (2.0 ** -8 + d + n))[:, None] * v).sum(0) \
                    + (w[:, None] * v).sum(0) * (wd + n + 3 * E) + 1e-36 * v.max()
                lse[t, h] = wd + n + 4 * E * np.log(total) + 3 * E * (big + np.log(total))
    return out, lse
