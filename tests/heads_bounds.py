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
