"""Error bounds of the operators on logits, element by element, counted from the
kernels' roundings.  For rows of one batch (at most 8128 columns, whatever their
alignment), whose lanes take their own maximum as reference: every exponent is
then formed about a value that is at least as large.

E = 2^-24, half a step of fp32; y = (z - max) / T <= 0 an element's exponent.  An
exponential is off by 2 E (one unit), by E |y| for every rounding of its argument
or of the factor log2(e) / T, and is 0 below 2^-126.  T is taken as fp32 holds it.
"""
import numpy as np
import torch

from oracle import reference as ref

E = 2.0 ** -24
FLUSH = 2.0 ** -126
ONE_BATCH = 8128


def stats(z: np.ndarray, temperature: float) -> dict:
    """Per row, [rows, 1]: maximum m, sum s, mean |y| and |y|^2 under p; y, p and
    ln p of all elements (0, 0, -inf where z is -inf)."""
    assert z.shape[1] <= ONE_BATCH
    m, s, lp = ref._log_softmax(z, temperature)
    with np.errstate(all="ignore"):
        y = np.where(z == -np.inf, 0.0, (m - z) / temperature)
        p = np.where(z == -np.inf, 0.0, np.exp(lp))
    return {"m": m, "s": s, "y": y, "p": p, "lp": lp,
            "mean": (p * y).sum(1, keepdims=True), "mean2": (p * y * y).sum(1, keepdims=True)}


def sum_error(st: dict) -> np.ndarray:
    """Relative error of S.  A lane adds its 32 terms in two chains of 16 and joins
    them: 17 E; a term has its exponential, the factor and the exponent's own
    rounding, and is brought to the row's maximum by another exponential with its
    exponent's rounding: 2 + 2 E and 3 E |y|.  What follows is in 64 bits."""
    return E * (17 + 4 + 3 * st["mean"])


def entropy_error(st: dict) -> np.ndarray:
    """Absolute error of H = ln S - t / S, t the sum of e^y y: the terms of t have
    those of S and the rounding of their sum and of y itself (two: 2 E |y|)."""
    t = E * ((17 + 4 + 4 + 2) * st["mean"] + 3 * st["mean2"])
    return sum_error(st) * (1 + st["mean"]) + t


def logprob_gradient_bound(z, tokens, dlogp, dentropy, temperature) -> np.ndarray:
    """(sum_t g_t - p (G + h (ln p + H))) / T in fp32, before its rounding to the
    output's type.  e^y: its argument has three roundings.  The weight is
    A + B y: A = G + h (H - ln S) three roundings of what it sums, the error of H,
    ln S (logf's two units, 4 E, and S's error); B four.  1 / (T S), stored S: S's error and
    four roundings.  A token's own g: four, its sum with the rest one."""
    z, dlogp = np.asarray(z, np.float64), np.asarray(dlogp, np.float64)
    st = stats(z, temperature)
    tokens = np.asarray(tokens)
    live = (tokens >= 0) & (tokens < z.shape[1])
    g = np.abs((dlogp * live).sum(1, keepdims=True))
    y, p = st["y"], st["p"]
    rel = E * (3 * y + 2 + 5) + sum_error(st)
    weight, extra = g, 3 * E * g
    if dentropy is not None:
        h = np.abs(np.asarray(dentropy, np.float64))[:, None]
        ln_s = np.log(st["s"])
        ent = (p * -np.where(p > 0, st["lp"], 0.0)).sum(1, keepdims=True)
        part = h * (ent + ln_s)
        extra = (3 * E * (g + part) + h * (entropy_error(st) + E * ent + 4 * E * ln_s
                                           + sum_error(st)) + h * y * 8 * E)
        weight = g + part + h * y
    own = np.zeros(z.shape)
    for r, c in zip(*np.nonzero(live)):
        own[r, tokens[r, c]] += abs(dlogp[r, c])
    bound = p * (weight * rel + extra) + own * 4 * E + (p * weight + own) * E
    return (bound + FLUSH * (weight + 1)) / temperature + FLUSH


def distill_gradient_bound(z, ids, teacher, dloss, tail, temperature) -> np.ndarray:
    """dloss / T (Q p - q) in fp32, before its rounding to the output's type: p as
    above with an exponential of 3 E and six factors, q by itself.  q: e^t with a
    tail (3 E); without, the exponent's two roundings, its sum over K entries
    (their own errors, log2 K additions in a wave and 3 between waves) and a
    division.  An entry of a column that others name too: an addition more.
    Outside the entries, with a tail: w (share Q - rest), w the softmax there,
    share and rest in 64 bits of S and of the tail's sum."""
    z = np.asarray(z, np.float64)
    ids, t = np.asarray(ids), np.asarray(teacher, np.float64)
    rows, cols = z.shape
    st = stats(z, temperature)
    g = np.abs(np.asarray(dloss, np.float64)) / temperature
    bound = np.zeros(z.shape)
    for r in range(rows):
        live = ids[r] >= 0
        if not live.any() or g[r] == 0.0 or st["s"][r, 0] == 0.0:
            continue
        at, x = ids[r][live], t[r][live]
        if tail:
            q, err, rest = np.exp(x), np.full(x.shape, 3.0), max(0.0, 1.0 - np.exp(x).sum())
        else:
            yt = (x.max() - x) / temperature
            q = np.exp(-yt)
            q, rest = q / q.sum(), 0.0
            err = (2 * yt + 3) + (q * (2 * yt + 3)).sum() + np.ceil(np.log2(ids.shape[1])) + 3 + 1
        named = np.zeros(cols, bool)
        named[at] = True
        s_err = sum_error(st)[r, 0]
        y, p = st["y"][r], st["p"][r]
        others = ~named & (z[r] != -np.inf)
        if tail and not others.any():
            rest = 0.0
        mass = q.sum() + rest
        p_err = mass * p * (E * (3 * y + 3 + 6) + s_err)
        q_err, count = np.zeros(cols), np.bincount(at, minlength=cols)
        np.add.at(q_err, at, q * E * (err + count[at]))
        q_all = np.bincount(at, weights=q, minlength=cols)
        row = np.where(named, p_err + q_err + 2 * E * (mass * p + q_all), p_err)
        if tail and others.any():
            # The tail's own maximum, sum and softmax.
            o = np.where(others, z[r], -np.inf)[None]
            ts = stats(o, temperature)
            w, share = ts["p"][0], p[others].sum()
            t_err = sum_error(ts)[0, 0]
            grad = abs(mass * share - rest)
            tail_row = w * (share * mass * (s_err + t_err)
                            + grad * (E * (3 * ts["y"][0] + 2 + 6) + t_err))
            row = np.where(named, row, tail_row)
        bound[r] = g[r] * (row + FLUSH * (mass + 2)) + FLUSH
    return bound


def rounded(bound: np.ndarray, want: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    """The bound with the rounding of the value that is off by as much."""
    if dtype == torch.float32:
        return bound
    return bound + (np.abs(want) + bound) * torch.finfo(dtype).eps / 2
