"""Inputs and error bounds shared by the tests of the operators on logits."""
import math

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 2.0 ** -24  # half a step of fp32


def half_step(dtype: str) -> float:
    return torch.finfo(DTYPES[dtype]).eps / 2


def sum_error(cols: int) -> float:
    """Relative error of S = sum 2^x: an addition of positive terms makes EPS,
    at most 16 in a batch's two partial sums and one per batch of 8192 columns
    (a handful more where batches are smaller and lanes are joined: 32); a term
    has its own, 2 EPS of the exponential and 3 roundings of x (difference,
    product, factor), 3 EPS ln 2 |x|, and sum p |x| <= log2(cols) + 1 about the
    maximum, plus 8 where a lane's reference is that far below it."""
    return (16 + cols / 2048 + 32 + 2 + 3 * math.log(2) * (math.log2(cols + 1) + 9)) * EPS


def entropy_error(cols: int) -> float:
    """Absolute error of ln S - ln 2 t / S, t = sum 2^x x: that of ln S, and
    every term of t off by the relative error of a sum's term, times
    sum p |x| <= log2(cols) + 9 bits."""
    return sum_error(cols) * (2 + math.log(2) * (math.log2(cols + 1) + 9))


def generator(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def make_logits(rows: int, cols: int, dtype: str, seed: int) -> torch.Tensor:
    g = generator(seed)
    z = torch.randn((rows, cols), generator=g) * 2.0
    for _ in range(6):
        z[torch.arange(rows), torch.randint(0, cols, (rows,), generator=g)] += 9.0
    return z.to(DTYPES[dtype])


def special_rows(cols: int, dtype: str, seed: int) -> tuple[torch.Tensor, list[str]]:
    """One row of each kind that a mask, an overflow or a tie can make."""
    base = make_logits(1, cols, dtype, seed)[0]
    low = torch.finfo(DTYPES[dtype]).min
    rows, names = [], []

    def add(name, edit):
        z = base.clone()
        edit(z)
        rows.append(z)
        names.append(name)

    add("plain", lambda z: None)
    add("empty", lambda z: z.fill_(-math.inf))
    add("all lowest", lambda z: z.fill_(low))
    add("lowest and -inf", lambda z: (z.fill_(low), z[::2].fill_(-math.inf)))
    add("masked by -inf", lambda z: z[cols // 3:].fill_(-math.inf))
    add("masked by lowest", lambda z: z[cols // 3:].fill_(low))
    add("one column left", lambda z: (z.fill_(-math.inf), z[cols // 2:cols // 2 + 1].fill_(3.0)))
    add("constant", lambda z: z.fill_(1.25))
    add("two values", lambda z: (z.fill_(-2.0), z[::3].fill_(0.5)))
    add("zeros of both signs", lambda z: (z.zero_(), z[::2].fill_(-0.0)))
    add("far from 0", lambda z: z.add_(1.0e4))
    add("huge", lambda z: z.mul_(2.0 ** 100))
    add("rising", lambda z: z.copy_(torch.linspace(-30, 30, cols)))
    add("falling", lambda z: z.copy_(torch.linspace(40, -90, cols)))
    add("peak last", lambda z: z[-1:].fill_(60.0))
    add("peak first", lambda z: z[:1].fill_(60.0))
    add("NaN", lambda z: z[cols // 2:cols // 2 + 1].fill_(math.nan))
    add("+inf", lambda z: z[-1:].fill_(math.inf))
    add("NaN and -NaN", lambda z: (z[-1:].fill_(math.nan), z[:1].fill_(math.nan).neg_()))
    return torch.stack(rows), names


def placed(t: torch.Tensor, gpu, offset: int = 0, gap: int = 0, fill=math.nan) -> torch.Tensor:
    """t on the GPU as a view `offset` elements into its allocation and with
    `gap` elements between rows, all of which hold `fill`."""
    rows, cols = t.shape
    flat = torch.full((offset + rows * (cols + gap) + 16,), fill, dtype=t.dtype, device=gpu)
    view = flat[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    view.copy_(t)
    return view


def as64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().double().numpy()


def assert_within(got, want, bound, what: str) -> None:
    """|got - want| <= bound where want is finite; elsewhere the same.  A value
    beyond fp32's largest has no other rounding to fp32 than the infinity."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    want = np.where(np.abs(want) >= 2.0 ** 128, np.copysign(np.inf, want), want)
    bound = np.broadcast_to(np.asarray(bound, np.float64), want.shape)
    assert got.shape == want.shape, f"{what}: {got.shape} {want.shape}"
    fine = np.isfinite(want)
    odd = ~fine & ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not odd.any(), f"{what}: {got[odd][:4]} for {want[odd][:4]} at {np.argwhere(odd)[:4]}"
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
        bad = fine & ~(off <= bound)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} values too far off; at {at} got {got[at]!r}, "
                             f"want {want[at]!r}, bound {bound[at]:.3g}")
