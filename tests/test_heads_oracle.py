"""The oracle of the operators on heads and paged caches: torch's autograd for the
gradients, complex numbers for the rotation, scaled_dot_product_attention for the
attention, and differences."""
import math

import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from oracle import heads as ref


def inputs(tokens=3, heads=2, dim=12, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((tokens, heads, dim), generator=g, dtype=torch.float64), g


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("pairs", [0, 1, 4, 6])
def test_rotation_is_a_complex_product(layout, pairs):
    x, g = inputs()
    pos = torch.tensor([0, 5, -100000])
    freq = torch.rand(pairs, generator=g, dtype=torch.float64)
    got = ref.rope(x.numpy(), pos.numpy(), freq.numpy(), layout, 1.5)
    a, b = ((x[..., :pairs], x[..., pairs:2 * pairs]) if layout == "half"
            else (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]))
    z = torch.complex(a, b) * torch.polar(torch.full((3, 1, pairs), 1.5, dtype=torch.float64),
                                          (pos.double()[:, None] * freq)[:, None])
    parts = (z.real, z.imag)
    turned = torch.cat(parts, -1) if layout == "half" else torch.stack(parts, -1).flatten(-2)
    np.testing.assert_allclose(got, torch.cat((turned, x[..., 2 * pairs:]), -1).numpy(), atol=1e-13)
    back = ref.rope(got, pos.numpy(), freq.numpy(), layout, 1 / 1.5, transposed=True)
    np.testing.assert_allclose(back, x.numpy(), atol=1e-13)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradients_of_the_normed_rotation(layout):
    x, g = inputs(5, 3, 10)
    w = torch.randn(10, generator=g, dtype=torch.float64)
    dy = torch.randn(x.shape, generator=g, dtype=torch.float64)
    pos, freq = torch.arange(5).numpy() * 7, np.array([1.0, 0.3, 0.01])

    def forward(x, w):
        n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        i, j = (slice(0, 3), slice(3, 6)) if layout == "half" else (slice(0, 6, 2), slice(1, 6, 2))
        angle = torch.from_numpy(pos[:, None, None] * freq)
        y = n.clone()
        y[..., i] = 0.8 * (n[..., i] * angle.cos() - n[..., j] * angle.sin())
        y[..., j] = 0.8 * (n[..., j] * angle.cos() + n[..., i] * angle.sin())
        return y

    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    (forward(a, b) * dy).sum().backward()
    got, r = ref.norm_rope(x.numpy(), w.numpy(), pos, freq, layout, 0.8)
    np.testing.assert_allclose(got, forward(x, w).numpy(), atol=1e-12)
    dx, dw = ref.norm_rope_bwd(x.numpy(), w.numpy(), r, dy.numpy(), pos, freq, layout, 0.8)
    np.testing.assert_allclose(dx, a.grad.numpy(), atol=1e-12)
    np.testing.assert_allclose(dw, b.grad.numpy(), atol=1e-12)
    # Against differences.
    step = torch.randn(x.shape, generator=g, dtype=torch.float64) * 1e-6
    change = ((forward(x + step, w) - forward(x - step, w)) * dy).sum() / 2
    assert abs(change.item() - (dx * step.numpy()).sum()) < 1e-13


def test_append_leaves_padding_out():
    cache, new = np.zeros((2, 3, 1, 2)), np.arange(8.0).reshape(4, 1, 2)
    got = ref.append(cache, new, [4, -1, 6, 0])
    assert got[1, 1, 0].tolist() == [0, 1] and got[0, 0, 0].tolist() == [6, 7]
    assert np.abs(got).sum() == 14


@pytest.mark.parametrize("window", [0, 3])
def test_attention_of_a_chunk(window):
    q, g = inputs(7, 4, 8)
    size, news, kvs = 4, [2, 4, 1], [9, 4, 0]
    k, v = (torch.randn((6, size, 2, 8), generator=g, dtype=torch.float64) for _ in range(2))
    table = np.array([[5, 0, 3], [2, -1, -1], [-1, -1, -1]])
    out, lse = ref.paged_attention(q.numpy(), k.numpy(), v.numpy(), table, [0, 2, 6, 7], kvs, 0.4,
                                   window)
    first = 0
    for b in range(2):
        new, kv = news[b], kvs[b]
        at = torch.from_numpy(table[b][: -(-kv // size)])
        ks, vs = (c[at].flatten(0, 1)[:kv].transpose(0, 1).repeat_interleave(2, 0) for c in (k, v))
        row = torch.arange(new)[:, None] + kv - new
        mask = torch.arange(kv) <= row
        if window:
            mask &= torch.arange(kv) > row - window
        qs = q[first:first + new].transpose(0, 1)
        want = torch.nn.functional.scaled_dot_product_attention(
            qs[None], ks[None], vs[None], attn_mask=mask, scale=0.4)[0]
        np.testing.assert_allclose(out[first:first + new], want.transpose(0, 1).numpy(),
                                   atol=1e-12)
        x = (0.4 * qs @ ks.transpose(1, 2)).masked_fill(~mask, -math.inf)
        np.testing.assert_allclose(lse[first:first + new], x.logsumexp(-1).T.numpy(), atol=1e-12)
        first += new
    assert (out[6] == 0).all() and (lse[6] == -math.inf).all()


def test_frequencies():
    plain, one = hip_lib.rope_frequencies(64, 10000.0)
    assert one == 1.0 and plain[0] == 1.0
    np.testing.assert_allclose(plain[-1], 10000.0 ** (-62 / 64), rtol=1e-6)
    linear, _ = hip_lib.rope_frequencies(64, scaling="linear", factor=4.0)
    np.testing.assert_allclose(linear, plain / 4, rtol=1e-6)
    ntk, _ = hip_lib.rope_frequencies(64, scaling="ntk", factor=4.0)
    np.testing.assert_allclose([ntk[0], ntk[-1]], [1.0, plain[-1] / 4], rtol=1e-6)
    yarn, magnitude = hip_lib.rope_frequencies(64, scaling="yarn", factor=4.0,
                                               original_length=2048)
    turns = plain * 2048 / (2 * math.pi)
    assert torch.equal(yarn[turns > 32], plain[turns > 32])
    np.testing.assert_allclose(yarn[turns < 1], plain[turns < 1] / 4, rtol=1e-6)
    assert magnitude == pytest.approx(1 + 0.1 * math.log(4))
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, base=0.0), dict(rot=8, factor=-1.0),
                dict(rot=8, scaling="other"), dict(rot=8, scaling="yarn", low=2.0, high=2.0)):
        with pytest.raises(ValueError):
            hip_lib.rope_frequencies(**bad)
