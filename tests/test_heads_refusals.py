"""What the operators on heads and paged caches refuse, on the host and before any
HIP call: the C entry points by status, the Python functions by exception.  No GPU."""
import ctypes
import math

import pytest
import torch

from credit_amd import hip_lib
from credit_amd.hip_lib import CreditHeads, CreditPages, CreditRotation

A, B, C, D, W = (n << 32 for n in range(1, 6))  # never dereferenced
NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, CONFIG = -1, -2, -3, -4, -5, -8
TYPES = ("f32", "bf16")


def heads(at, token=512, head=64, n=8):
    return CreditHeads(at, token, head, n)


def rotation(positions=W, inv_freq=W, rot=64, interleaved=0, magnitude=1.0):
    return CreditRotation(positions, inv_freq, rot, interleaved, magnitude)


def pages(at, page=8192, slot=512, head=64, n=100, size=16, n_heads=8):
    return CreditPages(at, page, slot, head, n, size, n_heads)


def calls():
    return {
        "rope": dict(q=heads(A), k=heads(B), rotation=rotation(), q_out=heads(C),
                     k_out=heads(D), tokens=10, dim=64, transposed=0, cfg=None),
        "qk_norm_rope_fwd": dict(q=heads(A), k=heads(B), q_weight=W, k_weight=W,
                                 rotation=rotation(), q_out=heads(C), k_out=heads(D), rstd=W,
                                 tokens=10, dim=64, eps=1e-6, cfg=None),
        "qk_norm_rope_bwd": dict(q=heads(A), k=heads(B), q_weight=W, k_weight=W,
                                 rotation=rotation(), rstd=W, dq_out=heads(C), dk_out=heads(D),
                                 dq=heads(C), dk=heads(D), dq_weight=W, dk_weight=W, tokens=10,
                                 dim=64, cfg=None),
        "paged_append": dict(k=heads(A), v=heads(B), q=heads(6 << 32), k_weight=W, q_weight=W,
                             rotation=rotation(), slots=W, k_cache=pages(C), v_cache=pages(D),
                             q_out=heads(7 << 32), tokens=10, dim=64, eps=1e-6, cfg=None),
        "paged_attention": dict(q=heads(A), k_cache=pages(C), v_cache=pages(D), pages=W,
                                pages_ld=20, cols=20, q_start=W, kv_len=W, out=heads(B), lse=W,
                                tokens=10, batch=3, dim=64, scale=0.125, window=0, cfg=None),
    }


def call(lib, op, dtype, **edit):
    args = {**calls()[op], **edit}
    passed = [ctypes.byref(v) if isinstance(v, ctypes.Structure) else v for v in args.values()]
    return getattr(lib, f"credit_{op}_{dtype}")(*passed)


def types(op):
    return ("bf16",) if op.startswith("paged") else TYPES


ROTATED = ("rope", "qk_norm_rope_fwd", "qk_norm_rope_bwd", "paged_append")


@pytest.mark.parametrize("op", calls())
def test_sizes_and_pointers(lib, op):
    for dtype in types(op):
        wide = 600 if op != "paged_attention" else 264
        for edit, status in ((dict(tokens=-1), SHAPE), (dict(tokens=1 << 31), SHAPE),
                             (dict(dim=0), SHAPE), (dict(dim=wide), SHAPE)):
            assert call(lib, op, dtype, **edit) == status, edit
        for name, value in calls()[op].items():
            if isinstance(value, CreditHeads):
                optional = {"rope": ("k", "k_out"), "paged_append": ("q", "q_out")}.get(op, ())
                assert call(lib, op, dtype, **{name: None}) == NULL, name
                for bad, status in ((heads(None), NULL), (heads(A, token=-1), SHAPE),
                                    (heads(A, head=-64), SHAPE), (heads(A, n=0), SHAPE),
                                    (heads(A + 1), ALIGN), (heads(A, token=1 << 60), SHAPE)):
                    assert call(lib, op, dtype, **{name: bad}) == status, (name, optional)
                assert hip_lib.last_error()
            elif isinstance(value, CreditPages):
                for bad, status in ((None, NULL), (pages(None), NULL), (pages(A, n=-1), SHAPE),
                                    (pages(A, size=0), SHAPE), (pages(A, n_heads=0), SHAPE),
                                    (pages(A, page=-1), SHAPE), (pages(A, slot=60), SHAPE),
                                    (pages(A, page=8000), SHAPE), (pages(A + 1), ALIGN)):
                    assert call(lib, op, dtype, **{name: bad}) == status, (name, status)
            elif value == W and name not in ("rstd", "lse", "k_weight", "q_weight", "pages"):
                assert call(lib, op, dtype, **{name: None}) == NULL, name
                assert call(lib, op, dtype, **{name: W + 1}) == ALIGN, name


@pytest.mark.parametrize("op", ROTATED)
def test_rotations(lib, op):
    for edit, status in ((dict(rot=3), SHAPE), (dict(rot=-2), SHAPE), (dict(rot=66), SHAPE),
                         (dict(positions=None), NULL), (dict(inv_freq=None), NULL),
                         (dict(positions=W + 4), ALIGN), (dict(inv_freq=W + 2), ALIGN),
                         (dict(magnitude=math.nan), CONFIG), (dict(magnitude=math.inf), CONFIG)):
        assert call(lib, op, types(op)[-1], rotation=rotation(**edit)) == status, edit


@pytest.mark.parametrize("op", calls())
def test_variants_and_cfg(lib, op):
    for variant, split, workspace, status in ((1, 0, None, UNSUPPORTED), (3, 2, None, UNSUPPORTED),
                                              (9, 0, None, CONFIG), (0, 2, None, UNSUPPORTED),
                                              (0, 65, None, CONFIG), (0, 0, W + 16, WORKSPACE)):
        cfg = hip_lib.CreditCfg(None, variant, split, workspace, 0)
        assert call(lib, op, types(op)[-1], cfg=ctypes.byref(cfg)) == status


@pytest.mark.parametrize("op", ["qk_norm_rope_fwd", "qk_norm_rope_bwd"])
def test_norms(lib, op):
    for dtype in TYPES:
        for name in ("q_weight", "k_weight"):
            assert call(lib, op, dtype, **{name: None}) == NULL
            assert call(lib, op, dtype, **{name: W + 1}) == ALIGN
        assert call(lib, op, dtype, rstd=W + 2) == ALIGN
    assert call(lib, "qk_norm_rope_bwd", "f32", rstd=None) == NULL
    for eps in (-1.0, math.nan, math.inf):
        assert call(lib, "qk_norm_rope_fwd", "f32", eps=eps) == CONFIG


def test_outputs_that_overlap(lib):
    """bf16, 10 tokens of 8 heads of 64: 10240 bytes."""
    def rope(**edit):
        return call(lib, "rope", "bf16", **edit)
    assert rope(q_out=heads(A + 2)) == CONFIG
    assert rope(q_out=heads(A + 128)) == CONFIG
    assert rope(q_out=heads(A, token=520)) == CONFIG
    assert rope(q_out=heads(B)) == CONFIG and rope(k_out=heads(A)) == CONFIG
    assert rope(q_out=heads(D)) == CONFIG
    assert rope(q_out=heads(C, head=32)) == SHAPE  # heads that overlap each other
    assert rope(q_out=heads(C, token=64)) == SHAPE
    assert rope(q_out=heads(C, n=7)) == SHAPE
    assert call(lib, "rope", "bf16", k=None) == NULL and rope(k_out=None) == NULL
    bwd = dict(dq=heads(A + 2))
    assert call(lib, "qk_norm_rope_bwd", "bf16", **bwd) == CONFIG
    # In place of dq_out, while q lies a little before it.
    assert call(lib, "qk_norm_rope_bwd", "bf16", q=heads(C - 128)) == CONFIG
    assert call(lib, "qk_norm_rope_bwd", "bf16", dq=heads(B)) == CONFIG
    assert call(lib, "qk_norm_rope_bwd", "bf16", dq=heads(D)) == CONFIG


def test_appends(lib):
    def append(**edit):
        return call(lib, "paged_append", "bf16", **edit)
    assert append(k_cache=pages(C, n_heads=4)) == SHAPE
    assert append(k_cache=pages(C, n=99)) == SHAPE
    assert append(v_cache=pages(D, size=8)) == SHAPE
    assert append(v_cache=pages(C + 128)) == CONFIG
    assert append(k=heads(C + 4096)) == CONFIG
    assert append(q_out=heads(C + 4096)) == CONFIG
    assert append(q_out=heads(A)) == CONFIG and append(q_out=heads(B)) == CONFIG
    assert append(q=None) == NULL and append(q_out=None) == NULL
    assert append(q=None, q_out=None) == CONFIG  # its weight is there
    assert append(k_weight=W + 1) == ALIGN
    assert append(eps=-1.0) == CONFIG


def test_attentions(lib):
    def attend(**edit):
        return call(lib, "paged_attention", "bf16", **edit)
    for edit, status in ((dict(dim=60), SHAPE), (dict(batch=-1), SHAPE),
                         (dict(batch=(1 << 20) + 1), SHAPE), (dict(q=heads(A, n=9)), SHAPE),
                         (dict(q=heads(A, n=12), out=heads(B, n=12)), SHAPE),
                         (dict(k_cache=pages(C, n=99)), SHAPE),
                         (dict(v_cache=pages(D, size=8)), SHAPE),
                         (dict(v_cache=pages(D, n_heads=4)), SHAPE), (dict(cols=-1), SHAPE),
                         (dict(pages_ld=19), SHAPE), (dict(pages=None), NULL),
                         (dict(pages=W + 2), ALIGN), (dict(lse=W + 2), ALIGN),
                         (dict(cols=1 << 27, pages_ld=1 << 27), SHAPE),
                         (dict(scale=0.0), CONFIG), (dict(scale=-1.0), CONFIG),
                         (dict(scale=math.nan), CONFIG), (dict(scale=math.inf), CONFIG),
                         (dict(window=-1), CONFIG), (dict(q=heads(A + 2)), ALIGN),
                         (dict(q=heads(A, token=516)), ALIGN), (dict(out=heads(B + 8)), ALIGN),
                         (dict(k_cache=pages(C + 8)), ALIGN),
                         (dict(k_cache=pages(C, page=8196)), ALIGN),
                         (dict(v_cache=pages(D, slot=516, page=8256)), ALIGN),
                         (dict(out=heads(A)), CONFIG), (dict(out=heads(C + 4096)), CONFIG),
                         (dict(tokens=1 << 28), SHAPE)):
        assert attend(**edit) == status, (edit, hip_lib.last_error())


def test_nothing_to_do(lib):
    for op in ("rope", "qk_norm_rope_fwd", "paged_append", "paged_attention"):
        nothing = {name: heads(None) for name, v in calls()[op].items()
                   if isinstance(v, CreditHeads)}
        assert call(lib, op, "bf16", tokens=0, **nothing) == 0
    assert call(lib, "paged_attention", "bf16", batch=0, pages=None, q_start=None,
                kv_len=None) == 0


def test_workspace_sizes(lib):
    assert hip_lib.workspace_bytes("qk_norm_rope_bwd", 100, 128) > 1024 * 128 * 4
    size = hip_lib.paged_attention_workspace_bytes
    assert size(1, 1, 32, 8, 128, 8192) > size(1, 1, 32, 8, 128, 1024) > 0
    assert size(1, 1, 32, 8, 128, 64) == 0 and size(0, 1, 32, 8, 128, 8192) == 0
    assert size(1, 1, 32, 5, 128, 8192) == 0 and size(8192, 1, 32, 8, 128, 8192) == 0


def test_python_refuses_before_the_library():
    x, pos, freq = torch.zeros(4, 2, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    cache = torch.zeros(3, 16, 2, 8)
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="q"):
        hip_lib.rope(x.half(), pos, freq, x)
    with pytest.raises(ValueError, match="heads"):
        hip_lib.rope(x[0], pos, freq, x)
    with pytest.raises(ValueError, match="on a GPU"):
        hip_lib.rope(x, pos, freq, x)
    with pytest.raises(ValueError, match="on a GPU"):
        hip_lib.qk_norm_rope_fwd(x, x, freq, freq, pos, freq, x, x)
    with pytest.raises(TypeError, match="k"):
        hip_lib.paged_append(x, x, pos, cache, cache)
    with pytest.raises(TypeError, match="q"):
        hip_lib.paged_attention(x, cache, cache, i32[None], i32, i32[:1], x)
    with pytest.raises(ValueError, match="on a GPU"):
        hip_lib.paged_attention(x.bfloat16(), cache.bfloat16(), cache.bfloat16(), i32[None], i32,
                                i32[:1], x.bfloat16())
