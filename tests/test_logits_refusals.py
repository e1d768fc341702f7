"""What the operators on logits refuse, on the host and before any HIP call:
the C entry points by status, the Python functions by exception.  No GPU."""
import ctypes
import math

import pytest
import torch

from credit_amd import hip_lib

FAKE = 0x100000  # never dereferenced: every call fails validation
TYPES = ("f32", "bf16")
SHAPE, ALIGN, NULL, UNSUPPORTED, CONFIG = -2, -3, -1, -4, -8

# Arguments by name, in order; None stands for NULL.
CALLS = {
    "token_logprob_fwd": dict(logits=FAKE, ld=64, tokens=FAKE, logp=FAKE, stats=FAKE,
                              entropy=FAKE, top_logp=FAKE, top_ids=FAKE, rows=4, cols=64,
                              n_tokens=1, n_top=5, temperature=1.0, cfg=None),
    "token_logprob_bwd": dict(logits=FAKE, ld=64, tokens=FAKE, stats=FAKE, entropy=FAKE,
                              dlogp=FAKE, dentropy=FAKE, dlogits=2 * FAKE, ldd=64, rows=4,
                              cols=64, n_tokens=1, temperature=1.0, cfg=None),
    "topk_distill_fwd": dict(logits=FAKE, ld=64, teacher_ids=FAKE, teacher=FAKE, loss=FAKE,
                             stats=FAKE, rows=4, cols=64, n_top=5, tail=1, temperature=1.0,
                             cfg=None),
    "topk_distill_bwd": dict(logits=FAKE, ld=64, teacher_ids=FAKE, teacher=FAKE, stats=FAKE,
                             dloss=FAKE, dlogits=2 * FAKE, ldd=64, rows=4, cols=64, n_top=5,
                             tail=1, temperature=1.0, cfg=None),
}
COMMON = [
    (dict(logits=None), NULL),
    (dict(stats=None), NULL),
    (dict(rows=-1), SHAPE),
    (dict(cols=0), SHAPE),
    (dict(cols=(1 << 29) + 1, ld=1 << 30), SHAPE),
    (dict(rows=1 << 31), SHAPE),
    (dict(ld=63), SHAPE),
    (dict(ld=0), SHAPE),
    (dict(ld=-64), SHAPE),
    (dict(ld=1 << 60), SHAPE),
    (dict(logits=FAKE + 1), ALIGN),
    (dict(temperature=0.0), CONFIG),
    (dict(temperature=-1.0), CONFIG),
    (dict(temperature=math.nan), CONFIG),
    (dict(temperature=math.inf), CONFIG),
    (dict(temperature=1e-5), CONFIG),
]
OWN = {
    "token_logprob_fwd": [(dict(tokens=None), NULL), (dict(logp=None), NULL),
                          (dict(top_logp=None), NULL), (dict(top_ids=None), NULL),
                          (dict(n_tokens=-1), SHAPE), (dict(n_tokens=257), SHAPE),
                          (dict(n_top=-1), SHAPE), (dict(n_top=65), SHAPE),
                          (dict(n_top=257, cols=1000, ld=1000), SHAPE)],
    "token_logprob_bwd": [(dict(tokens=None), NULL), (dict(dlogp=None), NULL),
                          (dict(entropy=None), NULL), (dict(dlogits=None), NULL),
                          (dict(n_tokens=257), SHAPE), (dict(ldd=63), SHAPE),
                          (dict(dlogits=2 * FAKE + 1), ALIGN),
                          (dict(dlogits=FAKE + 16), CONFIG),
                          (dict(dlogits=FAKE, ldd=128), CONFIG),
                          (dict(dlogits=FAKE + 64, rows=1), CONFIG)],
    "topk_distill_fwd": [(dict(teacher_ids=None), NULL), (dict(teacher=None), NULL),
                         (dict(loss=None), NULL), (dict(n_top=0), SHAPE),
                         (dict(n_top=257), SHAPE)],
    "topk_distill_bwd": [(dict(teacher_ids=None), NULL), (dict(teacher=None), NULL),
                         (dict(dloss=None), NULL), (dict(dlogits=None), NULL),
                         (dict(n_top=0), SHAPE), (dict(n_top=257), SHAPE),
                         (dict(ldd=63), SHAPE), (dict(dlogits=FAKE + 64), CONFIG)],
}


def call(lib, op, dtype, **edit):
    args = {**CALLS[op], **edit}
    return getattr(lib, f"credit_{op}_{dtype}")(*args.values())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op", CALLS)
def test_refused(lib, op, dtype):
    for edit, status in COMMON + OWN[op]:
        assert call(lib, op, dtype, **edit) == status, (edit, hip_lib.last_error())
        assert hip_lib.last_error()


@pytest.mark.parametrize("op", CALLS)
def test_staged_variant_and_bad_cfg(lib, op):
    for variant, split, workspace, status in ((2, 0, None, UNSUPPORTED), (9, 0, None, CONFIG),
                                              (0, 65, None, CONFIG), (0, 0, FAKE + 16, -5)):
        cfg = hip_lib.CreditCfg(None, variant, split, workspace, 0)
        assert call(lib, op, "f32", cfg=ctypes.byref(cfg)) == status


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op", CALLS)
def test_operands_off_their_alignment(lib, op, dtype):
    """Every pointer at half an element: of 8 bytes the columns', of 4 the rest."""
    columns = ("tokens", "teacher_ids", "top_ids")
    for name, value in CALLS[op].items():
        if value in (FAKE, 2 * FAKE):
            off = 1 if name in ("logits", "dlogits") else 4 if name in columns else 2
            assert call(lib, op, dtype, **{name: value + off}) == ALIGN, name


@pytest.mark.parametrize("op", ["token_logprob_bwd", "topk_distill_bwd"])
def test_gradients_have_no_parts(lib, op):
    cfg = hip_lib.CreditCfg(None, hip_lib.VARIANTS["split"], 4, None, 0)
    assert call(lib, op, "bf16", cfg=ctypes.byref(cfg)) == UNSUPPORTED


@pytest.mark.parametrize("op", CALLS)
def test_no_rows_is_a_noop(lib, op):
    nothing = {k: None for k, v in CALLS[op].items() if v is FAKE or v == 2 * FAKE}
    assert call(lib, op, "bf16", rows=0, **nothing) == 0


def test_python_refuses_before_the_library():
    z = torch.zeros(4, 64)
    tokens, out, stats = torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1), torch.zeros(4, 2)
    with pytest.raises(TypeError, match="logits"):
        hip_lib.token_logprob_fwd(z.half(), tokens, out, stats)
    with pytest.raises(ValueError, match="2-D"):
        hip_lib.token_logprob_fwd(z[0], tokens, out, stats)
    with pytest.raises(ValueError, match="contiguous"):
        hip_lib.token_logprob_fwd(torch.zeros(64, 4).t(), tokens, out, stats)
    with pytest.raises(ValueError, match="on a GPU"):
        hip_lib.token_logprob_fwd(z, tokens, out, stats)
    with pytest.raises(ValueError, match="on a GPU"):
        hip_lib.topk_distill_bwd(z, tokens, out, torch.zeros(4, 8), torch.zeros(4), z)
