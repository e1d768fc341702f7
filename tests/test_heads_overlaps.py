"""Outputs of the operators on heads that would share elements with another tensor of
the call are refused, the small ones among them, before any HIP call.  No GPU."""
import ctypes
import itertools

import pytest

from credit_amd import hip_lib
from tests.test_heads_refusals import CONFIG, call, heads, pages, rotation, types

def tensors(op):
    """The call's tensors by name, each at a place of its own."""
    at = itertools.count(6)

    def place():
        return next(at) << 32

    if op in ("rope", "qk_norm_rope_fwd"):
        names = {n: heads(place()) for n in ("q", "k", "q_out", "k_out")}
    elif op == "qk_norm_rope_bwd":
        names = {n: heads(place()) for n in ("q", "k", "dq_out", "dk_out", "dq", "dk")}
    elif op == "paged_append":
        names = {n: heads(place()) for n in ("k", "v", "q", "q_out")}
    else:
        names = {n: heads(place()) for n in ("q", "out")}
    if op.startswith("paged"):
        names.update({n: pages(place()) for n in ("k_cache", "v_cache")})
    small = {"rope": (), "qk_norm_rope_fwd": ("q_weight", "k_weight", "rstd"),
             "qk_norm_rope_bwd": ("q_weight", "k_weight", "rstd", "dq_weight", "dk_weight"),
             "paged_append": ("q_weight", "k_weight", "slots"),
             "paged_attention": ("pages", "q_start", "kv_len", "lse")}[op]
    names.update({n: place() for n in small})
    if op != "paged_attention":
        names["rotation"] = rotation(place(), place())
    return names


OUTPUTS = {"rope": ("q_out", "k_out"), "qk_norm_rope_fwd": ("q_out", "k_out", "rstd"),
           "qk_norm_rope_bwd": ("dq", "dk", "dq_weight", "dk_weight"),
           "paged_append": ("k_cache", "v_cache", "q_out"), "paged_attention": ("out", "lse")}
PAIRS = [(op, out, other) for op, outs in OUTPUTS.items() for out in outs
         for other in [*tensors(op), "positions", "inv_freq"]
         if other not in ("rotation", out)
         and not (op == "paged_attention" and other in ("positions", "inv_freq"))]


def address(value):
    return value.data if isinstance(value, ctypes.Structure) else value


@pytest.mark.parametrize("op,out,other", PAIRS)
def test_an_output_over_another_tensor(lib, op, out, other):
    for dtype in types(op):
        for ahead in (0, 16):  # the output begins in the other, or behind its first bytes
            names = tensors(op)
            if other in ("positions", "inv_freq"):
                to = getattr(names["rotation"], other)
            else:
                to = address(names[other])
            if isinstance(names[out], ctypes.Structure):
                names[out].data = to + ahead
                # Its own input's strides are what is allowed, so others are taken.
                names[out].head_stride *= 2
                for level in ("token_stride", "slot_stride", "page_stride"):
                    if hasattr(names[out], level):
                        setattr(names[out], level, 2 * getattr(names[out], level))
            else:
                names[out] = to + ahead
            if op == "paged_attention":
                names["batch"] = 8  # lengths of 32 bytes
            assert call(lib, op, dtype, **names) == CONFIG, (dtype, ahead)
            error = hip_lib.last_error()
            assert "overlaps" in error and out in error and other in error


def test_gradients_of_no_tokens_into_one_array(lib):
    names = tensors("qk_norm_rope_bwd")
    names["dk_weight"] = names["dq_weight"]
    assert call(lib, "qk_norm_rope_bwd", "f32", tokens=0, **names) == CONFIG
