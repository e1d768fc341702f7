"""Workspaces of the operators on heads at the ends of their sizes.  No GPU."""
import pytest

from credit_amd import hip_lib


@pytest.mark.parametrize("sizes", [
    (1 << 62, 1, 32, 8, 128, 8192), ((1 << 25) + 1, 1, 32, 8, 128, 1 << 20),
    (1, 1 << 40, 8, 8, 64, 8192), (1, (1 << 20) + 1, 8, 8, 64, 8192),
    (1, 1, 32, 8, 100, 8192), (1, 1, 32, 8, 264, 8192), (1, 1, 32, 8, 128, (1 << 30) + 1),
    (1, 1, 32, 8, 128, 1 << 62), (1 << 60, 1 << 20, 32, 8, 128, 1 << 40)], ids=str)
def test_sizes_that_a_call_refuses_take_none(lib, sizes):
    assert hip_lib.paged_attention_workspace_bytes(*sizes) == 0


def test_the_largest_sizes(lib):
    size = hip_lib.paged_attention_workspace_bytes
    assert size(1, 1, 32, 8, 128, 1 << 30) == size(1, 1, 32, 8, 128, 1 << 20) > 0
    assert size(1 << 25, 1, 32, 8, 128, 1 << 30) == 0  # more tiles than units: whole
