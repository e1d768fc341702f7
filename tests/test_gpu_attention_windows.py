"""Windows of attention over a paged cache at their ends: of one position, of as many
as there are and of more, where sequences have fewer positions than new tokens."""
import pytest

from credit_amd import hip_lib
from tests.heads_rules_lib import FEW, MANY, build, way
from tests.test_gpu_paged_attention import call, check, make

pytestmark = pytest.mark.gpu

# New tokens, positions, query heads, key heads: both sizes of tiles, whole and in parts.
SHAPES = {(FEW, False): ([9, 3, 30], [5, 0, 29], 4, 2),
          (FEW, True): ([9, 3, 60], [5, 0, 900], 4, 2),
          (MANY, False): ([200, 260], [70, 255], 32, 16),
          (MANY, True): ([200, 300], [70, 2200], 2, 1)}


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    return build(tmp_path_factory.mktemp("rules"))


@pytest.mark.parametrize("window", [1, 40, 254, 2 ** 30, 2 ** 31 - 40, 2 ** 31 - 1])
@pytest.mark.parametrize("which", SHAPES, ids=str)
def test_fewer_positions_than_new_tokens(gpu, rules, which, window):
    """Tokens in front of a sequence's first position see nothing, the others what the
    window leaves them."""
    args = make(*SHAPES[which], 64, 16)
    assert way(rules, args) == which
    out, lse = check(args, window)
    longest = args[3].shape[1] * args[1].shape[1]
    if window >= longest:  # hides nothing
        whole, whole_lse = call(args)
        assert (out == whole).all() and (lse == whole_lse).all()


def test_windows_beyond_32_bits(gpu):
    """They are none, or negative; their low 32 bits say nothing."""
    args = make([3, 20], [50, 80], 4, 2, 64, 16)
    want, want_lse = call(args)
    for window in (2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 70 + 5):
        out, lse = call(args, window)
        assert (out == want).all() and (lse == want_lse).all()
    for window in (-1, -2 ** 31 - 1, -2 ** 32 + 5):
        with pytest.raises(hip_lib.CreditError, match="window"):
            call(args, window)
