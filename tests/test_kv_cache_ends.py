"""CPU: what the cache calls' host side takes and refuses at the ends of its ranges."""
import math

import pytest
import torch

OK = 1 << 20          # an address that is never read: the checks come first


@pytest.mark.parametrize("theta,rest", [(0.0, 0.0), (1e4, -1e4), (1e4, math.nan), (math.inf, 0.0), (1e4, math.inf),
                                        (math.inf, -math.inf), (1.0, -2.0)])
def test_append_refuses_bases_that_are_no_base(theta, rest):
    from sparse_b200._lib import ROPE_APPEND, lib
    args = [OK] * 11 + [256] * 8 + [4, 2, 4, 2, 64, 64, 32, 8, theta, rest]
    assert lib.sb_rope_append_fp8(ROPE_APPEND.pack(*args), None) == -1
    assert b"bad shape" in lib.sb_last_error_string()


def test_a_base_is_taken_as_two_floats():
    from sparse_b200.ops import _two_floats
    for x in (1e4, 1e6, 1e4 * 8 ** (128 / 126), 1e4 / 3, 12345.678, 5e-41):
        hi, rest = _two_floats(x)
        assert hi == float(torch.tensor(x, dtype=torch.float32)) and abs(hi + float(torch.tensor(rest)) - x) <= 2.0 ** -48 * x + 2.0 ** -150
    assert _two_floats(1e4) == (1e4, 0.0)
    assert _two_floats(1e39)[0] == math.inf                # (which the call refuses)
