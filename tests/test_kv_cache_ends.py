"""CPU: what the cache calls' host side takes and refuses at the ends of its ranges."""
import math
import types

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


def _model_of_blocks(*blocks):
    """A model as far as `check_status` looks at it."""
    from sparse_b200.model import ShapedMoeModel
    m = object.__new__(ShapedMoeModel)
    m.layers = [types.SimpleNamespace(block=b) for b in blocks]
    m.attn_status = torch.ones(1, dtype=torch.int32)
    return m


def test_an_expired_wait_is_reported_once():
    m = _model_of_blocks(None)
    with pytest.raises(RuntimeError, match="status 1"):
        m.check_status()
    m.check_status()


def test_an_expired_wait_does_not_outlive_a_block_that_raises():
    class Block:
        calls = 0

        def check_status(self):
            self.calls += 1
            if self.calls == 1:
                raise RuntimeError("the block's")

    m = _model_of_blocks(Block())
    with pytest.raises(RuntimeError, match="the block's"):
        m.check_status()
    m.check_status()
