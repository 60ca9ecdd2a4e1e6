"""GPU: the quantised cache and the attention over it at the ends of what their formats hold, against
64-bit restatements.  Tolerances as in the tests of the ordinary range: with A = sum_j p_j |v_j| an
attention output is off by 2^-8 of itself and (2^-7 + 2^-10) A at most."""
import math

import pytest
import torch

from sparse_b200 import ops
from sparse_b200.kv_cache import CODES, SCALES, QuantizedCache
from test_gpu_kv_cache import BF, DEV, _attend, _bytes, _quantized, _rand, _want

pytestmark = pytest.mark.gpu

# (sequences, query heads, key heads): streamed alone or with the shared positions as rows of the same pass, one row
# tile of the tensor-core pass, two
ROWS = [(2, 4, 2), (40, 4, 2), (90, 4, 2)]


def _cache(k_codes, k_scales, v_codes, v_scales):
    return QuantizedCache(k_codes.view(CODES), k_scales.view(SCALES), v_codes.view(CODES), v_scales.view(SCALES))


# -- values of the smallest power of two -----------------------------------------------------------
@pytest.mark.parametrize("b,n_q,n_kv", ROWS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shared", [0, 70, 150])
def test_values_of_the_smallest_power_of_two(b, n_q, n_kv, d, shared):
    """Every row's scale byte is 0.  A code under 2^-6 stands for less than bf16's smallest step and an output may
    be less than its smallest normal: half a step of 2^-133 for each of the two roundings."""
    s_max = 170
    q, k = _rand(b, n_q, d, seed=1), _rand(b, n_kv, s_max, d, seed=2)
    v = (_rand(b, n_kv, s_max, d, seed=3).float() * 2.0 ** -121).to(BF)
    assert int(_bytes(_quantized(v)[1]).max()) == 0
    lens = [s_max - i % 17 for i in range(b)]
    got, kk, vv = _attend("fp8", q, k, v, lens, shared)
    want, tol = _want(q, kk, vv, lens, shared, d ** -0.5)
    assert bool(((got.double() - want).abs() <= tol + 2.0 ** -133).all())


def test_a_large_sum_of_weights_over_values_of_the_smallest_power_of_two():
    """Scores that lag behind the largest ones leave weights of up to e^5.5 in the sum of one pass of a CTA, some
    2^20: its inverse times 2^-127 is not a number that fp32 has many bits of.  All values are 2^-119, so is the output:
    2^-11 for a weight in 16 bits, 2^-10 for sums of ten thousand terms in 32, 2^-8 for the output."""
    d, s = 64, 2 ** 24
    k = torch.zeros(1, 1, s, d, dtype=torch.uint8, device=DEV)
    k.view(-1, 2, 128, d)[:, 1, :, 0] = int(torch.tensor(5.5).to(CODES).view(torch.uint8))      # every second tile
    v = torch.full((1, 1, s, d), int(torch.tensor(256.0).to(CODES).view(torch.uint8)), dtype=torch.uint8, device=DEV)
    one, least = (torch.full((1, 1, s), e, dtype=torch.uint8, device=DEV) for e in (127, 0))
    q = torch.zeros(1, 1, d, dtype=BF, device=DEV)
    q[..., 0] = 1.0
    got = ops.attn_decode_quantized(q, _cache(k, one, v, least), torch.tensor([s], dtype=torch.int32, device=DEV), scale=1.0)
    assert float((got.double() * 2.0 ** 119 - 1.0).abs().max()) <= 2.0 ** -8 + 2.0 ** -10 + 2.0 ** -11


@pytest.mark.parametrize("b,n_q,n_kv", ROWS)
@pytest.mark.parametrize("where", ["keys", "values"])
def test_rows_of_every_power_of_two_below_the_largest(b, n_q, n_kv, where):
    """One position counts at a time; its key, or its value, has one of the sizes 2^-126 .. 2^99 (bytes 0 to 218), on
    both sides of the border between shared and own positions."""
    d, shared, s_max = 64, 226, 300
    sizes = torch.exp2(torch.arange(-126, 100, device=DEV).double())
    k = torch.zeros(b, n_kv, s_max, d, dtype=BF, device=DEV)
    v = _rand(b, n_kv, s_max, d, seed=4)
    if where == "values":
        v[:, :, :226] = (v[:, :, :226].double() * sizes[None, None, :, None]).to(BF)
    q = torch.zeros(b, n_q, d, dtype=BF, device=DEV)
    lens = [s_max - i % 3 for i in range(b)]
    for at in (0, 1, 2, 60, 63, 64, 119, 126, 127, 128, 180, 190, 224, 225):
        k.zero_()
        size = float(sizes[at])
        for split in (shared, 0):
            src = torch.zeros(b, dtype=torch.long, device=DEV) if split else torch.arange(b, device=DEV)
            if where == "keys":
                # the query's largest value is 2^6 over the key's size, as far as bf16 goes: a score of 2^6
                k[src, :, at, 5] = size
                q[..., 5] = min(64.0 / size, 2.0 ** 127)
                score = float(q[0, 0, 5]) * size
            else:
                k[src, :, at, 5], q[..., 5], score = 300.0, 1.0, 300.0
            got, _, vv = _attend("fp8", q, k, v, lens, split, scale=1.0)
            if score < 64.0:
                # (sizes under 2^-121: the query cannot make up for them)
                mean, tol = _want(q, k.double(), vv, lens, split, 1.0)
                assert bool(((got.double() - mean).abs() <= tol).all()), (at, split)
                continue
            want = vv[src, :, at].repeat_interleave(n_q // n_kv, dim=1)
            # the others weigh exp(-64) each and are at most 2^102 times as large where values differ, exp(-300) then
            assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -133 if where == "values" else 1e-20)).all()), (at, split)


# -- bases that fp32 does not have -----------------------------------------------------------------
@pytest.mark.parametrize("theta", [1e4 * 8 ** (128 / 126), 1e4 / 3, 12345.678, 1e6 * 4 ** (64 / 62), 1e4])
@pytest.mark.parametrize("first", [0, 131072 - 2000, 2 ** 24 - 2001])
def test_append_angles_of_a_base_that_fp32_does_not_have(theta, first):
    """Pairs (1, 0): the outputs are the cosines and sines themselves, 2^-21 off at most, then rounded to bf16."""
    t, d = 2000, 128
    q = torch.zeros(t, 1, d, dtype=BF, device=DEV)
    q[..., :d // 2] = 1.0
    cache = QuantizedCache.zeros(1, 1, 1, d, d, DEV)
    pos = torch.arange(first, first + t, dtype=torch.int32, device=DEV)
    out = ops.rope_append_quantized(q, q, None, q, torch.full_like(pos, -1), pos, cache, theta)
    ang = pos.double()[:, None] * theta ** (-torch.arange(d // 2, device=DEV).double() / (d // 2))
    want = torch.cat([ang.cos(), ang.sin()], -1)
    assert bool(((out[:, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -21).all())


def test_bases_in_turn():
    """Each call has the angles of its own base, whichever was there before it."""
    q, c = _rand(3, 2, 64, seed=1), QuantizedCache.zeros(1, 1, 2, 64, 64, DEV)
    pos = torch.tensor([5, 1000, 99999], dtype=torch.int32, device=DEV)
    bases = [1e4, 1e4 * (1 + 2.0 ** -30), 5e5]
    outs = [ops.rope_append_quantized(q, q, None, q, pos * 0 - 1, pos, c, t) for t in bases]
    for t, want in list(zip(bases, outs))[::-1]:
        assert torch.equal(ops.rope_append_quantized(q, q, None, q, pos * 0 - 1, pos, c, t), want)
    for t in (0.0, -1.0, math.nan, math.inf, 1e39):
        with pytest.raises(RuntimeError):
            ops.rope_append_quantized(q, q, None, q, pos * 0 - 1, pos, c, t)


# -- e4m3's own NaN ----------------------------------------------------------------------------------
@pytest.mark.parametrize("b,n_q,n_kv", ROWS)
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_a_code_that_is_nan_reads_as_nan_everywhere(b, n_q, n_kv, dk, dv, code):
    """A cache that somebody filled by a cast of their own: read back, streamed and on the tensor cores the code is
    NaN, in its column where a value holds it, in the whole row where a key does."""
    s_max, shared = 200, 140
    k, v = _rand(b, n_kv, s_max, dk, seed=1), _rand(b, n_kv, s_max, dv, seed=2)
    q = _rand(b, n_q, dk, seed=3)
    lens = torch.full((b,), s_max - 1, dtype=torch.int32, device=DEV)
    lens[-1] = shared - 3                                  # ends before the later ones
    clean = ops.attn_decode_quantized(q, QuantizedCache(*_quantized(k), *_quantized(v)), lens, shared)
    group = n_q // n_kv
    for row, at, width in ((0, 0, dv), (0, 63, dv), (0, 64, dv), (0, 127, dv), (0, shared - 1, dv), (0, 7, dk), (0, shared - 2, dk),
                           (0, s_max - 1, dv), (1, 5, dv), (1, 150, dv), (1, 160, dk), (1, 6, dk)):
        for col in (0, 15, 16, width - 1):
            c = QuantizedCache(*_quantized(k), *_quantized(v))
            key = width == dk and at in (7, shared - 2, 160, 6)
            _bytes(c.k if key else c.v)[row, 1, at, col] = code
            want = clean.double().clone()
            # a shared position is sequence 0's and every sequence's that reaches it, another one its own's
            hit = (lens > at) & (torch.arange(b, device=DEV) == row if at >= shared else torch.tensor(row == 0, device=DEV))
            rows = hit.nonzero()[:, 0][:, None], torch.arange(group, 2 * group, device=DEV)[None]
            if key:
                want[rows] = math.nan
            else:
                want[..., col][rows] = math.nan
            got = ops.attn_decode_quantized(q, c, lens, shared)
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (row, at, col, key)
            assert torch.equal(got[~torch.isnan(got)], clean[~torch.isnan(got)]), (row, at, col, key)
    read, _ = ops.cache_read(c, 6, 1)
    assert bool(torch.isnan(read[1, 1, 0, col])) and int(torch.isnan(read).sum()) == 1


# -- scores of -inf, sizes up to the largest -----------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_q,n_kv", ROWS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shared", [1, 130, 200])
@pytest.mark.parametrize("own", ["-inf", "zero", "none"])
def test_shared_scores_of_minus_infinity_weigh_nothing(kind, b, n_q, n_kv, d, shared, own):
    """Shared positions whose every score is -inf: the own positions alone count; where there are none, or theirs are
    -inf too, zeros."""
    s_max = shared + 9
    q = torch.full((b, n_q, d), -3.0e38, dtype=BF, device=DEV)
    k, v = torch.full((b, n_kv, s_max, d), 3.0e38, dtype=BF, device=DEV), _rand(b, n_kv, s_max, d)
    if own == "zero":
        k[:, :, shared:] = 0.0
    lens = [shared if own == "none" else s_max - i % 9 for i in range(b)]
    got, _, vv = _attend(kind, q, k, v, lens, shared)
    if own != "zero":
        assert float(got.float().abs().max()) == 0.0
        return
    # scores of zero: the mean of the own positions
    want, tol = _want(torch.zeros_like(q), torch.zeros_like(vv[:, :, shared:]), vv[:, :, shared:], [n - shared for n in lens], 0, 1.0)
    assert bool(((got.double() - want).abs() <= tol).all())


# -- weights sum to one -------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_q,n_kv", ROWS)
@pytest.mark.parametrize("d", [64, 128])
def test_the_mean_of_equal_values_is_their_value(kind, b, n_q, n_kv, d):
    """All values 1: so is the output, whatever the probabilities are rounded to, as long as the sum that they are
    divided by is that of the rounded ones (half a step of bf16 below 1 is 2^-9).  The probabilities are 1 and, 63 times as
    often, 0.5 + 0.98 * 2^-9, which bf16 rounds to 0.5."""
    shared, s_max = 1280, 1290
    k = torch.zeros(b, n_kv, s_max, d, dtype=BF, device=DEV)
    k[..., 0], k[..., 1] = -0.6875, -0.46875               # exact in e4m3 too
    k[:, :, ::64] = 0.0
    v = torch.ones(b, n_kv, s_max, d, dtype=BF, device=DEV)
    q = torch.zeros(b, n_q, d, dtype=BF, device=DEV)
    q[..., 0], q[..., 1] = 1.0, 2.0 ** -8
    assert abs(math.exp(-0.6875 - 0.46875 / 256) - (0.5 + 0.98 * 2.0 ** -9)) < 2.0 ** -14
    got, _, _ = _attend(kind, q, k, v, [s_max - i % 3 for i in range(b)], shared, scale=1.0)
    assert bool((got == 1.0).all())


# -- several at once -----------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,b,n_q,n_kv,d,shared", [("fp8", 60, 8, 2, 64, 2000), ("bf16", 90, 4, 2, 64, 2000), ("fp8", 80, 16, 8, 128, 1500),
                                                      ("bf16", 40, 16, 16, 128, 1500)])
def test_calls_with_a_shared_prefix_on_their_own_streams(kind, b, n_q, n_kv, d, shared):
    """Launches of four streams run beside one another, those of a stream as close behind one another as they may: each
    CTA of the tensor-core pass finds its tensor memory, and every call gives the bits of a call alone."""
    s_max = shared + 40
    k, v = _rand(b, n_kv, s_max, d, seed=2), _rand(b, n_kv, s_max, d, seed=3)
    lens = torch.tensor([shared + i % 41 for i in range(b)], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = QuantizedCache(*_quantized(k), *_quantized(v))
    ck, cv = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()

    def call(q):
        if kind == "fp8":
            return ops.attn_decode_quantized(q, cache, lens, shared, status=status)
        return ops.attn_decode_shared(q, ck, cv, lens, shared, status=status)

    qs = [_rand(b, n_q, d, seed=i) for i in range(4)]
    want = [call(q) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in qs], []
    for _ in range(25):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, call(qs[i])))
    torch.cuda.synchronize()
    assert int(status) == 0 and all(torch.equal(out, want[i]) for i, out in got)
