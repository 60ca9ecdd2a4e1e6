"""GPU: the quantised key/value cache (write, read back) and decode attention over it and over
a shared prefix, against plain restatements in 64 bits.

Tolerances, from the roundings that the kernels make.  A code is off by at most half a step of
e4m3, 2^-4 of the value or half of the smallest step, 2^-10 of the row's power of two.
Attention: a probability may be rounded to bf16 before it is multiplied with a value (2^-8), and
so may the probabilities that their sum is made of; the result is rounded to bf16 (2^-8 of it).
With A = sum_j p_j |v_j| that is 2^-8 |out| + 2 * 2^-8 A.  Sums of products in fp32 (up to 192
terms, 2^-24 each) move a score of size S = sum |q k| scale by 192 * 2^-24 * S at most; S stays
below 60 here, so a probability by 7e-4 of itself: 2^-10 A for that and the exponentials."""
import math

import pytest
import torch

from sparse_b200 import ops
from sparse_b200.kv_cache import CODES, SCALES, QuantizedCache

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
BF = torch.bfloat16


def _rand(*shape, seed=0, dtype=BF):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _scale_of(rows):
    """Exponent e of fp64 rows [..., d]: least e >= -127 with max|row| <= 448 * 2^e, by trying all."""
    top = rows.abs().amax(-1, keepdim=True)
    e = torch.arange(-127, 128, dtype=torch.float64, device=rows.device)
    fits = top <= 448.0 * torch.exp2(e)
    return fits.to(torch.uint8).argmax(-1) - 127


def _quantized(rows):
    """(codes, scales) of bf16 rows, bit for bit what the cache has to hold."""
    e = _scale_of(rows.double())
    scaled = rows.double() * torch.exp2(-e.double()).unsqueeze(-1)
    # (under 2^120 the code 256 would stand for 2^128: codes stop at 240)
    scaled = torch.where(e.unsqueeze(-1) == 120, scaled.clamp(-240.0, 240.0), scaled)
    codes = scaled.float().to(CODES)
    return codes, (e + 127).to(torch.uint8).view(SCALES)


def _values(codes, scales):
    return codes.float().double() * scales.float().double().unsqueeze(-1)


def _random_cache(b, s, n, dk, dv, seed=0, level=1.0):
    k, v = _rand(b, n, s, dk, seed=seed) * level, _rand(b, n, s, dv, seed=seed + 1)
    return QuantizedCache(*_quantized(k), *_quantized(v))


def _bytes(t):
    return t.view(torch.uint8)


# -- write -----------------------------------------------------------------------------------
@pytest.mark.parametrize("t,n_q,n_kv,dk,dv,rope", [
    (1, 16, 16, 128, 128, 128), (7, 16, 16, 192, 128, 64), (33, 4, 2, 64, 64, 64), (300, 8, 1, 256, 16, 16),
    (5, 3, 3, 16, 256, 0), (2, 5, 5, 80, 96, 32)])
@pytest.mark.parametrize("packed", [True, False])
def test_append(t, n_q, n_kv, dk, dv, rope, packed):
    b, s_max, theta = 3, 320, 1.0e4
    off = 0 if packed else 3                       # an odd start: no 16-byte vectors
    fused = _rand(t, off + (n_q + n_kv) * dk + n_kv * dv, seed=t + dk)
    q = fused[:, off:off + n_q * dk].view(t, n_q, dk)
    k = fused[:, off + n_q * dk:off + (n_q + n_kv) * dk].view(t, n_kv, dk)
    v = fused[:, off + (n_q + n_kv) * dk:].view(t, n_kv, dv)
    seq = (torch.arange(t, device=DEV) % b).int()
    pos = (s_max - 1 - torch.arange(t, device=DEV)).int()
    cache = QuantizedCache.zeros(b, s_max, n_kv, dk, dv, DEV)
    before = fused.clone()
    out = ops.rope_append_quantized(q, k[..., :rope] if rope else None, k[..., rope:] if rope < dk else None, v, seq, pos,
                                    cache, theta)
    assert torch.equal(fused, before)

    ang = pos.double()[:, None, None] * theta ** (-2.0 * torch.arange(rope // 2, device=DEV).double() / max(rope, 1))

    def rotated(x):
        a, c = x[..., :rope // 2].double(), x[..., rope // 2:rope].double()
        return torch.cat([a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin(), x[..., rope:].double()], -1)

    want_q, want_k = rotated(q), rotated(k)
    # one rounding to bf16, behind fp32 products of values up to 5 with cosines that are 2^-22 off
    assert bool(((out.double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 5 * 2.0 ** -21).all())
    at = (seq.long(), slice(None), pos.long())
    codes_v, scales_v = _quantized(v)
    assert torch.equal(_bytes(cache.v)[at], _bytes(codes_v)) and torch.equal(_bytes(cache.v_scale)[at], _bytes(scales_v))
    e = _bytes(cache.k_scale)[at].double() - 127
    # (a row whose largest value stands at a border may take either power of two)
    sure = _scale_of(want_k * (1 - 1e-5)) == _scale_of(want_k * (1 + 1e-5))
    assert torch.equal(e[sure], _scale_of(want_k)[sure].double()) and float(sure.double().mean()) > 0.9
    got = _bytes(cache.k)[at].view(CODES).float().double() * torch.exp2(e)[..., None]
    assert bool(((got - want_k).abs() <= (2.0 ** -4 * want_k.abs()).clamp_min(2.0 ** -10 * torch.exp2(e)[..., None]) + 1e-5).all())
    if rope == 0:
        codes_k, scales_k = _quantized(k)
        assert torch.equal(_bytes(cache.k)[at], _bytes(codes_k)) and torch.equal(_bytes(cache.k_scale)[at], _bytes(scales_k))
    _bytes(cache.k)[at] = 0; _bytes(cache.k_scale)[at] = 0
    _bytes(cache.v)[at] = 0; _bytes(cache.v_scale)[at] = 0
    for x in (cache.k, cache.k_scale, cache.v, cache.v_scale):
        assert int(_bytes(x).max()) == 0, "rows that no token names are left as they were"


def test_append_shared_rotary_part_equals_repeated_one():
    t, n, rope, nope, dv = 11, 16, 64, 128, 128
    q, k_pe, kv = _rand(t, n, 192, seed=1), _rand(t, 1, rope, seed=2), _rand(t, n, nope + dv, seed=3)
    seq, pos = torch.zeros(t, dtype=torch.int32, device=DEV), torch.arange(t, dtype=torch.int32, device=DEV)
    caches = [QuantizedCache.zeros(1, 16, n, 192, dv, DEV) for _ in range(2)]
    outs = [ops.rope_append_quantized(q, k_pe if i == 0 else k_pe.expand(t, n, rope).contiguous(), kv[..., :nope],
                                      kv[..., nope:], seq, pos, c, 1e4) for i, c in enumerate(caches)]
    assert torch.equal(*outs)
    for name in QuantizedCache.__slots__:
        assert torch.equal(*(_bytes(getattr(c, name)) for c in caches))


def test_append_leaves_out_tokens_outside_the_cache():
    b, s, n = 2, 4, 2
    seq = torch.tensor([0, -1, 2, 1, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([-1, 0, 0, 4, 3], dtype=torch.int32, device=DEV)
    x = _rand(5, n, 64, seed=4)
    cache = QuantizedCache.zeros(b, s, n, 64, 64, DEV)
    q = ops.rope_append_quantized(x, x, None, x, seq, pos, cache, 1e4)
    assert bool(torch.isfinite(q).all())
    written = _bytes(cache.v_scale).float().sum(1) > 0
    assert written.nonzero().tolist() == [[1, 3]]


def test_append_of_special_rows():
    """Zeros, infinities, NaN, bf16's smallest and largest values, rows at the border of a power of two."""
    rows = torch.zeros(12, 64)
    rows[1, 5] = math.inf
    rows[2, 6] = math.nan
    rows[3] = 2.0 ** -133
    rows[4, 0], rows[4, 1] = 3.3895e38, 1.0
    rows[5, 0] = 448.0
    rows[6, 0] = 450.0
    rows[7, 0], rows[7, 1] = 1.75 * 2.0 ** -119, -2.0 ** -133
    rows[8, 0], rows[8, 1] = 1.0, 2.0 ** -17            # below the smallest step: half of it, to even
    rows[9] = -1.0
    rows[10, 0], rows[10, 1:5] = 448.0, torch.tensor([1.0625, 1.1875, 17.0, -19.0])      # ties
    rows[11, 63] = -math.inf
    rows = rows.to(BF).to(DEV).unsqueeze(1)
    t = rows.shape[0]
    cache = QuantizedCache.zeros(1, t, 1, 64, 64, DEV)
    pos = torch.arange(t, dtype=torch.int32, device=DEV)
    ops.rope_append_quantized(rows, None, rows, rows, torch.zeros_like(pos), pos, cache, 1e4)
    finite = torch.isfinite(rows.double()).all(-1)[:, 0]
    codes, scales = _quantized(torch.where(torch.isfinite(rows), rows, 0))
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert torch.equal(_bytes(c)[0, 0][finite], _bytes(codes)[:, 0][finite])
        assert torch.equal(_bytes(s)[0, 0][finite], _bytes(scales)[:, 0][finite])
        assert _bytes(s)[0, 0][~finite].tolist() == [255] * 3
    k, _ = ops.cache_read(cache, 0, t)
    assert bool(torch.isnan(k[0, 0][~finite]).all()) and bool(torch.isfinite(k[0, 0][finite]).all())


@pytest.mark.parametrize("pos", [4097, 131071, 1000003, 2 ** 24 - 1])
def test_append_angles_of_far_positions(pos):
    q = _rand(1, 2, 128, seed=pos % 97)
    cache = QuantizedCache.zeros(1, 1, 2, 128, 128, DEV)
    p = torch.tensor([pos], dtype=torch.int32, device=DEV)
    out = ops.rope_append_quantized(q, q, None, q, torch.zeros_like(p), p, cache, 1e6)
    ang = pos * 1e6 ** (-torch.arange(64, device=DEV).double() / 64)
    a, c = q[..., :64].double(), q[..., 64:].double()
    want = torch.cat([a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin()], -1)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 5 * 2.0 ** -21).all())


@pytest.mark.parametrize("pos", [2 ** 24 + 1, 2 ** 29 + 12345677, 2 ** 31 - 1, -(2 ** 24) - 3])
def test_append_angles_of_positions_that_fp32_does_not_have(pos):
    """Four sums of turns of at most 2^6, half an ulp each, are 2^-17 turns: 2^-14 rad."""
    q = _rand(1, 2, 128, seed=pos % 97)
    cache = QuantizedCache.zeros(1, 1, 2, 128, 128, DEV)
    p = torch.tensor([pos], dtype=torch.int32, device=DEV)
    out = ops.rope_append_quantized(q, q, None, q, torch.zeros_like(p), p, cache, 1e6)
    ang = pos * 1e6 ** (-torch.arange(64, device=DEV).double() / 64)
    a, c = q[..., :64].double(), q[..., 64:].double()
    want = torch.cat([a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin()], -1)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 5 * 2.0 ** -13).all())


# -- read back -------------------------------------------------------------------------------
@pytest.mark.parametrize("b,n,dk,dv,begin,count,shared", [
    (1, 1, 16, 16, 0, 1, 0), (3, 2, 64, 64, 3, 37, 11), (2, 16, 128, 128, 0, 40, 40), (2, 3, 192, 128, 39, 1, 40),
    (2, 2, 256, 240, 3, 30, 3), (1, 2, 80, 96, 0, 0, 0), (2, 2, 128, 128, 1, 39, 2)])
def test_read_back_is_exact(b, n, dk, dv, begin, count, shared):
    c = _random_cache(b, 40, n, dk, dv, seed=dk + begin)
    k, v = ops.cache_read(c, begin, count, shared)
    for got, codes, scales in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want = _values(codes, scales)
        want[:, :, :shared] = want[:1, :, :shared].clone()
        want = want[:, :, begin:begin + count]
        assert got.shape == want.shape and torch.equal(got.double(), want)


def test_read_back_of_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(1, 1, 1, 256).expand(1, 1, 256, 256).contiguous()
    scales = torch.arange(256, dtype=torch.uint8, device=DEV).view(1, 1, 256)
    c = QuantizedCache(codes.view(CODES), scales.view(SCALES), codes.view(CODES), scales.view(SCALES))
    k, v = ops.cache_read(c, 0, 256)
    want = _values(c.k, c.k_scale).float().to(BF)
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, posinf=1.0, neginf=-1.0), torch.nan_to_num(want, posinf=1.0, neginf=-1.0))


# -- attention -------------------------------------------------------------------------------
def _want(q, k, v, lens, shared, scale):
    """fp64: outputs and their tolerance; k, v [B, n_kv, S, d] fp64."""
    b, n_q, dk = q.shape
    n_kv = k.shape[1]
    out = torch.zeros(b, n_q, v.shape[-1], dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for i, n in enumerate(lens):
        n = max(0, min(n, k.shape[2]))
        if n == 0:
            continue
        kk, vv = (torch.cat([x[0, :, :min(shared, n)], x[i, :, shared:n]], 1) for x in (k, v))
        s = torch.einsum("hgd,hnd->hgn", q[i].double().view(n_kv, -1, dk), kk) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hgn,hnd->hgd", p, vv).reshape(n_q, -1)
        size[i] = torch.einsum("hgn,hnd->hgd", p, vv.abs()).reshape(n_q, -1)
    return out, 2.0 ** -8 * out.abs() + (2.0 ** -7 + 2.0 ** -10) * size


def _attend(kind, q, k, v, lens, shared, scale=None):
    """k, v [B, n_kv, S, d] bf16 -> (got, the values that the cache stands for)."""
    lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if kind == "bf16":
        ck, cv = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = ops.attn_decode_shared(q, ck, cv, lens, shared, scale, status)
        assert int(status) == 0
        return out, k.double(), v.double()
    c = QuantizedCache(*_quantized(k), *_quantized(v))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = ops.attn_decode_quantized(q, c, lens, shared, scale, status)
    assert int(status) == 0
    return out, _values(c.k, c.k_scale), _values(c.v, c.v_scale)


HEADS = [(16, 16, 128, 128), (16, 16, 192, 128), (4, 2, 64, 64), (8, 1, 128, 128), (20, 2, 64, 64), (12, 4, 192, 128),
         (40, 1, 128, 128)]


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("n_q,n_kv,dk,dv", HEADS)
@pytest.mark.parametrize("lens,shared,s_max", [
    ([1], 0, 1), ([0, 3, 65, 64, 63, 130], 0, 131), ([700], 0, 701), ([700, 0, 257], 0, 777), ([1025, 5, 1025], 5, 1030),
    ([300, 301, 200, 0, 299, 333], 300, 340), ([17, 17], 17, 17), ([129] * 9, 128, 140),
    # as many sequences as make the shared positions a pass of their own for all these heads
    ([130, 70, 0, 127, 128, 129, 131, 257] * 40, 128, 260), ([1000, 77, 0, 999, 1001, 1064, 1066, 1200] * 9, 1000, 1200)])
def test_attention(kind, n_q, n_kv, dk, dv, lens, shared, s_max):
    b = len(lens)
    q, k, v = _rand(b, n_q, dk, seed=b), _rand(b, n_kv, s_max, dk, seed=s_max), _rand(b, n_kv, s_max, dv, seed=7)
    got, kk, vv = _attend(kind, q, k, v, lens, shared)
    want, tol = _want(q, kk, vv, lens, shared, dk ** -0.5)
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())
    # of the whole: the roundings are independent of one another, so well inside the bound of each
    assert float((got.double() - want).norm()) <= 2.0 ** -8 * max(float(want.norm()), 1e-30)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("n_q,n_kv,shared,step", [(4, 2, 0, 31), (4, 4, 60, 7), (320, 160, 60, 211)])
def test_many_sequences_of_which_few_have_positions(kind, n_q, n_kv, shared, step):
    """Empty sequences before, between and behind the others; more tiles of the shared positions than SMs."""
    b, s_max, d = 1000 if n_kv < 100 else 300, 200, 64
    lens = [0] * b
    for i in range(step, b - 40, step):
        lens[i] = 1 + (i * 37) % s_max
    lens[0] = shared
    q, k, v = _rand(b, n_q, d, seed=5), _rand(b, n_kv, s_max, d, seed=6), _rand(b, n_kv, s_max, d, seed=7)
    got, kk, vv = _attend(kind, q, k, v, lens, shared)
    want, tol = _want(q, kk, vv, lens, shared, d ** -0.5)
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_q,n_kv,dk,dv,shared", [(1, 16, 16, 128, 128, 0), (2, 8, 2, 64, 64, 190), (5, 16, 4, 192, 128, 190),
                                                     (40, 4, 2, 128, 128, 190), (70, 8, 2, 64, 64, 257),
                                                     (90, 8, 8, 128, 128, 190), (150, 16, 16, 64, 64, 257),
                                                     (40, 48, 16, 128, 128, 190), (90, 16, 8, 192, 128, 193)])
def test_every_position_is_found(kind, b, n_q, n_kv, dk, dv, shared):
    """A key that answers the query alone: the output is its value, wherever it stands."""
    s_max = 300
    k = torch.zeros(b, n_kv, s_max, dk, dtype=BF, device=DEV)
    v = _rand(b, n_kv, s_max, dv, seed=3)
    q = torch.zeros(b, n_q, dk, dtype=BF, device=DEV)
    q[:, :, 0] = 1.0
    lens = [s_max - i % 3 for i in range(b)]
    for at in (0, 1, 7, 8, 15, 16, 31, 63, 64, 127, 128, 189, 190, 191, 255, 256, 257, 296):
        src = torch.zeros(b, dtype=torch.long, device=DEV) if at < shared else torch.arange(b, device=DEV)
        k.zero_()
        k[src, :, at, 0] = 64.0
        got, _, vv = _attend(kind, q, k, v, lens, shared, scale=1.0)
        want = vv[src, :, at].repeat_interleave(n_q // n_kv, dim=1)
        # the 299 others weigh exp(-64) each
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-20).all()), at


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_kv", [(2, 2), (40, 2), (200, 8)])
def test_masked_places_may_hold_anything(kind, b, n_kv):
    """NaN and infinities behind a sequence's end, and in the shared positions of a sequence that ends inside them,
    change nothing; a sequence that sees one has NaN."""
    n_q, d, s_max, shared = 2 * n_kv, 64, 200, 100
    lens = [150] * (b - 1) + [90]
    q, k, v = _rand(b, n_q, d, seed=1), _rand(b, n_kv, s_max, d, seed=2), _rand(b, n_kv, s_max, d, seed=3)
    clean, _, _ = _attend(kind, q, k, v, lens, shared)
    for x, bad in ((k, math.nan), (v, math.inf), (v, math.nan), (k, -math.inf)):
        y = x.clone()
        y[:, :, 150:] = bad
        y[1:, :, :shared] = bad                    # rows that nothing reads: shared ones stand in sequence 0
        args = (y, v) if x is k else (k, y)
        if kind == "fp8":
            ops_in = [(_quantized(torch.where(torch.isfinite(z), z, 0)), ~torch.isfinite(z).all(-1)) for z in args]
            for (codes, scales), at in ops_in:
                _bytes(scales)[at] = 255
            c = QuantizedCache(*ops_in[0][0], *ops_in[1][0])
            got = ops.attn_decode_quantized(q, c, torch.tensor(lens, dtype=torch.int32, device=DEV), shared)
        else:
            got = ops.attn_decode_shared(q, *(z.transpose(1, 2).contiguous() for z in args),
                                         torch.tensor(lens, dtype=torch.int32, device=DEV), shared)
        assert torch.equal(got, clean)
    # position 95 of sequence 0 is shared, but the last sequence ends before it
    y = v.clone()
    y[0, :, 95] = math.nan
    if kind == "fp8":
        codes, scales = _quantized(torch.where(torch.isfinite(y), y, 0))
        _bytes(scales)[0, :, 95] = 255
        got = ops.attn_decode_quantized(q, QuantizedCache(*_quantized(k), codes, scales),
                                        torch.tensor(lens, dtype=torch.int32, device=DEV), shared)
    else:
        got = ops.attn_decode_shared(q, k.transpose(1, 2).contiguous(), y.transpose(1, 2).contiguous(),
                                     torch.tensor(lens, dtype=torch.int32, device=DEV), shared)
    assert torch.equal(got[-1], clean[-1]) and bool(torch.isnan(got[:-1]).all())


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,shared,n_kv", [(2, 0, 2), (3, 200, 2), (40, 200, 2), (200, 200, 8)])
def test_scores_far_apart(kind, b, shared, n_kv):
    """Scores over hundreds, rising and falling with the position: the running maximum moves often."""
    n_q, d, s_max = 4 * n_kv, 64, 400
    for sign in (1.0, -1.0):
        k = torch.zeros(b, n_kv, s_max, d, dtype=BF, device=DEV)
        k[..., 0] = (sign * torch.arange(s_max, device=DEV) / 2).to(BF)
        v = _rand(b, n_kv, s_max, d, seed=5)
        q = torch.zeros(b, n_q, d, dtype=BF, device=DEV)
        q[:, :, 0] = torch.tensor([1.0, -1.0, 0.5, 4.0], device=DEV).repeat(n_kv)
        lens = [s_max - 7 * (i % 5) for i in range(b)]
        got, kk, vv = _attend(kind, q, k, v, lens, shared, scale=1.0)
        want, tol = _want(q, kk, vv, lens, shared, 1.0)
        # (scores up to 800: their fp32 products are exact here, the exponentials' arguments are off by 2^-14)
        assert bool(((got.double() - want).abs() <= tol + 2.0 ** -12 * want.abs()).all())


def test_values_of_very_different_size():
    """Quantised values whose powers of two span sixty binades: small ones with all the weight are not lost."""
    n, d, s = 2, 64, 96
    q = torch.zeros(1, n, d, dtype=BF, device=DEV)
    q[:, :, 0] = 1.0
    k = torch.zeros(1, n, s, d, dtype=BF, device=DEV)
    v = _rand(1, n, s, d, seed=9)
    k[:, :, ::2, 0] = -80.0                        # exp(-80) = 2^-115
    v[:, :, ::2] *= 2.0 ** 60
    got, kk, vv = _attend("fp8", q, k, v, [s], 0, scale=1.0)
    want, tol = _want(q, kk, vv, [s], 0, 1.0)
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_all_scores_minus_infinity_weigh_nothing(kind):
    """A query against keys whose every score is -inf: zeros, as the decode attention over the bf16 cache gives."""
    q = torch.full((1, 2, 64), -3.0e38, dtype=BF, device=DEV)
    k, v = torch.full((1, 2, 70, 64), 3.0e38, dtype=BF, device=DEV), _rand(1, 2, 70, 64)
    got, _, _ = _attend(kind, q, k, v, [70], 0)
    assert float(got.float().abs().max()) == 0.0


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_q,n_kv", [(40, 8, 4), (150, 32, 8)])
def test_strided_queries_and_repeats_give_the_same_bits(kind, b, n_q, n_kv):
    d, s = 128, 333
    fused = _rand(b, 3 + n_q * d + 11, seed=1)
    q = fused[:, 3:3 + n_q * d].view(b, n_q, d)
    k, v = _rand(b, n_kv, s, d, seed=2), _rand(b, n_kv, s, d, seed=3)
    lens = [(i * 29) % (s + 1) for i in range(b)]
    for shared in (0, 100):
        lens_ = [max(n, shared) for n in lens]
        a = _attend(kind, q, k, v, lens_, shared)[0]
        assert torch.equal(a, _attend(kind, q.contiguous(), k, v, lens_, shared)[0])
        assert torch.equal(a, _attend(kind, q, k, v, lens_, shared)[0])


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_q,n_kv,d", [(24, 4, 2, 64), (150, 16, 8, 128)])
def test_captured_call_follows_its_inputs(kind, b, n_q, n_kv, d):
    """A recorded call reads queries, lengths and cache as they are when it is replayed; two recordings do not
    share anything."""
    s, shared = 200, 64
    k, v = _rand(b, n_kv, s, d, seed=2), _rand(b, n_kv, s, d, seed=3)
    cache = QuantizedCache(*_quantized(k), *_quantized(v))
    ck, cv = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()

    def call(q, lens):
        if kind == "fp8":
            return ops.attn_decode_quantized(q, cache, lens, shared)
        return ops.attn_decode_shared(q, ck, cv, lens, shared)

    qs = [_rand(b, n_q, d, seed=i) for i in range(2)]
    lens = [torch.full((b,), n, dtype=torch.int32, device=DEV) for n in (200, 111)]
    call(qs[0], lens[0])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(qs[i], lens[i]))
        graphs.append(g)
    for step in range(3):
        for i in range(2):
            qs[i].copy_(_rand(b, n_q, d, seed=10 * step + i))
            lens[i].fill_(64 + 17 * step + i)
        want = [call(qs[i], lens[i]) for i in range(2)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_calls_on_their_own_streams():
    b, n_q, n_kv, d, s = 30, 8, 2, 64, 500
    k, v = _rand(b, n_kv, s, d, seed=2), _rand(b, n_kv, s, d, seed=3)
    cache = QuantizedCache(*_quantized(k), *_quantized(v))
    lens = torch.randint(0, s + 1, (b,), device=DEV).int()
    qs = [_rand(b, n_q, d, seed=i) for i in range(6)]
    want = [ops.attn_decode_quantized(q, cache, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [None] * len(qs)
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            got[i] = ops.attn_decode_quantized(qs[i], cache, lens)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_written_read_and_attended_together():
    """A prompt written in two chunks, positions one by one after it, the read-back and the attention of every step:
    all see the same cache."""
    b, n_q, n_kv, dk, dv, rope, s_max, theta = 3, 8, 4, 192, 128, 64, 80, 1e4
    cache = QuantizedCache.zeros(b, s_max, n_kv, dk, dv, DEV)
    past = 0
    for n in (33, 20, 1, 1, 1):
        t = b * n
        seq = torch.arange(b, dtype=torch.int32, device=DEV).repeat_interleave(n)
        pos = (torch.arange(n, dtype=torch.int32, device=DEV) + past).repeat(b)
        q, k_pe, kv = _rand(t, n_q, dk, seed=past), _rand(t, 1, rope, seed=past + 1), _rand(t, n_kv, dk - rope + dv, seed=past + 2)
        rotated = ops.rope_append_quantized(q, k_pe, kv[..., :dk - rope], kv[..., dk - rope:], seq, pos, cache, theta)
        past += n
        k, v = ops.cache_read(cache, 0, past)
        assert torch.equal(v[:, :, past - n:].double(),
                           _values(*_quantized(kv[..., dk - rope:].reshape(b, n, n_kv, dv).transpose(1, 2))))
        lens = torch.full((b,), past, dtype=torch.int32, device=DEV)
        last = rotated.view(b, n, n_q, dk)[:, -1]
        got = ops.attn_decode_quantized(last, cache, lens)
        want, tol = _want(last, k.double(), v.double(), [past] * b, 0, dk ** -0.5)
        assert bool(((got.double() - want).abs() <= tol).all())


def test_long_cache_offsets():
    """Codes beyond 2^31 bytes and positions near the end of a long cache."""
    n_kv, d, s_max = 8, 128, 2 ** 21 + 77                # 2.1 GB of key codes, as many of value codes
    cache = QuantizedCache.zeros(1, s_max, n_kv, d, d, DEV)
    pos = torch.tensor([s_max - 1, 5], dtype=torch.int32, device=DEV)
    x = _rand(2, n_kv, d, seed=1)
    ops.rope_append_quantized(x, None, x, x, torch.zeros_like(pos), pos, cache, 1e4)
    k, v = ops.cache_read(cache, s_max - 1, 1)
    assert torch.equal(v[0, :, 0].double(), _values(*_quantized(x[0])))
    lens = torch.tensor([s_max], dtype=torch.int32, device=DEV)
    q = x[:1] * 64
    got = ops.attn_decode_quantized(q, cache, lens, scale=1.0)
    # the query's own key outweighs the two million zero keys: 64 |k|^2 is above 3000
    want = v[0, :, 0]
    assert torch.equal(got[0], want)


# -- refusals that need tensors on the device ---------------------------------------------------
def test_wrappers_refuse_operands_that_do_not_fit():
    c = QuantizedCache.zeros(2, 8, 2, 64, 64, DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    q = _rand(2, 4, 64)
    for args, kw in (((q.float(), c, lens), {}), ((q[:1], c, lens), {}), ((q[..., :32], c, lens), {}),
                     ((q[:1].expand(2, 4, 64), c, lens), {}), ((q.transpose(1, 2).contiguous().transpose(1, 2), c, lens), {}),
                     ((q, c, lens.long()), {}), ((q, c, lens[:1]), {}), ((q, c, lens.cpu()), {}),
                     ((q, c, lens), {"shared_len": 9}), ((q, c, lens), {"shared_len": -1}), ((q[:, :3], c, lens), {}),
                     ((q, c, lens), {"status": lens.long()})):
        with pytest.raises(RuntimeError):
            ops.attn_decode_quantized(*args, **kw)
    for begin, count, shared in ((4, 5, 0), (-1, 2, 0), (0, -1, 0), (0, 4, 9)):
        with pytest.raises(RuntimeError):
            ops.cache_read(c, begin, count, shared)
    k, v = _rand(2, 2, 64), _rand(2, 2, 64)
    for args in ((q.float(), k, None, v, lens, lens), (q, k[..., :32], None, v, lens, lens), (q, k, k, v, lens, lens),
                 (q, k[..., :24], k[..., 24:], v, lens, lens), (q, _rand(2, 3, 64), None, v, lens, lens),
                 (q, k, None, v[..., :32], lens, lens), (q, k, None, v, lens.long(), lens), (q, k, None, v, lens, lens[:1]),
                 (q, k, None, v.cpu(), lens, lens), (q, None, None, v, lens, lens),
                 (q, k, None, v.transpose(1, 2).contiguous().transpose(1, 2), lens, lens)):
        with pytest.raises(RuntimeError):
            ops.rope_append_quantized(*args, c, 1e4)
    with pytest.raises(RuntimeError):
        ops.rope_append_quantized(q, k, None, v, lens, lens, c, 0.0)
    with pytest.raises(RuntimeError):
        ops.attn_decode_shared(q, _rand(2, 2, 2, 64).transpose(1, 2), _rand(2, 2, 2, 64), lens, 0)
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_q,n_kv,dk,dv,shared", [(18, 37, 37, 128, 128, 4500), (18, 37, 37, 64, 64, 4517),
                                                     (18, 37, 37, 192, 128, 2305), (150, 74, 74, 64, 64, 1281)])
@pytest.mark.parametrize("slope", [0.0, 0.02, -0.02])
def test_long_shared_prefix(kind, b, n_q, n_kv, dk, dv, shared, slope):
    """Many tiles per run of the tensor-core pass, with scores that keep rising (the accumulator is rescaled again and
    again), that keep falling, or that do neither."""
    s_max = shared + 20
    q, v = _rand(b, n_q, dk, seed=b), _rand(b, n_kv, s_max, dv, seed=7)
    k = _rand(b, n_kv, s_max, dk, seed=3) / 4
    if slope:
        q[:, :, 0], k[..., 0] = 1.0, (slope * torch.arange(s_max, device=DEV)).to(BF)
    lens = [shared + i % 21 for i in range(b)]
    got, kk, vv = _attend(kind, q, k, v, lens, shared, scale=1.0)
    want, tol = _want(q, kk, vv, lens, shared, 1.0)
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())
    assert float((got.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())


@pytest.mark.parametrize("kind,b,n_q,n_kv,d,shared", [("fp8", 64, 32, 4, 128, 4096), ("bf16", 40, 16, 16, 128, 2050),
                                                      ("fp8", 18, 6, 2, 64, 3000), ("bf16", 200, 8, 4, 64, 1500)])
def test_calls_back_to_back_end_in_time_with_the_same_bits(kind, b, n_q, n_kv, d, shared):
    """Hundreds of calls with nothing between them: no wait inside runs out, every one gives the same bits."""
    s_max = shared + 30
    q, k, v = _rand(b, n_q, d, seed=1), _rand(b, n_kv, s_max, d, seed=2), _rand(b, n_kv, s_max, d, seed=3)
    lens = torch.tensor([shared + i % 30 for i in range(b)], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    if kind == "fp8":
        cache = QuantizedCache(*_quantized(k), *_quantized(v))
        call = lambda: ops.attn_decode_quantized(q, cache, lens, shared, status=status)      # noqa: E731
    else:
        ck, cv = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        call = lambda: ops.attn_decode_shared(q, ck, cv, lens, shared, status=status)        # noqa: E731
    want, wrong = call(), torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(300):
        wrong += (call() != want).sum()
    assert int(status) == 0 and int(wrong) == 0


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("b,n_kv,shared", [(3, 2, 0), (3, 2, 77), (200, 8, 77)])
def test_a_scale_of_zero_weighs_all_positions_alike(kind, b, n_kv, shared):
    s_max = 140
    q, k, v = _rand(b, 2 * n_kv, 64, seed=1), _rand(b, n_kv, s_max, 64, seed=2), _rand(b, n_kv, s_max, 64, seed=3)
    lens = [77 + i % 64 for i in range(b)]
    got, kk, vv = _attend(kind, q, k, v, lens, shared, scale=0.0)
    want, tol = _want(q, kk, vv, lens, shared, 0.0)
    assert bool(((got.double() - want).abs() <= tol).all())


def test_shared_prefix_with_values_of_any_size():
    """Quantised rows with powers of two from the smallest to the largest, through the tensor-core pass: the operand
    that a code becomes is exact for every one of them."""
    b, n, d, shared = 130, 16, 64, 256
    q = torch.zeros(b, n, d, dtype=BF, device=DEV)
    q[:, :, 0] = 1.0
    k = torch.zeros(b, n, shared + 1, d, dtype=BF, device=DEV)
    v = _rand(b, n, shared + 1, d, seed=4)
    # every shared position is the one that counts for some query row: positions differ in their first 8 key bits
    sizes = torch.linspace(-120, 100, shared, device=DEV).round()
    v[0, :, :shared] = (v[0, :, :shared].double() * torch.exp2(sizes.double())[None, :, None]).to(BF)
    for at in (0, 1, 17, 100, 130, 150, 180, 200, 240, 255):
        k.zero_()
        k[0, :, at, 0] = 300.0
        got, _, vv = _attend("fp8", q, k, v, [shared + 1] * b, shared, scale=1.0)
        want = vv[0, :, at].expand(b, -1, -1)
        # the others weigh exp(-300): nothing, whatever their size
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs()).all()), at
