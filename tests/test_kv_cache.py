"""CPU: the quantised cache's container, and what its entry points refuse before they touch a device."""
import pytest
import torch

from sparse_b200.kv_cache import CODES, SCALES, QuantizedCache

OK = 1 << 20          # an address that is never read: the checks come first


def _cache(b=2, s=8, n=3, dk=64, dv=64):
    return QuantizedCache.zeros(b, s, n, dk, dv, torch.device("cpu"))


def test_an_empty_cache_reads_as_zero():
    c = _cache()
    assert c.k.dtype == CODES and c.v_scale.dtype == SCALES and c.k.shape == (2, 3, 8, 64) and c.v_scale.shape == (2, 3, 8)
    assert float((c.k.float() * c.k_scale.float().unsqueeze(-1)).abs().max()) == 0.0


def test_container_refuses_tensors_that_do_not_fit():
    c = _cache()
    for args in ((c.k[:, :2], c.k_scale, c.v, c.v_scale), (c.k, c.k_scale[:, :, :4], c.v, c.v_scale),
                 (c.k.view(torch.uint8), c.k_scale, c.v, c.v_scale), (c.k, c.k_scale.view(torch.uint8), c.v, c.v_scale),
                 (c.k.transpose(0, 1).contiguous().transpose(0, 1), c.k_scale, c.v, c.v_scale)):
        with pytest.raises(RuntimeError, match="QuantizedCache"):
            QuantizedCache(*args)


def _append(**over):
    from sparse_b200._lib import ROPE_APPEND, lib
    a = dict(q=OK, k_rot=OK, k_rest=OK, v=OK, seq=OK, pos=OK, q_out=OK, ck=OK, sk=OK, cv=OK, sv=OK)
    a.update({"stride%d" % i: 256 for i in range(8)}, T=4, B=2, n_q=4, n_kv=2, dk=64, dv=64, rope=32, s_max=8, theta=1e4, zero=0)
    a.update(over)
    return lib.sb_rope_append_fp8(ROPE_APPEND.pack(*(v or 0 for v in a.values())), None), lib.sb_last_error_string()


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(B=0), dict(n_q=0), dict(n_kv=0), dict(dk=8), dict(dk=72), dict(dv=272), dict(dv=0), dict(rope=8),
    dict(rope=80), dict(rope=-16), dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(s_max=0),
    dict(q=None), dict(k_rot=None), dict(k_rest=None), dict(v=None), dict(seq=None), dict(pos=None),
    dict(q_out=None), dict(ck=None), dict(sk=None), dict(cv=None), dict(sv=None), dict(q_out=OK + 2), dict(ck=OK + 8),
    dict(cv=OK + 1)])
def test_append_refuses(over):
    rc, msg = _append(**over)
    assert rc == -1 and b"sb_rope_append_fp8" in msg


def test_append_of_no_tokens_is_no_error():
    assert _append(T=0, q=None, k_rot=None)[0] == 0


def _read(**over):
    from sparse_b200._lib import CACHE_READ, lib
    a = dict(ck=OK, sk=OK, cv=OK, sv=OK, ok=OK, ov=OK, B=2, n_kv=2, dk=64, dv=64, s_max=8, begin=2, count=6, shared=3)
    a.update(over)
    return lib.sb_cache_read_fp8(CACHE_READ.pack(*(v or 0 for v in a.values())), None), lib.sb_last_error_string()


@pytest.mark.parametrize("over", [
    dict(B=-1), dict(B=65536), dict(n_kv=0), dict(dk=40), dict(dv=24), dict(s_max=0), dict(begin=-1), dict(count=-1),
    dict(count=7), dict(begin=9, count=0), dict(shared=9), dict(shared=-1), dict(ck=None), dict(sk=None), dict(cv=None), dict(sv=None),
    dict(ok=None), dict(ov=None), dict(ck=OK + 8), dict(ov=OK + 8)])
def test_read_refuses(over):
    rc, msg = _read(**over)
    assert rc == -1 and b"sb_cache_read_fp8" in msg


def test_read_of_nothing_is_no_error():
    assert _read(count=0, ck=None)[0] == 0 and _read(B=0)[0] == 0


def _attend(quantized, **over):
    from sparse_b200._lib import ATTN_CACHED, lib
    a = dict(q=OK, ck=OK, sk=OK, cv=OK, sv=OK, lens=OK, ws=OK, out=OK, status=0, q_stride=0, ws_bytes=1 << 30, B=2, n_q=4,
             n_kv=2, dk=64, dv=64, s_max=64, shared=16, scale=0.125)
    a.update(over)
    call = lib.sb_attn_decode_fp8 if quantized else lib.sb_attn_decode_shared
    return call(ATTN_CACHED.pack(*(v or 0 for v in a.values())), None), lib.sb_last_error_string()


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("over,want", [
    (dict(B=-1), -1), (dict(n_q=0), -1), (dict(n_kv=0), -1), (dict(n_q=5), -1), (dict(s_max=0), -1), (dict(shared=-1), -1),
    (dict(shared=65), -1), (dict(B=1 << 23), -1), (dict(q_stride=255), -1), (dict(q_stride=-256), -1), (dict(dk=128), -4), (dict(dv=32), -4),
    (dict(q=None), -1), (dict(ck=None), -1), (dict(cv=None), -1), (dict(lens=None), -1), (dict(ws=None), -1),
    (dict(out=None), -1), (dict(out=OK + 2), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(n_kv=65536, n_q=65536), -1), (dict(ck=OK + 8), -1), (dict(cv=OK + 4), -1), (dict(ws=OK + 8), -1), (dict(ws_bytes=0), -2)])
def test_attention_refuses(quantized, over, want):
    rc, msg = _attend(quantized, **over)
    assert rc == want and (b"sb_attn_decode_fp8" if quantized else b"sb_attn_decode_shared") in msg


def test_quantised_attention_refuses_missing_scales():
    assert _attend(True, sk=None)[0] == -1 and _attend(True, sv=None)[0] == -1


def test_missing_structs_are_refused():
    from sparse_b200._lib import lib
    for call in (lib.sb_rope_append_fp8, lib.sb_cache_read_fp8, lib.sb_attn_decode_fp8, lib.sb_attn_decode_shared):
        assert call(None, None) == -1 and b"null pointer" in lib.sb_last_error_string()
    assert lib.sb_cache_struct_bytes(3) == 0 and lib.sb_cache_struct_bytes(-1) == 0


def test_attention_of_no_sequences_is_no_error():
    assert _attend(True, B=0, q=None)[0] == 0 and _attend(False, B=0, ck=None)[0] == 0


def test_tensor_wrappers_refuse_before_any_launch():
    """CPU tensors, and operands whose shapes or types do not fit (there is no CPU path)."""
    from sparse_b200 import ops
    c, bf = _cache(), torch.bfloat16
    q, lens = torch.zeros(2, 3, 64, dtype=bf), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_quantized(q, c, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_shared(q, torch.zeros(2, 8, 3, 64, dtype=bf), torch.zeros(2, 8, 3, 64, dtype=bf), lens, 4)
    with pytest.raises(RuntimeError, match="caches"):
        ops.attn_decode_shared(q, torch.zeros(2, 8, 3, 64, dtype=bf), torch.zeros(2, 9, 3, 64, dtype=bf), lens, 4)
    with pytest.raises(RuntimeError, match="bf16"):
        ops.attn_decode_shared(q, torch.zeros(2, 8, 3, 64), torch.zeros(2, 8, 3, 64), lens, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rope_append_quantized(q, None, q, q, lens, lens, c, 1e4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.cache_read(c, 0, 4)
