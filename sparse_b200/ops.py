"""Tensor-level wrappers over the C ABI.

PyTorch is used for device memory and streams only; every computation below
is one call into libsparse_b200.  All functions run on the current CUDA stream
of the tensors' device and never synchronise.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import lib, check
from .kv_cache import QuantizedCache

_DT = {torch.bfloat16: _lib.SB_DTYPE_BF16, torch.float32: _lib.SB_DTYPE_F32}


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError("sparse_b200 ops need CUDA tensors (there is no CPU path)")
    if not t.is_contiguous():
        raise RuntimeError("sparse_b200 ops need contiguous tensors")
    return t.data_ptr()


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def pad_rows(n: int) -> int:
    """Row capacity the grouped GEMM wants for n rows (a whole number of tiles)."""
    return max(1, (max(n, 1) + _lib.SB_TILE_M - 1) // _lib.SB_TILE_M) * _lib.SB_TILE_M


def router_topk(x: torch.Tensor, wg: torch.Tensor, top_k: int,
                bias: Optional[torch.Tensor] = None,
                w_shared_gate: Optional[torch.Tensor] = None,
                renorm: bool = False, fp32_logits: bool = False,
                want_logits: bool = True):
    """-> (idx int32 [T,K], weights [T,K], logits [T,E] | None, shared_scale [T] | None)."""
    t, h = x.shape
    e = wg.shape[0]
    dev, dt = x.device, x.dtype
    idx = torch.empty((t, top_k), dtype=torch.int32, device=dev)
    w = torch.empty((t, top_k), dtype=dt, device=dev)
    logits = None
    if want_logits:
        logits = torch.empty((t, e), dtype=torch.float32 if fp32_logits else dt, device=dev)
    shared = torch.empty((t,), dtype=dt, device=dev) if w_shared_gate is not None else None
    bias_f = None
    if bias is not None:
        bias_f = bias.to(dt).to(torch.float32).contiguous()
    with torch.cuda.device(dev):
        check(lib.sb_router_topk(_ptr(x), _ptr(wg), _ptr(bias_f), _ptr(w_shared_gate), t, h, e,
                                 top_k, int(renorm), _DT[dt], int(fp32_logits), _ptr(idx), _ptr(w),
                                 _ptr(logits), _ptr(shared), _stream(x)), "sb_router_topk")
    return idx, w, logits, shared


def softmax_topk(logits: torch.Tensor, top_k: int, renorm: bool = False):
    t, e = logits.shape
    idx = torch.empty((t, top_k), dtype=torch.int32, device=logits.device)
    w = torch.empty((t, top_k), dtype=logits.dtype, device=logits.device)
    with torch.cuda.device(logits.device):
        check(lib.sb_softmax_topk(_ptr(logits), t, e, top_k, int(renorm), _DT[logits.dtype],
                                  _ptr(idx), _ptr(w), _stream(logits)), "sb_softmax_topk")
    return idx, w


class Permutation:
    """Outputs of `permute` (all device tensors)."""
    __slots__ = ("rows", "expert_offsets", "slot_of_item", "item_of_slot", "slot_scale",
                 "tile_table", "n_items", "r_cap")


def permute(x: torch.Tensor, item_expert: torch.Tensor, num_experts: int,
            items_per_row: int, item_scale: Optional[torch.Tensor] = None) -> Permutation:
    n = item_expert.numel()
    h = x.shape[1]
    dev = x.device
    p = Permutation()
    p.n_items, p.r_cap = n, pad_rows(n)
    p.rows = torch.empty((p.r_cap, h), dtype=torch.bfloat16, device=dev)
    p.expert_offsets = torch.empty((num_experts + 1,), dtype=torch.int32, device=dev)
    p.slot_of_item = torch.empty((max(n, 1),), dtype=torch.int32, device=dev)
    p.item_of_slot = torch.empty((max(n, 1),), dtype=torch.int32, device=dev)
    p.slot_scale = (torch.empty((p.r_cap,), dtype=torch.bfloat16, device=dev)
                    if item_scale is not None else None)
    p.tile_table = torch.empty((lib.sb_tile_table_ints(n, num_experts),), dtype=torch.int32, device=dev)
    ws_bytes = lib.sb_permute_workspace_bytes(n, num_experts)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        check(lib.sb_permute(_ptr(x), _ptr(item_expert), _ptr(item_scale), n, items_per_row, h,
                             num_experts, _ptr(ws), ws_bytes, _ptr(p.rows), _ptr(p.expert_offsets),
                             _ptr(p.slot_of_item), _ptr(p.item_of_slot), _ptr(p.slot_scale),
                             _ptr(p.tile_table), _stream(x)), "sb_permute")
    return p


def grouped_swiglu(rows: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
                   tile_table: Optional[torch.Tensor] = None, dense_rows: int = 0,
                   slot_of_expert: Optional[torch.Tensor] = None,
                   row_scale: Optional[torch.Tensor] = None,
                   status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """rows [R_cap,H]; w13 [S,2I,H]; w2 [S,H,I] -> (out [R_cap,H], h [R_cap,I])."""
    r_cap, h = rows.shape
    s, two_i, _ = w13.shape
    i = two_i // 2
    dev = rows.device
    hbuf = torch.empty((r_cap, i), dtype=torch.bfloat16, device=dev)
    out = torch.empty((r_cap, h), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        check(lib.sb_grouped_swiglu(_ptr(rows), _ptr(tile_table), dense_rows, _ptr(w13), _ptr(w2),
                                    _ptr(slot_of_expert), _ptr(row_scale), r_cap, h, i, s,
                                    _ptr(hbuf), _ptr(out), _ptr(status), _stream(rows)),
              "sb_grouped_swiglu")
    return out, hbuf


def dense_swiglu(rows: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor) -> torch.Tensor:
    """One SwiGLU FFN over all rows: rows [T,H]; w13 [1,2I,H]; w2 [1,H,I] -> [T,H], bf16.

    Up to `_lib.DECODE_MAX_TOKENS` rows the FFN is its weights' bytes, and the streaming
    kernels read them with every SM; the tile kernel would walk the output in 256-row
    tiles, for 10944 x 2048 eight of them in the down pass, on eight of the 74 CTA pairs
    (26 + 52 us for 134 MB at one row).  Operands are those of the tile kernel either way."""
    t, h = rows.shape
    i = w13.shape[1] // 2
    if w13.shape[1:] != (2 * i, h) or w2.shape[1:] != (h, i):
        raise RuntimeError("dense_swiglu: rows %s, w13 %s and w2 %s do not fit" % (
            tuple(rows.shape), tuple(w13.shape), tuple(w2.shape)))
    for v in (rows, w13, w2):
        if v.dtype != torch.bfloat16 or v.device != rows.device:
            raise RuntimeError("dense_swiglu needs bf16 operands on one device")
    if t > _lib.DECODE_MAX_TOKENS or h % 64 != 0 or i % 64 != 0 or any(
            _ptr(v) % 128 != 0 for v in (rows, w13, w2)):
        return grouped_swiglu(rows, w13, w2, dense_rows=t)[0][:t]
    hbuf = torch.empty((t, i), dtype=torch.bfloat16, device=rows.device)
    out = torch.empty((t, h), dtype=torch.bfloat16, device=rows.device)
    with torch.cuda.device(rows.device):
        check(lib.sb_decode_experts(_ptr(rows), None, 1, None, None, None, None, None, h, i, 1, None, None,
                                    _ptr(w13), _ptr(w2), None, i, t, _ptr(hbuf), _ptr(out), None, _stream(rows)),
              "sb_decode_experts(dense)")
    return out


def _streams(rows: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> bool:
    """Whether `sb_decode_linear` takes the operands: a few packed bf16 rows, whole 16-byte
    vectors, nothing that wants a gradient."""
    if rows.dim() != 2 or weight.dim() != 2 or not 0 < rows.shape[0] <= _lib.DECODE_MAX_TOKENS:
        return False
    n, k = weight.shape
    if not 0 < n <= 2 ** 27 or k == 0 or k % 32 != 0 or rows.shape[1] != k or (bias is not None and bias.shape != (n,)):
        return False
    operands = [v for v in (rows, weight, bias) if v is not None]
    if any(v.dtype != torch.bfloat16 or not v.is_cuda or v.device != rows.device or not v.is_contiguous()
           for v in operands):
        return False
    if torch.is_grad_enabled() and any(v.requires_grad for v in operands):
        return False
    return rows.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0


def linear(rows: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """rows [T,K] . weight [N,K]^T (+ bias): the weight-streaming kernel up to
    `_lib.DECODE_MAX_TOKENS` bf16 rows (8 MB of weights: 7 us through the library at one
    to eight rows, most of them not spent on the bytes), the library's GEMM above and
    for all operands that the kernel is not made for."""
    if not _streams(rows, weight, bias):
        return torch.nn.functional.linear(rows, weight, bias)
    (t, k), n = rows.shape, weight.shape[0]
    out = torch.empty((t, n), dtype=torch.bfloat16, device=rows.device)
    with torch.cuda.device(rows.device):
        check(lib.sb_decode_linear(_ptr(rows), _ptr(weight), _ptr(bias), t, n, k, _ptr(out), _stream(rows)),
              "sb_decode_linear")
    return out


def combine(rows_out: torch.Tensor, slot_of_item: torch.Tensor, idx: torch.Tensor,
            shared_out: Optional[torch.Tensor], tokens: int,
            shared_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`shared_scale` [T] bf16: the shared expert's scalar gate, applied to `shared_out`'s
    rows on the way (sb_combine_gated)."""
    h = rows_out.shape[1]
    k = idx.shape[1]
    out = torch.empty((tokens, h), dtype=torch.bfloat16, device=rows_out.device)
    with torch.cuda.device(rows_out.device):
        if shared_scale is None:
            check(lib.sb_combine(_ptr(rows_out), _ptr(slot_of_item), _ptr(idx), _ptr(shared_out), tokens,
                                 h, k, _ptr(out), _stream(rows_out)), "sb_combine")
        else:
            check(lib.sb_combine_gated(_ptr(rows_out), _ptr(slot_of_item), _ptr(idx), _ptr(shared_out),
                                       _ptr(shared_scale), tokens, h, k, _ptr(out), _stream(rows_out)),
                  "sb_combine_gated")
    return out


# The calls of a decode step, of which a layer makes several and whose kernels take a few
# microseconds: checks without tensor temporaries, the stream's handle without a Stream object, a
# device guard only where another device is current.
def _call(fn, what: str, device: int, args: bytes) -> None:
    """fn(args, stream) with `device` current, its current stream; raises on a status."""
    if torch._C._cuda_getDevice() == device:
        status = fn(args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = fn(args, torch._C._cuda_getCurrentRawStream(device))
    if status != 0:
        check(status, what)


# (the sizes of a serving loop's calls are few: one look-up instead of a call into the library)
_attn_workspace = functools.lru_cache(maxsize=1024)(lib.sb_attn_cached_workspace_bytes)


@functools.lru_cache(maxsize=64)
def _two_floats(x: float) -> Tuple[float, float]:
    """x as its fp32 rounding and what that leaves."""
    hi = ctypes.c_float(x).value
    return hi, x - hi


def _index(t: torch.Tensor, n: int, device: int, what: str) -> int:
    if t.dtype is not torch.int32 or t.get_device() != device or t.shape != (n,) or not t.is_contiguous():
        raise RuntimeError("%s must be a contiguous int32 tensor of %d elements on CUDA device %d" % (what, n, device))
    return t.data_ptr()


def _cache_device(cache: QuantizedCache) -> int:
    device = cache.k.get_device()
    if device < 0:
        raise RuntimeError("sparse_b200 ops need CUDA tensors (there is no CPU path)")
    return device


def _head_rows(view: Optional[torch.Tensor], t: int, heads: int, width: int, device: int) -> Tuple[int, int, int]:
    """Address, token stride and head stride (0: one head for all) of bf16 rows [t, heads or 1, width]."""
    if view is None:
        return 0, 0, 0
    shape = view.shape
    if len(shape) != 3 or shape[0] != t or shape[1] != heads and shape[1] != 1 or shape[2] != width or (
            view.dtype is not torch.bfloat16) or view.get_device() != device:
        raise RuntimeError("rope_append_quantized: needs bf16 [%d, %d or 1, %d] on the cache's device, got %s %s" % (
            t, heads, width, view.dtype, tuple(shape)))
    token, head, element = view.stride()
    if element != 1 and t > 0:
        raise RuntimeError("rope_append_quantized: the elements of a head must lie side by side")
    return view.data_ptr(), token, head if shape[1] > 1 else 0


def rope_append_quantized(q: torch.Tensor, k_rot: Optional[torch.Tensor], k_rest: Optional[torch.Tensor],
                          v: torch.Tensor, seq_of_token: torch.Tensor, pos_of_token: torch.Tensor,
                          cache: QuantizedCache, theta: float) -> torch.Tensor:
    """Rotary embedding of q and k, and k and v quantised into the cache; returns the rotated
    queries [T, n_q, dk].

    q [T, n_q, dk]; the first part of a key head, the rotated one, is k_rot [T, n_kv or 1, r]
    (one head: shared by all), the rest k_rest [T, n_kv or 1, dk - r] (None where nothing is
    left, as k_rot where nothing is rotated); v [T, n_kv or 1, dv].  All are bf16 views with any
    token and head strides.  Token t goes to row (seq_of_token[t], pos_of_token[t]), int32; one
    outside the cache is not stored.  Two tokens of a call must not name the same row.  `theta`,
    the base of the angles, is taken in 64 bits (to 48 of its bits)."""
    device = _cache_device(cache)
    b, n_kv, s_max, dk = cache.k.shape
    dv = cache.v.shape[3]
    rope = 0 if k_rot is None else k_rot.shape[-1]
    shape = q.shape
    if len(shape) != 3 or shape[1] < 1 or shape[2] != dk or rope > dk or (k_rest is None) != (rope == dk):
        raise RuntimeError("rope_append_quantized: q %s and a key of %d rotated and %s other elements for a cache of heads of %d"
                           % (tuple(shape), rope, None if k_rest is None else k_rest.shape[-1], dk))
    t, n_q, _ = shape
    q_ptr, q_token, q_head = _head_rows(q, t, n_q, dk, device)
    rot_ptr, rot_token, rot_head = _head_rows(k_rot, t, n_kv, rope, device)
    rest_ptr, rest_token, rest_head = _head_rows(k_rest, t, n_kv, dk - rope, device)
    v_ptr, v_token, v_head = _head_rows(v, t, n_kv, dv, device)
    seq = _index(seq_of_token, t, device, "rope_append_quantized: seq_of_token")
    pos = _index(pos_of_token, t, device, "rope_append_quantized: pos_of_token")
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    _call(lib.sb_rope_append_fp8, "sb_rope_append_fp8", device, _lib.ROPE_APPEND.pack(
        q_ptr, rot_ptr, rest_ptr, v_ptr, seq, pos, out.data_ptr(), cache.k.data_ptr(), cache.k_scale.data_ptr(),
        cache.v.data_ptr(), cache.v_scale.data_ptr(), q_token, q_head, rot_token, rot_head, rest_token, rest_head, v_token,
        v_head, t, b, n_q, n_kv, dk, dv, rope, s_max, *_two_floats(float(theta))))
    return out


def cache_read(cache: QuantizedCache, begin: int, count: int, shared_len: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Positions begin .. begin+count-1 of every sequence as bf16: (k [B, n_kv, count, dk],
    v [B, n_kv, count, dv]), exactly the values the codes stand for (but for those under bf16's
    smallest step, 2^-133).  Positions below `shared_len` are sequence 0's."""
    device = _cache_device(cache)
    b, n_kv, s_max, dk = cache.k.shape
    dv = cache.v.shape[3]
    if begin < 0 or count < 0 or begin + count > s_max or not 0 <= shared_len <= s_max:
        raise RuntimeError("cache_read: positions %d .. %d, %d of them shared, of a cache of %d" % (
            begin, begin + count, shared_len, s_max))
    k = cache.k.new_empty((b, n_kv, count, dk), dtype=torch.bfloat16)
    v = k.new_empty((b, n_kv, count, dv))
    _call(lib.sb_cache_read_fp8, "sb_cache_read_fp8", device, _lib.CACHE_READ.pack(
        cache.k.data_ptr(), cache.k_scale.data_ptr(), cache.v.data_ptr(), cache.v_scale.data_ptr(), k.data_ptr(),
        v.data_ptr(), b, n_kv, dk, dv, s_max, begin, count, shared_len))
    return k, v


def _decode_attention(name: str, call, q: torch.Tensor, cache_ptrs, seq_lens: torch.Tensor, b: int, n_kv: int, dk: int,
                      dv: int, s_max: int, shared_len: int, scale: Optional[float], status: Optional[torch.Tensor],
                      device: int) -> torch.Tensor:
    """Checks of the operands that both kinds of cache share, output and workspace, the call."""
    shape = q.shape
    if len(shape) != 3 or q.dtype is not torch.bfloat16 or q.get_device() != device or shape[0] != b or shape[2] != dk or (
            shape[1] < 1):
        raise RuntimeError("%s: q must be bf16 [%d, n_q, %d] on the cache's device, got %s %s on %s" % (
            name, b, dk, q.dtype, tuple(shape), q.device))
    n_q, seq_stride, packed = shape[1], 0, q.is_contiguous()
    if not packed:
        seq_stride, head_stride, element = q.stride()
        if element != 1 or (n_q > 1 and head_stride != dk) or (b > 1 and seq_stride < n_q * dk):
            raise RuntimeError("%s: the heads of a sequence's query must lie side by side, sequences apart" % name)
    if not 0 <= shared_len <= s_max:
        raise RuntimeError("%s: %d shared positions of a cache of %d" % (name, shared_len, s_max))
    if status is not None and (status.dtype != torch.int32 or status.get_device() != device or status.numel() < 1):
        raise RuntimeError("%s: status must be int32 on the cache's device" % name)
    lens = _index(seq_lens, b, device, name)
    out = torch.empty_like(q) if dv == dk and packed else q.new_empty((b, n_q, dv))
    ws_bytes = _attn_workspace(b, n_q, n_kv, dk, dv, s_max, shared_len) or 16
    ws = seq_lens.new_empty((ws_bytes + 3) // 4)          # (without a dtype of its own: half a microsecond less)
    _call(call, name, device, _lib.ATTN_CACHED.pack(
        q.data_ptr(), *cache_ptrs, lens, ws.data_ptr(), out.data_ptr(), 0 if status is None else status.data_ptr(),
        seq_stride if b > 1 else 0, ws_bytes, b, n_q, n_kv, dk, dv, s_max, shared_len, dk ** -0.5 if scale is None else scale))
    return out


def attn_decode_quantized(q: torch.Tensor, cache: QuantizedCache, seq_lens: torch.Tensor, shared_len: int = 0,
                          scale: Optional[float] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query per sequence, q [B, n_q, dk] bf16, against the first seq_lens[b] (int32)
    positions of its quantised cache -> [B, n_q, dv]; zeros where there are none.

    n_q is a multiple of the cache's heads.  `shared_len`: as many first positions are the
    same for the whole batch and stand in sequence 0's rows; they are read once.  `scale`
    (at least 0) defaults to dk ** -0.5; `status` (int32 on the device) becomes non-zero if a bounded
    wait gave up, and the outputs that depend on it NaN."""
    b, n_kv, s_max, dk = cache.k.shape
    ptrs = (cache.k.data_ptr(), cache.k_scale.data_ptr(), cache.v.data_ptr(), cache.v_scale.data_ptr())
    return _decode_attention("attn_decode_quantized", lib.sb_attn_decode_fp8, q, ptrs, seq_lens, b, n_kv, dk, cache.v.shape[3],
                             s_max, shared_len, scale, status, _cache_device(cache))


def attn_decode_shared(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, seq_lens: torch.Tensor,
                       shared_len: int, scale: Optional[float] = None,
                       status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`attn_decode_quantized` over a bf16 cache, cache_k [B, S, n_kv, dk] and cache_v
    [B, S, n_kv, dv]: the first `shared_len` positions of the batch stand in sequence 0's
    rows and are read once for all sequences.  Probabilities are rounded to bf16 before they are multiplied
    with values (`sb_attn_decode`, which the model uses where nothing is shared, keeps them in fp32)."""
    if cache_k.dim() != 4 or cache_v.dim() != 4 or cache_k.shape[:3] != cache_v.shape[:3]:
        raise RuntimeError("attn_decode_shared: caches [B, S, n_kv, d] do not fit: %s and %s" % (
            tuple(cache_k.shape), tuple(cache_v.shape)))
    device = cache_k.get_device()
    if cache_k.dtype != torch.bfloat16 or cache_v.dtype != torch.bfloat16 or cache_v.get_device() != device:
        raise RuntimeError("attn_decode_shared needs bf16 caches on one device")
    b, s_max, n_kv, dk = cache_k.shape
    return _decode_attention("attn_decode_shared", lib.sb_attn_decode_shared, q, (_ptr(cache_k), 0, _ptr(cache_v), 0), seq_lens, b,
                             n_kv, dk, cache_v.shape[3], s_max, shared_len, scale, status, device)


def slot_copy_async(dst: torch.Tensor, src: torch.Tensor, stream: torch.cuda.Stream,
                    kind: int) -> None:
    """Copy `src` (pinned host, peer or local device tensor) into the cache slot `dst`."""
    if dst.numel() * dst.element_size() != src.numel() * src.element_size():
        raise RuntimeError("slot copy size mismatch")
    if not dst.is_contiguous() or not src.is_contiguous():
        raise RuntimeError("slot copy needs contiguous tensors")
    check(lib.sb_slot_copy_async(dst.data_ptr(), src.data_ptr(), dst.numel() * dst.element_size(),
                                 kind, dst.device.index, stream.cuda_stream), "sb_slot_copy_async")
