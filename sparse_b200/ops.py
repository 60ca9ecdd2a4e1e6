"""Tensor-level wrappers over the C ABI.

PyTorch is used for device memory and streams only; every computation below
is one call into libsparse_b200.  All functions run on the current CUDA stream
of the tensors' device and never synchronise.
"""
from __future__ import annotations

import ctypes
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


def _rows3(t: torch.Tensor, what: str, like: torch.Tensor, heads, width: int) -> Tuple[int, int, int]:
    """Address, token stride and head stride of a bf16 [T, heads, width] view (one head: shared)."""
    if t.dim() != 3 or t.dtype != torch.bfloat16 or t.device != like.device or t.shape[0] != like.shape[0] or (
            t.shape[1] not in heads or t.shape[2] != width):
        raise RuntimeError("rope_append_quantized: %s must be bf16 [%d, %s, %d] on %s, got %s %s on %s" % (
            what, like.shape[0], " or ".join(map(str, heads)), width, like.device, t.dtype, tuple(t.shape), t.device))
    if t.stride(2) != 1 and t.shape[2] > 1 and t.shape[0] > 0:
        raise RuntimeError("rope_append_quantized: the elements of a head of %s must lie side by side" % what)
    return t.data_ptr(), t.stride(0), t.stride(1) if t.shape[1] > 1 else 0


def _index(t: torch.Tensor, n: int, device: torch.device, what: str) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.device != device or not t.is_contiguous():
        raise RuntimeError("%s must be a contiguous int32 tensor of %d elements on %s" % (what, n, device))
    return t.data_ptr()


def rope_append_quantized(q: torch.Tensor, k_rot: Optional[torch.Tensor], k_rest: Optional[torch.Tensor],
                          v: torch.Tensor, seq_of_token: torch.Tensor, pos_of_token: torch.Tensor,
                          cache: QuantizedCache, theta: float) -> torch.Tensor:
    """Rotary embedding of q and k, and k and v quantised into the cache; returns the rotated
    queries [T, n_q, dk].

    q [T, n_q, dk]; the first part of a key head, the rotated one, is k_rot [T, n_kv or 1, r]
    (one head: shared by all), the rest k_rest [T, n_kv or 1, dk - r] (None where nothing is
    left, as k_rot where nothing is rotated); v [T, n_kv or 1, dv].  All are bf16 views with any
    token and head strides.  Token t goes to row (seq_of_token[t], pos_of_token[t]), int32; one
    outside the cache is not stored."""
    if q.dim() != 3 or q.dtype != torch.bfloat16 or q.device != cache.device or not q.is_cuda:
        raise RuntimeError("rope_append_quantized: q must be bf16 [T, n_q, dk] on the cache's CUDA device")
    t, n_q, dk = q.shape
    b, n_kv, s_max, dk_cache = cache.k.shape
    dv = cache.v.shape[3]
    rope = k_rot.shape[-1] if k_rot is not None else 0
    if dk != dk_cache or rope > dk or n_q < 1:
        raise RuntimeError("rope_append_quantized: heads of %d and a cache of heads of %d" % (dk, dk_cache))
    if (k_rest is None) != (rope == dk):
        raise RuntimeError("rope_append_quantized: k_rest holds the %d unrotated elements of a key head" % (dk - rope))
    strides, ptrs = [], []
    for view, what, heads, width in ((q, "q", (n_q,), dk), (k_rot, "k_rot", (n_kv, 1), rope),
                                     (k_rest, "k_rest", (n_kv, 1), dk - rope), (v, "v", (n_kv, 1), dv)):
        ptr, token, head = _rows3(view, what, q, heads, width) if view is not None else (None, 0, 0)
        ptrs.append(ptr)
        strides += [token, head]
    seq, pos = (_index(x, t, q.device, "rope_append_quantized: " + n) for x, n in
                ((seq_of_token, "seq_of_token"), (pos_of_token, "pos_of_token")))
    out = torch.empty((t, n_q, dk), dtype=torch.bfloat16, device=q.device)
    with torch.cuda.device(q.device):
        check(lib.sb_rope_append_fp8(*ptrs, seq, pos, t, b, n_q, n_kv, dk, dv, rope, theta, s_max,
                                     (ctypes.c_int64 * 8)(*strides), out.data_ptr(), cache.k.data_ptr(),
                                     cache.k_scale.data_ptr(), cache.v.data_ptr(), cache.v_scale.data_ptr(), _stream(q)),
              "sb_rope_append_fp8")
    return out


def cache_read(cache: QuantizedCache, begin: int, count: int, shared_len: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Positions begin .. begin+count-1 of every sequence as bf16: (k [B, n_kv, count, dk],
    v [B, n_kv, count, dv]), exactly the values the codes stand for.  Positions below
    `shared_len` are sequence 0's."""
    b, n_kv, s_max, dk = cache.k.shape
    dv = cache.v.shape[3]
    if not cache.k.is_cuda:
        raise RuntimeError("sparse_b200 ops need CUDA tensors (there is no CPU path)")
    if begin < 0 or count < 0 or begin + count > s_max or not 0 <= shared_len <= s_max:
        raise RuntimeError("cache_read: positions %d .. %d, %d of them shared, of a cache of %d" % (
            begin, begin + count, shared_len, s_max))
    k = torch.empty((b, n_kv, count, dk), dtype=torch.bfloat16, device=cache.device)
    v = torch.empty((b, n_kv, count, dv), dtype=torch.bfloat16, device=cache.device)
    with torch.cuda.device(cache.device):
        check(lib.sb_cache_read_fp8(_ptr(cache.k), _ptr(cache.k_scale), _ptr(cache.v), _ptr(cache.v_scale), b, n_kv, dk, dv,
                                    s_max, begin, count, shared_len, k.data_ptr(), v.data_ptr(), _stream(k)),
              "sb_cache_read_fp8")
    return k, v


def _attn_operands(name: str, q: torch.Tensor, seq_lens: torch.Tensor, batch: int, n_kv: int, dk: int, dv: int, s_max: int,
                   shared_len: int, device: torch.device, status: Optional[torch.Tensor]):
    """Checks; -> (seq_lens, status, output, workspace) of a decode attention call."""
    if q.dim() != 3 or q.dtype != torch.bfloat16 or q.device != device or not q.is_cuda or q.shape[0] != batch or (
            q.shape[2] != dk or q.shape[1] < 1):
        raise RuntimeError("%s: q must be bf16 [%d, n_q, %d] on the cache's CUDA device, got %s %s on %s" % (
            name, batch, dk, q.dtype, tuple(q.shape), q.device))
    if batch > 0 and (q.stride(2) != 1 or (q.shape[1] > 1 and q.stride(1) != dk)) or (
            batch > 1 and q.stride(0) < q.shape[1] * dk):
        raise RuntimeError("%s: the heads of a sequence's query must lie side by side, sequences apart" % name)
    if not 0 <= shared_len <= s_max:
        raise RuntimeError("%s: %d shared positions of a cache of %d" % (name, shared_len, s_max))
    if status is not None and (status.dtype != torch.int32 or status.device != device):
        raise RuntimeError("%s: status must be int32 on %s" % (name, device))
    lens = _index(seq_lens, batch, device, name + ": seq_lens")
    n_q = q.shape[1]
    out = torch.empty((batch, n_q, dv), dtype=torch.bfloat16, device=device)
    ws_bytes = lib.sb_attn_cached_workspace_bytes(batch, n_q, n_kv, dv, s_max, shared_len)
    return lens, _ptr(status), out, torch.empty((max(ws_bytes, 16),), dtype=torch.uint8, device=device)


def attn_decode_quantized(q: torch.Tensor, cache: QuantizedCache, seq_lens: torch.Tensor, shared_len: int = 0,
                          scale: Optional[float] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query per sequence, q [B, n_q, dk] bf16, against the first seq_lens[b] (int32)
    positions of its quantised cache -> [B, n_q, dv]; zeros where there are none.

    n_q is a multiple of the cache's heads.  `shared_len`: as many first positions are the
    same for the whole batch and stand in sequence 0's rows; they are read once.  `scale`
    defaults to dk ** -0.5; `status` as in `grouped_swiglu`."""
    b, n_kv, s_max, dk = cache.k.shape
    dv = cache.v.shape[3]
    lens, st, out, ws = _attn_operands("attn_decode_quantized", q, seq_lens, b, n_kv, dk, dv, s_max, shared_len, cache.device,
                                       status)
    with torch.cuda.device(q.device):
        check(lib.sb_attn_decode_fp8(q.data_ptr(), q.stride(0) if b > 1 else 0, _ptr(cache.k), _ptr(cache.k_scale),
                                     _ptr(cache.v), _ptr(cache.v_scale), lens, b, q.shape[1], n_kv, dk, dv, s_max,
                                     shared_len, dk ** -0.5 if scale is None else scale, ws.data_ptr(), ws.numel(),
                                     out.data_ptr(), st, _stream(q)), "sb_attn_decode_fp8")
    return out


def attn_decode_shared(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, seq_lens: torch.Tensor,
                       shared_len: int, scale: Optional[float] = None,
                       status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`attn_decode_quantized` over a bf16 cache, cache_k [B, S, n_kv, dk] and cache_v
    [B, S, n_kv, dv]: the first `shared_len` positions of the batch stand in sequence 0's
    rows and are read once for all sequences."""
    if cache_k.dim() != 4 or cache_v.dim() != 4 or cache_k.shape[:3] != cache_v.shape[:3]:
        raise RuntimeError("attn_decode_shared: caches [B, S, n_kv, d] do not fit: %s and %s" % (
            tuple(cache_k.shape), tuple(cache_v.shape)))
    if any(c.dtype != torch.bfloat16 or c.device != cache_k.device for c in (cache_k, cache_v)):
        raise RuntimeError("attn_decode_shared needs bf16 caches on one device")
    b, s_max, n_kv, dk = cache_k.shape
    dv = cache_v.shape[3]
    lens, st, out, ws = _attn_operands("attn_decode_shared", q, seq_lens, b, n_kv, dk, dv, s_max, shared_len, cache_k.device,
                                       status)
    with torch.cuda.device(q.device):
        check(lib.sb_attn_decode_shared(q.data_ptr(), q.stride(0) if b > 1 else 0, _ptr(cache_k), _ptr(cache_v), lens, b,
                                        q.shape[1], n_kv, dk, dv, s_max, shared_len, dk ** -0.5 if scale is None else scale,
                                        ws.data_ptr(), ws.numel(), out.data_ptr(), st, _stream(q)), "sb_attn_decode_shared")
    return out


def slot_copy_async(dst: torch.Tensor, src: torch.Tensor, stream: torch.cuda.Stream,
                    kind: int) -> None:
    """Copy `src` (pinned host, peer or local device tensor) into the cache slot `dst`."""
    if dst.numel() * dst.element_size() != src.numel() * src.element_size():
        raise RuntimeError("slot copy size mismatch")
    if not dst.is_contiguous() or not src.is_contiguous():
        raise RuntimeError("slot copy needs contiguous tensors")
    check(lib.sb_slot_copy_async(dst.data_ptr(), src.data_ptr(), dst.numel() * dst.element_size(),
                                 kind, dst.device.index, stream.cuda_stream), "sb_slot_copy_async")
