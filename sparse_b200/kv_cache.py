"""A key/value cache in 8-bit floating point.

Half the bytes of the bf16 cache: what a decode step's attention reads, and what a
context of a given length takes of HBM.  Written by `ops.rope_append_quantized`, read by
`ops.attn_decode_quantized` and, as bf16, by `ops.cache_read`.

The row of a (sequence, head, position) is e4m3 codes and one power of two, the least
one (2^-127 or more) by which the row's largest magnitude is at most 448.  A row with an
infinity or a NaN has scale byte 255 and no e4m3 NaN among its codes; in a cache that somebody
filled by a cast of their own the codes 0x7f and 0xff read as NaN.  Heads come before positions,
unlike in the bf16 cache: a head's codes are then one run of bytes, and so are its scales, of which
a position has only one byte per head.
"""
from __future__ import annotations

import torch

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


class QuantizedCache:
    """k [B, n_kv, S, dk] and v [B, n_kv, S, dv] codes, k_scale and v_scale [B, n_kv, S]."""
    __slots__ = ("k", "k_scale", "v", "v_scale")

    def __init__(self, k: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor, v_scale: torch.Tensor):
        rows, device = k_scale.shape, k.get_device()
        if len(rows) != 3 or k.shape[:-1] != rows or v.shape[:-1] != rows or v_scale.shape != rows:
            raise RuntimeError("QuantizedCache: codes [B, n_kv, S, d] and scales [B, n_kv, S] do not fit: %s" % (
                [tuple(t.shape) for t in (k, k_scale, v, v_scale)],))
        if k.dtype is not CODES or v.dtype is not CODES or k_scale.dtype is not SCALES or v_scale.dtype is not SCALES or (
                v.get_device() != device) or k_scale.get_device() != device or v_scale.get_device() != device or not (
                k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise RuntimeError("QuantizedCache needs contiguous %s codes and %s scales on one device" % (CODES, SCALES))
        self.k, self.k_scale, self.v, self.v_scale = k, k_scale, v, v_scale

    @classmethod
    def zeros(cls, batch: int, max_seq: int, n_kv: int, dk: int, dv: int, device) -> "QuantizedCache":
        """A cache whose every position reads back as zero."""
        def z(*shape, dtype):
            return torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        return cls(z(batch, n_kv, max_seq, dk, dtype=CODES), z(batch, n_kv, max_seq, dtype=SCALES),
                   z(batch, n_kv, max_seq, dv, dtype=CODES), z(batch, n_kv, max_seq, dtype=SCALES))

    @property
    def device(self) -> torch.device:
        return self.k.device
