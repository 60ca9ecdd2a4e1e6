"""The measured calls of the quantised key/value cache and of decode attention over it.

Four kinds of work, told apart by a case's ``kind``:

* ``append``  one pass's keys and values rotated, quantised and written to the cache
              (`ops.rope_append_quantized`), queries rotated on the way;
* ``read``    cached positions back as bf16 (`ops.cache_read`), what the prompt pass
              of a later chunk attends to;
* ``decode``  one query per sequence against its quantised cache
              (`ops.attn_decode_quantized`);
* ``shared``  one query per sequence where the first positions are the same for the
              whole batch and lie in the cache of sequence 0 only
              (`ops.attn_decode_shared` over a bf16 cache, `ops.attn_decode_quantized`
              with a shared length over a quantised one).

A quantised cache holds, for every sequence, head and position, the row's values as
e4m3 codes and one power of two: the least one, 2^-127 or more, by which the row's
largest magnitude is at most 448.  Head layouts are those of the model shapes of
`sparse_b200.model` (16 heads of 128; 16 of 192/128 with 64 rotary; 4 of 64) and
generic layouts in which several query heads share a key head.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
# name -> query heads, key heads, key width, value width, rotary part of a key, rotary part shared by the heads
LAYOUTS = {
    "mha128": (16, 16, 128, 128, 128, False),
    "mla192": (16, 16, 192, 128, 64, True),
    "mha64": (4, 4, 64, 64, 64, False),
    "gqa128": (32, 8, 128, 128, 128, False),
    "gqa64": (8, 2, 64, 64, 64, False),
    "wide128": (32, 4, 128, 128, 128, False),
    "mqa128": (20, 1, 128, 128, 128, False),
}
ROOM = 40          # free positions behind the last one in use


def listed():
    return [
        # a decode step of eight sequences writes one position each: latency
        {"name": "append_8", "kind": "append", "layout": "mha128", "batch": 8, "tokens": 1, "past": 2048},
        # a later prompt chunk of eight sequences, 4096 tokens in all
        {"name": "append_8x512", "kind": "append", "layout": "mha128", "batch": 8, "tokens": 512, "past": 1024},
        # the whole prompt of one sequence, odd length, rotary key part shared by the heads
        {"name": "append_mla_1003", "kind": "append", "layout": "mla192", "batch": 1, "tokens": 1003, "past": 0},
        # a short context read back for a second prompt chunk
        {"name": "read_1x700", "kind": "read", "layout": "mha64", "batch": 1, "count": 700, "shared": 0},
        # eight sequences read back for a late prompt chunk, half of it a common prefix
        {"name": "read_8x4096", "kind": "read", "layout": "mha128", "batch": 8, "count": 4096, "shared": 2048},
        # one sequence generating
        {"name": "decode_1x1000", "kind": "decode", "layout": "mha128", "batch": 1, "context": 1000, "ragged": False},
        # a small batch of equally long contexts
        {"name": "decode_8x2048", "kind": "decode", "layout": "mha128", "batch": 8, "context": 2048, "ragged": False},
        # odd batch and length, keys wider than values
        {"name": "decode_mla_5x2751", "kind": "decode", "layout": "mla192", "batch": 5, "context": 2751, "ragged": False},
        # a serving batch: lengths from an empty slot to 16384, four query heads to a key head
        {"name": "decode_gqa_64_ragged", "kind": "decode", "layout": "gqa128", "batch": 64, "context": 16384,
         "ragged": True},
        # three short requests behind a common instruction
        {"name": "shared_3x500", "kind": "shared", "layout": "mha128", "batch": 3, "prefix": 500, "context": 40,
         "cache": "bf16"},
        # a batch behind a system prompt, bf16 cache
        {"name": "shared_32x8192", "kind": "shared", "layout": "mha128", "batch": 32, "prefix": 8192, "context": 300,
         "cache": "bf16"},
        # a large batch behind a long document, quantised, eight query heads to a key head: rows for the tensor cores
        {"name": "shared_fp8_64x16384", "kind": "shared", "layout": "wide128", "batch": 64, "prefix": 16384,
         "context": 1000, "cache": "fp8"},
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["append", "read", "decode", "shared"], [3, 2, 4, 4])[0]
    case = {"kind": kind, "layout": rng.choice(sorted(LAYOUTS))}
    if kind == "append":
        total = _log_uniform(rng, 1, 4096)
        batch = min(total, _log_uniform(rng, 1, 64))
        return {**case, "batch": batch, "tokens": total // batch, "past": rng.choice([0, _log_uniform(rng, 1, 32000)])}
    if kind == "read":
        batch, count = _log_uniform(rng, 1, 16), _log_uniform(rng, 1, 4096)
        return {**case, "batch": batch, "count": count, "shared": rng.choice([0, rng.randint(0, count)])}
    if kind == "decode":
        batch = _log_uniform(rng, 1, 128)
        # no more cached positions than 16 full contexts
        context = min(_log_uniform(rng, 1, 32768), 262144 // batch)
        return {**case, "batch": batch, "context": context, "ragged": rng.random() < 0.6}
    batch = _log_uniform(rng, 2, 128)
    context = min(_log_uniform(rng, 1, 2048), 65536 // batch)
    return {**case, "batch": batch, "prefix": _log_uniform(rng, 16, 16384), "context": context,
            "cache": rng.choice(["bf16", "fp8"])}


# -- inputs ----------------------------------------------------------------------------------
def _lens(case):
    """Cached positions of every sequence behind the shared ones, in order of length."""
    batch, context = case["batch"], case["context"]
    if case["kind"] == "decode" and not case["ragged"] or batch == 1:
        return [context] * batch
    return [context * i // (batch - 1) for i in range(batch)]


def _quantize(rows):
    """bf16 or fp32 rows [..., d] -> (e4m3 codes, e8m0 powers of two [...])."""
    rows = rows.to(F32)
    m, e = torch.frexp(rows.abs().amax(-1))                           # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(m == 0, torch.full_like(e, -127), e.clamp_min(-127))
    codes = torch.ldexp(rows, -e.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _random_rows(shape, gen, device):
    """Cached rows: N(0, 1) with a level of its own for every row."""
    level = torch.exp(0.5 * torch.randn((*shape[:-1], 1), generator=gen, device=device, dtype=F32))
    return (torch.randn(shape, generator=gen, device=device, dtype=F32) * level).to(BF16)


def _random_cache(case, s_max, n_kv, dk, dv, gen, device):
    """A full cache, filled sequence by sequence."""
    batch, bf16 = case["batch"], case.get("cache", "fp8") == "bf16"
    if bf16:
        k = torch.empty((batch, s_max, n_kv, dk), dtype=BF16, device=device)
        v = torch.empty((batch, s_max, n_kv, dv), dtype=BF16, device=device)
        for b in range(batch):
            k[b], v[b] = _random_rows(k[b].shape, gen, device), _random_rows(v[b].shape, gen, device)
        return {"k": k, "v": v}
    k = torch.empty((batch, n_kv, s_max, dk), dtype=torch.float8_e4m3fn, device=device)
    v = torch.empty((batch, n_kv, s_max, dv), dtype=torch.float8_e4m3fn, device=device)
    ks = torch.empty((batch, n_kv, s_max), dtype=torch.float8_e8m0fnu, device=device)
    vs = torch.empty((batch, n_kv, s_max), dtype=torch.float8_e8m0fnu, device=device)
    for b in range(batch):
        k[b], ks[b] = _quantize(_random_rows(k[b].shape, gen, device))
        v[b], vs[b] = _quantize(_random_rows(v[b].shape, gen, device))
    return {"k": k, "ks": ks, "v": v, "vs": vs}


def prepare(case, seed: int):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed + 29)
    n_q, n_kv, dk, dv, rope, one_rotary = LAYOUTS[case["layout"]]
    batch, kind = case["batch"], case["kind"]
    state = {"case": case, "theta": 1.0e4 if one_rotary else 1.0e6, "scale": 1.0 / math.sqrt(dk)}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device, dtype=F32).to(BF16)

    if kind == "append":
        n, past = case["tokens"], case["past"]
        t, s_max = batch * n, past + n + ROOM
        if one_rotary:
            # the projections of the model: queries and rotary key part, then keys and values per head
            proj, kv = normal(t, n_q * dk + rope), normal(t, n_kv * (dk - rope + dv)).view(t, n_kv, dk - rope + dv)
            state["q"] = proj[:, :n_q * dk].view(t, n_q, dk)
            state["k_rot"], state["k_rest"] = proj[:, n_q * dk:].view(t, 1, rope), kv[..., :dk - rope]
            state["v_in"] = kv[..., dk - rope:]
        else:
            proj = normal(t, (n_q + n_kv) * dk + n_kv * dv)
            k = proj[:, n_q * dk:(n_q + n_kv) * dk].view(t, n_kv, dk)
            state["q"] = proj[:, :n_q * dk].view(t, n_q, dk)
            state["k_rot"], state["k_rest"] = k[..., :rope], k[..., rope:] if rope < dk else None
            state["v_in"] = proj[:, (n_q + n_kv) * dk:].view(t, n_kv, dv)
        state["seq"] = torch.arange(batch, dtype=torch.int32, device=device).repeat_interleave(n)
        state["pos"] = (torch.arange(n, dtype=torch.int32, device=device) + past).repeat(batch)
        state["k"] = torch.zeros((batch, n_kv, s_max, dk), dtype=torch.float8_e4m3fn, device=device)
        state["v"] = torch.zeros((batch, n_kv, s_max, dv), dtype=torch.float8_e4m3fn, device=device)
        state["ks"] = torch.zeros((batch, n_kv, s_max), dtype=torch.float8_e8m0fnu, device=device)
        state["vs"] = torch.zeros((batch, n_kv, s_max), dtype=torch.float8_e8m0fnu, device=device)
        return state
    if kind == "read":
        state.update(_random_cache(case, case["count"] + ROOM, n_kv, dk, dv, gen, device))
        return state
    prefix = case.get("prefix", 0)
    state.update(_random_cache(case, prefix + case["context"] + ROOM, n_kv, dk, dv, gen, device))
    state["q"] = normal(batch, n_q, dk)
    order = torch.randperm(batch, generator=gen, device=device)
    state["lens"] = (torch.tensor(_lens(case), dtype=torch.int32, device=device) + prefix)[order]
    return state


# -- one pass --------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _run_own(state, case, kind)
    if kind == "append":
        return _append_plain(state, case)
    if kind == "read":
        return tuple(_read_plain(state[x], state[x + "s"], case) for x in ("k", "v"))
    return _attend_plain(state, case)


def _run_own(state, case, kind):
    from sparse_b200 import ops
    from sparse_b200.kv_cache import QuantizedCache

    if kind == "shared" and case["cache"] == "bf16":
        return ops.attn_decode_shared(state["q"], state["k"], state["v"], state["lens"], case["prefix"], state["scale"])
    cache = QuantizedCache(state["k"], state["ks"], state["v"], state["vs"])
    if kind == "append":
        q = ops.rope_append_quantized(state["q"], state["k_rot"], state["k_rest"], state["v_in"], state["seq"],
                                      state["pos"], cache, state["theta"])
        return q, *_written(state, case)
    if kind == "read":
        return ops.cache_read(cache, 0, case["count"], case["shared"])
    return ops.attn_decode_quantized(state["q"], cache, state["lens"], case.get("prefix", 0), state["scale"])


def _written(state, case):
    """The positions of an append, codes and powers of two."""
    return tuple(state[x].narrow(2, case["past"], case["tokens"]) for x in ("k", "ks", "v", "vs"))


def _rotate(x, pos, theta):
    """Pairs (i, i + half) of the last axis turned by pos * theta^(-i / half); angles in 64 bits."""
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, dtype=F64, device=x.device) / half)
    ang = (pos.to(F64).unsqueeze(1) * freq).unsqueeze(1)
    cos, sin = ang.cos().to(F32), ang.sin().to(F32)
    a, b = x[..., :half].to(F32), x[..., half:].to(F32)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _append_plain(state, case):
    rope = state["k_rot"].shape[-1]
    n_kv, seq, pos = state["v_in"].shape[1], state["seq"].long(), state["pos"].long()
    q = torch.cat([_rotate(state["q"][..., :rope], pos, state["theta"]), state["q"][..., rope:].to(F32)], -1).to(BF16)
    k = _rotate(state["k_rot"], pos, state["theta"]).expand(-1, n_kv, -1)
    if state["k_rest"] is not None:
        k = torch.cat([k, state["k_rest"].to(F32)], dim=-1)
    # (8-bit floating types have no indexed assignment: their bytes are moved)
    for name, rows in (("k", k), ("v", state["v_in"])):
        codes, scales = _quantize(rows)
        state[name].view(torch.uint8)[seq, :, pos] = codes.view(torch.uint8)
        state[name + "s"].view(torch.uint8)[seq, :, pos] = scales.view(torch.uint8)
    return q, *_written(state, case)


def _values(codes, scales):
    return codes.to(F32) * scales.to(F32).unsqueeze(-1)


def _read_plain(codes, scales, case):
    out = _values(codes[:, :, :case["count"]], scales[:, :, :case["count"]])
    out[:, :, :case["shared"]] = out[:1, :, :case["shared"]].clone()
    return out.to(BF16)


def _attend_plain(state, case):
    n_q, n_kv, dk, dv = LAYOUTS[case["layout"]][:4]
    batch, prefix, end = case["batch"], case.get("prefix", 0), case.get("prefix", 0) + case["context"]
    group = n_q // n_kv
    if "ks" in state:
        k = _values(state["k"][:, :, prefix:end], state["ks"][:, :, prefix:end])
        v = _values(state["v"][:, :, prefix:end], state["vs"][:, :, prefix:end])
        pk = _values(state["k"][0, :, :prefix], state["ks"][0, :, :prefix])
        pv = _values(state["v"][0, :, :prefix], state["vs"][0, :, :prefix])
    else:
        k, v = (state[x][:, prefix:end].transpose(1, 2).to(F32) for x in ("k", "v"))
        pk, pv = (state[x][0, :prefix].transpose(0, 1).to(F32) for x in ("k", "v"))
    q = state["q"].to(F32).view(batch, n_kv, group, dk) * state["scale"]
    lens = state["lens"].view(batch, 1, 1, 1)
    at = torch.arange(prefix, end, device=q.device)
    s = torch.where(at < lens, q @ k.transpose(-1, -2), -math.inf)
    # every sequence's rows against the shared positions at once
    rows = q.transpose(0, 1).reshape(n_kv, batch * group, dk)
    sp = (rows @ pk.transpose(-1, -2)).view(n_kv, batch, group, prefix).transpose(0, 1)
    m = s.amax(-1, keepdim=True)
    if prefix:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)                           # an empty sequence
    e, ep = torch.exp(s - m), torch.exp(sp - m)
    total = e.sum(-1, keepdim=True) + ep.sum(-1, keepdim=True)
    o = e @ v + (ep.transpose(0, 1).reshape(n_kv, batch * group, prefix) @ pv).view(
        n_kv, batch, group, dv).transpose(0, 1)
    return torch.where(total > 0, o / total, 0.0).reshape(batch, n_q, dv).to(BF16)


# -- what a pass cannot do without -----------------------------------------------------------
def work(case):
    n_q, n_kv, dk, dv, rope, one_rotary = LAYOUTS[case["layout"]]
    row = n_kv * (dk + dv + 2)                                        # quantised bytes of one position
    if case["kind"] == "append":
        keys = rope + n_kv * (dk - rope) if one_rotary else n_kv * dk
        t = case["batch"] * case["tokens"]
        return {"bytes": t * (2 * n_q * dk * 2 + 2 * keys + 2 * n_kv * dv + row + 8), "flops": 6 * t * (n_q + n_kv) * rope}
    if case["kind"] == "read":
        stored = case["shared"] + case["batch"] * (case["count"] - case["shared"])
        return {"bytes": stored * row + case["batch"] * case["count"] * n_kv * (dk + dv) * 2,
                "flops": case["batch"] * case["count"] * n_kv * (dk + dv)}
    if case.get("cache") == "bf16":
        row = n_kv * (dk + dv) * 2
    lens, prefix = _lens(case), case.get("prefix", 0)
    nbytes = (prefix + sum(lens)) * row + case["batch"] * (n_q * (dk + dv) * 2 + 4)
    return {"bytes": nbytes, "flops": 2 * n_q * (dk + dv) * (sum(lens) + prefix * case["batch"])}


# -- the definition in 64 bits ---------------------------------------------------------------
def _e4m3(x):
    """The nearest multiple of the step that a 3-bit mantissa leaves (2^-9 at least), ties to even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp_min(-9).to(F64))
    return torch.round(x / step) * step


def _exact_rows(rows):
    """fp64 rows -> the code values and powers of two of their quantised form."""
    top = rows.abs().amax(-1)
    e = torch.ceil(torch.log2(top.clamp_min(1e-60) / 448.0))
    # (the logarithm may be off by its last bit at an exact power of two)
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e).clamp_min(-127)
    return _e4m3(rows / torch.exp2(e).unsqueeze(-1)), torch.exp2(e)


def exact(case, seed: int):
    state = prepare(case, seed)
    n_q, n_kv, dk, dv, rope, _ = LAYOUTS[case["layout"]]
    batch = case["batch"]
    if case["kind"] == "append":
        n, t = case["tokens"], batch * case["tokens"]
        i = torch.arange(rope // 2, dtype=F64, device=state["q"].device)
        turn = torch.polar(torch.ones((), dtype=F64, device=i.device),
                           state["pos"].to(F64)[:, None, None] * torch.exp(-2.0 * i / rope * math.log(state["theta"])))

        def rotated(x):
            z = torch.complex(x[..., :rope // 2].to(F64), x[..., rope // 2:rope].to(F64)) * turn
            return torch.cat([z.real, z.imag, x[..., rope:].to(F64)], dim=-1)

        q, k = rotated(state["q"]), rotated(state["k_rot"]).expand(t, n_kv, rope)
        if state["k_rest"] is not None:
            k = torch.cat([k, state["k_rest"].to(F64)], dim=-1)
        out = [q]
        for rows in (k, state["v_in"].to(F64)):
            codes, scales = _exact_rows(rows)
            out += [codes.view(batch, n, n_kv, -1).transpose(1, 2), scales.view(batch, n, n_kv).transpose(1, 2)]
        return tuple(out)
    if case["kind"] == "read":
        outs = []
        for x in ("k", "v"):
            full = state[x].to(F32).to(F64) * state[x + "s"].to(F32).to(F64)[..., None]
            source = torch.arange(batch, device=full.device)[:, None].repeat(1, case["count"])
            source[:, :case["shared"]] = 0
            place = torch.arange(case["count"], device=full.device).expand(batch, -1)
            outs.append(full[source, :, place].transpose(1, 2))
        return tuple(outs)
    prefix, group = case.get("prefix", 0), n_q // n_kv
    out = torch.zeros((batch, n_q, dv), dtype=F64, device=state["q"].device)
    for b, end in enumerate(state["lens"].tolist()):
        if end == 0:
            continue

        def cached(x):
            if "ks" in state:
                parts = [(state[x][s, :, i:j].to(F32).to(F64) * state[x + "s"][s, :, i:j].to(F32).to(F64)[..., None])
                         for s, i, j in ((0, 0, prefix), (b, prefix, end))]
            else:
                parts = [state[x][s, i:j].to(F64).transpose(0, 1) for s, i, j in ((0, 0, prefix), (b, prefix, end))]
            return torch.cat(parts, dim=1)

        q = state["q"][b].to(F64).view(n_kv, group, dk)
        weight = torch.softmax(torch.einsum("hgd,hnd->hgn", q, cached("k")) * state["scale"], dim=-1)
        out[b] = torch.einsum("hgn,hnd->hgd", weight, cached("v")).reshape(n_q, dv)
    return out
