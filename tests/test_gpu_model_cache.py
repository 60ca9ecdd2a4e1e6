"""GPU: the shaped model with a quantised key/value cache and with a prompt prefix that the
batch shares, against itself.

Tolerances.  Two passes that round bf16 sums in another order differ by up to 2e-2 in a cached
row (the bound of the bf16 model's own test).  A quantised row adds a rounding to half a step of
e4m3 on each side, uniform within 2^-4 of the value at most: 2^-4 / sqrt(3) = 3.6 % rms each, 5.1 % for
the difference of two independent ones, 7.1 % with the 2e-2 in front of it."""
import dataclasses

import pytest
import torch

from sparse_b200 import ops, synth
from sparse_b200.model import TINY_MODEL, ModelConfig, ShapedMoeModel, greedy_decode_profiled

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
MLA = ModelConfig("mla-small", 2, 256, 16, 16, 192, 128, 64, 1.0e4, 1e-6, 512, synth.TINY, {0: 320}, "mla", 512, False)
GQA = dataclasses.replace(TINY_MODEL, name="tiny-gqa", n_kv_heads=2)


def _model(cfg, batch, max_seq, **kw):
    return ShapedMoeModel(cfg, DEV, batch, max_seq, seed=3, **kw)


def _rows(model, position):
    """The cached keys of one position in every layer, [layers, B, n_kv, dk] fp32."""
    if model.kv_cache == "fp8":
        return torch.stack([ops.cache_read(ly.cache, position, 1)[0][:, :, 0].float() for ly in model.layers])
    return torch.stack([ly.cache_k[:, position].float() for ly in model.layers])


def _prompt(b, s, shared, seed):
    ids = torch.randint(0, 512, (b, s), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))
    ids[:, :shared] = ids[:1, :shared].clone()
    return ids


def _near(a, b, bound):
    return float((a - b).norm() / b.norm()) < bound


@pytest.mark.parametrize("kv_cache", ["bf16", "fp8"])
@pytest.mark.parametrize("cfg", [TINY_MODEL, GQA, MLA], ids=lambda c: c.name)
@pytest.mark.parametrize("shared", [0, 21])
def test_decode_agrees_with_a_longer_prompt(cfg, kv_cache, shared):
    b, s = 5, 37
    ids = _prompt(b, s + 1, shared, 0)
    m1 = _model(cfg, b, 64, kv_cache=kv_cache)
    m1.prefill(ids)                                          # nothing shared, every sequence its own rows
    m2 = _model(cfg, b, 64, kv_cache=kv_cache, chunk_tokens=40)
    m2.prefill(ids[:, :s], shared)
    m2.cur_ids.copy_(ids[:, s])
    m2.decode_step(use_graph=False)
    bound = 0.071 if kv_cache == "fp8" else 2e-2
    assert _near(_rows(m2, s), _rows(m1, s), bound) and _near(_rows(m2, s - 1), _rows(m1, s - 1), bound)
    if shared:
        # the shared positions stand with sequence 0 only
        assert _near(_rows(m2, shared - 1)[:, 0], _rows(m1, shared - 1)[:, 0], bound)
        assert float(_rows(m2, shared - 1)[:, 1:].abs().max()) == 0.0
    m1.check_status(); m2.check_status()


@pytest.mark.parametrize("kv_cache", ["bf16", "fp8"])
@pytest.mark.parametrize("batch,shared", [(4, 0), (4, 9), (30, 17)])
def test_recorded_steps_equal_eager_steps(kv_cache, batch, shared):
    ids = _prompt(batch, 20, shared, 1)
    outs = []
    for use_graph in (False, True):
        m = _model(GQA, batch, 64, kv_cache=kv_cache)
        outs.append(greedy_decode_profiled(m, ids, torch.ones_like(ids), 12, None, None, False, use_graph=use_graph,
                                           shared_len=shared))
    assert torch.equal(*outs)


def test_another_shared_length_is_recorded_anew():
    """One model, requests with and without a common prefix in turn: each gives what a new model gives."""
    m, got = _model(TINY_MODEL, 4, 64, kv_cache="fp8"), []
    requests = [(0, 5), (16, 6), (16, 7), (3, 8), (0, 9)]
    for shared, seed in requests:
        got.append(greedy_decode_profiled(m, _prompt(4, 20, shared, seed), None, 8, None, None, False, shared_len=shared))
    for (shared, seed), out in zip(requests, got):
        want = greedy_decode_profiled(_model(TINY_MODEL, 4, 64, kv_cache="fp8"), _prompt(4, 20, shared, seed), None, 8, None,
                                      None, False, shared_len=shared)
        assert torch.equal(out, want)


def test_model_refuses():
    with pytest.raises(ValueError):
        _model(TINY_MODEL, 2, 32, kv_cache="int8")
    m, ids = _model(TINY_MODEL, 2, 32), _prompt(2, 10, 0, 2)
    for shared in (-1, 10, 11):
        with pytest.raises(RuntimeError):
            m.prefill(ids, shared)
    ids[1, 3] = (ids[0, 3] + 1) % 512
    with pytest.raises(RuntimeError, match="same"):
        m.prefill(ids, 4)
