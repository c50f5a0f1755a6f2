"""Served models with keys and values in 8 bits: every step's operators against plain implementations, on the cache as it is."""

import pytest
import torch

from nkipy_b200 import ops
from nkipy_b200.models import config as C
from nkipy_b200.models.engine import GenerationEngine, Sampling, StepEntry
from nkipy_b200.models.kv_cache import KVLayer, PagedKVCache, StateLayer
from nkipy_b200.models.speculative import DrafterLM, EagleConfig, SpeculativeEngine, random_drafter_weights
from nkipy_b200.models.transformer import TransformerLM
from nkipy_b200.models.weights import random_weights
from tests.test_quantized_kv import DEVICES, check_attention, oracle_quantize, oracle_turn

E4M3 = torch.float8_e4m3fn
KINDS = {
    "llama": dict(hidden_size=256, head_dim=64, num_heads=8, num_kv_heads=2, intermediate_size=512, vocab_size=512, num_layers=2),
    "qk-norm": dict(hidden_size=256, head_dim=128, num_heads=4, num_kv_heads=2, intermediate_size=512, vocab_size=512, num_layers=2,
                    qk_norm=True),
    "window": dict(hidden_size=256, head_dim=64, num_heads=8, num_kv_heads=1, intermediate_size=512, vocab_size=512, num_layers=2,
                   attn_bias=True, attention_sinks=True, sliding_window=16),
}


def model_of(kind, device):
    cfg = C.tiny(**KINDS[kind])
    return TransformerLM(cfg, random_weights(cfg, device=device, seed=1, std=0.05), device=device)


def ids(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


class Watched:
    """Stands in for the operators on a quantised cache and checks every call."""

    def __init__(self, monkeypatch, model):
        self.model, self.calls = model, {}
        for name in ("rope_kv_append", "paged_attn_decode", "rope_attn_decode", "flash_attn_prefill"):
            real = getattr(ops.quantized_kv, name)
            monkeypatch.setattr(ops.quantized_kv, name, lambda *a, _n=name, _r=real, **kw: self.check(_n, _r, a, kw))
        self.inside = False

    def check(self, name, real, a, kw):
        if self.inside:                       # a call that another of them makes
            return real(*a, **kw)
        self.inside = True
        try:
            out = real(*a, **kw)
        finally:
            self.inside = False
        self.calls[name] = self.calls.get(name, 0) + 1
        getattr(self, "_" + name)(out, *a, **kw)
        return out

    def _appended(self, qkv, pos, slots, cs, k, v, nq, nkv, dim, bias, k_norm_w, norm_eps):
        x = qkv.cpu().double()
        x = x.reshape(-1, *x.shape[-2:]).sum(0)
        if bias is not None:
            x = x + bias.cpu().double()
        x = x.view(-1, nq + 2 * nkv, dim)
        turned = oracle_turn(x[:, nq:nq + nkv], cs.cpu()[pos.cpu().long()], None if k_norm_w is None else k_norm_w.cpu(), norm_eps)
        for pages, rows in ((k, turned), (v, x[:, nq + nkv:])):
            values, scales = oracle_quantize(rows)
            on = slots.cpu() >= 0
            at = slots.cpu().long()[on]
            assert torch.equal(pages.values.cpu().double()[at // 32, :, at % 32], values[on])
            assert torch.equal(pages.scales.cpu().float().double()[at // 32, :, at % 32], scales[on])

    def _rope_kv_append(self, result, qkv, pos, slots, cs, k, v, nq, nkv, dim, *, bias=None, q_norm_w=None, k_norm_w=None, norm_eps=1e-6,
                        q_out=None):
        self._appended(qkv, pos, slots, cs, k, v, nq, nkv, dim, bias, k_norm_w, norm_eps)

    def _paged_attn_decode(self, result, q, k, v, table, lens, scale, *, q_len=1, window=0, sinks=None, **kw):
        m, dim = self.model, k.shape[3]
        check_attention(result.view(-1, m.nq, dim), q.view(-1, m.nq, dim), k, v, table, [(b * q_len, q_len, c) for b, c in enumerate(lens.tolist())
                                                                                      if c >= 0], scale, m.nq, m.nq // m.nkv,
                        None if sinks is None else sinks.cpu(), window=window)

    def _rope_attn_decode(self, result, qkv, pos, slots, cs, k, v, table, lens, scale, nq, nkv, *, bias=None, q_norm_w=None, k_norm_w=None,
                          norm_eps=1e-6, window=0, sinks=None, **kw):
        dim = k.shape[3]
        self._appended(qkv, pos, slots, cs, k, v, nq, nkv, dim, bias, k_norm_w, norm_eps)
        fresh = [ops.QuantizedPages.new(*(p.shape[:2]), dim, p.device) for p in (k, v)]
        self.inside = True
        q = ops.quantized_kv.rope_kv_append(qkv, pos, torch.full_like(slots, -1), cs, *fresh, nq, nkv, dim, bias=bias, q_norm_w=q_norm_w,
                                            k_norm_w=k_norm_w, norm_eps=norm_eps)
        self.inside = False
        self._paged_attn_decode(result, q, k, v, table, lens, scale, window=window, sinks=sinks)

    def _flash_attn_prefill(self, result, q, k, v, table, starts, new, lens, scale, *, max_q_len, causal=True, window=0, sinks=None, **kw):
        m, dim = self.model, k.shape[3]
        check_attention(result.view(-1, m.nq, dim), q.view(-1, m.nq, dim), k, v, table, list(zip(starts.tolist(), new.tolist(), lens.tolist())),
                        scale, m.nq, m.nq // m.nkv, None if sinks is None else sinks.cpu(), causal=causal, window=window)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_steps_of_a_scheduler(device, kind, monkeypatch):
    """Prompts in portions, mixed steps, single tokens, blocks that are given back and used again."""
    model = model_of(kind, device)
    engine = GenerationEngine(model, max_batch=4, max_seq_len=160, num_blocks=16, use_cuda_graph=False, enable_prefix_sharing=False,
                              kv_dtype=E4M3)
    seen = Watched(monkeypatch, model)
    a, b = engine.open_request(), engine.open_request()
    engine.run_step([StepEntry(a, ids(70, 1), [-1]), StepEntry(b, ids(5, 2))])
    engine.run_step([StepEntry(a, ids(1, 3), [0]), StepEntry(b, ids(40, 4), [-1])])          # a single token beside a portion
    engine.run_step([StepEntry(b, ids(1, 5), [0]), StepEntry(a, ids(1, 6), [0])])
    engine.release([a])
    c = engine.open_request()
    engine.run_step([StepEntry(c, ids(33, 7), [-1])])
    logits = engine.run_step([StepEntry(c, ids(1, 8), [0]), StepEntry(b, ids(1, 9), [0])])
    assert bool(logits.isfinite().all())
    assert seen.calls["rope_kv_append"] >= 6 and seen.calls["flash_attn_prefill"] >= 4
    assert seen.calls.get("rope_attn_decode", 0) + seen.calls.get("paged_attn_decode", 0) >= 4


@pytest.mark.parametrize("device", DEVICES)
def test_generate(device, monkeypatch):
    model = model_of("llama", device)
    engine = GenerationEngine(model, max_batch=3, max_seq_len=96, use_cuda_graph=False, kv_dtype=E4M3)
    seen = Watched(monkeypatch, model)
    out = engine.generate([ids(40, 1), ids(40, 1)[:33] + ids(9, 2)], 4)                       # the second shares a block
    assert [len(o) for o in out] == [4, 4] and engine.stats.cached_tokens == 0
    again = engine.generate([ids(40, 1)], 4)
    assert engine.stats.cached_tokens == 32 and len(again[0]) == 4
    assert sum(seen.calls.values()) >= 12


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_captured_steps_are_the_same(kind):
    """The captured decode step gives what launches one by one give, beside another engine's and with sampling."""
    model = model_of(kind, "cuda")
    prompts = [ids(70, 1), ids(3, 2), ids(33, 3)]
    engines = [GenerationEngine(model, max_batch=4, max_seq_len=160, use_cuda_graph=g, kv_dtype=E4M3) for g in (False, True, True)]
    outs = [e.generate(prompts, 12) for e in engines]
    assert outs[0] == outs[1] == outs[2]
    sampling = Sampling(0.8, 20, 0.9, 7)                       # random numbers go by the batch row: engines that have run as often
    assert engines[0].generate(prompts, 6, sampling=sampling) == engines[2].generate(prompts, 6, sampling=sampling)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_takes_half_the_bytes(device):
    model = model_of("llama", device)
    small, large = (model.new_cache(10, 2, 128, kv_dtype=t) for t in (E4M3, None))
    assert small.quantized and not large.quantized
    assert large.bytes() == 2 * 2 * 10 * 2 * 32 * 64 * 2 and small.bytes() == large.bytes() // 2 * 65 // 64


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads", [(4, 2), (8, 1)])                                           # the second: more than sixteen rows
def test_verified_drafts(device, heads, monkeypatch):
    cfg = C.tiny(num_heads=heads[0], num_kv_heads=heads[1], head_dim=64, num_layers=4)
    target = TransformerLM(cfg, random_weights(cfg, 0, 1, seed=5, std=0.05), device=device)
    ecfg = EagleConfig(hidden_size=cfg.hidden_size, target_hidden_size=cfg.hidden_size, num_heads=4, num_kv_heads=4, head_dim=64,
                       intermediate_size=256, draft_vocab_size=cfg.vocab_size, vocab_size=cfg.vocab_size, num_draft_tokens=3, ptd_token_id=3)
    drafter = DrafterLM(ecfg, random_drafter_weights(ecfg, seed=9, std=0.05), device)
    spec = SpeculativeEngine(target, drafter, max_batch=2, max_seq_len=96, kv_dtype=E4M3)
    assert spec.cache.quantized and not spec.dcache.quantized
    seen = Watched(monkeypatch, target)
    out = spec.generate([ids(19, 1), ids(33, 2)], 6)
    assert all(len(o) == 6 for o in out) and seen.calls["rope_kv_append"] >= 8


def test_other_models_refuse():
    with pytest.raises(ValueError):
        PagedKVCache.for_layers([KVLayer(2, 64, 128)], 4, 1, 4, "cpu", dtype=E4M3)
    with pytest.raises(ValueError):
        PagedKVCache.for_layers([KVLayer(2, 64, 64), StateLayer((2, 2))], 4, 1, 4, "cpu", dtype=E4M3)
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 96, 4, 1, 4, "cpu", dtype=E4M3)
    model = model_of("llama", "cpu")
    with pytest.raises(ValueError):
        GenerationEngine(model, max_batch=1, max_seq_len=64, kv_dtype=torch.float16)
    from nkipy_b200.models import registry

    cfg = C.tolenex_shape(256, layers=2, heads=4, kv_heads=2, ff=512, vocab=512, dim=32, vdim=64)
    arch = registry.for_config(cfg)
    hybrid = registry.build(arch, cfg, arch.random(cfg, 0, 1, "cpu", 0, "ep"), device="cpu")
    with pytest.raises(ValueError):
        GenerationEngine(hybrid, max_batch=1, max_seq_len=64, kv_dtype=E4M3)


def test_command_line(capsys):
    import argparse

    from nkipy_b200.models import runner

    ap = argparse.ArgumentParser()
    runner.add_common_args(ap)
    args = ap.parse_args(["--tiny", "--layers", "2", "-n", "3", "--prompt-len", "20", "--kv-dtype", "e4m3"])
    assert runner.kv_dtype(args) is E4M3 and runner.kv_dtype(ap.parse_args([])) is None
    assert runner.run_generation(C.llama3_8b(num_layers=2), args) == 0
    assert "Generated 3 tokens" in capsys.readouterr().out
