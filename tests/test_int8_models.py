"""Served models with weights in 8 bits, and generation under rules: the operators' calls of every step against plain implementations."""

import pytest
import torch

from nkipy_b200 import ops
from nkipy_b200.models import config as C
from nkipy_b200.models.engine import GenerationEngine, Sampling, StepEntry
from nkipy_b200.models.transformer import TransformerLM
from nkipy_b200.models.weights import random_weights
from tests.test_logit_rules import oracle, oracle_ids
from tests.test_quantized_linear import DEVICES, check_product, check_rows, oracle_numbers, oracle_product

E4M3 = torch.float8_e4m3fn
KINDS = {
    "llama": dict(hidden_size=256, head_dim=64, num_heads=8, num_kv_heads=2, intermediate_size=512, vocab_size=512, num_layers=2),
    "qk-norm": dict(hidden_size=256, head_dim=128, num_heads=4, num_kv_heads=2, intermediate_size=512, vocab_size=512, num_layers=2,
                    qk_norm=True),
    "window": dict(hidden_size=256, head_dim=64, num_heads=8, num_kv_heads=1, intermediate_size=512, vocab_size=512, num_layers=2,
                   attn_bias=True, attention_sinks=True, sliding_window=16),
}


def model_of(kind, device, quantize=True):
    cfg = C.tiny(**KINDS[kind])
    model = TransformerLM(cfg, random_weights(cfg, device=device, seed=1, std=0.05), device=device)
    return model.quantize_weights() if quantize else model


def ids(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


class Watched:
    """Checks every product in 8 bits, and the rows behind every norm."""

    def __init__(self, monkeypatch):
        self.products = self.norms = 0
        linear, norm = ops.quantized_linear.linear, ops.quantized_linear.add_rmsnorm

        def checked_linear(x, w, **kw):
            if type(x) is ops.QuantizedRows:
                q, sx = x.values.cpu(), x.scale.cpu()
            else:
                q, top = oracle_numbers(x.cpu())
                sx = (top / 127).float()
            before = None if kw.get("residual") is None else kw["residual"].cpu().clone()
            out = linear(x, w, **kw)
            parts = out.dim() == 3
            want, tol = oracle_product(q, sx, w.values.cpu(), w.scale.cpu(), gated=kw.get("gated", False), fp32=parts or kw.get("fp32_out", False),
                                       bias=None if kw.get("bias") is None else kw["bias"].cpu(), residual=before)
            # (partial sums: each is rounded to 32 bits, their sum of magnitudes is at most the sum over all of k)
            mass = (q.double().abs() @ w.values.cpu().double().abs().T) * sx.double()[:, None] * w.scale.cpu().double()
            check_product(out.double().sum(0) if parts else out, want, tol + (4 * 2.0 ** -24 * mass if parts else 0))
            self.products += 1
            return out

        def checked_norm(x, w, **kw):
            before = {k: v.cpu().double() for k, v in dict(kw, x=x).items() if torch.is_tensor(v) and k != "residual_out"}
            h, rows = norm(x, w, **kw)
            total = sum((before[k].reshape(rows.shape) for k in ("x", "residual_in") if k in before), torch.zeros(rows.shape, dtype=torch.float64))
            if "partials" in before:
                total = total + before["partials"].sum(0)
            if "bias" in before:
                total = total + before["bias"]
            total = total.to(torch.bfloat16).double()
            check_rows(rows, total * w.cpu().double(), 1 / torch.sqrt(total.square().mean(-1) + kw["eps"]), steps=64)
            self.norms += 1
            return h, rows

        monkeypatch.setattr(ops.quantized_linear, "linear", checked_linear)
        monkeypatch.setattr(ops.quantized_linear, "add_rmsnorm", checked_norm)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_steps_of_a_scheduler(device, kind, monkeypatch):
    model = model_of(kind, device)
    engine = GenerationEngine(model, max_batch=4, max_seq_len=160, num_blocks=16, use_cuda_graph=False, enable_prefix_sharing=False)
    seen = Watched(monkeypatch)
    a, b = engine.open_request(), engine.open_request()
    engine.run_step([StepEntry(a, ids(70, 1), [-1]), StepEntry(b, ids(5, 2))])
    engine.run_step([StepEntry(a, ids(1, 3), [0]), StepEntry(b, ids(90, 4), [-1])])
    logits = engine.run_step([StepEntry(b, ids(1, 5), [0]), StepEntry(a, ids(1, 6), [0])])
    assert bool(logits.isfinite().all())
    assert seen.products == 3 * (2 * 4 + 1) and seen.norms == 3 * 4


@pytest.mark.parametrize("device", DEVICES)
def test_logits_are_near_those_of_bf16_weights(device):
    """As far as 8 bits take them: every product adds an error of about 1 / (127 sqrt(12)) of its rows' and weights' largest numbers, some four
    of their root mean squares, on both sides: 1.3 % of a result each; nine products in a chain, whose errors are independent, some 4 %."""
    exact, model = model_of("llama", device, quantize=False), model_of("llama", device)
    rows = []
    for m in (exact, model):
        engine = GenerationEngine(m, max_batch=1, max_seq_len=64, use_cuda_graph=False)
        s = engine.open_request()
        rows.append(engine.run_step([StepEntry(s, ids(40, 1), list(range(40)))]).float().cpu())
    off = (rows[1] - rows[0]).norm() / rows[0].norm()
    assert 0 < float(off) < 0.08
    assert model.weight_bytes() < 0.75 * exact.weight_bytes()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("kv", [None, E4M3])
def test_captured_steps_are_the_same(kind, kv):
    model = model_of(kind, "cuda")
    prompts = [ids(70, 1), ids(3, 2), ids(33, 3)]
    outs = [GenerationEngine(model, max_batch=4, max_seq_len=160, use_cuda_graph=g, kv_dtype=kv).generate(prompts, 12) for g in (False, True)]
    assert outs[0] == outs[1]


def test_models_that_have_none():
    cfg = C.tiny(num_experts=4, top_k=2, moe_intermediate_size=64) if "num_experts" in C.ModelConfig.__dataclass_fields__ else None
    if cfg is not None and cfg.is_moe:
        with pytest.raises(ValueError):
            TransformerLM(cfg, random_weights(cfg, seed=1), device="cpu").quantize_weights()
    model = model_of("llama", "cpu")
    first = model.layers[0].qkv
    assert model.quantize_weights() is model and model.layers[0].qkv is first


@pytest.mark.parametrize("device", DEVICES)
def test_verified_drafts(device):
    from nkipy_b200.models.speculative import DrafterLM, EagleConfig, SpeculativeEngine, random_drafter_weights

    cfg = C.tiny(num_heads=4, num_kv_heads=2, head_dim=64, num_layers=4)
    target = TransformerLM(cfg, random_weights(cfg, 0, 1, seed=5, std=0.05), device=device).quantize_weights()
    ecfg = EagleConfig(hidden_size=cfg.hidden_size, target_hidden_size=cfg.hidden_size, num_heads=4, num_kv_heads=4, head_dim=64,
                       intermediate_size=256, draft_vocab_size=cfg.vocab_size, vocab_size=cfg.vocab_size, num_draft_tokens=3, ptd_token_id=3)
    drafter = DrafterLM(ecfg, random_drafter_weights(ecfg, seed=9, std=0.05), device)
    spec = SpeculativeEngine(target, drafter, max_batch=2, max_seq_len=96)
    out = spec.generate([ids(19, 1), ids(33, 2)], 6)
    assert all(len(o) == 6 for o in out)


# ------------------------------------------------------------------------------------------------ rules
class Chosen:
    """Follows every choice under rules by the oracle."""

    def __init__(self, monkeypatch):
        self.calls = 0
        real = ops.logit_rules.argmax

        def checked(logits, rules, out_ids=None):
            r = {k: v.cpu().clone() for k, v in ((f, getattr(rules, f)) for f in rules.__dataclass_fields__) if v is not None}
            got = real(logits, rules, out_ids)
            want, tokens = oracle(logits.cpu(), r)
            assert torch.equal(got.cpu(), oracle_ids(want))
            assert torch.equal(rules.tokens.cpu(), tokens)
            self.lens, self.tokens = r["lens"].tolist(), tokens
            self.calls += 1
            return got

        monkeypatch.setattr(ops.logit_rules, "argmax", checked)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quantize", [False, True])
def test_generation_under_rules(device, quantize, monkeypatch):
    model = model_of("llama", device, quantize)
    engine = GenerationEngine(model, max_batch=4, max_seq_len=128, use_cuda_graph=device == "cuda")
    prompts = [ids(40, 1), ids(5, 2), ids(33, 3)]
    plain = engine.generate(prompts, 8)
    assert engine.generate(prompts, 8, sampling=Sampling(presence=0.0)) == plain
    seen = Chosen(monkeypatch)
    out = engine.generate(prompts, 8, sampling=Sampling(repetition=1.3, frequency=0.4, presence=0.2, biases={7: 3.0, 9: -float("inf")}))
    assert seen.calls == 8
    assert seen.lens[:3] == [47, 12, 40]                                  # the last choice's: the prompt and seven of the answer
    for row, (p, o) in enumerate(zip(prompts, out)):
        assert seen.tokens[row, :len(p) + 7].tolist() == p + o[:7]
        assert 9 not in o
    # tokens that may not come again
    out = engine.generate(prompts, 12, sampling=Sampling(presence=1e9))
    assert all(len(set(o)) == 12 for o in out)


@pytest.mark.parametrize("device", DEVICES)
def test_generation_under_a_grammar(device):
    """Even tokens and odd ones in turn; one sequence may go on with nothing after its third token."""
    model = model_of("llama", device, False)
    engine = GenerationEngine(model, max_batch=3, max_seq_len=96, use_cuda_graph=device == "cuda")
    ends = ids(31, 2)
    prompts = [ids(20, 1), ends]

    def allowed(prompt, answer):
        if prompt == ends and len(answer) == 3:
            return []
        if len(answer) == 5:
            return None
        return torch.arange(512) % 2 == len(answer) % 2 if len(answer) < 2 else range(len(answer) % 2, 512, 2)

    for sampling in (Sampling(allowed=allowed), Sampling(temperature=0.9, top_k=50, seed=3, repetition=1.1, allowed=allowed)):
        out = engine.generate(prompts, 7, sampling=sampling)
        assert len(out[0]) == 7 and all(t % 2 == i % 2 for i, t in enumerate(out[0]) if i != 5)
        assert len(out[1]) == 3 and all(t % 2 == i % 2 for i, t in enumerate(out[1]))


def test_rows_are_free_after_a_grammar_that_fails():
    engine = GenerationEngine(model_of("llama", "cpu", False), max_batch=2, max_seq_len=64)
    prompts = [ids(20, 1), ids(9, 2)]
    plain = engine.generate(prompts, 4)

    def raises(prompt, answer):
        if len(answer) == 2:
            raise KeyError("no such state")

    for at in (0, 2):
        for bad in ([-1], [512], torch.tensor([3, 512])):
            with pytest.raises(ValueError):
                engine.generate(prompts, 4, sampling=Sampling(allowed=lambda p, a: bad if len(a) == at else None))
            assert not engine.active
    with pytest.raises(KeyError):
        engine.generate(prompts, 4, sampling=Sampling(allowed=raises))
    assert not engine.active and engine.generate(prompts, 4) == plain


def test_refusals_of_sampling():
    for kw in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("inf")), dict(repetition=float("nan")), dict(frequency=float("nan")),
               dict(presence=float("inf"))):
        with pytest.raises(ValueError):
            Sampling(**kw)
    engine = GenerationEngine(model_of("llama", "cpu", False), max_batch=1, max_seq_len=64)
    for bad in (512, -1):
        with pytest.raises(ValueError):
            engine.generate([ids(4, 1)], 2, sampling=Sampling(biases={bad: 1.0}))


def test_command_line(capsys):
    import argparse

    from nkipy_b200.models import runner

    ap = argparse.ArgumentParser()
    runner.add_common_args(ap)
    args = ap.parse_args(["--tiny", "--layers", "2", "-n", "3", "--prompt-len", "20", "--weight-dtype", "int8", "--repetition-penalty", "1.2",
                          "--frequency-penalty", "0.1", "--presence-penalty", "0.1"])
    assert runner.sampling_of(args).ruled and not runner.sampling_of(ap.parse_args([])).ruled
    assert runner.run_generation(C.llama3_8b(num_layers=2), args) == 0
    assert "Generated 3 tokens" in capsys.readouterr().out
    with pytest.raises(ValueError):
        runner.quantize_weights(args, object())


# ------------------------------------------------------------------------------------------------ weights that are replaced under an engine
@pytest.mark.parametrize("device", DEVICES)
def test_an_engine_whose_models_weights_are_replaced(device):
    """Neither the captured step nor the keys and values of the bf16 weights serve the quantised model."""
    prompts = [ids(100, 1), ids(7, 2)]
    model = model_of("llama", device, quantize=False)
    engine = GenerationEngine(model, max_batch=2, max_seq_len=160)
    engine.generate(prompts, 8)
    cached, graph = engine.stats.cached_tokens, engine._graph
    model.quantize_weights()
    out = engine.generate(prompts, 8)
    assert engine.stats.cached_tokens == cached and (device == "cpu" or engine._graph is not graph)
    assert out == GenerationEngine(model_of("llama", device), max_batch=2, max_seq_len=160).generate(prompts, 8)
    # the quantised model's own prefixes are found again, and every block is there
    assert engine.generate(prompts, 8) == out and engine.stats.cached_tokens == cached + 96
    assert engine.cache.allocator.num_free() == engine.cache.num_blocks


@pytest.mark.parametrize("device", DEVICES)
def test_open_sequences_do_not_outlive_their_weights(device):
    model = model_of("llama", device, quantize=False)
    engine = GenerationEngine(model, max_batch=2, max_seq_len=96)
    s, new = engine.open_request(), engine.open_request()
    engine.run_step([StepEntry(s, ids(40, 1), [-1])])
    engine.run_step([StepEntry(s, ids(1, 2), [-1])])
    model.quantize_weights()
    for call in (lambda: engine.run_step([StepEntry(s, ids(1, 3), [-1])]), lambda: engine.run_step([StepEntry(new, ids(4, 3), [-1])]),
                 lambda: engine.add_requests([ids(5, 3)]), engine.open_request, lambda: engine.prepare_decode(1), engine.step,
                 engine.decode_step_device):
        with pytest.raises(RuntimeError, match="weights were replaced"):
            call()
    engine.release([s])
    fresh = GenerationEngine(model, max_batch=2, max_seq_len=96)
    other = fresh.open_request()
    for tokens in (ids(40, 1), ids(1, 5)):             # (a sequence of which nothing was computed goes on)
        a, b = engine.run_step([StepEntry(new, tokens, [-1])]), fresh.run_step([StepEntry(other, tokens, [-1])])
        assert torch.equal(a, b)


def test_blocks_are_forgotten():
    from nkipy_b200.models.kv_cache import BlockAllocator

    a = BlockAllocator(6)
    tokens = list(range(70))
    held, _ = a.admit(tokens)
    a.publish(tokens, held, 70)
    gone, cached = a.admit(tokens[:40])
    assert cached == 32
    a.release(gone)
    a.release(held)
    assert len(a.evictable) == 2
    kept, _ = a.admit(tokens)
    a.forget()
    blocks, cached = a.admit(tokens)
    assert cached == 0 and not set(blocks) & set(kept)
    a.release(blocks)
    a.publish(tokens, kept, 70)
    assert a.admit(tokens[:40])[0][0] == kept[0]


@pytest.mark.parametrize("script", ["qwen3/evaluate.py", "gpt_oss/peagle/speculate.py"])
def test_commands_that_generate_without_rules_refuse_them(script):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for flag in ("--repetition-penalty", "--presence-penalty"):
        r = subprocess.run([sys.executable, os.path.join(root, "examples", "models", script), "--layers", "1", flag, "1.5"], capture_output=True, text=True,
                           cwd=root, env=dict(os.environ, PYTHONPATH=root), timeout=300)
        assert r.returncode and "penalties" in r.stderr.splitlines()[-1]


# ------------------------------------------------------------------------------------------------ decode steps of one and two sequences
class WatchedFew(Watched):
    """Sums of few rows come to the norm as [rows, columns], without an axis of parts."""

    def __init__(self, monkeypatch):
        norm = ops.quantized_linear.add_rmsnorm
        super().__init__(monkeypatch)
        self.whole = 0

        def checked_norm(x, w, **kw):
            before = {k: v.cpu().double() for k, v in dict(kw, x=x).items() if torch.is_tensor(v) and k != "residual_out"}
            h, rows = norm(x, w, **kw)
            total = sum((before[k].reshape(rows.shape) for k in ("x", "residual_in") if k in before),
                        torch.zeros(rows.shape, dtype=torch.float64))
            if "partials" in before:
                self.whole += before["partials"].dim() == 2
                total = total + (before["partials"] if before["partials"].dim() == 2 else before["partials"].sum(0))
            if "bias" in before:
                total = total + before["bias"]
            total = ops.quantized_linear.to_bf16(total)
            if h is not None:
                assert torch.equal(h.cpu().reshape(total.shape), total)
            check_rows(rows, total.double() * w.cpu().double(), 1 / torch.sqrt(total.double().square().mean(-1) + kw["eps"]), steps=64)
            self.norms += 1
            return h, rows

        monkeypatch.setattr(ops.quantized_linear, "add_rmsnorm", checked_norm)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("kv", [None, E4M3])
@pytest.mark.parametrize("batch", [1, 2, 4])
def test_decode_steps_of_few_sequences(device, kind, kv, batch, monkeypatch):
    """Every product and norm of decode steps with as many rows as the kernel for few tokens takes, and with more."""
    model = model_of(kind, device)
    engine = GenerationEngine(model, max_batch=batch, max_seq_len=96, use_cuda_graph=False, enable_prefix_sharing=False, kv_dtype=kv)
    seqs = [engine.open_request() for _ in range(batch)]
    engine.run_step([StepEntry(s, ids(30 + i, i), [-1]) for i, s in enumerate(seqs)])
    seen = WatchedFew(monkeypatch)
    for step in range(3):
        logits = engine.run_step([StepEntry(s, ids(1, 10 * step + i), [0]) for i, s in enumerate(seqs)])
        assert bool(logits.isfinite().all())
    assert seen.products == 3 * (2 * 4 + 1) and seen.norms == 3 * 4
    # (sums where k is divided: both layers' projection back, and the feed-forward's ahead of a norm in 8 bits)
    assert seen.whole == (3 * (2 * (model.split_o > 1) + (model.split_down > 1)) if batch <= 2 else 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("kv", [None, E4M3])
def test_a_sequence_decodes_alike_alone_and_beside_others(device, kind, kv):
    """The logits of one sequence's decode steps with one, two and four rows: products have the same bits, sums of parts and attention are rounded elsewhere."""
    model = model_of(kind, device)
    logits = []
    for batch in (1, 2, 4):
        engine = GenerationEngine(model, max_batch=batch, max_seq_len=96, enable_prefix_sharing=False, kv_dtype=kv)
        seqs = [engine.open_request() for _ in range(batch)]
        engine.run_step([StepEntry(s, ids(30 + i, i)) for i, s in enumerate(seqs)])
        logits.append(torch.stack([engine.run_step([StepEntry(s, ids(1, 10 * step + i), [0]) for i, s in enumerate(seqs)])[0].float().cpu()
                                   for step in range(3)]))
    # (a number of a row may go to its neighbour where a sum is rounded the other way: as far as 8 bits take the logits, 0.08, at the very most; another
    # position, cache page or row is off by more than 1)
    for other in logits[1:]:
        assert float((other - logits[0]).norm() / logits[0].norm()) < 0.08


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("kv", [None, E4M3])
@pytest.mark.parametrize("batch", [1, 2])
def test_captured_steps_of_few_sequences_are_the_same(kind, kv, batch):
    model = model_of(kind, "cuda")
    prompts = [ids(70, 1), ids(3, 2)][:batch]
    outs = [GenerationEngine(model, max_batch=batch, max_seq_len=160, use_cuda_graph=g, kv_dtype=kv).generate(prompts, 12) for g in (False, True)]
    assert outs[0] == outs[1]


@pytest.mark.parametrize("device", DEVICES)
def test_drawing_of_tokens_with_infinite_biases(device):
    """A token that is certain, two of them, one that may not come all the same, and nothing to draw from."""
    model = model_of("llama", device, False)
    engine = GenerationEngine(model, max_batch=2, max_seq_len=64)
    inf, prompts = float("inf"), [ids(9, 1), ids(20, 2)]
    for temperature in (0.0, 0.7, 2.0):
        warm = dict(temperature=temperature, seed=4)
        assert engine.generate(prompts, 4, sampling=Sampling(biases={7: inf, 9: 3.0}, **warm)) == [[7] * 4] * 2
        assert engine.generate(prompts, 4, sampling=Sampling(biases={7: inf}, top_k=5, top_p=0.9, **warm)) == [[7] * 4] * 2
        two = [t for o in (engine.generate(prompts, 24, sampling=Sampling(biases={7: inf, 500: inf}, **warm))) for t in o]
        assert set(two) == ({7, 500} if temperature else {7})
        out = engine.generate(prompts, 3, sampling=Sampling(biases={7: inf}, allowed=lambda p, a: [3, 5], **warm))
        assert {t for o in out for t in o} <= {3, 5}
        assert engine.generate(prompts, 3, sampling=Sampling(biases={t: -inf for t in range(512)}, **warm)) == [[], []]
    with pytest.raises(ValueError):
        Sampling(biases={3: float("nan")})


def test_forms_of_what_a_grammar_allows():
    """Ids and truth values as tensors, arrays, lists and other collections are the same masks; others are refused."""
    import numpy as np

    from nkipy_b200.models.engine import StepRules

    mask = np.arange(70) % 3 == 1
    some = np.flatnonzero(mask)
    forms = [mask, mask.tolist(), tuple(mask), torch.from_numpy(mask), some, some.astype(np.int32), some.astype(np.uint16), some.tolist(), tuple(some), set(some.tolist()),
             torch.from_numpy(some), torch.from_numpy(some).int(), range(1, 70, 3), (int(t) for t in some), {int(t): None for t in some}.keys()]
    for form in forms:
        rules = StepRules(Sampling(allowed=lambda p, a: form), 70, 2, 8, "cpu")
        rules.allow([1], [[1]], [[]])
        assert rules.rules.mask[0].tolist() == [-1] * 3
        assert torch.equal(rules.rules.mask[1:], ops.pack_mask(torch.from_numpy(mask)[None])), type(form)
    for none in ([], (), np.array([], dtype=np.int64), set(), torch.zeros(0), np.zeros(70, dtype=bool), iter([])):
        rules = StepRules(Sampling(allowed=lambda p, a: none), 70, 2, 8, "cpu")
        rules.allow([0], [[1]], [[]])
        assert rules.rules.mask.tolist() == [[0] * 3, [-1] * 3]
    for bad in (mask[:69], mask[None], [True] * 71, torch.ones(71, dtype=torch.bool), [1.5], np.array([2.0]), [70], {-1}, torch.tensor([3.0])):
        rules = StepRules(Sampling(allowed=lambda p, a: bad), 70, 2, 8, "cpu")
        with pytest.raises(ValueError):
            rules.allow([0], [[1]], [[]])


def test_quantising_goes_on_where_it_stopped(monkeypatch):
    model, whole = model_of("llama", "cpu", quantize=False), model_of("llama", "cpu")
    of, calls = ops.QuantizedWeight.of, []

    def short_of_memory(w):
        calls.append(w)
        if len(calls) == 4:
            raise torch.OutOfMemoryError("no more")
        return of(w)

    with monkeypatch.context() as m:
        m.setattr(ops.QuantizedWeight, "of", short_of_memory)
        with pytest.raises(torch.OutOfMemoryError):
            model.quantize_weights()
        assert not model.quantized
        model.quantize_weights()
    assert model.quantized and len(calls) == 4 * 2 + 1 + 1
    outs = [GenerationEngine(m, max_batch=1, max_seq_len=64).generate([ids(9, 1)], 4) for m in (model, whole)]
    assert outs[0] == outs[1]
