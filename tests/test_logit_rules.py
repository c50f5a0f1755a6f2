"""Penalties, biases and masks on logits, and the most likely token under them, against a plain implementation token by token."""

import math

import pytest
import torch

from nkipy_b200 import ops
from nkipy_b200.ops.logit_rules import mask_words

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF, F32 = torch.bfloat16, torch.float32
INF = math.inf


# ------------------------------------------------------------------------------------------------ oracle
def oracle(logits, r):
    """fp32 logits, and the tokens with the newest in its place: Python's numbers of 64 bits, one token after another."""
    B, V = logits.shape
    y = [[float(v) for v in row] for row in logits.float()]
    tokens = None if r.get("tokens") is None else r["tokens"].clone()
    for b in range(B):
        if tokens is not None:
            n = min(int(r["lens"][b]), tokens.shape[1])
            if n > 0 and r.get("ids") is not None:
                tokens[b, n - 1] = r["ids"][b]
            history = tokens[b, :max(n, 0)].tolist()
            prompt = int(r["prompt_lens"][b]) if r.get("prompt_lens") is not None else 0
            rep, freq, pres = (d if r.get(k) is None else float(r[k][b]) for k, d in (("repetition", 1.0), ("frequency", 0.0), ("presence", 0.0)))
            times, seen = {}, set()
            for i, t in enumerate(history):
                if 0 <= t < V:
                    seen.add(t)
                    times[t] = times.get(t, 0) + (i >= prompt)
            for t in seen:
                v = y[b][t]
                v = v / rep if v > 0 else v * rep
                v -= freq * times[t]
                y[b][t] = v - pres if times[t] else v
        if r.get("bias_ids") is not None:
            total = {}
            for t, v in zip(r["bias_ids"][b].tolist(), r["bias_values"][b].tolist()):
                if 0 <= t < V:
                    total[t] = total.get(t, 0.0) + v
            for t, v in total.items():
                y[b][t] += v
        m = -1 if r.get("mask") is None else (b if r.get("mask_rows") is None else int(r["mask_rows"][b]))
        if r.get("mask") is not None and 0 <= m < r["mask"].shape[0]:
            words = r["mask"][m].tolist()
            for t in range(V):
                if not (words[t // 32] >> (t % 32)) & 1:
                    y[b][t] = -INF
    return torch.tensor(y, dtype=torch.float64).float(), tokens


def oracle_ids(y):
    ids = []
    for row in y.tolist():
        best, at = -INF, -1
        for t, v in enumerate(row):
            if v > best:
                best, at = v, t
        ids.append(at)
    return torch.tensor(ids, dtype=torch.int32)


def make(seed, B, V, width=0, lens=None, penalties=True, biases=0, masks=None, ids=True):
    """Rules on the CPU as a dict."""
    g = torch.Generator().manual_seed(seed)
    r = {}
    if width:
        r["tokens"] = (V * torch.rand((B, width), generator=g) ** 4).int().clamp(max=V - 1)
        r["lens"] = torch.randint(1, width + 1, (B,), generator=g).int() if lens is None else torch.tensor(lens).int()
        r["prompt_lens"] = (r["lens"] * torch.rand((B,), generator=g)).int()
        if ids:
            r["ids"] = (V * torch.rand((B,), generator=g) ** 4).int().clamp(max=V - 1)
        if penalties:
            r["repetition"] = 1 + 0.3 * torch.rand((B,), generator=g)
            r["frequency"] = torch.randn((B,), generator=g) * 0.3
            r["presence"] = torch.randn((B,), generator=g) * 0.3
    if biases:
        r["bias_ids"] = torch.randint(-1, V, (B, biases), generator=g).int()
        r["bias_ids"][:, -1] = r["bias_ids"][:, 0]
        r["bias_values"] = torch.randn((B, biases), generator=g)
        r["bias_values"][:, biases // 2] = -INF
    if masks:
        allowed = torch.rand((B if masks == "rows" else 2, V), generator=g) < 0.3
        allowed[0] = False
        r["mask"] = ops.pack_mask(allowed)
        if masks == "shared":
            r["mask_rows"] = torch.randint(-1, 3, (B,), generator=g).int()
    return r


def there(r, device):
    return ops.LogitRules(**{k: v.to(device, copy=True) for k, v in r.items()})


def logits_of(seed, B, V, dtype):
    return (3 * torch.randn((B, V), generator=torch.Generator().manual_seed(seed + 1))).to(dtype)


def check(x, r, device, places=("new", "apart", "in place")):
    want, tokens = oracle(x, r)
    for place in places:
        rules, given = there(r, device), x.to(device, copy=True)
        out = {"new": None, "apart": torch.empty_like(given), "in place": given}[place]
        got = ops.apply_rules(given, rules, out=out)
        assert out is None or got is out
        assert torch.equal(got.cpu(), want.to(x.dtype)), place
        if place != "in place":
            assert torch.equal(given.cpu(), x)
        if tokens is not None:
            assert torch.equal(rules.tokens.cpu(), tokens)
    rules, given = there(r, device), x.to(device, copy=True)
    ids = ops.argmax(given, rules=rules)
    assert ids.dtype is torch.int32 and torch.equal(ids.cpu(), oracle_ids(want))
    if tokens is not None:
        assert torch.equal(rules.tokens.cpu(), tokens)
    assert torch.equal(given.cpu(), x)


CASES = [dict(width=20), dict(width=20, penalties=False), dict(biases=5), dict(masks="rows"), dict(masks="shared"), dict(width=40, biases=9, masks="rows"),
         dict(width=3, biases=1, masks="shared"), dict(width=700, biases=300), dict(width=20, ids=False)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,V", [(1, 1), (2, 31), (3, 33), (1, 1000), (5, 4099)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rules(device, dtype, B, V, case):
    check(logits_of(case, B, V, dtype), make(case * 10 + B, B, V, **CASES[case]), device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,V", [(1, 128256), (3, 151936), (2, 201088), (1, 300007), (40, 9001)])
def test_large_vocabularies(dtype, B, V):
    check(logits_of(V, B, V, dtype), make(B, B, V, width=1500, biases=20, masks="shared"), "cuda", places=("new", "in place"))


@pytest.mark.gpu
def test_many_rows_over_several_turns():
    """Slices of more tokens than counts are held for at a time."""
    B, V = 80, 210000
    g = torch.Generator().manual_seed(1)
    x = torch.randn((B, V), generator=g).to(BF)
    r = make(2, B, V, width=64, biases=4)
    rules = there(r, "cuda")
    got, ids = ops.apply_rules(x.cuda(), rules), ops.argmax(x.cuda(), rules=rules)
    for b in (0, 41, 79):
        want, _ = oracle(x[b:b + 1], {k: v[b:b + 1] for k, v in r.items()})
        assert torch.equal(got[b:b + 1].cpu(), want.to(BF))
        assert torch.equal(ids[b:b + 1].cpu(), oracle_ids(want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width,V,spread", [(4500, 5000, 1), (9001, 3001, 1), (20000, 700, 1), (20000, 40000, 30)])
def test_long_lists(device, width, V, spread):
    """More named tokens than a list holds, and more occurrences than half a word counts."""
    r = make(width, 2, V, width=width, lens=[width, width - 3], biases=2, masks="rows" if spread == 1 else None)
    g = torch.Generator().manual_seed(5)
    r["tokens"] = (V * torch.rand((2, width), generator=g) ** spread).int().clamp(max=V - 1)
    check(logits_of(width, 2, V, BF), r, device)


@pytest.mark.parametrize("device", DEVICES)
def test_without_rules(device):
    x = logits_of(0, 3, 1000, BF)
    check(x, {}, device)
    assert torch.equal(ops.argmax(x.to(device), rules=ops.LogitRules()), ops.argmax(x.to(device)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties_infinities_and_nan(device, dtype):
    V = 600
    low = float(torch.finfo(dtype).min)
    x = torch.zeros((8, V), dtype=dtype)
    x[0, [77, 300]] = 5                                  # a tie
    x[1] = -INF                                          # nothing
    x[2] = low                                           # the lowest value everywhere
    x[3] = torch.linspace(-1, 1, V).to(dtype)
    x[3, 10], x[3, 11] = float("nan"), INF
    x[4] = float("nan")
    x[5] = -1.0
    x[6, 0], x[6, 1] = -0.0, 0.0
    x[7, 5:] = INF
    ids = ops.argmax(x.to(device), rules=ops.LogitRules())
    assert ids.tolist() == [77, -1, 0, 11, -1, 0, 0, 5]
    allowed = torch.ones((8, V), dtype=torch.bool)
    allowed[0, 77], allowed[2, 0], allowed[5], allowed[7, 5] = False, False, False, False
    rules = ops.LogitRules(mask=ops.pack_mask(allowed).to(device))
    assert ops.argmax(x.to(device), rules=rules).tolist() == [300, -1, 1, 11, -1, -1, 0, 6]
    left = ops.apply_rules(x.to(device), rules).cpu()
    assert bool((left[5] == -INF).all()) and float(left[0, 77]) == -INF and bool(left[3, 10].isnan())
    # what is masked may be anything
    x[3, 10] = 0
    allowed[3, 11] = False
    assert ops.argmax(x.to(device), rules=ops.LogitRules(mask=ops.pack_mask(allowed).to(device))).tolist()[3] == V - 1


@pytest.mark.parametrize("device", DEVICES)
def test_ties_of_named_and_other_tokens(device):
    """A bias lifts a token to a value that others have, on either side of it and in the same piece of eight."""
    V = 100
    for at, others, want in ((18, [21, 40], 18), (18, [17, 40], 17), (90, [5], 5), (0, [1], 0), (15, [16], 15), (16, [15], 15)):
        x = torch.zeros((1, V))
        x[0, others] = 2.0
        rules = ops.LogitRules(bias_ids=torch.tensor([[at]]).int().to(device), bias_values=torch.tensor([[2.0]]).to(device))
        assert ops.argmax(x.to(device), rules=rules).tolist() == [want]


@pytest.mark.parametrize("device", DEVICES)
def test_lengths_and_ids_at_their_ends(device):
    """Rows without tokens, longer than their list, with ids outside of the vocabulary, the same id throughout, prompts of everything and of less than nothing."""
    B, V, width = 8, 300, 12
    x = logits_of(3, B, V, F32)
    r = make(4, B, V, width=width, lens=[0, -1, 1, width, width + 9, width, width, width])
    r["tokens"][5] = 7
    r["ids"][5] = 7
    r["tokens"][6, :6] = torch.tensor([-1, V, 2 ** 31 - 1, -2 ** 31, V - 1, 0]).int()
    r["ids"][4] = -5
    r["prompt_lens"][7], r["prompt_lens"][6] = width + 3, -4
    check(x, r, device)
    r["bias_ids"] = torch.tensor([[0, V, V - 1, -9, 0, 0]] * B).int()
    r["bias_values"] = torch.tensor([[1e8, 5.0, -2.0, INF, -1e8, 1.0]] * B)
    check(x, r, device)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_lie_apart(device):
    B, V = 4, 257
    for lead, dtype in ((0, BF), (1, BF), (8, F32), (3, F32)):
        x = logits_of(9, B, V + lead + 15, dtype)
        r = make(6, B, V, width=30, biases=6, masks="rows")
        want, tokens = oracle(x[:, lead:lead + V], r)
        wide = {k: torch.nn.functional.pad(v, (0, 5), value=3) if v.dim() == 2 else v for k, v in r.items()}
        rules = there(wide, device)
        for name in ("tokens", "bias_ids", "bias_values", "mask"):
            t = getattr(rules, name)
            setattr(rules, name, t[:, :t.shape[1] - 5])
        view = x.to(device, copy=True)[:, lead:lead + V]
        assert torch.equal(ops.argmax(view, rules=rules).cpu(), oracle_ids(want))
        assert torch.equal(ops.apply_rules(view, rules).cpu(), want.to(dtype))
        whole = view.new_full((B, V + 40), 4.0)
        ops.apply_rules(view, rules, out=whole[:, 8:8 + V])
        assert torch.equal(whole[:, 8:8 + V].cpu(), want.to(dtype))
        assert bool((whole[:, :8] == 4).all()) and bool((whole[:, 8 + V:] == 4).all())
        ops.apply_rules(view, rules, out=view)
        assert torch.equal(view.cpu(), want.to(dtype))


def test_masks_are_packed():
    allowed = torch.rand((3, 77), generator=torch.Generator().manual_seed(0)) < 0.5
    words = ops.pack_mask(allowed)
    assert words.shape == (3, mask_words(77)) and words.dtype is torch.int32
    for m in range(3):
        for t in range(77):
            assert bool((int(words[m, t // 32]) >> (t % 32)) & 1) == bool(allowed[m, t])
    assert torch.equal(ops.pack_mask(allowed[1]), words[1])
    assert ops.pack_mask(torch.ones(32, dtype=torch.bool)).tolist() == [-1]


def test_refusals():
    B, V = 2, 40
    x, r = torch.zeros((B, V)), make(0, B, V, width=6, biases=3, masks="rows")

    def bad(error, logits=x, out=None, **kw):
        rules = ops.LogitRules(**{**r, **kw})
        with pytest.raises(error):
            ops.apply_rules(logits, rules, out=out)
        if out is None:
            with pytest.raises(error):
                ops.argmax(logits, rules=rules)

    bad(TypeError, logits=x.half())
    bad(TypeError, logits=x.double())
    bad(ValueError, logits=x[0])
    bad(ValueError, logits=x.T)
    bad(ValueError, out=torch.zeros((B, V - 1)))
    bad(ValueError, out=torch.zeros((V, B)).T)
    bad(TypeError, out=x.to(BF))
    bad(ValueError, out=x.new_zeros(B * V + 1).as_strided((B, V), (V - 1, 1)))
    bad(TypeError, tokens=r["tokens"].long())
    bad(ValueError, tokens=r["tokens"][:1])
    bad(ValueError, tokens=None)
    bad(ValueError, lens=None)
    bad(ValueError, lens=r["lens"][:1])
    bad(TypeError, ids=r["ids"].long())
    bad(TypeError, repetition=r["repetition"].double())
    bad(ValueError, frequency=torch.zeros((B, 1)))
    bad(ValueError, bias_ids=None)
    bad(ValueError, bias_values=r["bias_values"][:, :2])
    bad(TypeError, bias_values=r["bias_values"].to(BF))
    bad(ValueError, mask=r["mask"][:, :1])
    bad(ValueError, mask=r["mask"][:1])
    bad(ValueError, mask=None, mask_rows=torch.zeros(B).int())
    bad(TypeError, mask_rows=torch.zeros(B))
    with pytest.raises(TypeError):
        ops.apply_rules(x, None)
    with pytest.raises(ValueError):
        ops.argmax(x, out_vals=torch.zeros(B), rules=ops.LogitRules())
    with pytest.raises(ValueError):
        ops.argmax(x, out_ids=torch.zeros(B + 1).int(), rules=ops.LogitRules())
    assert ops.apply_rules(x[:0], ops.LogitRules()).shape == (0, V) and ops.argmax(x[:0], rules=ops.LogitRules()).shape == (0,)


# ------------------------------------------------------------------------------------------------ captured, and on other streams
@pytest.mark.gpu
def test_captured_and_replayed():
    """A graph that goes on by a token at every replay: lengths, ids, penalties and masks are read when it runs."""
    B, V, width = 5, 5000, 30
    r = make(8, B, V, width=width, lens=[1, 5, 9, 2, 20], biases=4, masks="shared")
    rules = there(r, "cuda")
    x = logits_of(8, B, V, BF).cuda()
    ops.argmax(x, rules=there(r, "cuda"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = ops.argmax(x, rules=rules)
        rules.ids.copy_(ids)
        rules.lens.add_(1)
    state = {k: v.clone() for k, v in r.items()}
    for k, v in state.items():
        getattr(rules, k).copy_(v)
    for i in range(6):
        x.copy_(logits_of(20 + i, B, V, BF))
        graph.replay()
        want, state["tokens"] = oracle(x.cpu(), state)
        state["ids"], state["lens"] = oracle_ids(want), state["lens"] + 1
        assert torch.equal(ids.cpu(), state["ids"]) and torch.equal(rules.tokens.cpu(), state["tokens"])


@pytest.mark.gpu
def test_streams_beside_one_another():
    B, V = 3, 70001
    sets = [(logits_of(i, B, V, F32), make(i, B, V, width=300, biases=7)) for i in range(4)]
    want = [oracle_ids(oracle(x, r)[0]) for x, r in sets]
    given = [(x.cuda(), there(r, "cuda")) for x, r in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, (x, r) in zip(streams, given):
            with torch.cuda.stream(s):
                got.append(ops.argmax(x, rules=r))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------------------------------------ the end of a decode step
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,H,V", [(1, 64, 500), (5, 256, 1001), (64, 512, 4000)])
def test_from_the_last_layer_to_the_token(device, B, H, V):
    """Residual add, norm, vocabulary product in 8 bits, rules, most likely token: ids, of logits that are told apart by more than their tolerance."""
    g = torch.Generator().manual_seed(B)
    x, h = torch.randn((B, H), generator=g).to(BF), torch.randn((B, H), generator=g).to(BF)
    norm = (1 + 0.2 * torch.randn((H,), generator=g)).to(BF)
    w = ops.QuantizedWeight.of((torch.randn((V, H), generator=g) * 3 * H ** -0.5).to(BF))
    r = make(B, B, V, width=20, biases=3, masks="shared")
    rules = there(r, device)
    resid, rows = ops.add_rmsnorm(x.to(device), norm.to(device), residual_in=h.to(device), quantize=True)
    logits = ops.linear(rows, ops.QuantizedWeight(w.values.to(device), w.scale.to(device)), fp32_out=True)
    ids = ops.argmax(logits, rules=rules)
    # the same steps in 64 bits from the numbers, which are exact
    total = (x.double() + h.double()).to(BF)
    assert torch.equal(resid.cpu(), total)
    p = total.double() * norm.double()
    q = torch.round(127 * p / p.abs().amax(-1, keepdim=True))
    factor = p.abs().amax(-1) / 127 / torch.sqrt(total.double().square().mean(-1) + 1e-6)
    y = (q @ w.values.double().T) * factor[:, None] * w.scale.double()
    # (scale: 64 roundings, as for the rows; three more of the product)
    assert bool(((logits.cpu().double() - y).abs() <= 67 * 2.0 ** -24 * y.abs() + 1e-30).all())
    want, _ = oracle(y, r)
    top2 = want.double().nan_to_num(neginf=-1e30).topk(2, -1).values
    clear = ((top2[:, 0] - top2[:, 1]) > 1e-4) | (top2[:, 0] == -1e30)          # (nothing is left: -1)
    assert int(clear.sum()) >= B - 1
    assert torch.equal(ids.cpu()[clear], oracle_ids(want)[clear])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("biases,V", [(1, 50), (510, 3001), (512, 3008), (513, 700), (1500, 4003)])
def test_many_biases(device, dtype, biases, V):
    """As many as lie in shared memory, fewer and more; tokens with several; rows that start on sixteen bytes and others."""
    check(logits_of(biases, 3, V, dtype), make(biases, 3, V, width=30, biases=biases, masks="rows"), device)
    r = make(biases, 3, V, biases=biases)
    r["bias_ids"][:, ::3] = 7
    check(logits_of(biases, 3, V, dtype), r, device)


@pytest.mark.parametrize("device", DEVICES)
def test_more_named_tokens_than_are_listed(device):
    r = make(5, 2, 9000, width=4000)
    g = torch.Generator().manual_seed(6)
    r["tokens"] = torch.stack([torch.randperm(9000, generator=g)[:4000] for _ in range(2)]).int()
    r["lens"] = torch.tensor([4000, 1100], dtype=torch.int32)
    check(logits_of(5, 2, 9000, BF), r, device)


def test_rows_that_share_their_tokens():
    """Read they may be; the newest tokens have no place of their own in them."""
    tokens = torch.arange(6, dtype=torch.int32).expand(3, 6)
    rules = dict(tokens=tokens, lens=torch.tensor([6, 2, 0], dtype=torch.int32), presence=torch.ones(3))
    y = ops.apply_rules(torch.zeros((3, 8)), ops.LogitRules(**rules))
    assert (y != 0).sum(-1).tolist() == [6, 2, 0]
    with pytest.raises(ValueError):
        ops.apply_rules(torch.zeros((3, 8)), ops.LogitRules(**rules, ids=torch.zeros(3, dtype=torch.int32)))


@pytest.mark.parametrize("device", DEVICES)
def test_logits_are_rounded_once(device):
    """Sums beside the middle of two bf16 numbers, which 32 bits hold as the middle itself; and the middle."""
    middle, off = 2.0 ** -8, 2.0 ** -31
    x = torch.ones((1, 24), dtype=BF)
    x[0, 8:16], x[0, 16:] = -1.0, 1 + 2.0 ** -7
    add = torch.tensor([[middle + off, middle - off, middle, 2 ** -7, -off, off, 0, -middle / 2,
                         -middle - off, -middle + off, -middle, 0, -off, off, -2.0 ** -7, middle / 2,
                         middle + off, middle - off, middle, -middle, -middle - off, -middle + off, off, -off]])
    up, upper = 1 + 2.0 ** -7, 1 + 2.0 ** -6
    want = [up, 1, 1, up, 1, 1, 1, 1, -up, -1, -1, -1, -1, -1, -up, -1,          # (1 - 2^-9 lies in the middle: to the even one)
            upper, up, upper, 1, 1, up, up, up]
    rules = ops.LogitRules(bias_ids=torch.arange(24).int()[None].to(device), bias_values=add.to(device))
    for out in (None, x.to(device, copy=True)):
        assert ops.apply_rules(x.to(device) if out is None else out, rules, out=out).tolist() == [want]
    # penalties alike: 1 + 2^-8 + 2^-31 again; and numbers beyond the largest one
    x = torch.tensor([[1.0, 3.3895e38, -3.3895e38]], dtype=BF)
    rules = ops.LogitRules(tokens=torch.arange(3).int()[None].to(device), lens=torch.tensor([3]).int().to(device),
                           frequency=torch.tensor([-(middle + off)]).to(device))
    assert float(ops.apply_rules(x.to(device), rules)[0, 0]) == up
    rules.frequency = torch.tensor([3e38]).to(device)
    assert ops.apply_rules(x.to(device), rules).tolist()[0][2] == -INF
    # the choice compares 32 bits
    same = torch.ones((1, 2), dtype=BF)
    rules = ops.LogitRules(bias_ids=torch.tensor([[0, 1]]).int().to(device), bias_values=torch.tensor([[middle, middle + off]]).to(device))
    assert ops.argmax(same.to(device), rules=rules).tolist() == [0]
