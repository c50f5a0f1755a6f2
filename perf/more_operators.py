"""Operators of products in 8-bit whole numbers, and of the choice of a token under rules, for measuring them and comparing their outputs.

A row x of activations, or of a weight, is held as whole numbers and one factor: q = the whole number nearest to 127 x / max|x| (ties to
the even one), scale = max|x| / 127, so that x is about q * scale.  A row that is not finite has a scale of NaN and numbers of zero.

    rows      residual add and RMS norm, SwiGLU gate, or nothing, and then whole numbers and scales of the rows
    product   activations by a weight in 8 bits: q . w summed as whole numbers, times both scales; bias, residual, SwiGLU gate
    rules     penalties for repeated tokens, biases and masks on logits: the logits that are left, or the most likely token
    choose    the end of a decode step: residual add, norm, vocabulary product in 8 bits, rules, most likely token

    listed()              named cases
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   inputs on the GPU
    run(state)            one pass; `own`: through the framework's operators, otherwise by elementary torch operations
    work(case)            bytes and operations that a pass cannot do without
    exact(case, seed)     what `run` returns, in 64 bits

Rules of one row, in this order and rounded once at the end: a token that occurs in the row's tokens (those of its prompt too) is divided
by the repetition penalty where its logit is above zero and multiplied by it elsewhere; the frequency penalty times its occurrences
among the answer's tokens is taken off, and the presence penalty where there is one; then come the biases, of which several for one
token add up; a token whose bit of the mask is zero is minus infinity.  Where nothing is left the most likely token is -1.
"""

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5


def rows_case(form, tokens, width, splits=0, **name):
    """form "norm": bf16 rows and a residual; "gate": twice the width, gate and up, bf16 or that many fp32 partial sums; "plain": bf16 rows."""
    return dict(op="rows", form=form, tokens=tokens, width=width, splits=splits, **name)


def product_case(tokens, k, n, given="bf16", gated=False, bias=False, residual=False, fp32=False, **name):
    """given "bf16": rows that the product brings into 8 bits; "int8": rows that are; gated: n columns of gate and n of up."""
    return dict(op="product", tokens=tokens, k=k, n=n, given=given, gated=gated, bias=bias, residual=residual, fp32=fp32, **name)


def rules_case(batch, vocab, lo, hi, want="ids", fp32=False, penalties=True, biases=0, mask="none", **name):
    """batch rows of lo to hi tokens (0: no history); want "ids": the most likely token, "logits": all of them; biases: entries of a row;
    mask "rows": one of each row, "shared": few that rows point to, some to none."""
    return dict(op="rules", batch=batch, vocab=vocab, lo=lo, hi=hi, want=want, fp32=fp32, penalties=penalties, biases=biases, mask=mask, **name)


def choose_case(batch, hidden, vocab, lo, hi, biases=0, mask="none", **name):
    return dict(op="choose", batch=batch, hidden=hidden, vocab=vocab, lo=lo, hi=hi, penalties=True, biases=biases, mask=mask, **name)


def listed():
    return [
        # the newest token of one user's chat ahead of a layer's first projection: the latency of a launch
        rows_case("norm", 1, 4096, name="rows-1"),
        # a full prefill step of the serving benchmark
        rows_case("norm", 16384, 4096, name="rows-16384"),
        # the feed-forward of a decode step of the serving benchmark, gate and up left as two partial sums
        rows_case("gate", 64, 14336, splits=2, name="gate-64"),
        # the QKV projection of one user's chat
        product_case(1, 4096, 6144, name="product-1"),
        # the feed-forward's second projection in a decode step of the serving benchmark
        product_case(64, 14336, 4096, residual=True, name="product-64"),
        # gate and up projections of a packed step of continuous batching: one prompt of odd length and 24 single tokens
        product_case(414, 4096, 14336, given="int8", gated=True, name="gated-414"),
        # the same of half a prefill step of the serving benchmark
        product_case(8192, 4096, 14336, given="int8", gated=True, name="gated-8192"),
        # one user's chat with penalties; logits in 32 bits go on to a sampler
        rules_case(1, 128256, 203, 203, want="logits", fp32=True, name="rules-1"),
        # greedy decoding of the serving benchmark's batch, with a few biases
        rules_case(64, 128256, 1024, 2000, biases=9, name="rules-64"),
        # structured answers of many users: every row has a grammar's mask
        rules_case(128, 151936, 77, 1500, want="logits", mask="rows", name="rules-128"),
        # one user's chat from the last layer to the token
        choose_case(1, 4096, 128256, 203, 203, name="choose-1"),
        # the serving benchmark's batch, some rows with a grammar
        choose_case(64, 4096, 128256, 1024, 2000, biases=3, mask="shared", name="choose-64"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["rows", "product", "product", "rules", "choose"])
        if op == "rows":
            form = rng.choice(["norm", "gate", "plain"])
            c = rows_case(form, _log(rng, 1, 20000), _log(rng, 64, 16384), splits=rng.choice([0, 1, 2, 5]) if form == "gate" else 0)
        elif op == "product":
            k, n = (rng.choice([2048, 2880, 4096, 6144, 14336]) if rng.random() < 0.5 else _log(rng, 64, 16384) for _ in range(2))
            gated = rng.random() < 0.3
            bias, residual, fp32 = (not gated and rng.random() < 0.3 for _ in range(3))
            c = product_case(_log(rng, 1, 9000), k, n, given=rng.choice(["bf16", "int8"]), gated=gated, bias=bias, residual=residual and not fp32,
                             fp32=fp32)
        else:
            batch, hi = _log(rng, 1, 160), _log(rng, 1, 9000)
            vocab = rng.choice([32000, 128256, 151936, 201088]) if rng.random() < 0.5 else _log(rng, 500, 200000)
            lo, biases, mask = rng.randint(max(hi // 3, 1), hi), rng.choice([0, 0, 1, 40, 300]), rng.choice(["none", "rows", "shared"])
            if op == "rules":
                if rng.random() < 0.2:
                    lo = hi = 0
                c = rules_case(batch, vocab, lo, hi, want=rng.choice(["ids", "logits"]), fp32=rng.random() < 0.5,
                               penalties=hi > 0 and rng.random() < 0.8, biases=biases, mask=mask)
            else:
                c = choose_case(batch, rng.choice([1024, 2048, 2880, 4096]), vocab, lo, hi, biases=biases, mask=mask)
        if _cost(c) <= max(_cost(x) for x in listed() if x["op"] == op):
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _lengths(c):
    """Tokens of every row: spread over the case's range, its ends among them."""
    n = c["batch"]
    return [c["hi"] - (c["hi"] - c["lo"]) * ((7 * i) % n) // max(n - 1, 1) for i in range(n)]


def _rules_bytes(c):
    words = 4 * -(-c["vocab"] // 32)
    return 4 * sum(_lengths(c)) + 8 * c["batch"] * c["biases"] + words * {"none": 0, "rows": c["batch"], "shared": min(c["batch"], 3)}[c["mask"]]


def work(c):
    if c["op"] == "rows":
        t, w = c["tokens"], c["width"]
        if c["form"] == "norm":                       # rows, residual, new residual, whole numbers and scale
            return {"bytes": t * (7 * w + 4) + 2 * w, "flops": 8 * t * w}
        per = {"plain": 2, "gate": 8 * c["splits"] if c["splits"] else 4}[c["form"]]
        return {"bytes": t * (per * w + w + 4), "flops": (5 if c["form"] == "plain" else 12 + 2 * c["splits"]) * t * w}
    if c["op"] == "product":
        m, k, n, f = c["tokens"], c["k"], c["n"], 2 if c["gated"] else 1
        x = m * (2 * k if c["given"] == "bf16" else k + 4)
        out = m * n * (4 if c["fp32"] else 2) + (2 * m * n if c["residual"] else 0) + (2 * n if c["bias"] else 0)
        return {"bytes": x + f * n * (k + 4) + out, "flops": 2 * f * m * n * k}
    cells = c["batch"] * c["vocab"]
    if c["op"] == "rules":
        e = 4 if c["fp32"] else 2
        return {"bytes": cells * e * (2 if c["want"] == "logits" else 1) + _rules_bytes(c), "flops": 3 * cells}
    h = c["hidden"]
    return {"bytes": c["batch"] * 6 * h + c["vocab"] * (h + 4) + 4 * cells + _rules_bytes(c), "flops": 2 * cells * h}


# ------------------------------------------------------------------------------------------------ inputs
def _rows(g, shape, size=1.0):
    """bf16 rows as a layer gives them: columns of unequal size, a few of them large."""
    spread = torch.exp(0.6 * torch.randn(shape[-1:], generator=g, device=DEV))
    return (size * torch.randn(shape, generator=g, device=DEV) * spread).to(torch.bfloat16)


def _weight(g, n, k):
    """A weight's whole numbers and scales, as `_eighths` would give them for normal weights."""
    q = (32 * torch.randn((n, k), generator=g, device=DEV, dtype=torch.float16)).round_().clamp_(-127, 127).to(torch.int8)
    q[:, 0] = 127
    return q, (torch.rand((n,), generator=g, device=DEV) + 0.5) * k ** -0.5 / 32


def _aligned(q):
    """The same numbers with rows that start on 16 bytes, as a program keeps them."""
    n, k = q.shape
    if k % 16 == 0:
        return q
    wide = torch.zeros((n, (k + 15) // 16 * 16), dtype=torch.int8, device=q.device)
    wide[:, :k] = q
    return wide[:, :k]


def _rules(c, g, r):
    """Tokens, penalties, biases and masks of a batch."""
    B, V, lens = c["batch"], c["vocab"], _lengths(c)
    s = {}
    u = lambda *shape: torch.rand(shape, generator=g, device=DEV)  # noqa: E731
    if c["hi"]:
        # few tokens make up much of a text; the place of the newest one is written by the call
        s["tokens"] = (V * u(B, c["hi"] + 5) ** 6).int().clamp(max=V - 1)
        s["ids"] = (V * u(B) ** 6).int().clamp(max=V - 1)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["prompts"] = torch.tensor([n * r.randint(0, 9) // 10 for n in lens], dtype=torch.int32, device=DEV)
    if c["penalties"] and c["hi"]:
        s["repetition"] = 1 + 0.1 * torch.randint(0, 5, (B,), generator=g, device=DEV).float()
        s["frequency"] = 0.25 * torch.randint(-1, 5, (B,), generator=g, device=DEV).float()
        s["presence"] = 0.25 * torch.randint(-1, 5, (B,), generator=g, device=DEV).float()
    if c["biases"]:
        n = c["biases"]
        at = (V * u(B, n)).int().clamp(max=V - 1)
        at[:, n // 2:][u(B, n - n // 2) < 0.3] = -1                       # rows with fewer
        at[:, n - 1] = at[:, 0]                                           # the same token twice
        s["bias_ids"], s["bias_values"] = at, 4 * u(B, n) - 2
        s["bias_values"][u(B, n) < 0.1] = -math.inf                       # tokens that are not wanted at all
    if c["mask"] != "none":
        G, words = (B if c["mask"] == "rows" else min(B, 3)), -(-V // 32)
        # a grammar leaves a few tokens, or most of them
        few = u(G, 1) < 0.6
        bits = u(G, words * 32) < torch.where(few, 20.0 / V, 0.9)
        bits[0, :] = bits[0, :] & (torch.arange(words * 32, device=DEV) >= V)         # one that leaves nothing
        s["mask"] = (bits.view(G, words, 32).long() << torch.arange(32, device=DEV)).sum(-1).to(torch.int32)
        if c["mask"] == "shared":
            s["mask_rows"] = torch.randint(-1, G, (B,), generator=g, device=DEV).int()
    return s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = random.Random(seed)
    s = {"case": c}
    if c["op"] == "rows":
        t, w = c["tokens"], c["width"]
        if c["form"] == "norm":
            s["x"], s["residual"] = _rows(g, (t, w)), _rows(g, (t, w), 2.0)
            s["norm"] = (1 + 0.2 * torch.randn((w,), generator=g, device=DEV)).to(torch.bfloat16)
        elif c["form"] == "gate" and c["splits"]:
            s["x"] = 2 * c["splits"] ** -0.5 * torch.randn((c["splits"], t, 2 * w), generator=g, device=DEV)
        else:
            s["x"] = _rows(g, (t, 2 * w if c["form"] == "gate" else w))
    elif c["op"] == "product":
        m, k, n = c["tokens"], c["k"], c["n"]
        x = _rows(g, (m, k))
        if c["given"] == "int8":
            q, s["x_scale"] = _eighths(x.double())
            s["x"] = _aligned(q)
        else:
            s["x"] = x
        w, s["w_scale"] = _weight(g, 2 * n if c["gated"] else n, k)
        s["w"] = _aligned(w)
        s["bias"] = _rows(g, (n,), 0.2) if c["bias"] else None
        s["residual"] = _rows(g, (m, n)) if c["residual"] else None
    else:
        if c["op"] == "rules":
            logits = 3 * torch.randn((c["batch"], c["vocab"]), generator=g, device=DEV)
            s["logits"] = logits if c["fp32"] else logits.to(torch.bfloat16)
        else:
            h = c["hidden"]
            s["x"], s["residual"] = _rows(g, (c["batch"], h)), _rows(g, (c["batch"], h), 2.0)
            s["norm"] = (1 + 0.2 * torch.randn((h,), generator=g, device=DEV)).to(torch.bfloat16)
            s["w"], s["w_scale"] = _weight(g, c["vocab"], h)
            s["w_scale"] *= 3                                             # logits as wide as a model's
        s["rules"] = _rules(c, g, r)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from nkipy_b200 import ops

    c = s["case"]
    if c["op"] == "rows":
        if c["form"] == "norm":
            h, q = ops.add_rmsnorm(s["x"], s["norm"], residual_in=s["residual"], eps=EPS, quantize=True)
            return dict(values=q.values, scale=q.scale, residual=h)
        q = ops.silu_mul(s["x"], quantize=True) if c["form"] == "gate" else ops.quantize_rows(s["x"])
        return dict(values=q.values, scale=q.scale)
    if c["op"] == "product":
        x = ops.QuantizedRows(s["x"], s["x_scale"]) if c["given"] == "int8" else s["x"]
        return ops.linear(x, ops.QuantizedWeight(s["w"], s["w_scale"]), bias=s["bias"], residual=s["residual"], gated=c["gated"],
                          fp32_out=c["fp32"])
    d = s["rules"]
    rules = ops.LogitRules(tokens=d.get("tokens"), lens=d.get("lens"), prompt_lens=d.get("prompts"), ids=d.get("ids"),
                           repetition=d.get("repetition"), frequency=d.get("frequency"), presence=d.get("presence"),
                           bias_ids=d.get("bias_ids"), bias_values=d.get("bias_values"), mask=d.get("mask"), mask_rows=d.get("mask_rows"))
    if c["op"] == "rules":
        if c["want"] == "ids":
            return _chosen(s, ids=ops.argmax(s["logits"], rules=rules))
        return _chosen(s, logits=ops.apply_rules(s["logits"], rules))
    h, x = ops.add_rmsnorm(s["x"], s["norm"], residual_in=s["residual"], eps=EPS, quantize=True)
    logits = ops.linear(x, ops.QuantizedWeight(s["w"], s["w_scale"]), fp32_out=True)
    return _chosen(s, ids=ops.argmax(logits, rules=rules), logits=logits, residual=h)


def _chosen(s, **more):
    return dict(more, tokens=s["rules"]["tokens"]) if "tokens" in s["rules"] else more


def _eighths(x):
    """Whole numbers and scales of rows in 64 bits, and the scale rounded once: a number next to a half could fall on its other side in 32."""
    top = x.abs().amax(-1, keepdim=True)
    q = torch.nan_to_num(127 * (x / top), nan=0.0, posinf=0.0, neginf=0.0).round()
    scale = torch.where(top.isfinite(), top / 127, torch.nan)
    return torch.where(top.isfinite(), q, 0.0).to(torch.int8), scale.squeeze(-1).float()


def _normed(s):
    """(residual stream, whole numbers of its norm, their scales).  The norm's factor is one for the row and leaves the numbers alone."""
    h = (s["x"].double() + s["residual"].double()).to(torch.bfloat16)
    q, scale = _eighths(h.double() * s["norm"].double())
    hf = h.float()
    return h, q, scale * torch.rsqrt((hf * hf).mean(-1) + EPS)


def _whole(q, w):
    """q . w of whole numbers; sums below 2^24, which is what they are in earnest, are exact in 32 bits."""
    return q.float() @ w.float().T


def _plain_product(s):
    c = s["case"]
    q, sx = (s["x"], s["x_scale"]) if c["given"] == "int8" else _eighths(s["x"].double())
    y = _whole(q, s["w"]) * sx[:, None] * s["w_scale"]
    if c["gated"]:
        gate, up = y[:, :c["n"]], y[:, c["n"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y if c["fp32"] else y.to(torch.bfloat16)


def _ruled(d, logits):
    """Logits in 64 bits under the rules; writes the newest tokens to their places."""
    B, V = logits.shape
    y = logits.double()
    if "tokens" in d:
        t = d["tokens"]
        t.scatter_(1, (d["lens"] - 1).long()[:, None], d["ids"][:, None])
        at = torch.arange(t.shape[1], device=DEV)
        there = at < d["lens"][:, None]
        seen = torch.zeros((B, V), device=DEV).scatter_add_(1, t.long(), there.float()) > 0
        count = torch.zeros((B, V), device=DEV).scatter_add_(1, t.long(), (there & (at >= d["prompts"][:, None])).float())
        if "repetition" in d:
            rep = d["repetition"].double()[:, None]
            y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
            y = y - d["frequency"].double()[:, None] * count - d["presence"].double()[:, None] * (count > 0)
    if "bias_ids" in d:
        on = d["bias_ids"] >= 0
        y = y.scatter_add(1, d["bias_ids"].clamp(min=0).long(), torch.where(on, d["bias_values"].double(), 0.0))
    if "mask" in d:
        bits = ((d["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=DEV)) & 1).bool().flatten(1)[:, :V]
        if "mask_rows" in d:
            rows = d["mask_rows"].long()
            bits = bits[rows.clamp(min=0)] | (rows < 0)[:, None]
        y = torch.where(bits, y, -math.inf)
    return y


def _first_largest(y):
    """Lowest index of the largest value of every row, as 32 bits hold it; -1 where all are minus infinity."""
    y = y.float()
    top = y.amax(-1, keepdim=True)
    at = torch.where(y == top, torch.arange(y.shape[1], device=DEV), y.shape[1]).amin(-1)
    return torch.where(top.squeeze(-1) == -math.inf, -1, at).int()


def _plain(s):
    c = s["case"]
    if c["op"] == "rows":
        if c["form"] == "norm":
            h, q, scale = _normed(s)
            return dict(values=q, scale=scale, residual=h)
        x = s["x"].double()
        if c["form"] == "gate":
            x = x.sum(0) if c["splits"] else x
            gate, up = x[:, :c["width"]], x[:, c["width"]:]
            x = gate / (1 + torch.exp(-gate)) * up
        q, scale = _eighths(x)
        return dict(values=q, scale=scale)
    if c["op"] == "product":
        return _plain_product(s)
    if c["op"] == "rules":
        y = _ruled(s["rules"], s["logits"])
        if c["want"] == "ids":
            return _chosen(s, ids=_first_largest(y))
        return _chosen(s, logits=y.to(s["logits"].dtype))
    h, q, scale = _normed(s)
    logits = _whole(q, s["w"]) * scale[:, None] * s["w_scale"]
    return _chosen(s, ids=_first_largest(_ruled(s["rules"], logits)), logits=logits, residual=h)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_eighths(x):
    """By a search among the halves between whole numbers: |x| / max|x| against (k + 1/2) / 127, both times 254 max|x|."""
    top = x.abs().amax(-1)
    k = torch.floor(127 * x.abs() / top[:, None]).nan_to_num(0.0)
    left = 254 * x.abs() - (2 * k + 1) * top[:, None]                     # whole number of 2^-n: exact for short x
    k = k + ((left > 0) | ((left == 0) & (k % 2 == 1))).double()
    return torch.copysign(k, x) + 0.0, top / 127


def _swish(g, u):
    return u * g * torch.special.expit(g)


def _exact_norm(s):
    h = (s["x"].double() + s["residual"].double()).to(torch.bfloat16).double()
    q, scale = _exact_eighths(h * s["norm"].double())
    return h, q, scale / torch.sqrt(h.square().sum(-1) / h.shape[1] + EPS)


def _exact_rules(s, logits):
    """Row by row, token by token of what the rules name."""
    c, d = s["case"], {k: v.cpu() for k, v in s["rules"].items()}
    y = logits.double().cpu()
    V = c["vocab"]
    for b in range(c["batch"]):
        row = y[b]
        if "tokens" in d:
            n, p = int(d["lens"][b]), int(d["prompts"][b])
            d["tokens"][b, n - 1] = d["ids"][b]
            if "repetition" in d:
                rep, fr, pr = (float(d[k][b]) for k in ("repetition", "frequency", "presence"))
                all_ids = torch.unique(d["tokens"][b, :n]).long()
                row[all_ids] = torch.where(row[all_ids] > 0, row[all_ids] / rep, row[all_ids] * rep)
                ids, times = torch.unique(d["tokens"][b, p:n], return_counts=True)
                row[ids.long()] -= fr * times.double() + pr
        if "bias_ids" in d:
            for i, v in zip(d["bias_ids"][b].tolist(), d["bias_values"][b].tolist()):
                if i >= 0:
                    row[i] += v
        if "mask" in d:
            m = int(d["mask_rows"][b]) if "mask_rows" in d else b
            if m >= 0:
                words = d["mask"][m].numpy().view("uint8")
                left = torch.zeros((len(words), 8), dtype=torch.bool)
                for j in range(8):
                    left[:, j] = torch.from_numpy((words >> j) & 1).bool()
                row[~left.flatten()[:V]] = -math.inf
    best, at = y.float().numpy().max(1), y.float().numpy().argmax(1)
    ids = torch.where(torch.from_numpy(best) == -math.inf, -1, torch.from_numpy(at)).int()
    return y.to(DEV), ids.to(DEV), d.get("tokens")


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rows":
        if c["form"] == "norm":
            h, q, scale = _exact_norm(s)
            return dict(values=q.to(torch.int8), scale=scale, residual=h)
        x = s["x"].double()
        if c["form"] == "gate":
            x = x.sum(0) if c["splits"] else x
            x = _swish(x[:, :c["width"]], x[:, c["width"]:])
        q, scale = _exact_eighths(x)
        return dict(values=q.to(torch.int8), scale=scale)
    if c["op"] == "product":
        if c["given"] == "int8":
            x = s["x"].double() * s["x_scale"].double()[:, None]
        else:
            q, scale = _exact_eighths(s["x"].double())
            x = q * scale[:, None]
        y = x @ (s["w"].double() * s["w_scale"].double()[:, None]).T
        y = _swish(y[:, :c["n"]], y[:, c["n"]:]) if c["gated"] else y
        for more in (s["bias"], s["residual"]):
            y = y if more is None else y + more.double()
        return y
    if c["op"] == "rules":
        y, ids, tokens = _exact_rules(s, s["logits"])
        out = dict(ids=ids) if c["want"] == "ids" else dict(logits=y)
    else:
        h, q, scale = _exact_norm(s)
        logits = (q @ s["w"].double().T) * (scale[:, None] * s["w_scale"].double())
        _, ids, tokens = _exact_rules(s, logits)
        out = dict(ids=ids, logits=logits, residual=h)
    return dict(out, tokens=tokens.to(DEV)) if tokens is not None else out
