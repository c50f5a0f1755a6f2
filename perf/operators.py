"""Operators of a key / value cache held in 8 bits, for measuring them and comparing their outputs.

A page of 32 tokens of one kv head holds e4m3 values [32, dim] and one power of two per token: a head's row x is kept as
e4m3(x / 2^e), e the smallest whole number for which the row's largest magnitude is at most 448 * 2^e (between -64 and 64).

    append   rotate queries and keys of new tokens, write keys and values to their places in the pages
    decode   attention of the newest one to four tokens of every sequence over its pages
    step     both for one new token per sequence, from the partial sums of the QKV projection
    prompt   causal attention of packed prompts, or portions behind cached tokens, over their pages

    listed()              named cases
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   inputs on the GPU
    run(state)            one pass; `own`: through the framework's operators, otherwise by elementary torch operations
    work(case)            bytes and operations that a pass cannot do without
    exact(case, seed)     what `run` returns, in 64 bits
"""

import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 32
LOG2_MIN, LOG2_MAX = -64, 64
EPS = 1e-6

HEADS = {"a": (32, 8, 128), "b": (32, 4, 128), "c": (64, 8, 64), "d": (16, 16, 64), "e": (5, 1, 128)}


def case_of(op, heads, batch, lo, hi, new=1, splits=0, window=0, sinks=False, norm=False, bias=False, **name):
    """batch sequences of lo to hi tokens in the cache (prompt: ahead of the new ones); new: their new tokens (prompt: at most, down to
    half of it); splits: partial sums of the projection, 0: finished bf16."""
    nq, nkv, dim = HEADS[heads]
    return dict(op=op, nq=nq, nkv=nkv, dim=dim, batch=batch, lo=lo, hi=hi, new=new, splits=splits, window=window, sinks=sinks,
                norm=norm, bias=bias, **name)


def listed():
    return [
        # the new token of one user's chat: the latency of a launch
        case_of("append", "a", 1, 203, 203, splits=8, name="append-1"),
        # a packed step of continuous batching: one prompt of odd length, queries and keys normed per head
        case_of("append", "b", 1, 0, 0, new=390, norm=True, name="append-390"),
        # a full prefill step of the serving benchmark
        case_of("append", "a", 16, 0, 0, new=1024, name="append-16384"),
        # one user's chat
        case_of("decode", "a", 1, 203, 203, name="decode-1"),
        # the serving benchmark: 64 sequences of 1024 tokens
        case_of("decode", "a", 64, 1024, 1024, name="decode-64"),
        # a few long documents
        case_of("decode", "a", 7, 3500, 7000, name="decode-long"),
        # two drafted tokens checked at once, heads of 64 with sinks
        case_of("decode", "c", 37, 1000, 2000, new=2, sinks=True, name="verify-37"),
        # the attention of a decode step from the projection's partial sums: the serving benchmark
        case_of("step", "a", 64, 1024, 1024, splits=6, name="step-64"),
        # the same of a sliding-window layer for one user, heads of 64 with biases and sinks
        case_of("step", "c", 1, 130, 130, splits=8, window=128, sinks=True, bias=True, name="step-1-window"),
        # time to the first token of one short prompt
        case_of("prompt", "a", 1, 0, 0, new=77, name="prompt-77"),
        # a full prefill step of the serving benchmark
        case_of("prompt", "a", 16, 0, 0, new=1024, name="prompt-16x1024"),
        # portions of long documents behind what is cached already, heads of 64 with sinks
        case_of("prompt", "c", 3, 4000, 8000, new=500, sinks=True, name="prompt-portions"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op, heads = rng.choice(["append", "decode", "step", "prompt"]), rng.choice(sorted(HEADS))
        nq, nkv, dim = HEADS[heads]
        sinks, norm, bias = (rng.random() < 0.3 for _ in range(3))
        window = _log(rng, 16, 2000) if rng.random() < 0.3 else 0
        if op == "append":
            batch, new, splits = _log(rng, 1, 64), _log(rng, 1, 1500), 0
            if rng.random() < 0.4:
                batch, new, splits = _log(rng, 1, 128), 1, rng.randint(1, 9)
            hi = _log(rng, 1, 4000)
            c = case_of(op, heads, batch, rng.randint(0, hi), hi, new=new, splits=splits, norm=norm, bias=bias)
        elif op == "prompt":
            hi = _log(rng, 1, 8000) if rng.random() < 0.5 else 0
            c = case_of(op, heads, _log(rng, 1, 16), hi // 2, hi, new=_log(rng, 1, 2000), window=window, sinks=sinks)
        else:
            batch, hi = _log(rng, 1, 160), _log(rng, 4, 9000)
            new = rng.randint(1, min(4, 16 // (nq // nkv))) if op == "decode" else 1
            c = case_of(op, heads, batch, rng.randint(max(hi // 3, new), max(hi, new)), max(hi, new), new=new, window=window, sinks=sinks,
                        **(dict(splits=rng.randint(1, 9), norm=norm, bias=bias) if op == "step" else {}))
        full = c["batch"] * nq * c["new"] * (c["hi"] + c["new"])              # scores of the plain form
        if full <= 6e8 and c["batch"] * (c["hi"] + c["new"]) <= 70000 and _cost(c) <= max(_cost(x) for x in listed() if x["op"] == op):
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _lengths(c):
    """(tokens in the cache ahead of the new ones, new tokens) of every sequence: spread over the case's range, its ends among them."""
    n = c["batch"]
    at = [c["hi"] - (c["hi"] - c["lo"]) * ((7 * i) % n) // max(n - 1, 1) for i in range(n)]
    if c["op"] == "prompt":
        return at, [max(c["new"] - (c["new"] // 2) * ((5 * i) % n) // max(n, 1), 1) for i in range(n)]
    if c["op"] == "append":
        return at, [c["new"]] * n
    return [x - c["new"] for x in at], [c["new"]] * n


def _pairs(c):
    """(keys seen by all queries together, keys read at least once) of one query head."""
    pairs = read = 0
    for have, new in zip(*_lengths(c)):
        for i in range(new):
            end = have + i + 1
            pairs += min(end, c["window"]) if c["window"] else end
        read += min(have + new, c["window"] + new - 1) if c["window"] else have + new
    return pairs, read


def work(c):
    nq, nkv, dim = c["nq"], c["nkv"], c["dim"]
    tokens = sum(_lengths(c)[1])
    width = (nq + 2 * nkv) * dim
    kept = 2 * nkv * (dim + 1)
    flops = bytes_ = 0
    if c["op"] in ("append", "step"):
        bytes_ += tokens * (width * (4 * c["splits"] if c["splits"] else 2) + dim * 4 + kept + 8)
        flops += tokens * width * (3 + c["splits"])
    if c["op"] != "append":
        pairs, read = _pairs(c)
        flops += 4 * pairs * nq * dim
        bytes_ += (read - (tokens if c["op"] == "step" else 0)) * kept
    bytes_ += tokens * nq * dim * (4 if c["op"] in ("decode", "prompt") else 2)
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------------------------------------ inputs
def _rows(g, shape):
    """bf16 keys or values as a projection gives them: columns of unequal size, a few of them large."""
    spread = torch.exp(0.6 * torch.randn(shape[-1:], generator=g, device=DEV))
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(torch.bfloat16)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = random.Random(seed)
    nq, nkv, dim, op = c["nq"], c["nkv"], c["dim"], c["op"]
    have, new = _lengths(c)
    total = [a + b for a, b in zip(have, new)]
    tokens, B = sum(new), c["batch"]
    pages = [-(-n // PAGE) for n in total]
    pool = sum(pages) + 3
    ids = list(range(pool))
    r.shuffle(ids)
    table, n = torch.zeros((B, max(pages)), dtype=torch.int32), 0
    for b, k in enumerate(pages):
        table[b, :k] = torch.tensor(ids[n:n + k], dtype=torch.int32)
        n += k
    starts = [sum(new[:b]) for b in range(B)]
    pos = torch.cat([torch.arange(a, a + k, dtype=torch.int32) for a, k in zip(have, new)])
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    slots = table[seq, (pos // PAGE).long()] * PAGE + pos % PAGE
    s = {"case": c, "max_new": max(new), "table": table.to(DEV), "positions": pos.to(DEV), "slots": slots.to(torch.int32).to(DEV),
         "lens": torch.tensor(total, dtype=torch.int32, device=DEV), "starts": torch.tensor(starts, dtype=torch.int32, device=DEV),
         "new": torch.tensor(new, dtype=torch.int32, device=DEV)}
    for name in ("k", "v"):
        values, scales = _quantized(_rows(g, (pool, nkv, PAGE, dim)).double())
        s[name], s[name + "_scale"] = values, scales
    if op in ("append", "step"):
        width = (nq + 2 * nkv) * dim
        if c["splits"]:
            s["qkv"] = torch.randn((c["splits"], tokens, width), generator=g, device=DEV) * c["splits"] ** -0.5
        else:
            s["qkv"] = _rows(g, (tokens, width))
        inv = 1.0 / 500000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        ang = torch.arange(max(total), dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], -1).float().to(DEV)
        s["bias"] = (0.2 * torch.randn((width,), generator=g, device=DEV)).to(torch.bfloat16) if c["bias"] else None
        for name in ("q_norm", "k_norm"):
            s[name] = (1 + 0.2 * torch.randn((dim,), generator=g, device=DEV)).to(torch.bfloat16) if c["norm"] else None
    else:
        s["q"] = (1.5 * torch.randn((tokens, nq * dim), generator=g, device=DEV)).to(torch.bfloat16)
    s["sinks"] = torch.randn((nq,), generator=g, device=DEV) if c["sinks"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else _plain(s)


def _outputs(s, **more):
    """The state's pages as the values they stand for, beside `more`."""
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return dict(more, k=s["k"].view(f8), v=s["v"].view(f8), k_scale=s["k_scale"].view(e8), v_scale=s["v_scale"].view(e8))


def _own(s):
    from nkipy_b200 import ops

    c, scale = s["case"], s["case"]["dim"] ** -0.5
    k, v = ops.QuantizedPages(s["k"], s["k_scale"]), ops.QuantizedPages(s["v"], s["v_scale"])
    if c["op"] == "append":
        q = ops.rope_kv_append(s["qkv"], s["positions"], s["slots"], s["cos_sin"], k, v, c["nq"], c["nkv"], c["dim"], bias=s["bias"],
                               q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], norm_eps=EPS)
        return _outputs(s, q=q)
    if c["op"] == "step":
        o = ops.rope_attn_decode(s["qkv"], s["positions"], s["slots"], s["cos_sin"], k, v, s["table"], s["lens"], scale, c["nq"], c["nkv"],
                                 bias=s["bias"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], norm_eps=EPS, window=c["window"],
                                 sinks=s["sinks"])
        return _outputs(s, o=o)
    if c["op"] == "decode":
        return ops.paged_attn_decode(s["q"], k, v, s["table"], s["lens"], scale, q_len=c["new"], window=c["window"], sinks=s["sinks"])
    return ops.flash_attn_prefill(s["q"], k, v, s["table"], s["starts"], s["new"], s["lens"], scale, max_q_len=s["max_new"],
                                  window=c["window"], sinks=s["sinks"])


def _pow2(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantized(x):
    """(e4m3 values, power-of-two scales) of rows in 64 bits: next to a border of e4m3, 32 bits could fall on its other side."""
    m, e = torch.frexp(x.abs().amax(-1))                       # 448 is 0.875 * 2^9
    e = (e - 9 + (m > 0.875).int()).clamp(LOG2_MIN, LOG2_MAX)
    e = torch.where(m == 0, LOG2_MIN, e)
    y = x * _pow2(-e)[..., None]
    step = _pow2((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)    # three bits behind the leading one, from 2^-6 on
    y = (torch.round(y / step) * step).clamp(-448, 448)
    return y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _rotate(x, cs, w):
    """Rows [tokens, heads, dim]: optional norm, then rotate-halves RoPE, in x's type."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    h = x.shape[-1] // 2
    cos, sin = cs[:, None, :h].to(x.dtype), cs[:, None, h:].to(x.dtype)
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    c = s["case"]
    nq, nkv, dim = c["nq"], c["nkv"], c["dim"]
    x = s["qkv"].double()
    x = x.sum(0) if c["splits"] else x
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x.view(x.shape[0], nq + 2 * nkv, dim)
    cs = s["cos_sin"][s["positions"].long()]
    q = _rotate(x[:, :nq].float(), cs, s["q_norm"]).to(torch.bfloat16).reshape(x.shape[0], nq * dim)
    at = s["slots"].long()
    for name, rows in (("k", _rotate(x[:, nq:nq + nkv], cs, s["k_norm"])), ("v", x[:, nq + nkv:])):
        values, scales = _quantized(rows)
        s[name].view(torch.uint8)[at // PAGE, :, at % PAGE] = values.view(torch.uint8)
        s[name + "_scale"].view(torch.uint8)[at // PAGE, :, at % PAGE] = scales.view(torch.uint8)
    return q


def _gathered(s, name):
    """Cached rows of all sequences in 32 bits, [batch, kv heads, tokens, dim], padded to the longest."""
    at = s["table"].long()
    x = s[name].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    x = x * s[name + "_scale"].view(torch.uint8)[at].view(torch.float8_e8m0fnu).float()[..., None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend(s, q, pos):
    """q [batch, new, heads, dim] in 32 bits at positions pos [batch, new] -> the same shape."""
    c = s["case"]
    nq, nkv, dim = c["nq"], c["nkv"], c["dim"]
    B, n = pos.shape
    k, v = _gathered(s, "k"), _gathered(s, "v")
    q = q.view(B, n, nkv, nq // nkv, dim).permute(0, 2, 3, 1, 4).reshape(B, nkv, -1, dim)
    sc = ((q @ k.transpose(-1, -2)) * dim ** -0.5).view(B, nkv, nq // nkv, n, -1)
    at = torch.arange(k.shape[2], device=DEV)
    seen = at <= pos[..., None]
    if c["window"]:
        seen = seen & (at > pos[..., None] - c["window"])
    sc = sc.masked_fill(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, nkv, nq // nkv, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    o = (p / total).view(B, nkv, -1, p.shape[-1]) @ v
    return o.view(B, nkv, nq // nkv, n, dim).permute(0, 3, 1, 2, 4).reshape(B, n, nq, dim)


def _plain(s):
    c = s["case"]
    nq, dim, B = c["nq"], c["dim"], c["batch"]
    if c["op"] == "append":
        return _outputs(s, q=_append(s))
    if c["op"] == "step":
        q = _append(s)
        o = _attend(s, q.float().view(B, 1, nq, dim), (s["lens"] - 1).long()[:, None])
        return _outputs(s, o=o.to(torch.bfloat16).view(B, nq * dim))
    n = s["max_new"]
    i = torch.arange(n, device=DEV)
    rows = (s["starts"].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)       # shorter ones are padded with rows of the next
    o = _attend(s, s["q"].float()[rows].view(B, n, nq, dim), (s["lens"] - s["new"]).long()[:, None] + i)
    return o[i < s["new"][:, None]].to(torch.bfloat16).reshape(-1, nq * dim)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _e4m3_grid():
    """All finite magnitudes of e4m3, in the order of their codes."""
    codes = [((8 + m) * 2.0 ** (e - 10)) if e else m * 2.0 ** -9 for e in range(16) for m in range(8)]
    return torch.tensor(codes[:127], dtype=torch.float64, device=DEV)


def _exact_rows(x):
    """Values and scales of rows, by a search among all values of e4m3."""
    grid = _e4m3_grid()
    scales = torch.tensor([2.0 ** e for e in range(LOG2_MIN, LOG2_MAX + 1)], dtype=torch.float64, device=DEV)
    scale = scales[torch.searchsorted(grid[-1] * scales, x.abs().amax(-1).contiguous()).clamp(max=len(scales) - 1)]
    y = (x.abs() / scale[..., None]).contiguous()
    up = torch.searchsorted(grid, y).clamp(max=len(grid) - 1)
    low = (up - 1).clamp(min=0)
    over, under = grid[up] - y, y - grid[low]
    code = torch.where((over < under) | ((over == under) & (up % 2 == 0)), up, low)
    return torch.copysign(grid[code], x), scale


def exact(c, seed):
    s = prepare(c, seed)
    nq, nkv, dim, B = c["nq"], c["nkv"], c["dim"], c["batch"]
    K, V = s["k"].double(), s["v"].double()
    KS, VS = s["k_scale"].float().double(), s["v_scale"].float().double()
    have, new = _lengths(c)
    if c["op"] in ("append", "step"):
        x = s["qkv"].double()
        if c["splits"]:
            x = x.sum(0)
        if s["bias"] is not None:
            x = x + s["bias"].double()
        x = x.view(-1, nq + 2 * nkv, dim)
        cs = s["cos_sin"].double()[s["positions"].long()]
        turn = torch.complex(cs[:, None, :dim // 2], cs[:, None, dim // 2:])

        def turned(y, w):
            if w is not None:
                y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / dim + EPS) * w.double()
            z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)

        q = turned(x[:, :nq], s["q_norm"])
        page, off = (s["slots"] // PAGE).long(), (s["slots"] % PAGE).long()
        K[page, :, off], KS[page, :, off] = _exact_rows(turned(x[:, nq:nq + nkv], s["k_norm"]))
        V[page, :, off], VS[page, :, off] = _exact_rows(x[:, nq + nkv:])
        if c["op"] == "append":
            return dict(q=q.reshape(-1, nq * dim), k=K, v=V, k_scale=KS, v_scale=VS)
        q = q.to(torch.bfloat16).double()              # what attention is given
    else:
        q = s["q"].double().view(-1, nq, dim)
    out, row = torch.empty_like(q), 0
    for b, (h, n) in enumerate(zip(have, new)):
        pages = s["table"][b, :-(-(h + n) // PAGE)].long()
        k = (K[pages] * KS[pages][..., None]).transpose(1, 2).reshape(-1, nkv, dim)[:h + n]
        v = (V[pages] * VS[pages][..., None]).transpose(1, 2).reshape(-1, nkv, dim)[:h + n]
        at, mine = torch.arange(h + n, device=DEV), torch.arange(h, h + n, device=DEV)[:, None]
        hidden = at > mine
        if c["window"]:
            hidden |= at <= mine - c["window"]
        for j in range(nq):
            sc = q[row:row + n, j] @ k[:, j * nkv // nq].T / math.sqrt(dim)
            sc[hidden] = -math.inf
            if s["sinks"] is not None:
                sc = torch.cat([sc, s["sinks"][j].double().expand(n, 1)], 1)
            p = torch.softmax(sc, -1)[:, :h + n]
            out[row:row + n, j] = p @ v[:, j * nkv // nq]
        row += n
    out = out.view(-1, nq * dim)
    return dict(o=out, k=K, v=V, k_scale=KS, v_scale=VS) if c["op"] == "step" else out
