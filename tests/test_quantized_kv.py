"""Keys and values in 8 bits against plain implementations in 64 bits: what is stored, byte by byte, and attention over it."""

import math

import pytest
import torch

from nkipy_b200 import ops

PAGE = 32
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ------------------------------------------------------------------------------------------------ oracles
def oracle_quantize(x):
    """(values, scales) that rows [..., dim] in 64 bits stand for, by comparison with every value e4m3 has.  Rows that are not finite:
    zeros and NaN."""
    codes = torch.arange(127, dtype=torch.uint8).view(F8).double()
    tops = torch.tensor([448.0 * 2.0 ** e for e in range(-64, 65)], dtype=torch.float64)
    values, scales = [], []
    for rows in x.double().reshape(-1, x.shape[-1]).split(256):
        fine = rows.isfinite().all(-1)
        rows = torch.where(fine[:, None], rows, 0.0)
        scale = (tops < rows.abs().amax(-1, keepdim=True)).sum(-1).clamp(max=128)
        scale = tops[scale] / 448.0
        gap = ((rows.abs() / scale[:, None])[..., None] - codes).abs()
        tied = gap == gap.min(-1, keepdim=True).values                  # one code, or two neighbours: the even one
        n = torch.arange(127).expand_as(tied)
        pick = torch.where(tied & ((n % 2 == 0) | (tied.sum(-1, keepdim=True) == 1)), n, -1).max(-1).values
        values.append(torch.copysign(codes[pick], rows))
        scales.append(torch.where(fine, scale, math.nan))
    return torch.cat(values).reshape(x.shape), torch.cat(scales).reshape(x.shape[:-1])


def stored(pages):
    return pages.values.cpu().double(), pages.scales.cpu().float().double()


def fill(pages, rows):
    """Rows [blocks, heads, 32, dim] into the pages, by the oracle."""
    v, s = oracle_quantize(rows)
    pages.values.copy_(v.float().to(F8))
    byte = torch.where(s.isnan(), 255, torch.log2(s.nan_to_num(1.0)).round().int() + 127)
    pages.scales.view(torch.uint8).copy_(byte.to(torch.uint8))


def cached(pages, table_row, ctx):
    """[ctx, heads, dim] of one sequence in 64 bits; NaN rows whole; blocks outside the pool are zeros."""
    v, s = stored(pages)
    rows = []
    for b in table_row[:-(-ctx // PAGE)].tolist():
        rows.append(v[b] * s[b][..., None] if 0 <= b < v.shape[0] else torch.zeros_like(v[0]))
    return torch.cat([r.transpose(0, 1) for r in rows])[:ctx] if rows else torch.zeros((0, v.shape[1], v.shape[3]), dtype=torch.float64)


def oracle_attend(q, k, v, scale, pos, causal=True, window=0, chunk=0, sinks=None):
    """One query head's row q [dim] at position pos over k, v [tokens, dim] in 64 bits: (result, tolerance).

    Tolerance: the result is rounded to bf16 (2^-8 of it); weights to f16 (2^-11 each), exponentials by the special-function unit and
    sums in 32 bits (2^-19), and scores in 32 bits, where a tensor core cuts each of the up to eight partial sums behind 2^-22 of what
    it holds: 2^-19 of sum |q k|, which moves a weight by that much of itself, and the sum of weights too.  f16's steps end at 2^-24:
    with the largest weight at 2^6 or above, a weight is off by up to 2^-31 of the largest besides (which takes a value's scale in, so
    that it may be that of the largest value), for every token."""
    n = k.shape[0]
    at = torch.arange(n)
    seen = at <= pos if causal else torch.ones(n, dtype=torch.bool)
    if window:
        seen &= at > pos - window
    if chunk:
        seen &= at >= (pos // chunk) * chunk
    if not seen.any():
        return torch.zeros_like(q), torch.zeros_like(q)
    k, v = k[seen], v[seen]
    if k.isnan().any() or v.isnan().any():
        return torch.full_like(q, math.nan), torch.zeros_like(q)
    s = k @ q * scale
    top = s.max() if sinks is None else max(s.max(), sinks)
    p = torch.exp(s - top)
    total = p.sum() + (0.0 if sinks is None else math.exp(sinks - top))
    p = p / total
    o = p @ v
    moved = 2.0 ** -19 * float((k.abs() @ q.abs()).max()) * scale
    return o, 2.0 ** -8 * o.abs() + (p @ v.abs()) * (2.0 ** -11 + 2.0 ** -19 + 2 * moved) + n * 2.0 ** -30 * float(v.abs().max()) + 1e-30


def check_attention(out, q, k_pages, v_pages, table, spans, scale, nq, group, sinks=None, **masks):
    """out, q [tokens, nq, dim]; spans: (first row, new tokens, context) per sequence."""
    out, q = out.cpu().double(), q.cpu().double()
    for b, (row, n, ctx) in enumerate(spans):
        k, v = cached(k_pages, table[b].cpu(), max(ctx, 0)), cached(v_pages, table[b].cpu(), max(ctx, 0))
        for i in range(n):
            for h in range(nq):
                want, tol = oracle_attend(q[row + i, h], k[:, h // group], v[:, h // group], scale, ctx - n + i,
                                          sinks=None if sinks is None else float(sinks[h]), **masks)
                got = out[row + i, h]
                assert torch.equal(got.isnan(), want.isnan()), (b, i, h)
                assert bool(((got - want).abs() <= tol)[~want.isnan()].all()), (b, i, h, float((got - want).abs().max()), float(tol.max()))


def pool(g, blocks, nkv, dim, device, spread=0.5):
    k, v = ops.QuantizedPages.new(blocks, nkv, dim, device), ops.QuantizedPages.new(blocks, nkv, dim, device)
    for pages in (k, v):
        fill(pages, torch.randn((blocks, nkv, PAGE, dim), generator=g, dtype=torch.float64)
             * torch.exp(spread * torch.randn((blocks, nkv, PAGE, 1), generator=g, dtype=torch.float64)))
    return k, v


def shuffled_table(g, contexts, extra=0):
    """Block table of sequences with these contexts over shuffled blocks; (table, blocks)."""
    need = [max(-(-c // PAGE), 1) for c in contexts]
    ids = torch.randperm(sum(need) + extra, generator=g).to(torch.int32)
    table, n = torch.zeros((len(contexts), max(need)), dtype=torch.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = ids[n:n + k]
        n += k
    return table, sum(need) + extra


# ------------------------------------------------------------------------------------------------ what is stored
def rope_table(dim, n):
    ang = torch.arange(n, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    return torch.cat([ang.cos(), ang.sin()], -1).float()


def oracle_turn(x, cs, w, eps):
    """Rows [T, heads, dim] in 64 bits: norm, rotation."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    h = x.shape[-1] // 2
    c, s = cs[:, None, :h].double(), cs[:, None, h:].double()
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def append_case(g, T, nq, nkv, dim, splits, norm, bias):
    W = (nq + 2 * nkv) * dim
    if splits:
        qkv = torch.randn((splits, T, W), generator=g) * torch.exp(torch.randn((W,), generator=g))
    else:
        qkv = (torch.randn((T, W), generator=g) * torch.exp(torch.randn((W,), generator=g))).to(torch.bfloat16)
    b = torch.randn((W,), generator=g).to(torch.bfloat16) if bias else None
    qw, kw = ((1 + 0.3 * torch.randn((dim,), generator=g)).to(torch.bfloat16) if norm else None for _ in range(2))
    return qkv, b, qw, kw


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,nq,nkv,dim,splits,norm,bias", [
    (1, 4, 2, 128, 3, False, False), (5, 5, 1, 64, 0, True, True), (3, 16, 2, 64, 9, True, False), (70, 2, 2, 128, 0, False, True),
    (257, 4, 2, 128, 0, True, False), (300, 3, 1, 64, 2, False, True), (259, 2, 1, 128, 0, False, False), (260, 2, 2, 64, 0, False, False)])
def test_append_stores_the_nearest_values(device, T, nq, nkv, dim, splits, norm, bias):
    g = torch.Generator().manual_seed(T * 7 + dim)
    qkv, b, qw, kw = append_case(g, T, nq, nkv, dim, splits, norm, bias)
    blocks, cs = -(-T // PAGE) + 3, rope_table(dim, 500)
    k, v = pool(g, blocks, nkv, dim, device)
    before = [*stored(k), *stored(v)]
    slots = torch.randperm(blocks * PAGE, generator=g)[:T].to(torch.int32)
    slots[T // 2] = -1                                                     # nothing is stored for it
    pos = torch.randint(0, 500, (T,), generator=g).to(torch.int32)
    to = lambda t: None if t is None else t.to(device)                     # noqa: E731
    q = ops.rope_kv_append(to(qkv), to(pos), to(slots), to(cs), k, v, nq, nkv, dim, bias=to(b), q_norm_w=to(qw), k_norm_w=to(kw),
                           norm_eps=1e-5)
    x = qkv.double().sum(0) if splits else qkv.double()
    x = (x + (b.double() if bias else 0.0)).view(T, nq + 2 * nkv, dim)
    rows = cs[pos.long()]
    want = before
    for i, (y, w) in enumerate(((x[:, nq:nq + nkv], kw), (x[:, nq + nkv:], None))):
        if i == 0:
            y = oracle_turn(y, rows, w, 1e-5)
        values, scales = oracle_quantize(y)
        for t in range(T):
            if slots[t] >= 0:
                want[2 * i][slots[t] // PAGE, :, slots[t] % PAGE] = values[t]
                want[2 * i + 1][slots[t] // PAGE, :, slots[t] % PAGE] = scales[t]
    for a, b_ in zip([*stored(k), *stored(v)], want):
        assert torch.equal(a, b_)
    qr = oracle_turn(x[:, :nq], rows, qw, 1e-5)
    big = x[:, :nq].abs().amax(-1, keepdim=True) if qw is None else (qr.abs().amax(-1, keepdim=True) * 2)
    # rounded to bf16 (2^-8), from sums, norm and rotation in 32 bits: a dozen roundings of at most the head's largest terms
    assert bool(((q.cpu().double().view(T, nq, dim) - qr).abs() <= 2.0 ** -8 * qr.abs() + 2.0 ** -19 * big).all())


@pytest.mark.parametrize("device", DEVICES)
def test_append_rounds_ties_and_ends_of_the_range(device):
    dim, nkv = 64, 1
    rows = torch.zeros((14, dim), dtype=torch.float32)
    rows[0, 0] = 448.0                                                     # scale 1 and its neighbours
    rows[1, 0] = 448.0 + 2.0 ** -15
    rows[2, 0], rows[2, 1:5] = 448.0, torch.tensor([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])      # ties: to 16, 20, 0, 2^-8
    rows[3, 0], rows[3, 1:3] = -448.0, torch.tensor([17.0 + 2.0 ** -19, -(17.0 - 2.0 ** -19)])
    rows[4] = 0.0
    rows[5, 3] = 1e-30                                                     # below what scales reach
    rows[6, 3] = 3e38                                                      # beyond it: saturates
    rows[7, 5] = math.inf
    rows[8, 6], rows[8, 1] = math.nan, 3.0
    rows[9, 7], rows[9, 1] = -math.inf, 3.0
    rows[10, 0], rows[10, 1] = 2.0 ** -60, 2.0 ** -70
    rows[11] = torch.linspace(-448, 448, dim)
    rows[12] = 2.0 ** torch.linspace(-12, 8, dim)
    rows[13] = 447.9 * 2.0 ** 64
    T = rows.shape[0]
    for splits in (0, 1, 2):
        qkv = torch.cat([torch.zeros((T, dim)), rows, rows.flip(0)], 1)
        if splits == 0:
            qkv = qkv.to(torch.bfloat16)
            want = qkv.double()
        else:
            parts = [qkv] if splits == 1 else [qkv * 0.5, qkv * 0.5]
            qkv = torch.stack(parts)
            want = qkv.double().sum(0)
        k, v = ops.QuantizedPages.new(2, nkv, dim, device), ops.QuantizedPages.new(2, nkv, dim, device)
        slots = (torch.arange(T, dtype=torch.int32) * 3) % 64
        ops.rope_kv_append(qkv.to(device), None, slots.to(device), None, k, v, 1, nkv, dim)
        for pages, col in ((k, dim), (v, 2 * dim)):
            values, scales = oracle_quantize(want[:, col:col + dim])
            gv, gs = stored(pages)
            at = slots.long()
            assert torch.equal(gv[at // PAGE, 0, at % PAGE], values)
            assert torch.equal(gs[at // PAGE, 0, at % PAGE].nan_to_num(-1), scales.nan_to_num(-1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 200])
def test_append_rounds_rotations_beside_a_tie(device, T):
    """Rotations that 32 bits put on the other side of the middle between two values of e4m3: the products' roundings move their difference
    by more than one of its steps."""
    g = torch.Generator().manual_seed(33)
    dim, h, n = 64, 32, 3000000
    a, d = ((1 + torch.randint(0, 128, (2, n), generator=g) / 128) * (1 - 2 * torch.randint(0, 2, (2, n), generator=g))).unbind(0)
    a = 2 * a
    c, tie = 0.5 + 0.5 * torch.rand(n, generator=g), 1 + (1 + 2 * torch.randint(0, 8, (n,), generator=g)) / 16
    s = ((a.double() * c.double() - tie) / d.double()).float()
    exact, rough = a.double() * c.double() - d.double() * s.double(), a * c - d * s      # (products of 8 and 24 bits: exact)
    odd = (((rough > tie) & (exact < tie)) | ((rough < tie) & (exact > tie))) & (s.abs() < 1)
    a, c, d, s, exact = (t[odd][:T * h].view(T, h) for t in (a, c, d, s, exact))
    k, v = (ops.QuantizedPages.new(-(-T // PAGE), 1, dim, device) for _ in range(2))
    x = torch.zeros((T, 3, dim))
    x[:, 1] = torch.cat([a, d], -1)
    at = torch.arange(T, dtype=torch.int32, device=device)
    ops.rope_kv_append(x.view(T, -1).to(torch.bfloat16).to(device), at, at, torch.cat([c, s], -1).to(device), k, v, 1, 1, dim)
    turned = torch.cat([exact, d.double() * c.double() + a.double() * s.double()], -1)
    want, scale = oracle_quantize(turned)
    assert torch.equal(k.values.view(-1, dim)[:T].cpu().double(), want)
    assert torch.equal(k.scales.view(-1)[:T].cpu().float().double(), scale)


def test_dequantize_gives_what_is_stored():
    g = torch.Generator().manual_seed(3)
    k, _ = pool(g, 3, 2, 64, "cpu")
    v, s = stored(k)
    assert torch.equal(k.dequantize().double(), v * s[..., None])
    assert torch.equal(k.dequantize(torch.tensor([2, 0])).double(), (v * s[..., None])[[2, 0]])
    assert k.nbytes == 3 * 2 * 32 * 65


# ------------------------------------------------------------------------------------------------ attention of single tokens
DECODE = [
    # nq, nkv, dim, q_len, contexts, masks
    (4, 2, 128, 1, [1, 31, 32, 33, 64, 65, 200], {}),
    (8, 1, 64, 2, [2, 40, 97, 513], {}),
    (5, 1, 128, 3, [3, 34, 100], dict(window=17)),
    (16, 1, 64, 1, [0, 7, 300, -1], dict(sinks=True)),
    (4, 4, 64, 4, [4, 129, 1000], dict(chunk=48)),
    (2, 1, 128, 1, [1500], dict(window=700, sinks=True)),
    (2, 2, 64, 1, [3000], {}),
    (32, 2, 128, 1, [700, 5, 2100], {}),
    (6, 1, 64, 4, [70, 4], {}),                                             # more than sixteen query rows per kv head
    (2, 1, 128, 3, [2, 1, 0], {}),                                          # new tokens ahead of position 0
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nq,nkv,dim,q_len,contexts,masks", DECODE)
def test_decode(device, nq, nkv, dim, q_len, contexts, masks):
    g = torch.Generator().manual_seed(nq * 131 + dim + len(contexts))
    masks = dict(masks)
    table, blocks = shuffled_table(g, contexts, extra=2)
    k, v = pool(g, blocks, nkv, dim, device)
    sinks = torch.randn((nq,), generator=g) if masks.pop("sinks", False) else None
    B = len(contexts)
    q = (2 * torch.randn((B * q_len, nq * dim), generator=g)).to(torch.bfloat16)
    lens = torch.tensor(contexts, dtype=torch.int32)
    for splits in (0, 1, 3):
        out = ops.paged_attn_decode(q.to(device), k, v, table.to(device), lens.to(device), dim ** -0.5, q_len=q_len,
                                    sinks=None if sinks is None else sinks.to(device), num_splits=splits, **masks)
        check_attention(out.view(-1, nq, dim), q.view(-1, nq, dim), k, v, table, [(b * q_len, q_len, c) for b, c in enumerate(contexts)],
                        dim ** -0.5, nq, nq // nkv, sinks, **masks)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_sees_nothing_of_what_is_masked(device, dim):
    """NaN rows behind the context, before the window and in pages of other sequences; blocks that are not in the pool."""
    g = torch.Generator().manual_seed(dim)
    contexts, nq, nkv = [37, 150], 4, 2
    table, blocks = shuffled_table(g, contexts, extra=3)
    k, v = pool(g, blocks, nkv, dim, device)
    lens = torch.tensor(contexts, dtype=torch.int32)
    q = torch.randn((2, nq * dim), generator=g).to(torch.bfloat16)
    hidden = torch.ones((blocks, PAGE), dtype=torch.bool)
    for b, c in enumerate(contexts):
        for j in range(max(c - 60, 0), c):
            hidden[table[b, j // PAGE], j % PAGE] = False
    for pages in (k, v):
        raw = pages.scales.view(torch.uint8).cpu()
        raw[hidden[:, None].expand(raw.shape)] = 255
        pages.scales.view(torch.uint8).copy_(raw)
        values = pages.values.view(torch.uint8).cpu()
        values[hidden[:, None].expand(raw.shape)] = 0
        pages.values.view(torch.uint8).copy_(values)
    for splits in (1, 4):
        out = ops.paged_attn_decode(q.to(device), k, v, table.to(device), lens.to(device), dim ** -0.5, window=60, num_splits=splits)
        assert bool(out.isfinite().all())
        check_attention(out.view(-1, nq, dim), q.view(-1, nq, dim), k, v, table, [(0, 1, 37), (1, 1, 150)], dim ** -0.5, nq, 2, window=60)
    # a row that is seen and not finite takes its kv head's queries along, and no others
    at = int(table[0, 1]), 0
    for pages in (k, v):
        saved = pages.scales.view(torch.uint8).clone()
        pages.scales.view(torch.uint8)[at[0], 1, at[1]] = 255
        pages.values.view(torch.uint8)[at[0], 1, at[1]] = 0
        out = ops.paged_attn_decode(q.to(device), k, v, table.to(device), lens.to(device), dim ** -0.5, window=60).view(2, nq, dim)
        assert bool(out[0, 2:].isnan().all()) and bool(out[0, :2].isfinite().all()) and bool(out[1].isfinite().all())
        pages.scales.view(torch.uint8).copy_(saved)


@pytest.mark.parametrize("device", DEVICES)
def test_blocks_outside_the_pool_read_as_zeros(device):
    g = torch.Generator().manual_seed(5)
    k, v = pool(g, 4, 1, 64, device)
    table = torch.tensor([[1, 9, 3], [-1, 2, 0]], dtype=torch.int32)
    lens = torch.tensor([90, 70], dtype=torch.int32)
    q = torch.randn((2, 2 * 64), generator=g).to(torch.bfloat16)
    out = ops.paged_attn_decode(q.to(device), k, v, table.to(device), lens.to(device), 0.125)
    check_attention(out.view(2, 2, 64), q.view(2, 2, 64), k, v, table, [(0, 1, 90), (1, 1, 70)], 0.125, 2, 2)
    out = ops.flash_attn_prefill(q.to(device), k, v, table.to(device), torch.tensor([0, 1], dtype=torch.int32, device=device),
                                 torch.tensor([1, 1], dtype=torch.int32, device=device), lens.to(device), 0.125, max_q_len=1)
    check_attention(out.view(2, 2, 64), q.view(2, 2, 64), k, v, table, [(0, 1, 90), (1, 1, 70)], 0.125, 2, 2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_far_apart(device, dim):
    """Rows of 2^-50 to 2^50 beside one another, queries of unequal size."""
    g = torch.Generator().manual_seed(dim + 1)
    nq, nkv, ctx = 2, 1, 100
    table, blocks = shuffled_table(g, [ctx])
    k, v = ops.QuantizedPages.new(blocks, nkv, dim, device), ops.QuantizedPages.new(blocks, nkv, dim, device)
    at = torch.randint(-50, 51, (blocks, nkv, PAGE, 1), generator=g).double()
    fill(v, torch.randn((blocks, nkv, PAGE, dim), generator=g, dtype=torch.float64) * 2.0 ** at)
    fill(k, torch.randn((blocks, nkv, PAGE, dim), generator=g, dtype=torch.float64) * 2.0 ** -at.abs().sqrt())
    q = (torch.randn((1, nq * dim), generator=g) * torch.tensor([1e-3, 3e4]).repeat_interleave(dim)).to(torch.bfloat16)
    lens = torch.tensor([ctx], dtype=torch.int32, device=device)
    scale = 1e-4
    out = ops.paged_attn_decode(q.to(device), k, v, table.to(device), lens, scale)
    check_attention(out.view(1, nq, dim), q.view(1, nq, dim), k, v, table, [(0, 1, ctx)], scale, nq, nq)


# ------------------------------------------------------------------------------------------------ attention of prompts
PROMPTS = [
    # nq, nkv, dim, (cached, new) per sequence, masks
    (2, 1, 128, [(0, 1), (0, 33), (40, 5), (0, 130)], {}),
    (4, 2, 64, [(0, 300)], {}),
    (2, 2, 128, [(100, 257)], {}),
    (3, 1, 64, [(0, 64), (31, 1), (500, 70)], dict(sinks=True)),
    (2, 1, 128, [(10, 200), (0, 90)], dict(window=50)),
    (2, 1, 64, [(200, 140)], dict(window=129, sinks=True)),
    (2, 1, 128, [(60, 150)], dict(chunk=70)),
    (1, 1, 64, [(0, 70), (0, 200)], dict(causal=False)),
    (2, 1, 128, [(0, 140), (33, 5)], dict(causal=False)),
    (8, 4, 64, [(0, 70)] * 41 + [(129, 3), (0, 1)], {}),                     # more pieces than SMs
    (6, 1, 128, [(3 * i, 1 + 11 * i) for i in range(24)], {}),               # of every length
    (5, 1, 64, [(0, 60), (300, 60)], dict(window=1)),
    (8, 1, 64, [(2100, 5), (0, 3), (1300, 20)], {}),                         # few rows over long contexts, divided among works
    (4, 2, 128, [(3000, 2), (40, 1)], dict(sinks=True)),
    (2, 1, 128, [(2500, 33), (1, 300)], dict(window=700)),
    (2, 1, 64, [(1600, 4)], dict(causal=False)),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nq,nkv,dim,spans,masks", PROMPTS)
def test_prompts(device, nq, nkv, dim, spans, masks):
    g = torch.Generator().manual_seed(nq * 17 + dim + len(spans))
    masks = dict(masks)
    contexts = [a + n for a, n in spans]
    table, blocks = shuffled_table(g, contexts, extra=2)
    k, v = pool(g, blocks, nkv, dim, device)
    sinks = torch.randn((nq,), generator=g) if masks.pop("sinks", False) else None
    new = [n for _, n in spans]
    total = sum(new)
    q = (2 * torch.randn((total + 3, nq * dim), generator=g)).to(torch.bfloat16)
    starts = [sum(new[:b]) for b in range(len(new))]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)       # noqa: E731
    out = torch.full((total + 3, nq * dim), 7.0, dtype=torch.bfloat16, device=device)
    ops.flash_attn_prefill(q.to(device), k, v, table.to(device), i32(starts), i32(new), i32(contexts), dim ** -0.5, max_q_len=max(new),
                           sinks=None if sinks is None else sinks.to(device), out=out, **masks)
    check_attention(out.view(-1, nq, dim), q.view(-1, nq, dim), k, v, table, list(zip(starts, new, contexts)), dim ** -0.5, nq, nq // nkv,
                    sinks, **masks)
    assert bool((out[total:] == 7.0).all())                                  # rows behind the last sequence


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spans", [[(0, 5)], [(0, 1), (700, 9), (1400, 3), (50, 60)], [(383, 1), (384, 1), (511, 2)]])
def test_prompts_with_room_in_their_tables(device, dim, spans):
    """Tables as wide as the longest sequence may become: what is divided goes by what a sequence has."""
    g = torch.Generator().manual_seed(dim + len(spans))
    nq, nkv = 4, 2
    contexts, new = [a + n for a, n in spans], [n for _, n in spans]
    table, blocks = shuffled_table(g, contexts)
    k, v = pool(g, blocks, nkv, dim, device)
    wide = torch.zeros((len(spans), 512), dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q, sinks = torch.randn((sum(new), nq * dim), generator=g).to(torch.bfloat16), torch.randn((nq,), generator=g)
    starts = [sum(new[:b]) for b in range(len(new))]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)        # noqa: E731
    for window in (0, 600):
        out = ops.flash_attn_prefill(q.to(device), k, v, wide.to(device), i32(starts), i32(new), i32(contexts), dim ** -0.5, max_q_len=max(new),
                                     sinks=sinks.to(device), window=window)
        check_attention(out.view(-1, nq, dim), q.view(-1, nq, dim), k, v, table, list(zip(starts, new, contexts)), dim ** -0.5, nq, 2, sinks,
                        window=window)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_with_tokens_ahead_of_the_first(device, dim):
    """Contexts shorter than the new tokens, or empty: rows that see nothing are zero (with or without sinks), pieces without a tile lie
    among others."""
    g = torch.Generator().manual_seed(dim + 2)
    nq, nkv = 4, 1
    spans = [(70, 3), (90, 0), (200, 130), (1, 0), (150, -1), (65, 65), (300, 10)]
    contexts = [c for _, c in spans]
    table, blocks = shuffled_table(g, contexts)
    k, v = pool(g, blocks, nkv, dim, device)
    new = [n for n, _ in spans]
    starts = [sum(new[:b]) for b in range(len(new))]
    q = torch.randn((sum(new), nq * dim), generator=g).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)        # noqa: E731
    for sinks in (None, torch.randn((nq,), generator=g)):
        out = ops.flash_attn_prefill(q.to(device), k, v, table.to(device), i32(starts), i32(new), i32(contexts), dim ** -0.5,
                                     max_q_len=max(new), sinks=None if sinks is None else sinks.to(device))
        check_attention(out.view(-1, nq, dim), q.view(-1, nq, dim), k, v, table, list(zip(starts, new, contexts)), dim ** -0.5, nq, nq, sinks)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_see_nothing_of_later_tokens(device, dim):
    g = torch.Generator().manual_seed(dim + 9)
    nq, nkv, n = 2, 1, 150
    table, blocks = shuffled_table(g, [n], extra=1)
    k, v = pool(g, blocks, nkv, dim, device)
    for pages, j in ((k, 120), (v, 90), (k, 149 + 3)):                       # the last one behind the context
        blk = int(table[0, j // PAGE]) if j < n else int(table[0, -1])
        pages.scales.view(torch.uint8)[blk, 0, j % PAGE] = 255
        pages.values.view(torch.uint8)[blk, 0, j % PAGE] = 0
    q = torch.randn((n, nq * dim), generator=g).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)        # noqa: E731
    out = ops.flash_attn_prefill(q.to(device), k, v, table.to(device), i32([0]), i32([n]), i32([n]), dim ** -0.5, max_q_len=n).view(n, nq, dim)
    assert bool(out[:90].isfinite().all()) and bool(out[90:].isnan().all())
    check_attention(out, q.view(n, nq, dim), k, v, table, [(0, n, n)], dim ** -0.5, nq, nq)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nq,nkv,dim,splits,norm,bias,masks", [
    (4, 2, 128, 3, False, False, {}), (8, 1, 64, 8, False, True, dict(window=40, sinks=True)), (5, 1, 128, 1, True, False, {}),
    (16, 16, 64, 10, True, True, dict(sinks=True))])
def test_step_is_append_and_attention(device, nq, nkv, dim, splits, norm, bias, masks):
    g = torch.Generator().manual_seed(nq + dim + splits)
    masks = dict(masks)
    contexts = [1, 33, 64, 130, 0]                                           # the last row is inactive
    table, blocks = shuffled_table(g, contexts)
    one, two = pool(g, blocks, nkv, dim, device), None
    two = tuple(ops.QuantizedPages(p.values.clone(), p.scales.clone()) for p in one)
    qkv, b, qw, kw = append_case(g, len(contexts), nq, nkv, dim, splits, norm, bias)
    sinks = torch.randn((nq,), generator=g).to(device) if masks.pop("sinks", False) else None
    to = lambda t: None if t is None else t.to(device)                       # noqa: E731
    lens = torch.tensor(contexts, dtype=torch.int32)
    pos = (lens - 1).clamp(min=0)
    slots = torch.tensor([int(table[i, p // PAGE]) * PAGE + p % PAGE for i, p in enumerate(pos.tolist())], dtype=torch.int32)
    slots[-1] = -1
    cs, lens, table_d = to(rope_table(dim, 200)), to(lens), to(table)
    more = dict(bias=to(b), q_norm_w=to(qw), k_norm_w=to(kw), norm_eps=1e-5)
    out = ops.rope_attn_decode(to(qkv), to(pos), to(slots), cs, *one, table_d, lens, dim ** -0.5, nq, nkv, sinks=sinks, **masks, **more)
    q = ops.rope_kv_append(to(qkv), to(pos), to(slots), cs, *two, nq, nkv, dim, **more)
    for a, c in zip(one, two):
        assert torch.equal(a.values.view(torch.uint8), c.values.view(torch.uint8))
        assert torch.equal(a.scales.view(torch.uint8), c.scales.view(torch.uint8))
    check_attention(out.view(-1, nq, dim), q.view(-1, nq, dim), *one, table, [(i, 1, c) for i, c in enumerate(contexts)], dim ** -0.5, nq,
                    nq // nkv, None if sinks is None else sinks.cpu(), **masks)


@pytest.mark.parametrize("device", DEVICES)
def test_values_that_are_not_finite_stay_with_their_head_and_token(device):
    """From the projection through the pages to attention: what is not finite reaches the rows that see it, and no others."""
    g = torch.Generator().manual_seed(77)
    nq, nkv, dim, n = 4, 2, 64, 40
    k, v = pool(g, 3, nkv, dim, device)
    table, slots = torch.tensor([[2, 0]], dtype=torch.int32), torch.cat([torch.arange(64, 96), torch.arange(8)]).int()
    x = torch.randn((n, (nq + 2 * nkv) * dim), generator=g).to(torch.bfloat16)
    head = x.view(n, nq + 2 * nkv, dim)
    head[30, nq, 5], head[35, nq + nkv + 1, 63], head[20, 1, 7] = math.inf, math.nan, math.nan      # K of head 0, V of head 1, a query
    cs, i32 = rope_table(dim, n), lambda t: torch.tensor(t, dtype=torch.int32, device=device)       # noqa: E731
    q = ops.rope_kv_append(x.to(device), torch.arange(n, dtype=torch.int32).to(device), slots.to(device), cs.to(device), k, v, nq, nkv, dim)
    out = ops.flash_attn_prefill(q, k, v, table.to(device), i32([0]), i32([n]), i32([n]), 0.125, max_q_len=n).view(n, nq, dim).cpu()
    lost = torch.zeros((n, nq), dtype=torch.bool)
    lost[30:, :2], lost[35:, 2:], lost[20, 1] = True, True, True
    assert torch.equal(out.isnan().any(-1), lost) and torch.equal(out.isnan().all(-1), lost)
    last = ops.paged_attn_decode(q[-1:], k, v, table.to(device), i32([n]), 0.125, window=5).view(nq, dim).cpu()
    assert bool(last[:2].isfinite().all()) and bool(last[2:].isnan().all())


@pytest.mark.parametrize("device", DEVICES)
def test_tables_that_are_part_of_larger_ones(device):
    g = torch.Generator().manual_seed(78)
    nq, nkv, dim, contexts = 4, 2, 64, [70, 1, 600]
    table, blocks = shuffled_table(g, contexts)
    k, v = pool(g, blocks, nkv, dim, device)
    wide = torch.full((5, table.shape[1] + 7), -9, dtype=torch.int32)
    wide[1:4, 3:3 + table.shape[1]] = table
    part = wide.to(device)[1:4, 3:3 + table.shape[1]]
    q = torch.randn((3, nq * dim), generator=g).to(torch.bfloat16)
    lens, one = torch.tensor(contexts, dtype=torch.int32, device=device), torch.ones(3, dtype=torch.int32, device=device)
    spans = [(b, 1, c) for b, c in enumerate(contexts)]
    for out in (ops.paged_attn_decode(q.to(device), k, v, part, lens, 0.125), ops.paged_attn_decode(q.to(device), k, v, part, lens, 0.125, num_splits=3),
                ops.flash_attn_prefill(q.to(device), k, v, part, torch.arange(3, dtype=torch.int32, device=device), one, lens, 0.125, max_q_len=1)):
        check_attention(out.view(3, nq, dim), q.view(3, nq, dim), k, v, table, spans, 0.125, nq, nq // nkv)
    # one row for all sequences
    same = table[2:].to(device).expand(3, -1)
    out = ops.paged_attn_decode(q.to(device), k, v, same, lens, 0.125)
    check_attention(out.view(3, nq, dim), q.view(3, nq, dim), k, v, table[2:].expand(3, -1), spans, 0.125, nq, nq // nkv)


@pytest.mark.parametrize("device", DEVICES)
def test_packed_steps(device):
    """Single tokens first, then prompts, then rows of padding."""
    g = torch.Generator().manual_seed(79)
    nq, nkv, dim = 4, 2, 128
    spans = [(0, 1, 40), (1, 1, 333), (2, 1, 1), (3, 50, 50), (53, 20, 90)]
    table, blocks = shuffled_table(g, [c for *_, c in spans])
    k, v = pool(g, blocks, nkv, dim, device)
    q = torch.randn((80, nq * dim), generator=g).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)        # noqa: E731
    out = ops.packed_attention(q.to(device), k, v, table.to(device), i32([s for s, *_ in spans]), i32([n for _, n, _ in spans]),
                               i32([c for *_, c in spans]), dim ** -0.5, max_q_len=50, singles=3)
    check_attention(out.view(80, nq, dim), q.view(80, nq, dim), k, v, table, spans, dim ** -0.5, nq, nq // nkv)


class Work:
    """Appended tokens, a step, decode attention in parts and prompts in parts, over pages of their own."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.nq, self.nkv, self.dim, contexts = 4, 2, 128, [900, 33, 2000]
        self.contexts = contexts
        table, blocks = shuffled_table(g, contexts)
        self.k, self.v = pool(g, blocks, self.nkv, self.dim, "cuda")
        W = (self.nq + 2 * self.nkv) * self.dim
        self.parts, self.rows = torch.randn((3, 3, W), generator=g).cuda(), torch.randn((20, W), generator=g).to(torch.bfloat16).cuda()
        pos = torch.tensor(contexts) - 1
        self.slots = torch.tensor([int(table[b, p // PAGE]) * PAGE + p % PAGE for b, p in enumerate(pos.tolist())], dtype=torch.int32).cuda()
        back = torch.arange(pos[2] - 19, pos[2] + 1)
        self.long = (table[2, back // PAGE].long() * PAGE + back % PAGE).int().cuda()
        self.pos, self.back, self.table = pos.int().cuda(), back.int().cuda(), table.cuda()
        self.lens, self.cs = torch.tensor(contexts, dtype=torch.int32).cuda(), rope_table(self.dim, 2000).cuda()
        self.at = [torch.tensor([x], dtype=torch.int32).cuda() for x in (0, 20, 2000)]

    def run(self):
        heads = self.nq, self.nkv
        a = ops.rope_attn_decode(self.parts, self.pos, self.slots, self.cs, self.k, self.v, self.table, self.lens, 0.1, *heads, num_splits=4)
        q = ops.rope_kv_append(self.rows, self.back, self.long, self.cs, self.k, self.v, *heads, self.dim)
        b = ops.paged_attn_decode(q[:3], self.k, self.v, self.table, self.lens, 0.1, num_splits=5)
        c = ops.flash_attn_prefill(q, self.k, self.v, self.table[2:], *self.at, 0.1, max_q_len=20)
        return a, b, c

    def change(self, other):
        """The other's inputs in this one's tensors."""
        self.parts.copy_(other.parts)
        self.rows.copy_(other.rows)


@pytest.mark.gpu
def test_captured_and_on_several_streams():
    """Graphs replayed beside one another and beside eager calls: the results are those of calls one after another, bit by bit."""
    works = [Work(s) for s in range(4)]
    [w.run() for w in works]
    want = [[t.clone() for t in w.run()] for w in works]                     # (a second run stores the same bytes)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for w in works[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(w.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in works]
    got = [[] for _ in works]
    for _ in range(10):
        for i, (w, st) in enumerate(zip(works, streams)):
            with torch.cuda.stream(st):
                if i < 2:
                    graphs[i].replay()
                    got[i].append([t.clone() for t in outs[i]])
                else:
                    got[i].append(w.run())
    torch.cuda.synchronize()
    for rounds, w in zip(got, want):
        for one in rounds:
            assert all(torch.equal(a, b) for a, b in zip(one, w))
    works[0].change(works[1])                                                # a replayed graph reads what is there then
    graphs[0].replay()
    graphs[0].replay()                                                       # (the tokens that the first one appended take part in its step)
    torch.cuda.synchronize()
    now = [t.clone() for t in outs[0]]
    assert all(torch.equal(a, b) for a, b in zip(now, works[0].run())) and not torch.equal(now[0], want[0][0])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_pools_beyond_32_bits(dim):
    """Blocks whose bytes lie behind 2^32."""
    g = torch.Generator().manual_seed(80 + dim)
    nkv, nq, n = 8, 16, 130
    blocks = (1 << 32) // (nkv * PAGE * dim) + 50
    empty = lambda *shape: torch.empty(shape, dtype=torch.uint8, device="cuda")       # noqa: E731
    k, v = (ops.QuantizedPages(empty(blocks, nkv, PAGE, dim).view(F8), empty(blocks, nkv, PAGE).view(E8)) for _ in range(2))
    used = torch.tensor([blocks - 1, 0, blocks - 20, blocks - 3, 7], dtype=torch.int32)       # the last ones, and the first ones between them
    pos = torch.arange(n, dtype=torch.int32)
    slots = used[pos.long() // PAGE] * PAGE + pos % PAGE
    x = torch.randn((n, (nq + 2 * nkv) * dim), generator=g).to(torch.bfloat16)
    q = ops.rope_kv_append(x.cuda(), pos.cuda(), slots.cuda(), rope_table(dim, n).cuda(), k, v, nq, nkv, dim)
    small = tuple(ops.QuantizedPages(p.values.view(torch.uint8)[used.cuda().long()].view(F8), p.scales.view(torch.uint8)[used.cuda().long()].view(E8))
                  for p in (k, v))
    i32 = lambda t: torch.tensor(t, dtype=torch.int32).cuda()                # noqa: E731
    out = ops.flash_attn_prefill(q, k, v, used[None].cuda(), i32([0]), i32([n]), i32([n]), 0.1, max_q_len=n)
    check_attention(out.view(n, nq, dim), q.view(n, nq, dim), *small, torch.arange(5)[None], [(0, n, n)], 0.1, nq, 2)
    last = ops.paged_attn_decode(q[-1:], k, v, used[None].cuda(), i32([n]), 0.1, num_splits=2)
    check_attention(last.view(1, nq, dim), q[-1:].view(1, nq, dim), *small, torch.arange(5)[None], [(0, 1, n)], 0.1, nq, 2)
    step = ops.rope_attn_decode(x[None, -1:].float().cuda(), pos[-1:].cuda(), slots[-1:].cuda(), rope_table(dim, n).cuda(),
                                k, v, used[None].cuda(), i32([n]), 0.1, nq, nkv)
    check_attention(step.view(1, nq, dim), q[-1:].view(1, nq, dim), *small, torch.arange(5)[None], [(0, 1, n)], 0.1, nq, 2)


@pytest.mark.gpu
def test_kernels_are_counted():
    w = Work(9)
    w.run()
    heads, n = (w.nq, w.nkv), []
    for f in (lambda: ops.rope_kv_append(w.rows, w.back, w.long, w.cs, w.k, w.v, *heads, w.dim),
              lambda: ops.rope_attn_decode(w.parts, w.pos, w.slots, w.cs, w.k, w.v, w.table, w.lens, 0.1, *heads),
              lambda: ops.paged_attn_decode(w.parts[0, :, :w.nq * w.dim].bfloat16().contiguous(), w.k, w.v, w.table, w.lens, 0.1)):
        before = ops.launch_count()
        f()
        n.append(ops.launch_count() - before)
    assert n == [1, 2, 1]


# ------------------------------------------------------------------------------------------------ refusals
def test_pages_are_checked():
    good = ops.QuantizedPages.new(2, 1, 64)
    with pytest.raises(TypeError):
        ops.QuantizedPages(good.values.float(), good.scales)
    with pytest.raises(TypeError):
        ops.QuantizedPages(good.values, good.scales.view(torch.uint8))
    with pytest.raises(ValueError):
        ops.QuantizedPages(good.values[:1], good.scales)
    with pytest.raises(ValueError):
        ops.QuantizedPages.new(2, 1, 96)
    with pytest.raises(ValueError):
        ops.QuantizedPages(good.values[:, :, :16].contiguous(), good.scales[:, :, :16].contiguous())
    two = ops.QuantizedPages.new(2, 3, 64)
    with pytest.raises(ValueError):
        ops.QuantizedPages(two.values.transpose(0, 1), two.scales.transpose(0, 1).contiguous())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    shifted = lambda t: torch.empty((t.numel() + 1,), dtype=t.dtype, device=device)[1:].view(t.shape)        # noqa: E731
    k, v = (ops.QuantizedPages.new(4, 2, 64, device) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)        # noqa: E731
    q = torch.zeros((2, 4 * 64), dtype=torch.bfloat16, device=device)
    table, lens = i32([[0, 1], [2, 3]]), i32([40, 50])
    plain = torch.zeros((4, 2, 32, 64), dtype=torch.bfloat16, device=device)
    decode = lambda q=q, k=k, v=v, t=table, n=lens, **kw: ops.paged_attn_decode(q, k, v, t, n, 0.1, **kw)       # noqa: E731
    for kw, err in [(dict(k=plain), TypeError), (dict(v=plain), TypeError), (dict(v=ops.QuantizedPages.new(4, 1, 64, device)), ValueError),
                    (dict(q=q.float()), TypeError), (dict(q=q[:1]), ValueError), (dict(q=q[:, :3 * 64].contiguous()), ValueError),
                    (dict(t=table.long()), TypeError), (dict(n=lens.long()), TypeError), (dict(n=lens[:1]), ValueError),
                    (dict(t=table[0]), ValueError), (dict(window=-1), ValueError), (dict(chunk=-2), ValueError), (dict(q_len=0), ValueError),
                    (dict(mods=ops.ScoreMods(softcap=3.0)), ValueError), (dict(sinks=torch.zeros((3,), device=device)), ValueError),
                    (dict(out=torch.empty_like(q, dtype=torch.float32)), TypeError), (dict(out=q[:1]), ValueError),
                    *([] if device == "cpu" else [(dict(q=shifted(q)), ValueError), (dict(out=shifted(q)), ValueError),
                                                  (dict(num_splits=2, scratch=torch.zeros((8,), device=device)), ValueError)])]:
        with pytest.raises(err):
            decode(**kw)
    prompt = lambda s=i32([0, 1]), n=i32([1, 1]), c=lens, **kw: ops.flash_attn_prefill(       # noqa: E731
        q, k, v, table, s, n, c, 0.1, **{"max_q_len": 1, **kw})
    for kw, err in [(dict(s=i32([0])), ValueError), (dict(n=lens.float()), TypeError), (dict(max_q_len=0), ValueError), (dict(out=q.float()), TypeError),
                    (dict(mods=ops.ScoreMods(keep_first=3)), ValueError)]:
        with pytest.raises(err):
            prompt(**kw)
    qkv = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device=device)
    cs = torch.zeros((64, 64), device=device)
    append = lambda x=qkv, pos=i32([0, 1]), s=i32([0, 1]), c=cs, nq=4, nkv=2, d=64, **kw: ops.rope_kv_append(       # noqa: E731
        x, pos, s, c, k, v, nq, nkv, d, **kw)
    for kw, err in [(dict(x=qkv[:, :-8].contiguous()), ValueError), (dict(x=qkv.half()), TypeError), (dict(pos=i32([0])), ValueError),
                    (dict(s=i32([0, 1]).long()), TypeError), (dict(c=cs.double()), TypeError), (dict(c=cs[:, :32].contiguous()), ValueError),
                    (dict(c=cs[:0]), ValueError), (dict(nkv=4, nq=0), ValueError), (dict(nq=3), ValueError), (dict(d=128), ValueError),
                    (dict(bias=torch.zeros((8 * 64,), device=device)), TypeError), (dict(pos=None), ValueError),
                    (dict(k_norm_w=torch.zeros((32,), dtype=torch.bfloat16, device=device)), ValueError)]:
        with pytest.raises(err):
            append(**kw)
    with pytest.raises(ValueError):
        ops.rope_attn_decode(qkv, i32([0, 1]), i32([0, 1]), cs, k, v, table, lens, 0.1, 4, 2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 3])
def test_partial_sums_that_lie_apart(device, T):
    """Slices of a larger buffer: partial sums further apart than their rows; rows apart are refused."""
    g = torch.Generator().manual_seed(90)
    nq, nkv, dim, W = 2, 1, 64, 4 * 64
    whole = torch.randn((3, T + 2, W), generator=g).to(device)
    at = torch.arange(T, dtype=torch.int32, device=device)
    one, two = (tuple(ops.QuantizedPages.new(1, nkv, dim, device) for _ in range(2)) for _ in range(2))
    cs = rope_table(dim, T).to(device)
    a = ops.rope_kv_append(whole[:, 1:1 + T], at, at, cs, *one, nq, nkv, dim)
    b = ops.rope_kv_append(whole[:, 1:1 + T].contiguous(), at, at, cs, *two, nq, nkv, dim)
    assert torch.equal(a, b) and all(torch.equal(x.values.view(torch.uint8), y.values.view(torch.uint8)) for x, y in zip(one, two))
    for bad in (torch.zeros((3, T, 2 * W), device=device)[..., ::2], torch.zeros((3, 2, 2 * W), device=device)[:, :, :W],
                torch.zeros((2, 2 * W), dtype=torch.bfloat16, device=device)[:, :W]):
        with pytest.raises(ValueError):
            ops.rope_kv_append(bad, at[:1].expand(bad.shape[-2]).contiguous(), None, None, *one, nq, nkv, dim)


@pytest.mark.parametrize("blocks,heads", [(0, 1), (1, 0)])
@pytest.mark.parametrize("device", DEVICES)
def test_pools_have_a_page(device, blocks, heads):
    with pytest.raises(ValueError):
        ops.QuantizedPages.new(blocks, heads, 64, device)


def test_parts_of_a_sequence_are_bounded():
    pages = ops.QuantizedPages.new(2, 1, 64)
    with pytest.raises(ValueError):
        ops.paged_attn_decode(torch.zeros((1, 64), dtype=torch.bfloat16), pages, pages, torch.zeros((1, 1), dtype=torch.int32),
                              torch.ones(1, dtype=torch.int32), 0.1, num_splits=100000)


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused(monkeypatch):
    w = Work(3)
    q = torch.zeros((3, w.nq * w.dim), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.paged_attn_decode(q, w.k, w.v, w.table, w.lens, 0.1)
    with pytest.raises(ValueError):
        ops.paged_attn_decode(q.cuda(), w.k, w.v, w.table.cpu(), w.lens, 0.1)
    with pytest.raises(ValueError):
        ops.rope_kv_append(w.rows.cpu(), w.back, w.long, w.cs, w.k, w.v, w.nq, w.nkv, w.dim)
    with pytest.raises(ValueError):
        ops.flash_attn_prefill(q.cuda(), w.k, w.v, w.table, w.lens.cpu(), w.lens, w.lens, 0.1, max_q_len=1)
    cpu = ops.QuantizedPages(w.v.values.cpu(), w.v.scales.cpu())
    with pytest.raises(ValueError):
        ops.paged_attn_decode(q.cuda(), w.k, cpu, w.table, w.lens, 0.1)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)              # the pages' device is not the current one
    for call in (lambda: ops.paged_attn_decode(q.cuda(), w.k, w.v, w.table, w.lens, 0.1), w.run,
                 lambda: ops.flash_attn_prefill(q.cuda(), w.k, w.v, w.table, w.lens, w.lens, w.lens, 0.1, max_q_len=1)):
        with pytest.raises(ValueError):
            call()
