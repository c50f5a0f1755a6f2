"""Keys and values in 8 bits at their edges: scratch, queries and scales of unusual sizes, masks that part two query tiles, bytes that nobody sees."""

import math
import subprocess
import sys

import pytest
import torch

from nkipy_b200 import ops
from nkipy_b200.ops import _lib
from nkipy_b200.ops import quantized_kv as Q
from tests.test_quantized_kv import DEVICES, cached, fill, oracle_quantize, oracle_turn, pool, rope_table, shuffled_table, stored


# ------------------------------------------------------------------------------------------------ scratch
class Library:
    """Stands in for the kernel library: sizes are right once it is initialised."""

    def __init__(self, sms=148):
        self.sms, self.ready = sms, False

    def nkb_init(self):
        self.ready = True
        return 0

    def nkb_q8_attn_decode_scratch_floats(self, *sizes):
        return 1000 if self.ready else 10

    def nkb_q8_attn_prefill_scratch_floats(self, *sizes):
        return 2000 if self.ready else 20


@pytest.fixture
def fresh_library(monkeypatch):
    """A library that no call has reached yet, and sizes that no call has asked for."""
    def forget():
        Q._decode_floats.cache_clear()
        Q._prefill_floats.cache_clear()

    fake = Library()
    forget()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(_lib, "_initialised", False)
    yield fake
    forget()


def test_sizes_of_scratch_are_asked_of_an_initialised_library(fresh_library):
    assert Q._decode_floats(1, 8, 128, 4, 4) == 1000
    fresh_library.ready = _lib._initialised = False
    assert Q._prefill_floats(1, 100, 32, 8, 128, 32) == 2000


def test_no_size_is_kept_of_a_library_without_a_device(fresh_library, monkeypatch):
    monkeypatch.setattr(fresh_library, "nkb_init", lambda: -1)
    for _ in range(2):
        with pytest.raises(_lib.KernelLibraryError):
            Q._decode_floats(1, 8, 128, 4, 4)
        with pytest.raises(_lib.KernelLibraryError):
            Q._prefill_floats(1, 100, 32, 8, 128, 32)


@pytest.mark.gpu
def test_scratch_of_a_new_process():
    """A cache that is the process's first use of the library has room for what its steps take."""
    code = """
from nkipy_b200 import ops
from nkipy_b200.ops import _lib, quantized_kv as Q
sizes = [(8, 32, 1, 32), (8, 32, 1, 250), (1, 16, 3, 400), (4, 4, 2, 77)]
first = [Q.decode_scratch(ops.QuantizedPages.new(1, nkv, 128, "cuda"), nq, batch, pages).numel() for nkv, nq, batch, pages in sizes]
_lib.ensure_init()
Q._decode_floats.cache_clear()
again = [Q.decode_scratch(ops.QuantizedPages.new(1, nkv, 128, "cuda"), nq, batch, pages).numel() for nkv, nq, batch, pages in sizes]
assert first == again, (first, again)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


@pytest.mark.gpu
def test_kernels_refuse_scratch_that_is_too_small(monkeypatch):
    """The library looks at the size by itself: here the caller believes in a smaller one."""
    g = torch.Generator().manual_seed(1)
    table, blocks = shuffled_table(g, [900])
    k, v = pool(g, blocks, 2, 64, "cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")       # noqa: E731
    q = torch.zeros((1, 4 * 64), dtype=torch.bfloat16, device="cuda")
    small = torch.zeros((Q.COUNTERS + 8,), device="cuda")
    monkeypatch.setattr(Q, "_decode_floats", lambda *sizes: small.numel())
    with pytest.raises(_lib.KernelLibraryError):
        ops.paged_attn_decode(q, k, v, table.cuda(), i32(900), 0.1, num_splits=4, scratch=small)
    monkeypatch.setattr(Q, "_prefill_floats", lambda *sizes: small.numel())
    monkeypatch.setattr(Q, "_scratch", lambda *a: small)
    with pytest.raises(_lib.KernelLibraryError):
        ops.flash_attn_prefill(q, k, v, table.cuda(), i32(0), i32(1), i32(900), 0.1, max_q_len=1)
    assert not bool(small.any())


# ------------------------------------------------------------------------------------------------ attention, all rows of a sequence at once
def attend(q, k, v, scale, pos0, causal=True, window=0, chunk=0, sink=None, weights=2.0 ** -11, lost=2.0 ** -30, keep_first=0, softcap=0.0):
    """One query head's rows q [n, dim] at positions pos0 on, over k, v [tokens, dim], in 64 bits: (results, tolerances).

    As `test_quantized_kv.oracle_attend` has it: 2^-8 of the result for its rounding to bf16; of every weight `weights` for its own rounding
    (f16: 2^-11, bf16: 2^-8), 2^-19 for exponential and sum, and twice what 2^-19 of the largest sum |q k| moves it by; `lost` of the largest
    value that the row sees, for every token that it sees, for weights that end above nothing."""
    pos, at = pos0 + torch.arange(q.shape[0])[:, None], torch.arange(k.shape[0])
    if not len(k):
        return torch.zeros_like(q), torch.zeros_like(q)
    seen = at <= pos if causal else torch.ones((q.shape[0], k.shape[0]), dtype=torch.bool)
    if window:
        seen = seen & (at > pos - window)
    if chunk:
        seen = seen & (at >= pos - pos % chunk)
    if keep_first:
        seen = seen | ((at < keep_first) & (at <= pos))
    lost_rows = (seen & (k.isnan() | v.isnan()).any(-1)).any(-1)              # tokens that stand for NaN take the rows that see them along
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    s = q @ k.T * scale
    s = (softcap * torch.tanh(s / softcap) if softcap else s).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        top = top.clamp(min=sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True) + (0.0 if sink is None else torch.exp(sink - top))
    p = torch.where(total > 0, p / total, 0.0)
    o = (p @ v).masked_fill(lost_rows[:, None], math.nan)
    moved = 2.0 ** -19 * (q.abs() @ k.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True) * abs(scale)
    largest = v.abs().amax(-1).expand(seen.shape).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    return o, 2.0 ** -8 * o.abs().nan_to_num(0.0) + (p @ v.abs()) * (weights + 2.0 ** -19 + 2 * moved) + seen.sum(-1, keepdim=True) * lost * largest + 1e-30


def check_rows(out, q, k, v, spans, scale, group, sinks=None, **masks):
    """out, q [tokens, heads, dim]; k, v: a sequence's rows [context, kv heads, dim] each; spans: (first row, new tokens, context)."""
    out, q = out.cpu().double(), q.cpu().double()
    for b, (row, n, ctx) in enumerate(spans):
        for h in range(q.shape[1]):
            want, tol = attend(q[row:row + n, h], k[b][:, h // group].double(), v[b][:, h // group].double(), scale, ctx - n,
                               sink=None if sinks is None else float(sinks[h]), **masks)
            got = out[row:row + n, h]
            assert torch.equal(got.isnan(), want.isnan()), (b, h)
            err = (got - want).abs().nan_to_num(0.0)
            assert bool((err <= tol).all()), (b, h, float((err / tol).max()))


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------------ masks that part two query tiles
CHUNKS = [
    # nq, nkv, (cached, new) per sequence, masks
    (1, 1, [(200, 700)], dict(chunk=512)),                                   # the second 128 rows of a pair begin four key tiles later
    (2, 2, [(0, 1500), (77, 300)], dict(chunk=1100)),
    (4, 1, [(900, 300)], dict(chunk=1000)),
    (1, 1, [(100, 800)], dict(chunk=512, window=300)),
    (1, 1, [(130, 700)], dict(chunk=400, causal=False)),
    (2, 1, [(1500, 40), (0, 200)], dict(chunk=700)),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("nq,nkv,spans,masks", CHUNKS)
def test_chunks_that_begin_between_query_tiles(device, dim, bits, nq, nkv, spans, masks):
    g = torch.Generator().manual_seed(dim + nq)
    contexts, new = [a + n for a, n in spans], [n for _, n in spans]
    table, blocks = shuffled_table(g, contexts)
    q = torch.randn((sum(new), nq * dim), generator=g).to(torch.bfloat16)
    if bits == 8:
        pages = pool(g, blocks, nkv, dim, device)
        k, v = ([cached(p, table[b], c) for b, c in enumerate(contexts)] for p in pages)
    else:
        pages = [torch.randn((blocks, nkv, 32, dim), generator=g).to(torch.bfloat16) for _ in range(2)]
        k, v = ([p[table[b, :-(-c // 32)].long()].transpose(1, 2).reshape(-1, nkv, dim)[:c] for b, c in enumerate(contexts)] for p in pages)
        pages = [p.to(device) for p in pages]
    starts = [sum(new[:b]) for b in range(len(new))]
    out = ops.flash_attn_prefill(q.to(device), *pages, table.to(device), i32(starts, device), i32(new, device), i32(contexts, device),
                                 dim ** -0.5, max_q_len=max(new), **masks)
    check_rows(out.view(-1, nq, dim), q.view(-1, nq, dim), k, v, list(zip(starts, new, contexts)), dim ** -0.5, nq // nkv,
               **masks, weights=2.0 ** -11 if bits == 8 else 2.0 ** -8)


# ------------------------------------------------------------------------------------------------ queries and keys of unusual sizes
def prompt(q, pages, table, spans, scale, device, **masks):
    """Rows [tokens, heads, dim] of `spans` (first row, new tokens, context)."""
    n, heads, dim = q.shape
    out = ops.flash_attn_prefill(q.reshape(n, heads * dim).to(device), *pages, table.to(device), *(i32([s[j] for s in spans], device) for j in (0, 1, 2)),
                                 scale, max_q_len=max(s[1] for s in spans), **{m: x.to(device) if m == "sinks" else x for m, x in masks.items()})
    return out.view(n, heads, dim)


def rows_of(pages, table, spans):
    """Keys and values of every sequence, [context, kv heads, dim] in 64 bits."""
    return ([cached(p, table[b], ctx) for b, (_, _, ctx) in enumerate(spans)] for p in pages)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("nq,nkv,spans,masks", [
    (4, 2, [(0, 200, 200), (200, 33, 350), (233, 1, 77)], {}),
    (2, 1, [(0, 140, 300)], dict(window=50)),
    (8, 1, [(0, 5, 2100), (5, 3, 1000)], {}),                               # divided among works
    (4, 4, [(70 * i, 70, 70) for i in range(40)], {}),
    (4, 1, [(0, 130, 260)], dict(chunk=100)),
])
def test_queries_that_are_zero_or_tiny(device, dim, sinks, nq, nkv, spans, masks):
    """Rows of zeros see the mean of their values, rows next to zero the same within the tolerance."""
    g = torch.Generator().manual_seed(dim + nq)
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    pages = pool(g, blocks, nkv, dim, device)
    q = torch.randn((sum(n for _, n, _ in spans), nq, dim), generator=g).to(torch.bfloat16)
    size = torch.randint(0, 4, q.shape[:2], generator=g)
    q = torch.where(size[..., None] == 0, q, q * torch.tensor([0.0, 0.0, 1e-20, 1e-38])[size][..., None]).to(torch.bfloat16)
    q[:, -1] = 0.0                                                          # a head of zeros
    s = torch.randn((nq,), generator=g) if sinks else None
    out = prompt(q, pages, table, spans, dim ** -0.5, device, **masks, **({"sinks": s} if sinks else {}))
    check_rows(out, q, *rows_of(pages, table, spans), spans, dim ** -0.5, nq // nkv, s, **masks)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys", [0.0, 2.0 ** -60, 2.0 ** -30, 2.0 ** 60])
def test_keys_that_are_zero_or_far_from_one(device, dim, keys):
    g = torch.Generator().manual_seed(dim)
    spans, nq = [(0, 150, 250), (150, 5, 1500)], 2
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    k, v = pool(g, blocks, 1, dim, device)
    fill(k, torch.randn((blocks, 1, 32, dim), generator=g, dtype=torch.float64) * keys)
    for size in (0.0, 1e-30, 2.0 ** -60, 1.0):
        if size * keys > 2.0 ** 10:
            continue
        q = (torch.randn((155, nq, dim), generator=g) * size).to(torch.bfloat16)
        for scale in (dim ** -0.5, 1e-6):
            out = prompt(q, (k, v), table, spans, scale, device)
            check_rows(out, q, *rows_of((k, v), table, spans), spans, scale, nq)
            one = ops.paged_attn_decode(q[149:151].reshape(2, -1).to(device), k, v, table.to(device), i32([250, 1500], device), scale)
            check_rows(one.view(2, nq, dim), q[149:151], *rows_of((k, v), table, spans), [(0, 1, 250), (1, 1, 1500)], scale, nq)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [-1.0, -0.05, 0.0, 1e-30, -1e-40])
def test_scales_of_scores(device, dim, scale):
    g = torch.Generator().manual_seed(dim)
    spans, nq = [(0, 150, 250), (150, 5, 1500)], 2
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    pages = pool(g, blocks, 1, dim, device)
    q = torch.randn((155, nq, dim), generator=g).to(torch.bfloat16)
    check_rows(prompt(q, pages, table, spans, scale, device), q, *rows_of(pages, table, spans), spans, scale, nq)
    one = ops.paged_attn_decode(q[149:151].reshape(2, -1).to(device), *pages, table.to(device), i32([250, 1500], device), scale)
    check_rows(one.view(2, nq, dim), q[149:151], *rows_of(pages, table, spans), [(0, 1, 250), (1, 1, 1500)], scale, nq)


@pytest.mark.parametrize("device", DEVICES)
def test_scales_that_are_not_finite_are_refused(device):
    g = torch.Generator().manual_seed(0)
    table, blocks = shuffled_table(g, [40])
    pages, q = pool(g, blocks, 1, 64, device), torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    for scale in (math.nan, math.inf, -math.inf):
        with pytest.raises(ValueError):
            prompt(q, pages, table, [(0, 1, 40)], scale, device)
        with pytest.raises(ValueError):
            ops.paged_attn_decode(q[0].to(device), *pages, table.to(device), i32([40], device), scale)
        with pytest.raises(ValueError):
            ops.rope_attn_decode(torch.zeros((1, 1, 3 * 64), device=device), i32([39], device), i32([-1], device), None, *pages, table.to(device),
                                 i32([40], device), scale, 1, 1)


# ------------------------------------------------------------------------------------------------ scale bytes that no row has
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("byte,stands_for", [(0, 63), (1, 63), (62, 63), (192, 191), (254, 191)])
def test_scales_outside_the_range_stand_for_its_ends(device, byte, stands_for):
    g = torch.Generator().manual_seed(byte)
    dim, nq, spans = 64, 2, [(0, 1, 40)]
    table, blocks = shuffled_table(g, [40])
    k, v = pool(g, blocks, 1, dim, device)
    v.scales.view(torch.uint8)[...] = byte
    want = v.values.float() * 2.0 ** (stands_for - 127)
    assert torch.equal(v.dequantize(), want) and torch.equal(v.dequantize(torch.tensor([1], device=device)), want[1:2])
    keys, _ = rows_of((k, v), table, spans)
    values = [want.cpu()[table[0].long()].transpose(1, 2).reshape(-1, 1, dim)[:40]]
    q = torch.randn((1, nq, dim), generator=g).to(torch.bfloat16)
    for out in (prompt(q, (k, v), table, spans, 0.125, device),
                ops.paged_attn_decode(q.view(1, -1).to(device), k, v, table.to(device), i32([40], device), 0.125).view(1, nq, dim)):
        check_rows(out, q, keys, values, spans, 0.125, nq)


# ------------------------------------------------------------------------------------------------ bytes that nobody sees
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("byte", [0x7f, 0xff, 0x7e])
@pytest.mark.parametrize("q_len,masks", [(1, {}), (1, dict(window=45)), (3, {}), (4, dict(window=40)), (2, dict(chunk=48))])
def test_bytes_that_nobody_sees(device, dim, byte, q_len, masks):
    """Behind a context, before a window and in other blocks: e4m3's NaN or largest number, with any scale."""
    g = torch.Generator().manual_seed(dim + byte + q_len)
    nq, nkv, contexts = 4, 2, [37, 150, 64, 700, q_len]
    table, blocks = shuffled_table(g, contexts, extra=2)
    pages = pool(g, blocks, nkv, dim, device)
    spans = [(b * q_len, q_len, c) for b, c in enumerate(contexts)]
    k, v = rows_of(pages, table, spans)
    seen = torch.zeros((blocks, 32), dtype=torch.bool)
    for b, c in enumerate(contexts):
        first = c - q_len
        lo = max(first - masks.get("window", c) + 1, first - first % masks["chunk"] if "chunk" in masks else 0, 0)
        for j in range(lo, c):
            seen[table[b, j // 32], j % 32] = True
    for p in pages:
        values, scales = p.values.view(torch.uint8).cpu(), p.scales.view(torch.uint8).cpu()
        values[~seen[:, None].expand(scales.shape)] = byte
        scales[~seen[:, None].expand(scales.shape)] = torch.randint(0, 256, (int((~seen).sum()) * nkv,), generator=g).to(torch.uint8)
        p.values.view(torch.uint8).copy_(values)
        p.scales.view(torch.uint8).copy_(scales)
    q = torch.randn((len(contexts) * q_len, nq, dim), generator=g).to(torch.bfloat16)
    for splits in (1, 4):
        out = ops.paged_attn_decode(q.view(q.shape[0], -1).to(device), *pages, table.to(device), i32(contexts, device), 0.1, q_len=q_len,
                                    num_splits=splits, **masks)
        check_rows(out.view(q.shape), q, k, v, spans, 0.1, 2, **masks)
    check_rows(prompt(q, pages, table, spans, 0.1, device, **masks), q, k, v, spans, 0.1, 2, **masks)
    if q_len == 1 and "chunk" not in masks:                                  # the step: nothing appended, queries as they are
        qkv = torch.cat([q.float().view(5, -1), torch.zeros((5, 2 * nkv * dim))], -1)[None].to(device)
        out = ops.rope_attn_decode(qkv, i32([0] * 5, device), i32([-1] * 5, device), None, *pages, table.to(device), i32(contexts, device), 0.1, nq,
                                   nkv, **masks)
        check_rows(out.view(q.shape), q, k, v, spans, 0.1, 2, **masks)


# ------------------------------------------------------------------------------------------------ values of very different sizes
def stored_rows(g, pages, table, spans, sizes):
    """Random rows in the pages, the sequences' tokens times their sizes (one tensor of them per sequence)."""
    rows = torch.randn(pages.values.shape, generator=g, dtype=torch.float64)
    for b, (_, _, ctx) in enumerate(spans):
        at = torch.arange(ctx)
        rows[table[b, at // 32].long(), :, at % 32] *= sizes[b][:, None, None]
    fill(pages, rows)


def zeros_and_large(g, dim, large, places, device):
    """Pages of three sequences whose values are zero or large, by thirds or halves of their tokens; (pages, table, contexts)."""
    contexts = [700, 900, 64]
    table, blocks = shuffled_table(g, contexts)
    k, v = (ops.QuantizedPages.new(blocks, 1, dim, device) for _ in range(2))
    spans = [(0, 0, c) for c in contexts]
    stored_rows(g, k, table, spans, [torch.full((c,), 0.5, dtype=torch.float64) for c in contexts])
    stored_rows(g, v, table, spans, [torch.tensor(places)[torch.arange(c) * len(places) // c].double() * large for c in contexts])
    return (k, v), table, contexts


LARGE = [2.0 ** 40, 2.0 ** 60, 2.0 ** 70]
PLACES = [[0.0, 1.0], [1.0, 0.0], [0.0, 1.0, 0.0]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("places", PLACES)
def test_rows_of_zeros_count_beside_large_values(device, dim, large, places):
    """Tokens whose values are zero, and with them their scales the smallest, take their part of the denominator."""
    g = torch.Generator().manual_seed(dim)
    pages, table, contexts = zeros_and_large(g, dim, large, places, device)
    q = torch.randn((3, 2, dim), generator=g).to(torch.bfloat16)
    spans = [(b, 1, c) for b, c in enumerate(contexts)]
    for splits in (1, 4):
        out = ops.paged_attn_decode(q.view(3, -1).to(device), *pages, table.to(device), i32(contexts, device), 0.3, num_splits=splits)
        check_rows(out.view(q.shape), q, *rows_of(pages, table, spans), spans, 0.3, 2)


# ------------------------------------------------------------------------------------------------ sizes far apart within a prompt
# The 128 tokens of a tile are brought to its largest scale, which may be that of a token that a row does not see.  What that may cost a row is
# 2^-30 of its largest value for a token, as elsewhere, times 2^12 by which the tile's scale may be above what the row sees before the row
# is computed by itself.  Keys: 2^18 above, 2^-25 of f16 behind 2^6 at that scale is 2^(18 - 31) of the row's largest scale, whose largest key is 224
# or more: 2^-20.8 of it for an element.  A row's sum |q| is at most some 3.4 of sum |q k| over the largest key here (normal numbers, 64
# or 128 of them, the largest 2.7 of their deviation), so that scores are off by 2^-19 of the latter, which `moved` has.
FAR = 2.0 ** -18


FAR_SPANS = [
    # nq, nkv, spans, masks
    (4, 2, [(0, 200, 200), (200, 33, 350), (233, 1, 77)], {}),
    (1, 1, [(0, 300, 700)], dict(window=150)),
    (2, 1, [(0, 140, 300)], dict(window=50)),
    (8, 1, [(0, 5, 2100), (5, 3, 1000)], {}),                               # divided among works
    (16, 4, [(0, 9, 1200)], dict(window=700)),
    (4, 4, [(70 * i, 70, 70) for i in range(40)], {}),
    (2, 1, [(0, 150, 300)], dict(chunk=100)),
    (2, 1, [(0, 40, 300)], dict(causal=False, window=130)),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("nq,nkv,spans,masks", FAR_SPANS)
def test_prompts_with_sizes_far_apart(device, dim, sinks, nq, nkv, spans, masks):
    """Values of 2^-40 to 2^40 and keys of 2^-30 to 1 beside one another, some tokens zero."""
    g = torch.Generator().manual_seed(dim + nq + len(spans))
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    k, v = (ops.QuantizedPages.new(blocks, nkv, dim, device) for _ in range(2))
    sizes = lambda lo, hi: [2.0 ** torch.randint(lo, hi + 1, (c,), generator=g).double() * (torch.rand((c,), generator=g) > 0.1)       # noqa: E731
                            for _, _, c in spans]
    stored_rows(g, k, table, spans, sizes(-30, 0))
    stored_rows(g, v, table, spans, sizes(-40, 40))
    q = torch.randn((sum(n for _, n, _ in spans), nq, dim), generator=g).to(torch.bfloat16)
    s = torch.randn((nq,), generator=g) if sinks else None
    out = prompt(q, (k, v), table, spans, dim ** -0.5, device, **masks, **({"sinks": s} if sinks else {}))
    check_rows(out, q, *rows_of((k, v), table, spans), spans, dim ** -0.5, nq // nkv, s, **masks, lost=FAR)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", ["keys", "values", "both"])
@pytest.mark.parametrize("up", [2.0 ** 9, 2.0 ** 13, 2.0 ** 19, 2.0 ** 30, 2.0 ** 60])
def test_large_tokens_beside_what_a_row_sees(device, dim, what, up):
    """Tokens that are far larger than the others: rows ahead of them, and behind the window that shows them, do not notice."""
    g = torch.Generator().manual_seed(dim)
    nq, nkv = 4, 2
    spans, masks = [(0, 290, 290), (290, 100, 600), (390, 1, 129)], dict(window=200)
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    k, v = pool(g, blocks, nkv, dim, device)
    q = torch.randn((391, nq, dim), generator=g).to(torch.bfloat16)
    plain = rows_of((k, v), table, spans)
    want = [[attend(q[r:r + n, h].double(), ks[:, h // 2], vs[:, h // 2], 0.1, c - n, lost=FAR, **masks) for h in range(nq)]
            for (r, n, c), ks, vs in zip(spans, *plain)]
    large = [[200, 255, 256], [310, 599], [128]]                             # positions
    for pages, name in ((k, "keys"), (v, "values")):
        if what in (name, "both"):
            scales = pages.scales.view(torch.uint8).cpu()
            for b, at in enumerate(large):
                for j in at:
                    scales[table[b, j // 32], :, j % 32] += int(math.log2(up))
            pages.scales.view(torch.uint8).copy_(scales.clamp(max=190))
    out = prompt(q, (k, v), table, spans, 0.1, device, **masks).cpu().double()
    check = 0
    for b, (r, n, c) in enumerate(spans):
        pos = c - n + torch.arange(n)
        free = torch.ones(n, dtype=torch.bool)
        for j in large[b]:
            free &= (pos < j) | (pos >= j + 200)
        check += int(free.sum())
        for h in range(nq):
            o, tol = want[b][h]
            assert bool(((out[r:r + n, h] - o).abs() <= tol)[free].all()), (b, h)
    assert check == 289


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("places", PLACES)
@pytest.mark.parametrize("new", [[3, 150, 5], [3, 4, 5]])                   # the second: divided among works
def test_rows_of_zeros_count_beside_large_values_of_prompts(device, dim, large, places, new):
    g = torch.Generator().manual_seed(dim)
    pages, table, contexts = zeros_and_large(g, dim, large, places, device)
    spans = [(sum(new[:b]), n, c) for b, (n, c) in enumerate(zip(new, contexts))]
    q = torch.randn((sum(new), 2, dim), generator=g).to(torch.bfloat16)
    check_rows(prompt(q, pages, table, spans, 0.3, device), q, *rows_of(pages, table, spans), spans, 0.3, 2, lost=FAR)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spans,masks", [([(0, 200, 500), (200, 30, 90), (230, 9, 7)], {}), ([(0, 4, 1500), (4, 5, 700)], dict(window=300))])
def test_sizes_far_apart_beside_what_is_lost(device, dim, spans, masks):
    """Tokens that stand for NaN, blocks outside the pool, contexts shorter than the new tokens, rows behind the last sequence."""
    g = torch.Generator().manual_seed(dim)
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    k, v = (ops.QuantizedPages.new(blocks, 1, dim, device) for _ in range(2))
    for pages, up in ((k, 20), (v, 40)):
        stored_rows(g, pages, table, spans, [2.0 ** torch.randint(-up, 1, (c,), generator=g).double() for _, _, c in spans])
        lost = torch.rand((blocks, 1, 32), generator=g) < 0.004
        raw = pages.scales.view(torch.uint8).cpu().masked_fill(lost, 255)
        pages.scales.view(torch.uint8).copy_(raw)
        values = pages.values.view(torch.uint8).cpu().masked_fill(lost[..., None], 0)
        pages.values.view(torch.uint8).copy_(values)
    table[0, 2], table[1, -1] = -1, blocks + 5
    total = sum(n for _, n, _ in spans)
    q = torch.randn((total + 2, 2, dim), generator=g).to(torch.bfloat16)
    out = torch.full((total + 2, 2 * dim), 7.0, dtype=torch.bfloat16, device=device)
    got = prompt(q, (k, v), table, spans, 0.2, device, out=out, **masks)
    check_rows(got, q, *rows_of((k, v), table, spans), spans, 0.2, 2, **masks, lost=FAR)
    assert bool((out[total:] == 7.0).all())


# ------------------------------------------------------------------------------------------------ sinks
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
def test_sinks_of_minus_infinity_are_none(device, dim):
    """Also where a row sees nothing: its result is zero."""
    g = torch.Generator().manual_seed(dim)
    nq, contexts = 4, [40, 0, 700, -1, 3]
    table, blocks = shuffled_table(g, contexts)
    pages = pool(g, blocks, 2, dim, device)
    sinks = torch.tensor([-math.inf, 0.5, -math.inf, torch.finfo(torch.float32).min])
    q = torch.randn((5, nq, dim), generator=g).to(torch.bfloat16)
    spans = [(b, 1, max(c, 0)) for b, c in enumerate(contexts)]
    lens, some = i32(contexts, device), sinks.to(device)
    for splits in (1, 4):
        out = ops.paged_attn_decode(q.view(5, -1).to(device), *pages, table.to(device), lens, 0.3, sinks=some, num_splits=splits)
        check_rows(out.view(q.shape), q, *rows_of(pages, table, spans), spans, 0.3, 2, sinks)
    spans = [(0, 3, 40), (3, 9, 4), (12, 5, 0), (17, 2, 900)]
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    pages = pool(g, blocks, 2, dim, device)
    q = torch.randn((19, nq, dim), generator=g).to(torch.bfloat16)
    for window in (0, 2):
        out = prompt(q, pages, table, spans, 0.3, device, sinks=sinks, window=window)
        check_rows(out, q, *rows_of(pages, table, spans), spans, 0.3, 2, sinks, window=window)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spans,lost", [([(0, 100, 100), (100, 33, 33)], [1, 0]), ([(0, 5, 1500), (5, 3, 700)], [46, 3])])
def test_blocks_outside_the_pool_beside_small_rows(device, dim, spans, lost):
    """Zeros that stand for such a block have no say in the scale of the tile that it is in."""
    g = torch.Generator().manual_seed(dim)
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    pages = [ops.QuantizedPages.new(blocks, 1, dim, device) for _ in range(2)]
    for p in pages:
        stored_rows(g, p, table, spans, [torch.full((c,), 2.0 ** -40, dtype=torch.float64) for _, _, c in spans])
    table[0, lost[0]], table[1, lost[1]] = -1, blocks + 5
    q = (torch.randn((sum(n for _, n, _ in spans), 2, dim), generator=g) * 2.0 ** 37).to(torch.bfloat16)
    check_rows(prompt(q, pages, table, spans, 0.3, device), q, *rows_of(pages, table, spans), spans, 0.3, 2)
    lens, last = i32([c for _, _, c in spans], device), torch.stack([q[r + n - 1] for r, n, _ in spans])
    out = ops.paged_attn_decode(last.reshape(2, -1).to(device), *pages, table.to(device), lens, 0.3)
    check_rows(out.view(last.shape), last, *rows_of(pages, table, spans), [(b, 1, c) for b, (_, _, c) in enumerate(spans)], 0.3, 2)


# ------------------------------------------------------------------------------------------------ results in the place of queries
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("spans,q_len", [([(0, 200, 260), (200, 40, 40)], 0), ([(0, 4, 1500), (4, 4, 700)], 4)])
def test_results_in_the_place_of_queries(device, spans, q_len):
    g = torch.Generator().manual_seed(len(spans))
    nq, nkv, dim = 8, 1, 64
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    k, v = (ops.QuantizedPages.new(blocks, nkv, dim, device) for _ in range(2))
    stored_rows(g, k, table, spans, [2.0 ** torch.randint(-30, 1, (c,), generator=g).double() for _, _, c in spans])
    stored_rows(g, v, table, spans, [2.0 ** torch.randint(-40, 41, (c,), generator=g).double() for _, _, c in spans])
    q = torch.randn((sum(n for _, n, _ in spans), nq, dim), generator=g).to(torch.bfloat16)
    both = q.reshape(q.shape[0], -1).to(device).clone()
    want = prompt(q, (k, v), table, spans, 0.125, device)
    lens = i32([c for _, _, c in spans], device)
    if q_len:                                                               # decode of more than sixteen rows goes the prompts' way
        ops.paged_attn_decode(both, k, v, table.to(device), lens, 0.125, q_len=q_len, out=both)
    else:
        ops.flash_attn_prefill(both, k, v, table.to(device), *(i32([s[j] for s in spans], device) for j in (0, 1)), lens, 0.125,
                               max_q_len=max(n for _, n, _ in spans), out=both)
    assert torch.equal(both.view(q.shape), want)
    check_rows(both.view(q.shape), q, *rows_of((k, v), table, spans), spans, 0.125, nq, lost=FAR)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spans,masks,mods", [
    ([(0, 700, 900)], dict(chunk=512), dict(softcap=20.0)), ([(0, 900, 900), (900, 200, 1300)], dict(chunk=700), dict(softcap=20.0)),
    ([(0, 600, 1100)], dict(window=300), dict(softcap=20.0, keep_first=70)), ([(0, 400, 900)], dict(window=64), dict(keep_first=130)),
    ([(0, 500, 500)], dict(window=128), dict(softcap=20.0))])
def test_modified_scores_over_16_bit_pages_with_masks_that_part_query_tiles(device, dim, spans, masks, mods):
    """Capped scores and kept first tokens take turns by key tiles of 64, the kept ones ahead (see test_query_turns.py)."""
    g = torch.Generator().manual_seed(dim)
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    pages = [torch.randn((blocks, 1, 32, dim), generator=g).to(torch.bfloat16) for _ in range(2)]
    k, v = ([p[table[b, :-(-c // 32)].long()].transpose(1, 2).reshape(-1, 1, dim)[:c] for b, (_, _, c) in enumerate(spans)] for p in pages)
    q = torch.randn((sum(n for _, n, _ in spans), 2, dim), generator=g).to(torch.bfloat16)
    out = prompt(q, [p.to(device) for p in pages], table, spans, dim ** -0.5, device, mods=ops.ScoreMods(**mods), **masks)
    # (a capped score comes from a polynomial or an exponential of the special-function unit: 2^-19 of the cap, as weights have it)
    check_rows(out, q, k, v, spans, dim ** -0.5, 2, weights=2.0 ** -8 + 2.0 ** -19 * mods.get("softcap", 0.0), **masks, **mods)


# ------------------------------------------------------------------------------------------------ norms of rows of any size
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("T,splits", [(3, 0), (3, 2), (70, 0), (200, 0), (200, 3)])
@pytest.mark.parametrize("eps", [1e-6, 1e-60])
def test_norms_of_rows_whose_squares_leave_32_bits(device, dim, T, splits, eps):
    """Queries and keys of 1e-25 to 1e25, however many tokens a call has."""
    g = torch.Generator().manual_seed(dim + T)
    nq, nkv, size = 3, 1, 10.0 ** torch.tensor([-25.0, 0.0, 18.0, 25.0])
    x = torch.randn((T, nq + 2 * nkv, dim), generator=g) * size[torch.randint(0, 4, (T, nq + 2 * nkv, 1), generator=g)]
    x = torch.stack([x * 0.25 for _ in range(splits)]) if splits else x.to(torch.bfloat16)
    w = [(1 + 0.3 * torch.randn((dim,), generator=g)).to(torch.bfloat16) for _ in range(2)]
    cs, pos = rope_table(dim, 300), torch.arange(T, dtype=torch.int32)
    k, v = (ops.QuantizedPages.new(-(-T // 32), nkv, dim, device) for _ in range(2))
    q = ops.rope_kv_append(x.reshape(*x.shape[:-2], -1).to(device), pos.to(device), pos.to(device), cs.to(device), k, v, nq, nkv, dim,
                           q_norm_w=w[0].to(device), k_norm_w=w[1].to(device), norm_eps=eps).cpu().double().view(T, nq, dim)
    y = x.double().sum(0) if splits else x.double()
    want = oracle_turn(y[:, :nq], cs[:T], w[0], eps)
    # rounded to bf16; a dozen roundings of 32 bits of at most twice the head's largest
    assert bool(((q - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)).all())
    values, scales = oracle_quantize(oracle_turn(y[:, nq:nq + nkv], cs[:T], w[1], eps))
    got, s = stored(k)
    assert torch.equal(got[pos.long() // 32, :, pos.long() % 32], values) and torch.equal(s[pos.long() // 32, :, pos.long() % 32], scales)


@pytest.mark.gpu
@pytest.mark.parametrize("spans", [[(0, 150, 250), (150, 90, 90)], [(0, 4, 1500), (4, 5, 700)]])
def test_rows_computed_once_more_beside_other_calls(spans):
    """Captured, replayed beside eager calls on another stream, and after other prompts: the same bits."""
    g = torch.Generator().manual_seed(7)
    table, blocks = shuffled_table(g, [c for _, _, c in spans])
    works = []
    for _ in range(2):
        k, v = (ops.QuantizedPages.new(blocks, 2, 128, "cuda") for _ in range(2))
        stored_rows(g, k, table, spans, [2.0 ** torch.randint(-30, 1, (c,), generator=g).double() for _, _, c in spans])
        stored_rows(g, v, table, spans, [2.0 ** torch.randint(-40, 41, (c,), generator=g).double() for _, _, c in spans])
        q = torch.randn((sum(n for _, n, _ in spans), 4 * 128), generator=g).to(torch.bfloat16).cuda()
        at = [i32([s[j] for s in spans], "cuda") for j in (0, 1, 2)]
        works.append(lambda q=q, k=k, v=v, t=table.cuda(), at=at: ops.flash_attn_prefill(q, k, v, t, *at, 0.1, max_q_len=max(s[1] for s in spans)))
    want = [w().clone() for w in works]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = works[0]()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            graph.replay()
            got[0].append(out.clone())
        with torch.cuda.stream(streams[1]):
            got[1].append(works[1]().clone())
    torch.cuda.synchronize()
    assert all(torch.equal(a, w) for outs, w in zip(got, want) for a in outs)
