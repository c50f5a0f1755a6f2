"""Micro-benchmark cases of keys and values in 8 bits, at the shapes of `attn-decode` and `attn-prefill`."""
from __future__ import annotations

import torch

from . import QuantizedPages, flash_attn_prefill, paged_attn_decode, rope_attn_decode, rope_kv_append
from .quantized_kv import PAGE, quantize_rows

NQ, NKV, D = 32, 8, 128
TOKEN = 2 * NKV * (D + 1)                # bytes of a token's keys and values


def _result(name, args, timer, fns, bytes, flops, **shape):
    return dict(case=name, us=timer(fns, args.iters, args.warmup, not args.no_graph), bytes=bytes, flops=flops, shape=shape)


def _rows(*shape):
    return torch.randn(*shape, device="cuda").to(torch.bfloat16)


def _pools(blocks, sets):
    """Pages of normal values."""
    pages = lambda: QuantizedPages(*quantize_rows(torch.randn(blocks, NKV, PAGE, D, device="cuda")))       # noqa: E731
    return [(pages(), pages()) for _ in range(sets)]


def _batch(B, ctx):
    pages = -(-ctx // PAGE)
    return torch.arange(B * pages, device="cuda", dtype=torch.int32).reshape(B, pages), torch.full((B,), ctx, device="cuda", dtype=torch.int32)


def append(tokens):
    def case(args, timer, sets_for):
        W, blocks = (NQ + 2 * NKV) * D, -(-tokens // PAGE)
        bytes = tokens * (W * 2 + NQ * D * 2 + TOKEN + 8)
        sets = sets_for(bytes, args.sets)
        qkv, cs = [_rows(tokens, W) for _ in range(sets)], torch.randn(tokens, D, device="cuda")
        at = torch.arange(tokens, device="cuda", dtype=torch.int32)
        fns = [lambda x=x, kv=kv: rope_kv_append(x, at, at, cs, *kv, NQ, NKV, D) for x, kv in zip(qkv, _pools(blocks, sets))]
        return _result(f"quantized-append-{tokens}", args, timer, fns, bytes, 0.0, tokens=tokens, nq=NQ, nkv=NKV, head_dim=D, sets=sets)
    return case


def attn_decode(args, timer, sets_for):
    B, ctx = 64, 1056
    table, lens = _batch(B, ctx)
    sets = sets_for(B * ctx * TOKEN, args.sets)
    q = _rows(B, NQ * D)
    fns = [lambda kv=kv: paged_attn_decode(q, *kv, table, lens, D ** -0.5, num_splits=args.kv_splits) for kv in _pools(table.numel(), sets)]
    return _result("quantized-attn-decode", args, timer, fns, B * ctx * TOKEN + 4 * q.numel(), 4.0 * B * NQ * ctx * D, batch=B, context=ctx,
                   nq=NQ, nkv=NKV, head_dim=D, sets=sets, kv_splits=args.kv_splits)


def step(args, timer, sets_for):
    B, ctx, parts = 64, 1056, 4
    table, lens = _batch(B, ctx)
    sets = sets_for(B * ctx * TOKEN, args.sets)
    W = (NQ + 2 * NKV) * D
    qkv, cs = torch.randn(parts, B, W, device="cuda"), torch.randn(ctx, D, device="cuda")
    pos, slots = lens - 1, table[:, -1].contiguous() * PAGE + (ctx - 1) % PAGE
    fns = [lambda kv=kv: rope_attn_decode(qkv, pos, slots, cs, *kv, table, lens, D ** -0.5, NQ, NKV) for kv in _pools(table.numel(), sets)]
    return _result("quantized-step", args, timer, fns, B * ctx * TOKEN + 4 * qkv.numel() + 2 * B * NQ * D, 4.0 * B * NQ * ctx * D, batch=B,
                   context=ctx, nq=NQ, nkv=NKV, head_dim=D, partials=parts, sets=sets, launches_per_call=2)


def attn_prefill(args, timer, sets_for):
    B, S = args.batch or 8, args.seq or 2048
    table, lens = _batch(B, S)
    sets = sets_for(B * S * TOKEN, args.sets)
    q, starts = _rows(B * S, NQ * D), torch.arange(B, device="cuda", dtype=torch.int32) * S
    fns = [lambda kv=kv: flash_attn_prefill(q, *kv, table, starts, lens, lens, D ** -0.5, max_q_len=S) for kv in _pools(table.numel(), sets)]
    return _result("quantized-attn-prefill", args, timer, fns, B * S * TOKEN + 4 * q.numel(), 2.0 * B * NQ * S * S * D, batch=B, seq=S, nq=NQ,
                   nkv=NKV, head_dim=D, causal=True, sets=sets)


CASES = {"quantized-append-64": append(64), "quantized-append-16384": append(16384), "quantized-attn-decode": attn_decode,
         "quantized-step": step, "quantized-attn-prefill": attn_prefill}
