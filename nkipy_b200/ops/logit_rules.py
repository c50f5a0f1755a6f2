"""Rules on logits ahead of the choice of a token: penalties for repeated tokens, biases and masks.

They are reached through `apply_rules`, which gives the logits that are left, and `argmax` with rules, which chooses the most likely token
without writing them.  A row's tokens are its state: the list of ids that a scheduler keeps anyway, into which a call writes the
newest.  No file of the reference corresponds to these (it decodes greedily, examples/models/qwen3/kernels/sampling.py:113-147).
"""

from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from . import _count_launch, _stream
from .quantized_linear import _on_gpu, to_bf16

_ARGS = struct.Struct("15P5q6i")          # NkbLogitRules of csrc/kernels/rules_args.h


@dataclass(slots=True)
class LogitRules:
    """What is done to the logits [rows, vocab] of a step, in 64 bits and rounded once (`apply_rules` to their type, `argmax` to fp32), in this order:

    tokens int32 [rows, width], lens int32 [rows]: the ids of every row so far, the newest included (lens beyond the width count as the
        width; a length below one: no tokens).  ids int32 [rows]: the newest, which the call writes to tokens[b, lens[b] - 1]; None: it
        is there already.  prompt_lens int32 [rows]: how many of them are the prompt's; None: none.  Ids outside the vocabulary count for
        nothing.
    repetition fp32 [rows], above zero: a token that is among the row's is divided by it where its logit is above zero, and multiplied
        elsewhere.
    frequency, presence fp32 [rows]: taken off a token that is among the answer's, as often as it is there, and once.
    bias_ids int32 [rows, n], bias_values fp32 [rows, n]: added to single tokens; several for one token add up.  Negative ids: none.
    mask int32 [masks, words]: bit t % 32 of word t // 32 says whether token t may come (zero: its logit becomes minus infinity).
        mask_rows int32 [rows]: a row's mask, outside of them: none; None: row b has mask b.

    All on the logits' device.  Rows of the matrices may lie apart; the vectors are contiguous."""
    tokens: Optional[torch.Tensor] = None
    lens: Optional[torch.Tensor] = None
    prompt_lens: Optional[torch.Tensor] = None
    ids: Optional[torch.Tensor] = None
    repetition: Optional[torch.Tensor] = None
    frequency: Optional[torch.Tensor] = None
    presence: Optional[torch.Tensor] = None
    bias_ids: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    mask: Optional[torch.Tensor] = None
    mask_rows: Optional[torch.Tensor] = None


def mask_words(vocab: int) -> int:
    """Words of a mask."""
    return -(-vocab // 32)


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool [masks, vocab] (or [vocab]) as the words of `LogitRules.mask`."""
    vocab = allowed.shape[-1]
    bits = torch.zeros((*allowed.shape[:-1], mask_words(vocab) * 32), dtype=torch.int64, device=allowed.device)
    bits[..., :vocab] = allowed
    words = (bits.unflatten(-1, (-1, 32)) << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _vector(t, name, dtype, shape, index):
    if t is None:
        return 0
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{name} wants {dtype}, not {t.dtype}")
    raise ValueError(f"{name} wants to be contiguous {list(shape)}, on the logits' device")


def _matrix(t, name, dtype, rows, index):
    """(address, elements from one row to the next); rows None: any number."""
    if t is None:
        return 0, 0
    if t.dtype is not dtype:
        raise TypeError(f"{name} wants {dtype}, not {t.dtype}")
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or t.get_device() != index:
        raise ValueError(f"{name} wants rows of neighbouring numbers, one for each of the logits', on their device")
    ld, column = t.stride()
    if column != 1 and shape[1] > 1:
        raise ValueError(f"{name} wants rows of neighbouring numbers, one for each of the logits', on their device")
    return t.data_ptr(), ld


def _packed(logits, rules: LogitRules, out, out_ids) -> bytes:
    if not isinstance(rules, LogitRules):
        raise TypeError("rules are LogitRules")
    f32 = logits.dtype is torch.float32
    if not f32 and logits.dtype is not torch.bfloat16:
        raise TypeError(f"rules want bf16 or fp32 logits, not {logits.dtype}")
    shape = logits.shape
    if len(shape) != 2 or shape[1] < 1 or shape[0] > 65535:
        raise ValueError("rules want logits [rows, vocab], of 65535 rows at most, with neighbouring columns")
    (B, V), (ld, column), at, index, r, rows = shape, logits.stride(), logits.data_ptr(), logits.get_device(), rules, shape[:1]
    if column != 1 and V > 1:
        raise ValueError("rules want logits [rows, vocab], of 65535 rows at most, with neighbouring columns")
    out_at, out_ld = _matrix(out, "out", logits.dtype, B, index)
    if out is not None:
        if out.shape != shape or (B > 1 and out_ld < V):
            raise ValueError("out wants the logits' shape")
        if out_at == at and B > 1 and out_ld != ld:
            raise ValueError("rows of out that lie over the logits want to be the same ones")
    i32, number = torch.int32, torch.float32
    tokens = tokens_ld = width = lens = prompts = ids = rep = freq = pres = bias_ids = bias_values = bias_ld = biases = mask = mask_ld = masks = 0
    mask_rows = 0
    if r.tokens is not None:
        if r.lens is None:
            raise ValueError("tokens want lens")
        tokens, tokens_ld = _matrix(r.tokens, "tokens", i32, B, index)
        width = r.tokens.shape[1]
        lens, prompts = _vector(r.lens, "lens", i32, rows, index), _vector(r.prompt_lens, "prompt_lens", i32, rows, index)
        ids = _vector(r.ids, "ids", i32, rows, index)
        if ids and B > 1 and tokens_ld < width:
            raise ValueError("rows of tokens that ids are written to want memory of their own")
        rep = _vector(r.repetition, "repetition", number, rows, index)
        freq, pres = _vector(r.frequency, "frequency", number, rows, index), _vector(r.presence, "presence", number, rows, index)
    elif r.lens is not None or r.ids is not None or r.prompt_lens is not None:
        raise ValueError("lens, prompt_lens and ids belong to tokens")
    elif r.repetition is not None or r.frequency is not None or r.presence is not None:
        raise ValueError("penalties want the rows' tokens")
    if r.bias_ids is not None or r.bias_values is not None:
        if r.bias_ids is None or r.bias_values is None:
            raise ValueError("biases want ids and values")
        (bias_ids, bias_ld), (bias_values, values_ld) = (_matrix(r.bias_ids, "bias_ids", i32, B, index),
                                                         _matrix(r.bias_values, "bias_values", number, B, index))
        if r.bias_ids.shape != r.bias_values.shape or (B > 1 and bias_ld != values_ld):
            raise ValueError("biases want as many values as ids, laid out the same")
        biases = r.bias_ids.shape[1]
    if r.mask is not None:
        mask, mask_ld = _matrix(r.mask, "mask", i32, None if r.mask_rows is not None else B, index)
        masks, words = r.mask.shape
        if words < mask_words(V):
            raise ValueError(f"mask wants {mask_words(V)} words for a vocabulary of {V}")
        mask_rows = _vector(r.mask_rows, "mask_rows", i32, rows, index)
    elif r.mask_rows is not None:
        raise ValueError("mask_rows belong to masks")
    return _ARGS.pack(at, out_at, _vector(out_ids, "out_ids", i32, rows, index), tokens, lens, prompts, ids, rep, freq, pres, bias_ids,
                      bias_values, mask, mask_rows, _stream() if index >= 0 else 0, ld, out_ld, tokens_ld, bias_ld, mask_ld, B, V, width,
                      biases, masks, f32)


def _reference(logits, r: LogitRules) -> torch.Tensor:
    """Logits under the rules in 64 bits; writes the newest tokens."""
    y = logits.double().clone()
    B, V = y.shape
    for b in range(B):
        row = y[b]
        if r.tokens is not None:
            n = min(int(r.lens[b]), r.tokens.shape[1])
            if n > 0:
                if r.ids is not None:
                    r.tokens[b, n - 1] = r.ids[b]
                ids = r.tokens[b, :n].long()
                inside = (ids >= 0) & (ids < V)
                seen = torch.bincount(ids[inside], minlength=V) > 0
                answer = torch.arange(n) >= (int(r.prompt_lens[b]) if r.prompt_lens is not None else 0)
                times = torch.bincount(ids[inside & answer], minlength=V).double()
                rep, freq, pres = (d if t is None else float(t[b]) for t, d in ((r.repetition, 1.0), (r.frequency, 0.0), (r.presence, 0.0)))
                hit = row[seen]
                hit = torch.where(hit > 0, hit / rep, hit * rep) - freq * times[seen]
                row[seen] = torch.where(times[seen] > 0, hit - pres, hit)
        if r.bias_ids is not None:
            total = {}
            for t, v in zip(r.bias_ids[b].tolist(), r.bias_values[b].double().tolist()):
                if 0 <= t < V:
                    total[t] = total.get(t, 0.0) + v
            for t, v in total.items():
                row[t] += v
        m = -1 if r.mask is None else (b if r.mask_rows is None else int(r.mask_rows[b]))
        if r.mask is not None and 0 <= m < r.mask.shape[0]:
            t = torch.arange(V)
            row[((r.mask[m][t // 32] >> (t % 32)) & 1) == 0] = float("-inf")
    return y


def apply_rules(logits: torch.Tensor, rules: LogitRules, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits [rows, vocab] (bf16 or fp32) under the rules, in their type.  out: where they go; the logits themselves, whose
    untouched pieces are not even read then, or apart from them."""
    if out is None:
        out = torch.empty_strided(logits.shape, (logits.shape[-1], 1), dtype=logits.dtype, device=logits.device) if logits.dim() == 2 else logits
    args = _packed(logits, rules, out, None)
    if not logits.shape[0]:
        return out
    if not _on_gpu(logits.get_device()):
        y = _reference(logits, rules)
        return out.copy_(to_bf16(y) if out.dtype is torch.bfloat16 else y)
    rc = _lib.lib().nkb_logit_rules(args)
    if rc:
        _lib.check(rc, "nkb_logit_rules")
    _count_launch()
    return out


def argmax(logits: torch.Tensor, rules: LogitRules, out_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 [rows]: the first of the largest values that the rules leave, as 32 bits hold them; -1 where none is above minus infinity."""
    if out_ids is None:
        out_ids = torch.empty_strided((logits.shape[0],), (1,), dtype=torch.int32, device=logits.device)
    args = _packed(logits, rules, None, out_ids)
    if not logits.shape[0]:
        return out_ids
    if not _on_gpu(logits.get_device()):
        y = _reference(logits, rules).float().nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
        top, at = y.max(-1)
        first = torch.where(y == top[:, None], torch.arange(y.shape[1]), y.shape[1]).amin(-1)
        return out_ids.copy_(torch.where(top == float("-inf"), -1, first))
    rc = _lib.lib().nkb_logit_rules(args)
    if rc:
        _lib.check(rc, "nkb_logit_rules")
    _count_launch()
    return out_ids
