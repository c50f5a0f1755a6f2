"""Keys and values kept in 8 bits: the pages, and the operators that write and read them.

A page of 32 tokens of one kv head is e4m3 values ``[32, dim]`` and one power of two per token.  A head's row x is kept as
``e4m3(x / 2^e)`` (nearest, ties to even) and e, the smallest whole number with ``max|x| <= 448 * 2^e``, between -64 and 64: rows
beyond 448 * 2^64 saturate, and what is below 2^-74 becomes zero.  A row that holds a value which is not finite stands for NaN as a whole
(scale NaN, values 0), so that a NaN in a masked place has no way into a sum.  Scale bytes that no row has stand for the nearest that
one may have.  What no query of a call sees, behind a context or before a window, may be any bytes; what one of them sees has no e4m3
NaN among its values.

One scale per token and head, because tokens are appended one at a time: a scale that several tokens shared would have to be
guessed, or change what is stored already.  A power of two, because e4m3 is a floating type: another factor would keep no more
bits, and this one is undone without a rounding.

The values are rounded once, from sums, norms and rotations in 64 bits, so that a token has the same bytes whichever kernel, or the
reference on the CPU, writes them.

These functions are reached through `rope_kv_append`, `paged_attn_decode`, `rope_attn_decode`, `flash_attn_prefill` and
`packed_attention`, which take a `QuantizedPages` wherever they take a cache tensor.  No file of the reference corresponds to
them (its cache is dense and bf16, examples/models/qwen3/qwen3.py:52-71).
"""

from __future__ import annotations

import functools
import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib

PAGE = 32
LOG2_MIN, LOG2_MAX = -64, 64
DIMS = (64, 128)


class QuantizedPages:
    """Keys or values of one layer: e4m3 `values` [blocks, kv heads, 32, dim] and power-of-two `scales` [blocks, kv heads, 32]
    (torch.float8_e8m0fnu), both contiguous and on one device."""
    __slots__ = ("values", "scales", "shape", "device", "index", "at")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype is not torch.float8_e4m3fn or scales.dtype is not torch.float8_e8m0fnu:
            raise TypeError("QuantizedPages wants float8_e4m3fn values and float8_e8m0fnu scales")
        shape = values.shape
        if len(shape) != 4:
            raise ValueError("QuantizedPages wants values [blocks, kv heads, 32, dim]")
        blocks, heads, page, dim = shape
        if page != PAGE or scales.shape != (blocks, heads, PAGE):
            raise ValueError("QuantizedPages wants values [blocks, kv heads, 32, dim] and scales [blocks, kv heads, 32]")
        if dim not in DIMS:
            raise ValueError("QuantizedPages has heads of 64 or 128 columns")
        index = values.get_device()
        if not values.is_contiguous() or not scales.is_contiguous() or scales.get_device() != index:
            raise ValueError("QuantizedPages wants contiguous tensors on one device")
        self.at = v, s = values.data_ptr(), scales.data_ptr()
        if (v | s) & 15 or not v:
            raise ValueError("QuantizedPages wants tensors that start on 16 bytes, of a block and a head at least")
        # shape as of a cache tensor; index: of the CUDA device, -1: the CPU; at: where the tensors start
        self.values, self.scales, self.shape, self.index, self.device = values, scales, shape, index, values.device

    @property
    def is_cuda(self) -> bool:
        return self.index >= 0

    @classmethod
    def new(cls, num_blocks: int, kv_heads: int, dim: int, device="cpu") -> "QuantizedPages":
        """Pages of zeros."""
        values = torch.zeros((num_blocks, kv_heads, PAGE, dim), dtype=torch.uint8, device=device)
        scales = torch.full((num_blocks, kv_heads, PAGE), 127, dtype=torch.uint8, device=device)
        return cls(values.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.scales.numel()

    def dequantize(self, blocks: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values that the pages (of the given blocks) stand for, fp32 [blocks, kv heads, 32, dim]."""
        v, s = self.values.view(torch.uint8), self.scales.view(torch.uint8)
        if blocks is not None:
            v, s = v[blocks], s[blocks]
        s = torch.where(s == 255, s, s.clamp(127 + LOG2_MIN, 127 + LOG2_MAX))
        return v.view(torch.float8_e4m3fn).float() * s.view(torch.float8_e8m0fnu).float()[..., None]


# --------------------------------------------------------------------------- reference on the CPU
def _pow2(e: torch.Tensor) -> torch.Tensor:
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values, scales) of rows [..., dim], computed in 64 bits."""
    x = x.double()
    fine = x.isfinite().all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    m, e = torch.frexp(x.abs().amax(-1))                          # 448 is 0.875 * 2^9
    e = torch.where(m == 0, LOG2_MIN, e - 9 + (m > 0.875).int()).clamp(LOG2_MIN, LOG2_MAX)
    y = x * _pow2(-e)[..., None]
    step = _pow2((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    y = (torch.round(y / step) * step).clamp(-448.0, 448.0)
    scales = torch.where(fine, e + 127, 255).to(torch.uint8)
    return y.float().to(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def _ref_append(qkv, positions, slots, cos_sin, k_pages, v_pages, nq, nkv, dim, bias, q_norm_w, k_norm_w, eps, q_out):
    T = qkv.shape[-2]
    x = qkv.double()
    x = x.reshape(-1, T, x.shape[-1]).sum(0) if qkv.dtype == torch.float32 else x
    if bias is not None:
        x = x + bias.double()
    x = x.reshape(T, nq + 2 * nkv, dim)

    def turn(t, w):
        if w is not None:
            t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w.to(t.dtype)
        if cos_sin is not None:
            cs = cos_sin[positions.long().clamp(0, cos_sin.shape[0] - 1)].to(t.dtype)[:, None]
            h = dim // 2
            t = torch.cat([t[..., :h] * cs[..., :h] - t[..., h:] * cs[..., h:], t[..., h:] * cs[..., :h] + t[..., :h] * cs[..., h:]], -1)
        return t

    q_out.copy_(turn(x[:, :nq], q_norm_w).reshape(q_out.shape))
    if slots is not None:
        at = slots.long()
        on = (at >= 0) & (at < k_pages.shape[0] * PAGE)
        at = at[on]
        for pages, rows in ((k_pages, turn(x[:, nq:nq + nkv], k_norm_w)), (v_pages, x[:, nq + nkv:])):
            values, scales = quantize_rows(rows[on])
            pages.values.view(torch.uint8)[at // PAGE, :, at % PAGE] = values.view(torch.uint8)
            pages.scales.view(torch.uint8)[at // PAGE, :, at % PAGE] = scales.view(torch.uint8)
    return q_out


def _ref_rows(pages: QuantizedPages, table_row: torch.Tensor, ctx: int) -> torch.Tensor:
    """[ctx, kv heads, dim] of one sequence; blocks outside the pool read as zeros."""
    blocks = table_row[:(ctx + PAGE - 1) // PAGE].long()
    inside = (blocks >= 0) & (blocks < pages.shape[0])
    x = pages.dequantize(torch.where(inside, blocks, 0)).masked_fill(~inside[:, None, None, None], 0.0)
    return x.permute(0, 2, 1, 3).reshape(-1, pages.shape[1], pages.shape[3])[:ctx]


def _ref_attend(q, k_pages, v_pages, table_row, ctx, scale, pos0, causal, window, chunk, sinks):
    """q [n, nq, dim] fp32 at positions pos0, pos0 + 1, ... of one sequence -> the same shape."""
    n, nq, dim = q.shape
    if ctx <= 0:
        return torch.zeros_like(q)
    k, v = _ref_rows(k_pages, table_row, ctx), _ref_rows(v_pages, table_row, ctx)
    group = nq // k.shape[1]
    lost = v.isnan().any(-1)
    s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(group, 1)) * scale
    s = s.masked_fill(lost.T.repeat_interleave(group, 0)[:, None], float("nan"))
    at, pos = torch.arange(ctx), pos0 + torch.arange(n)[:, None]
    seen = at <= pos if causal else torch.ones((n, ctx), dtype=torch.bool)
    if window > 0:
        seen = seen & (at > pos - window)
    if chunk > 0:
        seen = seen & (at >= pos - pos % chunk)
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks.float()[:, None, None])
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks.float()[:, None, None] - top)
    o = torch.einsum("hqk,khd->hqd", p, v.masked_fill(lost[..., None], 0.0).repeat_interleave(group, 1))
    return torch.where(total == 0, 0.0, o / total).transpose(0, 1)


# --------------------------------------------------------------------------- checks of arguments
# (a call has a few microseconds on the host: each check is one line that passes, and the reason is looked for when it does not)
def _pair(k_cache, v_cache) -> Tuple[int, int, int]:
    """(blocks, kv heads, dim) of a layer's pages."""
    if type(k_cache) is not QuantizedPages or type(v_cache) is not QuantizedPages:
        raise TypeError("keys and values are both QuantizedPages, or neither is")
    if k_cache.shape != v_cache.shape or k_cache.index != v_cache.index:
        raise ValueError("keys and values want pages of one shape on one device")
    blocks, nkv, _, dim = k_cache.shape
    return blocks, nkv, dim


def _want(t: torch.Tensor, name: str, dtype, shape, index: int) -> None:
    """A contiguous tensor of this type and shape on device `index` (-1: the CPU)."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return
    if t.dtype is not dtype:
        raise TypeError(f"{name} wants {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has the shape {tuple(t.shape)}, not {tuple(shape)}")
    raise ValueError(f"{name} wants to be contiguous and on the pages' device")


def _want_rows(t: torch.Tensor, name: str, shape, index: int) -> int:
    """Address of bf16 rows that kernels read or write in pieces of sixteen bytes."""
    _want(t, name, torch.bfloat16, shape, index)
    at = t.data_ptr()
    if at & 15 and index >= 0:
        raise ValueError(f"{name} wants to start on 16 bytes")
    return at


def _on_gpu(index: int) -> bool:
    """Whether the kernels run (CUDA); they are launched on the current device's current stream."""
    if index < 0:
        return False
    if index != torch._C._cuda_getDevice():
        raise ValueError("the pages are on another device than the current one")
    if not _lib._initialised:
        _lib.ensure_init()
    return True


def _check_heads(nq: int, nkv: int) -> int:
    if nq < 1 or nkv < 1 or nq % nkv:
        raise ValueError("query heads are a multiple of the kv heads")
    return nq // nkv


def _check_table(block_table, context_lens, index: int) -> Tuple[int, int, int]:
    """(sequences, blocks of a row, entries from one row to the next)"""
    shape = block_table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError("block_table wants [sequences, blocks]")
    if block_table.dtype is not torch.int32:
        raise TypeError(f"block_table wants torch.int32, not {block_table.dtype}")
    B, width = shape
    step, column = (width, 1) if block_table.is_contiguous() else block_table.stride()
    if block_table.get_device() != index or (column != 1 and width > 1):
        raise ValueError("block_table wants neighbouring columns and to be on the pages' device")
    _want(context_lens, "context_lens", torch.int32, (B,), index)
    return B, width, step


def _check_qkv(qkv, positions, slots, cos_sin, k_cache, nq, nkv, head_dim, bias, q_norm_w, k_norm_w) -> Tuple[int, int, int, int]:
    """(tokens, partial sums, elements between them, rows of cos_sin)"""
    index, shape = k_cache.index, qkv.shape
    _check_heads(nq, nkv)
    if nkv != k_cache.shape[1] or head_dim != k_cache.shape[3]:
        raise ValueError("the pages have other kv heads than the projection")
    W = (nq + 2 * nkv) * head_dim
    parts = 1
    if len(shape) == 3 and qkv.dtype is torch.float32:
        parts = shape[0]
    elif len(shape) != 2 or qkv.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("qkv is bf16 [T, W] or fp32 partial sums [S, T, W]")
    T = shape[-2]
    if shape[-1] != W or parts < 1:
        raise ValueError(f"qkv has the shape {tuple(shape)}, not [..., {W}]")
    stride = T * W
    if not qkv.is_contiguous():                                   # partial sums may lie apart
        stride = qkv.stride(0)
        if len(shape) == 2 or qkv.stride(-1) != 1 or (T > 1 and qkv.stride(-2) != W):
            raise ValueError("qkv wants rows that follow one another")
    if qkv.get_device() != index:
        raise ValueError("qkv wants to be on the pages' device")
    rows = 0
    if cos_sin is not None:
        rows = cos_sin.shape[0]
        _want(cos_sin, "cos_sin", torch.float32, (rows, head_dim), index)
        if not rows or positions is None:
            raise ValueError("a rotation wants positions and rows of cos and sin")
    if positions is not None:
        _want(positions, "positions", torch.int32, (T,), index)
    if slots is not None:
        _want(slots, "slots", torch.int32, (T,), index)
    if bias is not None:
        _want(bias, "bias", torch.bfloat16, (W,), index)
    if q_norm_w is not None:
        _want(q_norm_w, "q_norm_w", torch.bfloat16, (head_dim,), index)
    if k_norm_w is not None:
        _want(k_norm_w, "k_norm_w", torch.bfloat16, (head_dim,), index)
    return T, parts, stride, rows


def _check_masks(mods, scale: float, window: int, chunk: int, sinks, nq: int, index: int) -> None:
    if mods:
        raise ValueError("attention over QuantizedPages takes no score modifications")
    if not math.isfinite(scale):
        raise ValueError("scale is a finite number")
    if window < 0 or chunk < 0:
        raise ValueError("window and chunk are not negative")
    if sinks is not None:
        _want(sinks, "sinks", torch.float32, (nq,), index)


def _result(out: Optional[torch.Tensor], q: torch.Tensor, index: int) -> torch.Tensor:
    """Like q."""
    if out is None:
        return torch.empty_like(q)
    _want_rows(out, "out", q.shape, index)
    return out


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _floats(scratch: Optional[torch.Tensor]) -> int:
    return 0 if scratch is None else scratch.numel()


# NkbQ8Append and NkbQ8Attn of csrc/kernels/q8_args.h: packed, a call takes a quarter of the time that as many arguments do
_APPEND, _ATTN = struct.Struct("14Pqd8i"), struct.Struct("13P2q12ifi")


MAX_SPLITS = 1024
COUNTERS = 16384                     # words of the scratch of attention that count
_SCRATCH = {}


def _scratch(device: torch.device, floats: int) -> torch.Tensor:
    """Partial results of divided sequences, behind arrival counters that are zero between calls: one per device and stream.  A graph
    that is captured gets its own, cleared whenever it runs: it may run beside other graphs, and ahead of the call that would have
    cleared a shared one."""
    if torch._C._cuda_isCurrentStreamCapturing():
        buf = torch.empty((floats,), dtype=torch.float32, device=device)
        buf[:COUNTERS].zero_()
        return buf
    key = (device.index, _stream())
    buf = _SCRATCH.get(key)
    if buf is None or buf.numel() < floats:
        buf = _SCRATCH[key] = torch.zeros((floats,), dtype=torch.float32, device=device)
    return buf


# (sizes go by the device's SMs, which the library knows once it is initialised)
@functools.lru_cache(maxsize=4096)
def _decode_floats(B: int, nkv: int, D: int, group: int, num_splits: int) -> int:
    _lib.ensure_init()
    floats = _lib.lib().nkb_q8_attn_decode_scratch_floats(B, nkv, D, group, num_splits)
    if floats < 0:
        raise _lib.KernelLibraryError(f"nkb_q8_attn_decode_scratch_floats failed with code {floats}")
    return floats


@functools.lru_cache(maxsize=4096)
def _prefill_floats(B: int, max_q_len: int, nq: int, nkv: int, D: int, width: int) -> int:
    _lib.ensure_init()
    floats = _lib.lib().nkb_q8_attn_prefill_scratch_floats(B, max_q_len, nq, nkv, D, width)
    if floats < 0:
        raise _lib.KernelLibraryError(f"nkb_q8_attn_prefill_scratch_floats failed with code {floats}")
    return floats


@functools.lru_cache(maxsize=4096)
def _prefill_launches(B: int, max_q_len: int, nq: int, nkv: int, width: int) -> int:
    """Parts of blocks are joined by a second one."""
    return _lib.lib().nkb_q8_attn_prefill_launches(B, max_q_len, nq, nkv, width)


def _pick_splits(ctas: int, max_pages: int, sms: int = 148) -> int:
    """Parts that decode attention makes of a sequence on average."""
    return 1 if ctas >= sms else max(min(sms // ctas, max(max_pages // 8, 1), 16), 1)


def _splits(num_splits: int, scratch, B: int, nkv: int, D: int, group: int, max_pages: int, device):
    """(parts of a sequence, scratch for their results or None).  The caller holds the scratch until the launch: a graph's own is free for
    another tensor of the call otherwise."""
    if num_splits <= 0:
        num_splits = _pick_splits(B * nkv, max_pages)
    if num_splits <= 1:
        return 1, None
    need = _decode_floats(B, nkv, D, group, num_splits)
    if scratch is None:
        scratch = _scratch(device, need)
    elif (scratch.dtype is not torch.float32 or scratch.numel() < need or scratch.device != device or not scratch.is_contiguous()
          or scratch.data_ptr() & 15):
        raise ValueError(f"scratch wants {need} contiguous fp32 values on {device} from 16 bytes on, the first {COUNTERS} zero before "
                         "the first call")
    return num_splits, scratch


def decode_scratch(pages: QuantizedPages, nq: int, max_batch: int, max_pages: int) -> Optional[torch.Tensor]:
    """Scratch for every decode attention of up to max_batch sequences of max_pages pages, for a caller that keeps its own: steps that
    are captured into a graph share it, one behind another.  None on the CPU."""
    if not pages.is_cuda:
        return None
    nkv, D = pages.shape[1], pages.shape[3]
    floats = max(_decode_floats(b, nkv, D, nq // nkv, _pick_splits(b * nkv, max_pages)) for b in range(1, max_batch + 1))
    return torch.zeros((max(floats, COUNTERS),), dtype=torch.float32, device=pages.device)


# --------------------------------------------------------------------------- operators
def rope_kv_append(qkv, positions, slots, cos_sin, k_cache, v_cache, nq, nkv, head_dim, *, bias=None, q_norm_w=None, k_norm_w=None,
                   norm_eps=1e-6, q_out=None) -> torch.Tensor:
    """`ops.rope_kv_append` onto quantised pages: norms and rotations are rounded once, at the end.  A slot that is negative or
    outside the pages stores nothing; two tokens of a call have different slots."""
    blocks = _pair(k_cache, v_cache)[0]
    T, parts, stride, rows = _check_qkv(qkv, positions, slots, cos_sin, k_cache, nq, nkv, head_dim, bias, q_norm_w, k_norm_w)
    if q_out is None:
        q_out = qkv.new_empty((T, nq * head_dim), dtype=torch.bfloat16)
    else:
        _want_rows(q_out, "q_out", (T, nq * head_dim), k_cache.index)
    if not _on_gpu(k_cache.index):
        return _ref_append(qkv, positions, slots, cos_sin, k_cache, v_cache, nq, nkv, head_dim, bias, q_norm_w, k_norm_w, norm_eps, q_out)
    partial, at = qkv.dtype is torch.float32, qkv.data_ptr()
    rc = _lib.lib().nkb_q8_append(_APPEND.pack(
        0 if partial else at, at if partial else 0, _p(bias), _p(positions), _p(slots), _p(cos_sin), _p(q_norm_w), _p(k_norm_w),
        q_out.data_ptr(), *k_cache.at, *v_cache.at, _stream(), stride, norm_eps, parts, T, nq, nkv, head_dim, rows, blocks, 0))
    if rc:
        _lib.check(rc, "nkb_q8_append")
    _count_launch()
    return q_out


def paged_attn_decode(q, k_cache, v_cache, block_table, context_lens, scale, *, q_len=1, window=0, chunk=0, sinks=None, mods=None,
                      num_splits=0, scratch=None, out=None) -> torch.Tensor:
    """`ops.paged_attn_decode` over quantised pages."""
    blocks, nkv, D = _pair(k_cache, v_cache)
    index = k_cache.index
    B, width, table_step = _check_table(block_table, context_lens, index)
    nq = q.shape[-1] // D
    group = _check_heads(nq, nkv)
    _check_masks(mods, scale, window, chunk, sinks, nq, index)
    if q_len < 1 or num_splits > MAX_SPLITS:
        raise ValueError(f"q_len is at least one, num_splits at most {MAX_SPLITS}")
    q_at = _want_rows(q, "q", (B * q_len, nq * D), index)
    out = _result(out, q, index)
    if not B:
        return out
    if not _on_gpu(index):
        qf, res = q.float().reshape(B, q_len, nq, D), out.view(B, q_len, nq, D)
        for b in range(B):
            ctx = min(int(context_lens[b]), width * PAGE)
            res[b] = _ref_attend(qf[b], k_cache, v_cache, block_table[b], ctx, scale, ctx - q_len, True, window, chunk, sinks)
        return out
    if q_len * group > 16:          # more rows than a fragment of the decode kernel has
        q_start = torch.arange(0, B * q_len, q_len, device=k_cache.device, dtype=torch.int32)
        return flash_attn_prefill(q, k_cache, v_cache, block_table, q_start, torch.full_like(q_start, q_len), context_lens, scale,
                                  max_q_len=q_len, window=window, chunk=chunk, sinks=sinks, out=out)
    num_splits, scratch = _splits(num_splits, scratch, B, nkv, D, group, width, k_cache.device)
    rc = _lib.lib().nkb_q8_attn_decode(_ATTN.pack(
        q_at, *k_cache.at, *v_cache.at, block_table.data_ptr(), 0, 0, context_lens.data_ptr(), out.data_ptr(), _p(sinks), _p(scratch), _stream(),
        table_step, _floats(scratch), B, B * q_len, q_len, nq, nkv, D, blocks, width, 1, window, chunk, num_splits, scale, 0))
    if rc:
        _lib.check(rc, "nkb_q8_attn_decode")
    _count_launch()
    return out


def rope_attn_decode(qkv_partials, positions, slots, cos_sin, k_cache, v_cache, block_table, context_lens, scale, nq, nkv, *, bias=None,
                     q_norm_w=None, k_norm_w=None, norm_eps=1e-6, window=0, sinks=None, num_splits=0, scratch=None,
                     out=None) -> torch.Tensor:
    """`ops.rope_attn_decode` over quantised pages: `rope_kv_append`, and attention that fetches the older pages meanwhile.  The new token
    takes part as it is kept, in 8 bits.  slots[b] is the place of sequence b's position context_lens[b] - 1, which no other sequence of the
    call sees, or negative."""
    blocks, _, D = _pair(k_cache, v_cache)
    index = k_cache.index
    B, width, table_step = _check_table(block_table, context_lens, index)
    if qkv_partials.dtype is not torch.float32 or qkv_partials.shape[-2] != B:
        raise ValueError("rope_attn_decode wants fp32 partials [S, B, W], one token per sequence")
    if index < 0 or not B or nkv < 1 or nq // nkv > 16:
        q = rope_kv_append(qkv_partials, positions, slots, cos_sin, k_cache, v_cache, nq, nkv, D, bias=bias, q_norm_w=q_norm_w,
                           k_norm_w=k_norm_w, norm_eps=norm_eps)
        return paged_attn_decode(q, k_cache, v_cache, block_table, context_lens, scale, window=window, sinks=sinks, num_splits=num_splits,
                                 scratch=scratch, out=out)
    _, parts, stride, rows = _check_qkv(qkv_partials, positions, slots, cos_sin, k_cache, nq, nkv, D, bias, q_norm_w, k_norm_w)
    _check_masks(None, scale, window, 0, sinks, nq, index)
    if num_splits > MAX_SPLITS:
        raise ValueError(f"num_splits is at most {MAX_SPLITS}")
    if out is None:
        out = qkv_partials.new_empty((B, nq * D), dtype=torch.bfloat16)
    else:
        _want_rows(out, "out", (B, nq * D), index)
    _on_gpu(index)
    num_splits, scratch = _splits(num_splits, scratch, B, nkv, D, nq // nkv, width, k_cache.device)
    # the queries lie where their results come: who writes a result has read, or waited for those who read, its queries
    q_at, stream, pages = out.data_ptr(), _stream(), (*k_cache.at, *v_cache.at)
    rc = _lib.lib().nkb_q8_step(
        _APPEND.pack(0, qkv_partials.data_ptr(), _p(bias), _p(positions), _p(slots), _p(cos_sin), _p(q_norm_w), _p(k_norm_w), q_at, *pages, stream,
                     stride, norm_eps, parts, B, nq, nkv, D, rows, blocks, 0),
        _ATTN.pack(q_at, *pages, block_table.data_ptr(), 0, 0, context_lens.data_ptr(), q_at, _p(sinks), _p(scratch), stream,
                   table_step, _floats(scratch), B, B, 1, nq, nkv, D, blocks, width, 1, window, 0, num_splits, scale, 0))
    if rc:
        _lib.check(rc, "nkb_q8_step")
    _count_launch(2)
    return out


def flash_attn_prefill(q, k_cache, v_cache, block_table, q_start, q_lens, context_lens, scale, *, max_q_len, causal=True, window=0,
                       chunk=0, sinks=None, mods=None, out=None) -> torch.Tensor:
    """`ops.flash_attn_prefill` over quantised pages.  Rows of q that belong to no sequence are left as they are in `out`, which may be q.  What a
    row does not see costs it no more than 2^-18 of its largest value for a token and 2^-20 of its largest key, whatever its size."""
    blocks, nkv, D = _pair(k_cache, v_cache)
    index = k_cache.index
    B, width, table_step = _check_table(block_table, context_lens, index)
    nq, total = q.shape[-1] // D, q.shape[0]
    _check_heads(nq, nkv)
    _check_masks(mods, scale, window, chunk, sinks, nq, index)
    q_at = _want_rows(q, "q", (total, nq * D), index)
    _want(q_start, "q_start", torch.int32, (B,), index)
    _want(q_lens, "q_lens", torch.int32, (B,), index)
    out = _result(out, q, index)
    if not B or not total:
        return out
    if max_q_len < 1:
        raise ValueError("max_q_len is at least one")
    if not _on_gpu(index):
        qf, res = q.float().reshape(-1, nq, D), out.view(-1, nq, D)
        for b in range(B):
            n, at, ctx = int(q_lens[b]), int(q_start[b]), min(int(context_lens[b]), width * PAGE)
            if n > 0:
                res[at:at + n] = _ref_attend(qf[at:at + n], k_cache, v_cache, block_table[b], ctx, scale, ctx - n, causal, window, chunk,
                                             sinks)
        return out
    if abs(out.data_ptr() - q_at) < 2 * q.numel():      # (queries may be read again behind their results)
        q = q.clone()
        q_at = q.data_ptr()
    floats = _prefill_floats(B, max_q_len, nq, nkv, D, width)
    scratch = _scratch(k_cache.device, floats)
    rc = _lib.lib().nkb_q8_attn_prefill(_ATTN.pack(
        q_at, *k_cache.at, *v_cache.at, block_table.data_ptr(), q_start.data_ptr(), q_lens.data_ptr(), context_lens.data_ptr(), out.data_ptr(),
        _p(sinks), scratch.data_ptr(), _stream(), table_step, scratch.numel(), B, total, max_q_len, nq, nkv, D, blocks,
        width, 1 if causal else 0, window, chunk, 1, scale, 0))
    if rc:
        _lib.check(rc, "nkb_q8_attn_prefill")
    _count_launch(_prefill_launches(B, max_q_len, nq, nkv, width))
    return out


from . import _count_launch, _stream  # noqa: E402  (defined above the import of this module)
