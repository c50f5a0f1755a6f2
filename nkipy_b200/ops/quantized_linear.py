"""Products of rows and weights in 8-bit whole numbers.

A row x, of activations or of a weight, is held as ``q``, the whole numbers nearest to ``127 x / max|x|`` (ties to the even one), and one
factor ``scale = max|x| / 127``: x is about ``q * scale``, off by half a scale at most.  A row with a value that is not finite has the
scale NaN and zeros, a row of zeros the scale 0.

A factor for every token and every output channel, because both leave the sum over k: ``y = (sum_k q_x q_w) * scale_x * scale_w``, whose
sum is exact.  The numbers of a row are decided exactly too (quant_rows.cu), so a row has the same numbers whichever kernel, or the
reference on the CPU, made them.  Behind a norm they come from the products h * w of the residual stream and the norm's weights, which
are exact (of rows whose largest product is 2^-125 or more); the norm's factor is one for the row and goes into its scale.

    QuantizedRows     rows of activations: `quantize_rows`, or `rmsnorm`, `add_rmsnorm` and `silu_mul` with quantize=True
    QuantizedWeight   a weight, which `linear` takes in the place of a bf16 one

No file of the reference corresponds to these (its products are bf16, examples/models/qwen3/kernels/transformer_layer.py:16-120).
"""

from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _lib
from . import _count_launch, _stream, mixers

MAX_K = 131071                       # 128 * 128 * k stays below 2^31
FEW_ROWS, FEW_BYTES = 2, 98304       # rows, and bytes of them in 8 bits, that the kernel for few tokens takes (gemm_i8_few.cu)
# NkbQuantRows and NkbGemmI8 of csrc/kernels/i8_args.h
_ROWS, _GEMM = struct.Struct("9P3q4i3fi"), struct.Struct("8P4q8i")


class _Quantized:
    """int8 `values` [rows, k] and fp32 `scale` [rows] on one device.  Rows start on 16 bytes: values that do not lie so are copied."""
    __slots__ = ("values", "scale", "shape", "index", "device", "ld", "at")

    def __init__(self, values: torch.Tensor, scale: torch.Tensor):
        if values.dtype is not torch.int8 or scale.dtype is not torch.float32:
            raise TypeError(f"{type(self).__name__} wants int8 values and fp32 scales")
        shape = values.shape
        if len(shape) != 2 or scale.shape != shape[:1] or not 1 <= shape[1] <= MAX_K:
            raise ValueError(f"{type(self).__name__} wants values [rows, k] of at most {MAX_K} columns and scales [rows]")
        index = values.get_device()
        if scale.get_device() != index or (shape[0] > 1 and scale.stride(0) != 1):
            raise ValueError(f"{type(self).__name__} wants scales that follow one another, on the values' device")
        ld, column = values.stride()
        if (column != 1 and shape[1] > 1) or ld < shape[1] or ld & 15 or values.data_ptr() & 15:
            values = _padded(shape[0], shape[1], values.device).copy_(values)
            ld = values.stride(0)
        # index: of the CUDA device, -1: the CPU; ld: numbers from one row to the next; at: where values and scales start
        self.values, self.scale, self.shape, self.index, self.device, self.ld = values, scale, shape, index, values.device, ld
        self.at = values.data_ptr(), scale.data_ptr()

    @classmethod
    def _made(cls, values: torch.Tensor, scale: torch.Tensor, ld: int, index: int):
        """Of tensors that are known to lie as they should."""
        self = cls.__new__(cls)
        self.values, self.scale, self.shape, self.index, self.device, self.ld = values, scale, values.shape, index, values.device, ld
        self.at = values.data_ptr(), scale.data_ptr()
        return self

    @property
    def is_cuda(self) -> bool:
        return self.index >= 0

    @property
    def nbytes(self) -> int:
        return self.values.numel() + 4 * self.scale.numel()

    def dequantize(self) -> torch.Tensor:
        """The values that the rows stand for, fp32 [rows, k]."""
        return self.values.float() * self.scale[:, None]


class QuantizedRows(_Quantized):
    """Rows of activations [tokens, k] in 8 bits."""
    __slots__ = ()


class QuantizedWeight(_Quantized):
    """A weight [n, k] in 8 bits with a scale for every output channel; for a gated product [2 n, k], gate rows and then up rows.

    Weights may be fetched while the kernel before the product still runs (`linear`, weights_static): a program that writes the
    values of an existing one says weights_static=False in the product behind that."""
    __slots__ = ()

    @classmethod
    def of(cls, w: torch.Tensor) -> "QuantizedWeight":
        """From bf16 or fp32 [n, k]."""
        r = quantize_rows(w)
        return cls(r.values, r.scale)


def _padded(rows: int, k: int, device) -> torch.Tensor:
    """int8 [rows, k] whose rows start on 16 bytes."""
    ld = (k + 15) // 16 * 16
    t = torch.empty((rows, ld), dtype=torch.int8, device=device)
    if ld == k:
        return t
    t[:, k:].zero_()
    return t[:, :k]


def _want(t: torch.Tensor, name: str, dtype, shape, index: int) -> int:
    """Address of a contiguous tensor of this type and shape on device `index`."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{name} wants {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has the shape {tuple(t.shape)}, not {tuple(shape)}")
    raise ValueError(f"{name} wants to be contiguous and on the others' device")


def _on_gpu(index: int) -> bool:
    """Whether the kernels run (CUDA); they are launched on the current device's current stream."""
    if index < 0:
        return False
    if index != torch._C._cuda_getDevice():
        raise ValueError("the tensors are on another device than the current one")
    if not _lib._initialised:
        _lib.ensure_init()
    return True


_BF16, _F32 = torch.bfloat16, torch.float32


def to_bf16(y: torch.Tensor) -> torch.Tensor:
    """Numbers in 64 bits rounded to bf16 once: on the way through 32 bits to odd, since to the nearest they may come to lie in the middle of two
    bf16 numbers that they are not in the middle of."""
    f = y.float()
    d, bits = f.double(), f.view(torch.int32)
    bits = torch.where((d == y) | y.isnan(), bits, (bits - (d.abs() > y.abs()).int()) | 1)
    return bits.view(torch.float32).to(_BF16)


# --------------------------------------------------------------------------- rows
def _numbers(x: torch.Tensor):
    """(whole numbers, largest magnitude) of rows in 64 bits; zeros and NaN where a row is not finite in 32."""
    fine = x.float().isfinite().all(-1, keepdim=True)
    top = torch.where(fine, x, 0.0).abs().amax(-1, keepdim=True)
    q = torch.round(127 * (x / top))
    return torch.where(fine & (top > 0), q, 0.0).to(torch.int8), torch.where(fine, top, torch.nan).squeeze(-1)


def _launch_rows(form, rows, width, device, index, x=0, partials=0, bias=0, residual=0, w=0, residual_out=0, x_ld=0, split_stride=0,
                 splits=0, eps=0.0, limit=0.0, alpha=0.0, late=0) -> QuantizedRows:
    # (the kernel writes the columns up to the next sixteen, too)
    ld = (width + 15) & -16
    values = torch.empty_strided((rows, width), (ld, 1), dtype=torch.int8, device=device) if ld == width else \
        torch.empty((rows, ld), dtype=torch.int8, device=device)[:, :width]
    scale = torch.empty_strided((rows,), (1,), dtype=_F32, device=device)
    rc = _lib.lib().nkb_quant_rows(_ROWS.pack(
        x, partials, bias, residual, w, residual_out, values.data_ptr(), scale.data_ptr(), _stream(), x_ld, ld, split_stride, form, rows,
        width, splits, eps, limit, alpha, late))
    if rc:
        _lib.check(rc, "nkb_quant_rows")
    _count_launch()
    return QuantizedRows._made(values, scale, ld, index)


def _check_rows(x: torch.Tensor):
    """(rows, columns, elements from one row to the next) of rows to be brought into 8 bits."""
    if x.dtype is not _BF16 and x.dtype is not _F32:
        raise TypeError(f"quantize_rows wants bf16 or fp32, not {x.dtype}")
    shape = x.shape
    if len(shape) != 2 or not 1 <= shape[1] <= MAX_K:
        raise ValueError(f"quantize_rows wants [rows, k] of at most {MAX_K} columns")
    ld, column = x.stride()
    if column != 1 and shape[1] > 1:
        raise ValueError("quantize_rows wants neighbouring columns")
    return shape[0], shape[1], ld


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """bf16 or fp32 rows [rows, k] (they may lie apart) in 8 bits."""
    rows, width, ld = _check_rows(x)
    index = x.get_device()
    if not _on_gpu(index):
        q, top = _numbers(x.double())
        return QuantizedRows(q, (top / 127).float())
    # (late: they may become a weight, which a product right behind fetches ahead of its wait)
    return _launch_rows(0 if x.dtype is _BF16 else 1, rows, width, x.device, index, x=x.data_ptr(), x_ld=ld, late=1)


def add_rmsnorm(x, w, *, residual_in=None, partials=None, bias=None, residual_out=None, eps=1e-6, hidden=None, rows=None):
    """`ops.add_rmsnorm` whose normed rows are brought into 8 bits.  The residual stream, the sum rounded to bf16, is what the norm sees,
    whether it is wanted or not; sums of more than two addends are taken in 64 bits."""
    ref = x if x is not None else partials
    if ref is None or w is None:
        raise ValueError("quantised rows come from x or partial sums, and from a norm")
    index, hidden = ref.get_device(), ref.shape[-1] if hidden is None else hidden
    if not 1 <= hidden <= MAX_K:
        raise ValueError(f"quantised rows have at most {MAX_K} columns")
    if rows is None:
        rows = x.numel() // hidden if x is not None else partials.shape[-2]
    splits, stride, parts_at, n = 0, 0, 0, rows * hidden
    if partials is not None:
        if partials.dtype is not _F32:
            raise TypeError("partials must be fp32")
        splits = partials.shape[0] if partials.dim() == 3 else 1
        stride = partials.stride(0) if partials.dim() == 3 else 0
        one = partials[0] if partials.dim() == 3 and splits else partials
        if not splits or one.shape != (rows, hidden) or partials.get_device() != index or not one.is_contiguous():
            raise ValueError("partials wants [splits, rows, hidden] with neighbouring rows, on the others' device")
        parts_at = partials.data_ptr()
    x_at = residual_at = bias_at = 0
    if x is not None:
        if x.numel() != n:
            raise ValueError(f"x wants {rows} rows of {hidden}")
        x_at = _want(x, "x", _BF16, x.shape, index)
    if residual_in is not None:
        if residual_in.numel() != n:
            raise ValueError(f"residual_in wants {rows} rows of {hidden}")
        residual_at = _want(residual_in, "residual_in", _BF16, residual_in.shape, index)
    w_at = _want(w, "w", _BF16, (hidden,), index)
    if bias is not None:
        bias_at = _want(bias, "bias", _BF16, (hidden,), index)
    if residual_out is not None:
        if residual_out.numel() != n:
            raise ValueError(f"residual_out wants {rows} rows of {hidden}")
        _want(residual_out, "residual_out", _BF16, residual_out.shape, index)
    elif x is not None and residual_in is not None and len(x.shape) == 2:
        residual_out = torch.empty_like(x)
    elif residual_in is not None or partials is not None:
        residual_out = torch.empty((rows, hidden), dtype=_BF16, device=ref.device)
    if not _on_gpu(index):
        h = torch.zeros((rows, hidden), dtype=torch.float64)
        if partials is not None:
            h = h + (partials.double().sum(0) if partials.dim() == 3 else partials.double())
        for t in (x, bias, residual_in):
            if t is not None:
                h = h + t.double().reshape(-1, hidden)
        h = to_bf16(h)
        if residual_out is not None:
            residual_out.copy_(h.reshape(residual_out.shape))
        q, top = _numbers(h.double() * w.double())
        scale = (top / 127).float() * torch.rsqrt(h.float().square().mean(-1) + eps)
        return residual_out, QuantizedRows(q, scale)
    return residual_out, _launch_rows(2, rows, hidden, ref.device, index, x=x_at, partials=parts_at, bias=bias_at, residual=residual_at, w=w_at,
                                      residual_out=0 if residual_out is None else residual_out.data_ptr(), x_ld=hidden,
                                      split_stride=stride, splits=splits, eps=eps)


def silu_mul(gate_up, limit: float = 0.0, alpha: float = 1.702, bias=None) -> QuantizedRows:
    """`ops.silu_mul` whose rows are brought into 8 bits; bf16 [T, 2 I], or fp32 (partial sums) [S, T, 2 I]."""
    if gate_up.dtype is not _BF16 and gate_up.dtype is not _F32:
        raise TypeError(f"silu_mul wants bf16 or fp32, not {gate_up.dtype}")
    index, f32 = gate_up.get_device(), gate_up.dtype is torch.float32
    if gate_up.dim() != 2 and not (f32 and gate_up.dim() == 3 and gate_up.shape[0]):
        raise ValueError("silu_mul wants [T, 2 I], or fp32 partial sums [S, T, 2 I]")
    rows, two = gate_up.shape[-2:]
    width = two // 2
    if two % 2 or not 1 <= width <= MAX_K:
        raise ValueError(f"silu_mul wants gate and up of at most {MAX_K} columns")
    if gate_up.stride(-1) != 1:
        raise ValueError("silu_mul wants neighbouring columns")
    bias_at = 0 if bias is None else _want(bias, "bias", _BF16, (two,), index)
    if not _on_gpu(index):
        v = gate_up.double() if gate_up.dim() == 2 else gate_up.double().sum(0)
        if bias is not None:
            v = v + bias.double()
        g, u = v[:, :width], v[:, width:]
        if limit > 0:
            limit, alpha = torch.tensor([limit, alpha], dtype=_F32).tolist()         # (as the kernel has them)
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
            y = (u + 1) * g / (1 + torch.exp(-alpha * g))
        else:
            y = g / (1 + torch.exp(-g)) * u
        q, top = _numbers(y)
        return QuantizedRows(q, (top / 127).float())
    deep, at = gate_up.dim() == 3, gate_up.data_ptr()
    return _launch_rows(4 if f32 else 3, rows, width, gate_up.device, index, x=0 if f32 else at, partials=at if f32 else 0, bias=bias_at,
                        x_ld=gate_up.stride(-2), split_stride=gate_up.stride(0) if deep else 0,
                        splits=(gate_up.shape[0] if deep else 1) if f32 else 0, limit=limit, alpha=alpha)


# --------------------------------------------------------------------------- products
def effective_splits(k: int, splits: int) -> int:
    """Partial sums that a product asked for `splits` of them really has: whole slabs of 128 k, none of them empty."""
    slabs = -(-k // 128)
    return -(-slabs // -(-slabs // max(1, min(splits, slabs))))


def linear(x, w: QuantizedWeight, *, bias=None, residual=None, out=None, splits: int = 1, gated: bool = False, weights_static: bool = True,
           act: str = "silu", fp32_out: bool = False, out_act=None) -> torch.Tensor:
    """`ops.linear` with a weight in 8 bits; x: `QuantizedRows`, or bf16 or fp32 rows, which are brought into 8 bits first.

    The sum is exact; it is rounded to 32 bits and multiplied by both scales, and the result is rounded once more, to bf16, at the
    end.  Rows of other types than bf16 and fp32 are refused, and so is out_act."""
    if type(w) is not QuantizedWeight:
        raise TypeError("rows in 8 bits want a QuantizedWeight")
    if out_act is not None:
        raise ValueError("products in 8 bits have no out_act")
    N = w.shape[0] // 2 if gated else w.shape[0]
    if gated and (w.shape[0] % 2 or act not in ("silu", "gelu_tanh")):
        raise ValueError("a gated product wants gate and up rows, and silu or gelu_tanh")
    index = w.index
    given = type(x) is QuantizedRows
    if given:
        M, K = x.shape
        if x.index != index:
            raise ValueError("rows and weight want to be on one device")
    else:
        M, K, x_ld = _check_rows(x)
        if x.get_device() != index:
            raise ValueError("rows and weight want to be on one device")
    if K != w.shape[1]:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)} w {tuple(w.shape)}")
    if gated and (bias is not None or residual is not None or fp32_out or splits > 1):
        raise ValueError("a gated product has no bias, residual, fp32_out or splits")
    if splits > 1 and residual is not None:
        raise ValueError("partial sums have no residual")
    dtype = _F32 if fp32_out or splits > 1 else _BF16
    parts = effective_splits(K, splits) if splits > 1 else 0
    bias_at = 0 if bias is None else _want(bias, "bias", _BF16, (N,), index)
    if out is None:
        out = torch.empty((parts, M, N) if parts else (M, N), dtype=dtype, device=w.device)
    elif parts:
        if out.dtype is not dtype or not out.is_contiguous() or out.get_device() != index or out.numel() < parts * M * N:
            raise ValueError("split-K output must be fp32 with room for [S, M, N]")
        out = out.view(-1)[:parts * M * N].view(parts, M, N)
    else:
        if out.dtype is not dtype:
            raise TypeError(f"out wants {dtype}, not {out.dtype}")
        if out.shape != (M, N) or out.get_device() != index or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError("out wants [M, N] with neighbouring columns, on the weight's device")
    ldo = N if out.is_contiguous() else max(out.stride(-2), N)
    if residual is not None:
        if residual.dtype is not torch.bfloat16:
            raise TypeError(f"residual wants torch.bfloat16, not {residual.dtype}")
        if residual.shape != (M, N) or residual.get_device() != index:
            raise ValueError("residual wants [M, N] on the weight's device")
        if residual.stride() != out.stride():
            residual = residual.contiguous() if ldo == N else torch.empty_strided((M, N), (ldo, 1), dtype=residual.dtype,
                                                                                  device=residual.device).copy_(residual)
    if not M or not N:
        return out
    if not _on_gpu(index):
        return _reference(x if given else quantize_rows(x), w, bias, residual, out, parts, gated, act, N)
    stream, form = _stream(), 0 if given or x.dtype is _BF16 else 1
    more = (bias_at, 0 if residual is None else residual.data_ptr(), out.data_ptr(), stream)
    ends = (w.ld, ldo, out.stride(0) if parts else 0, M, N, K, gated, mixers.ACTIVATIONS[act][0] if gated else 0, dtype is _F32, parts,
            weights_static)
    if M <= FEW_ROWS and not parts and M * ((K + 511) & -512) <= FEW_BYTES:
        if given:
            rows, at, q_ld = None, x.at, x.ld
        else:
            rows, at, q_ld = _ROWS.pack(x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, stream, x_ld, 0, 0, form, M, K, 0, 0.0, 0.0, 0.0, 0), (0, 0), 0
        rc = _lib.lib().nkb_gemm_i8_few(rows, _GEMM.pack(at[0], w.at[0], at[1], w.at[1], *more, q_ld, *ends))
        if rc:
            _lib.check(rc, "nkb_gemm_i8_few")
        _count_launch()
        return out
    if given:
        (q_at, scale_at), q_ld, rows = x.at, x.ld, None
    else:
        # numbers and scales in one piece of memory; both launches by one call
        q_ld = (K + 15) & -16
        buffer = torch.empty_strided((M * (q_ld + 4),), (1,), dtype=torch.int8, device=w.device)
        q_at = buffer.data_ptr()
        scale_at = q_at + M * q_ld
        rows = _ROWS.pack(x.data_ptr(), 0, 0, 0, 0, 0, q_at, scale_at, stream, x_ld, q_ld, 0, form, M, K, 0, 0.0, 0.0, 0.0, 0)
    rc = _lib.lib().nkb_linear_i8(rows, _GEMM.pack(q_at, w.at[0], scale_at, w.at[1], *more, q_ld, *ends))
    if rc:
        _lib.check(rc, "nkb_linear_i8")
    _count_launch(1 if given else 2)
    return out


def _reference(x, w, bias, residual, out, parts, gated, act, N):
    q, v = x.values.double(), w.values.double()

    def part(a, b):
        return (q[:, a:b] @ v[:, a:b].T).float() * x.scale[:, None] * w.scale

    if parts:
        step = -(-(-(-x.shape[1] // 128)) // parts) * 128
        for s in range(parts):
            out[s] = part(s * step, (s + 1) * step)
        if bias is not None:
            out[0] += bias.float()
        return out
    y = part(0, x.shape[1])
    if gated:
        y = mixers.ACTIVATIONS[act][1](y[:, :N]) * y[:, N:]
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return out.copy_(y)
