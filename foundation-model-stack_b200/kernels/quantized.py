"""Quantised linear layers: rows and weights of 8 bits, weights of 4 bits, and the products over them.

``QuantizedRows``: rows of e4m3 (``torch.float8_e4m3fn``: largest value 448) with one float32 scale a row, so that row r stands for
values[r] * scales[r].  ``quantize_rows`` makes them of any rows, ``add_rmsnorm_quantized`` behind the residual sum and the norm.
``E4M3Weight``: a matrix of such rows, one scale an output channel; ``linear_e4m3`` multiplies rows with it.

``Int4Weight``: whole numbers q of 0 to 15 with one bfloat16 scale s and one whole zero point z for every ``group_size``
consecutive input channels of an output channel, which stand for (q - z) * s; ``linear_int4`` multiplies bfloat16 rows with it.

Weights are laid out once, when a model is loaded, and what made them has finished when their constructor returns: the
products ask for a weight's bytes before the kernel in front of them is done, which is right for constants only.  A weight's
tensors must not be written afterwards.  All launches go to the current device's current stream; tensors of another device are
refused.  ``linear``, ``gated_linear`` and ``activated_linear`` (kernels/ops.py) take these weights too.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import ops
from .build import load_library

E4M3 = torch.float8_e4m3fn
INT4_FEW_ROWS = 8  # rows up to which the 4-bit product runs on mma.sync and has a gated form (csrc/gemm_int4.cu)


def _on_device(what: str, *tensors) -> None:
    """Every tensor lies on the current device, whose stream the launch goes to (that it is contiguous the launch itself sees to)."""
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ops.KernelError(f"{what}: a tensor on the CPU reached a CUDA kernel; this library has no CPU path")
        if device is None:
            device = ops._device()
        if t.get_device() != device:
            raise ops.KernelError(f"{what}: a tensor lies on {t.device}, the current device is cuda:{device}")


def _settled(t: torch.Tensor) -> None:
    """What was launched for ``t`` is done."""
    if t.is_cuda:
        if torch.cuda.is_current_stream_capturing():
            raise ops.KernelError("weights are laid out before a graph is captured, not in it")
        torch.cuda.current_stream(t.device).synchronize()


def _pitch(dim: int) -> int:
    return (dim + 15) // 16 * 16


class QuantizedRows:
    """``values`` [rows, pitch] e4m3 (pitch: dim rounded up to 16, zeros behind a row's last value), ``scales`` [rows] float32."""

    __slots__ = ("values", "scales", "dim")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, dim: int) -> None:
        if values.dtype != E4M3 or values.dim() != 2 or dim <= 0 or values.shape[1] != _pitch(dim):
            raise ops.KernelError(f"rows of {dim} e4m3 values lie {_pitch(dim)} apart: {values.dtype} {tuple(values.shape)} is something else")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (values.shape[0],) or scales.device != values.device:
            raise ops.KernelError(f"one float32 scale a row: {scales.dtype} {tuple(scales.shape)} on {scales.device} for {values.shape[0]} rows on {values.device}")
        self.values, self.scales, self.dim = values, scales, int(dim)

    @classmethod
    def of(cls, values: torch.Tensor, scales: torch.Tensor) -> "QuantizedRows":
        """Of e4m3 ``values`` [rows, dim] as they are; where dim is no multiple of 16, or the rows lie otherwise, of a copy."""
        if values.dtype != E4M3 or values.dim() != 2:
            raise ops.KernelError(f"e4m3 rows are [rows, dim] {E4M3}: {values.dtype} {tuple(values.shape)} is something else")
        dim = values.shape[1]
        if _pitch(dim) != dim or not values.is_contiguous() or values.data_ptr() % 16:
            rows = torch.zeros((values.shape[0], _pitch(dim)), dtype=torch.uint8, device=values.device)
            rows[:, :dim] = values.view(torch.uint8)
            values = rows.view(E4M3)
        return cls(values, scales.contiguous(), dim)

    @property
    def shape(self):
        return (self.values.shape[0], self.dim)

    @property
    def device(self):
        return self.values.device

    def dequantize(self) -> torch.Tensor:
        """The float32 rows that they stand for."""
        return self.values[:, : self.dim].float() * self.scales[:, None]


class E4M3Weight:
    """A matrix [out, in] of e4m3 with one scale an output channel."""

    __slots__ = ("rows",)

    def __init__(self, rows: QuantizedRows) -> None:
        _settled(rows.values)
        self.rows = rows

    @property
    def shape(self):
        return self.rows.shape

    @property
    def device(self):
        return self.rows.device

    def dequantize(self) -> torch.Tensor:
        return self.rows.dequantize()

    def tensors(self):
        return {"values": self.rows.values, "scales": self.rows.scales}


class Int4Weight:
    """A matrix [out, in] of 4 bits.  ``blocks`` [out / 16, in / 128, 256 + 16 per] int32: 16 rows by 128 input channels each, the
    values and behind them ``per`` (1, 2 or 4) words a row with scale and zero point, laid out as csrc/gemm_int4.cu says.  Made by
    ``pack_int4``."""

    __slots__ = ("blocks", "shape", "per")

    def __init__(self, blocks: torch.Tensor, shape, per: int) -> None:
        out, dim = (int(v) for v in shape)
        if blocks.dtype != torch.int32 or per not in (1, 2, 4) or tuple(blocks.shape) != (-(-out // 16), -(-dim // 128), 256 + 16 * per):
            raise ops.KernelError(f"the packed blocks of a {out} x {dim} matrix are not {blocks.dtype} {tuple(blocks.shape)}")
        _settled(blocks)
        self.blocks, self.shape, self.per = blocks, (out, dim), int(per)

    @property
    def device(self):
        return self.blocks.device

    def dequantize(self) -> torch.Tensor:
        """The float32 matrix that it stands for."""
        out, dim = self.shape
        n16, kb = self.blocks.shape[:2]
        row = torch.arange(16, device=self.device)[:, None]
        words = self.blocks[:, :, :256].reshape(n16, kb, 16, 4, 4)[:, :, row, torch.arange(4, device=self.device)[None, :] ^ (row // 2 % 4)]
        q = torch.stack([(words >> (4 * (i // 2) + 16 * (i % 2))) & 15 for i in range(8)], dim=-1)  # [.., row, piece, word, 8]
        q = q.permute(0, 2, 1, 4, 3, 5).reshape(n16 * 16, kb * 128)[:out, :dim].float()
        groups = self.blocks[:, :, 256:].reshape(n16, kb, self.per, 16).permute(0, 3, 1, 2).reshape(n16 * 16, kb * self.per)
        groups = groups.repeat_interleave(128 // self.per, dim=1)[:out, :dim]
        return (q - ((groups & -65536).view(torch.float32) - 128.0)) * (groups << 16).view(torch.float32)

    def tensors(self):
        return {"blocks": self.blocks}


# ---- rows to 8 bits ------------------------------------------------------------------------------------------------
def _empty_rows(n: int, dim: int, device) -> QuantizedRows:
    out = QuantizedRows.__new__(QuantizedRows)  # nothing to check: a decode step makes some hundred of them
    pitch = (dim + 15) // 16 * 16
    out.values = torch.empty_strided((n, pitch), (pitch, 1), dtype=E4M3, device=device)  # 0.9 us less of the host's time than torch.empty
    out.scales = torch.empty_strided((n,), (1,), dtype=torch.float32, device=device)
    out.dim = dim
    return out


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """Rows [rows, dim] (float32 or bfloat16) as e4m3: scale = max |x| / 448, value = x * 448 / max |x| to the nearest, ties to even.  A row of
    zeros (or one whose scale would lie below 2^-110) gets scale 0 and zeros; one with a NaN or an
    infinity a scale that is not finite, and what a product makes of it is not finite either."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ops.KernelError(f"quantize_rows: rows are [rows, dim], not {tuple(x.shape)}")
    _on_device("quantize_rows", x)
    n, dim = x.shape
    out = _empty_rows(n, dim, x.device)
    ops._call("quantize_rows", "fms_quantize_rows", x, ops._code(x.dtype), out.values, out.scales, n, dim, (dim + 15) // 16 * 16,
              ops._stream())
    return out


def add_rmsnorm_quantized(residual: torch.Tensor, delta: Optional[torch.Tensor], gain: torch.Tensor, eps: float,
                          rows: Optional[torch.Tensor] = None) -> QuantizedRows:
    """``add_rmsnorm`` whose result leaves as e4m3 rows: residual (float32, in place) += delta; y = gain * rmsnorm(residual);
    scale = max |y| / 448, value = y * 448 / max |y|.  With ``rows`` (int32) only those rows are computed and the residual is not
    written.  ``delta`` is float32 or bfloat16 or None, ``gain`` float32 or bfloat16.  Rows of zeros and rows that are not
    finite: as ``quantize_rows``, the scale of the latter NaN."""
    shape = residual.shape
    if residual.dtype != torch.float32 or len(shape) != 2 or shape[1] == 0:
        raise ops.KernelError(f"the residual stream is float32 [rows, dim], not {residual.dtype} {tuple(shape)}")
    n_all, dim = shape
    if delta is not None and delta.shape != shape:
        raise ops.KernelError(f"add_rmsnorm_quantized: the sublayer's output is {tuple(delta.shape)}, the stream {tuple(shape)}")
    if gain.shape != shape[1:]:
        raise ops.KernelError(f"add_rmsnorm_quantized: a gain of {tuple(gain.shape)} for rows of {dim}")
    if rows is not None and (rows.dtype != torch.int32 or rows.dim() != 1):
        raise ops.KernelError(f"add_rmsnorm_quantized: rows are a vector of int32, not {rows.dtype} {tuple(rows.shape)}")
    _on_device("add_rmsnorm_quantized", residual, delta, gain, rows)
    n = n_all if rows is None else rows.shape[0]
    out = _empty_rows(n, dim, residual.device)
    ops._call("quantize_rows", "fms_add_rmsnorm_quantized", residual, delta, ops.F32 if delta is None else ops._code(delta.dtype), gain,
              ops._code(gain.dtype), float(eps), out.values, out.scales, rows, n, dim, (dim + 15) // 16 * 16, n_all, ops._stream())
    return out


# ---- weights ---------------------------------------------------------------------------------------------------------
def e4m3_weight(values: torch.Tensor, scales: torch.Tensor) -> E4M3Weight:
    """A weight of e4m3 ``values`` [out, in] and float32 ``scales`` [out], as a quantised checkpoint has them."""
    return E4M3Weight(QuantizedRows.of(values, scales))


def quantize_e4m3(weight: torch.Tensor) -> E4M3Weight:
    """A float32 or bfloat16 matrix [out, in] rounded to e4m3, one scale an output channel (``quantize_rows``)."""
    return E4M3Weight(quantize_rows(weight))


def pack_int4(q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group_size: int = 128) -> Int4Weight:
    """A weight that stands for (q - zeros) * scales: ``q`` [out, in] whole numbers of 0 to 15, ``scales`` [out, groups] (kept in
    bfloat16), ``zeros`` [out, groups] whole numbers of 0 to 15, or None: 8 throughout.  Groups are ``group_size`` consecutive
    input channels, a multiple of 32, or all of them; the last may be shorter.  ``in`` is a multiple of 8."""
    if q.dim() != 2 or q.shape[0] == 0 or q.shape[1] == 0 or q.is_floating_point() or q.is_complex():
        raise ops.KernelError(f"pack_int4: q is [out, in] whole numbers, not {q.dtype} {tuple(q.shape)}")
    out, dim = q.shape
    if dim % 8:
        raise ops.KernelError(f"pack_int4: {dim} input channels, a multiple of 8 is wanted")
    if group_size <= 0 or (group_size % 32 and group_size < dim):
        raise ops.KernelError(f"pack_int4: groups of {group_size}: a multiple of 32, or all {dim} input channels")
    group_size = min(int(group_size), (dim + 31) // 32 * 32)
    n_groups = -(-dim // group_size)
    if tuple(scales.shape) != (out, n_groups) or not scales.is_floating_point():
        raise ops.KernelError(f"pack_int4: scales are [{out}, {n_groups}], not {scales.dtype} {tuple(scales.shape)}")
    if zeros is not None and (tuple(zeros.shape) != (out, n_groups) or zeros.is_floating_point()):
        raise ops.KernelError(f"pack_int4: zero points are [{out}, {n_groups}] whole numbers, not {zeros.dtype} {tuple(zeros.shape)}")
    for name, t in (("values", q), ("zero points", zeros)):
        if t is not None and (int(t.min()) < 0 or int(t.max()) > 15):
            raise ops.KernelError(f"pack_int4: {name} of 4 bits are 0 to 15; there are {int(t.min())} to {int(t.max())}")
    device = q.device
    n16, kb = -(-out // 16), -(-dim // 128)
    if (out, dim) != (n16 * 16, kb * 128):
        wide = torch.zeros((n16 * 16, kb * 128), dtype=q.dtype, device=device)
        wide[:out, :dim] = q
        q = wide
    parts = q.reshape(n16, 16, kb, 4, 4, 8)  # 16 rows; of a block's k: words, pieces, values
    words = torch.zeros((n16, 16, kb, 4, 4), dtype=torch.int32, device=device)
    for i in range(8):
        words |= parts[..., i].to(torch.int32) << (4 * (i // 2) + 16 * (i % 2))
    words = words.permute(0, 2, 1, 4, 3)  # block of rows, block of k, row, piece, word
    row = torch.arange(16, device=device)[:, None]
    words = words[:, :, row, torch.arange(4, device=device)[None, :] ^ (row // 2 % 4)]
    scale_bits = scales.to(device=device, dtype=torch.bfloat16).contiguous().view(torch.int16).to(torch.int32) & 0xFFFF
    z = torch.full((out, n_groups), 8.0, device=device) if zeros is None else zeros.to(device=device, dtype=torch.float32)
    zero_bits = (z + 128.0).contiguous().view(torch.int32) & -65536  # 128 + z has no bits below bfloat16's
    per = 1 if group_size % 128 == 0 or n_groups == 1 else (2 if group_size % 64 == 0 else 4)
    at = torch.arange(kb * per, device=device) * (128 // per) // group_size  # the group of a part of a block; behind the last column: any
    groups = torch.zeros((n16 * 16, kb * per), dtype=torch.int32, device=device)
    groups[:out] = (scale_bits | zero_bits)[:, at.clamp(max=n_groups - 1)]
    groups = groups.view(n16, 16, kb, per).permute(0, 2, 3, 1).reshape(n16, kb, per * 16)
    return Int4Weight(torch.cat((words.reshape(n16, kb, 256), groups), dim=2), (out, dim), per)


def quantize_int4(weight: torch.Tensor, group_size: int = 128) -> Int4Weight:
    """A matrix [out, in] rounded to 4 bits: a group's 15 steps span its values and zero, scale = (high - low) / 15 in bfloat16,
    zero point = -low / scale and value = w / scale + zero point, each to the nearest."""
    if weight.dim() != 2 or not weight.is_floating_point() or weight.numel() == 0:
        raise ops.KernelError(f"quantize_int4: a matrix [out, in] is wanted, not {weight.dtype} {tuple(weight.shape)}")
    out, dim = weight.shape
    if group_size <= 0 or (group_size % 32 and group_size < dim):
        raise ops.KernelError(f"quantize_int4: groups of {group_size}: a multiple of 32, or all {dim} input channels")
    group_size = min(int(group_size), (dim + 31) // 32 * 32)
    n_groups = -(-dim // group_size)
    q = torch.empty((out, dim), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((out, n_groups), dtype=torch.bfloat16, device=weight.device)
    zeros = torch.empty((out, n_groups), dtype=torch.uint8, device=weight.device)
    for first in range(0, out, 4096):  # some rows at a time: the float32 copies of a whole matrix would be eight times its bytes
        w = torch.zeros((min(4096, out - first), n_groups * group_size), dtype=torch.float32, device=weight.device)
        w[:, :dim] = weight[first:first + 4096]
        w = w.view(w.shape[0], n_groups, group_size)
        low, high = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
        scale = ((high - low) / 15.0).to(torch.bfloat16)
        step = torch.where(scale > 0, scale.float(), torch.ones_like(low))
        zero = (-low / step).round().clamp(0, 15)
        values = ((w / step[:, :, None]).round() + zero[:, :, None]).clamp(0, 15)
        q[first:first + 4096] = values.view(w.shape[0], -1)[:, :dim].to(torch.uint8)
        scales[first:first + 4096], zeros[first:first + 4096] = scale, zero.to(torch.uint8)
    return pack_int4(q, scales, zeros, group_size)


# ---- products --------------------------------------------------------------------------------------------------------
def _bias(what: str, bias: Optional[torch.Tensor], out: int):
    """A bias as the products add it to their float32 sums, and its dtype's code: bfloat16 and float32 as they are, others in float32."""
    if bias is None:
        return None, ops.BF16
    if tuple(bias.shape) != (out,):
        raise ops.KernelError(f"{what}: a bias of {tuple(bias.shape)} for {out} output channels")
    if bias.dtype not in (torch.bfloat16, torch.float32):
        bias = bias.to(torch.float32)
    return bias, ops._code(bias.dtype)


def _rows_for(what: str, x, weight: E4M3Weight) -> QuantizedRows:
    if not isinstance(weight, E4M3Weight):
        raise ops.KernelError(f"{what}: the weight is an E4M3Weight, not {type(weight).__name__}")
    if isinstance(x, torch.Tensor):
        x = quantize_rows(x)
    if x.dim != weight.shape[1]:
        raise ops.KernelError(f"{what}: rows of {x.dim} values, weights of {weight.shape[1]}")
    _on_device(what, x.values, x.scales, weight.rows.values, weight.rows.scales)
    return x


_scratch_sizes = {}  # (entry, device, sizes) -> floats


def _scratch(library: str, name: str, device, rows: int, *sizes):
    """Scratch memory for the sums that several thread blocks share, and its floats: of one call alone, so that calls at once and
    captured graphs do not meet in it."""
    sizes = (min(rows, 257),) + sizes  # more than 256 rows want none
    key = (name, device) + sizes
    floats = _scratch_sizes.get(key)
    if floats is None:
        entry = getattr(load_library(library), name)
        entry.restype, entry.argtypes = ctypes.c_long, [ctypes.c_long] * len(sizes)
        floats = _scratch_sizes[key] = entry(*sizes)
    return (torch.empty_strided((floats,), (1,), dtype=torch.float32, device=device) if floats else None), floats


def linear_e4m3(x, weight: E4M3Weight, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Rows ``x`` (``QuantizedRows``; a tensor is quantised first) times weight [out, in] transposed (+ bias,
    bfloat16 or float32), summed in float32, in bfloat16 or float32."""
    x = _rows_for("linear_e4m3", x, weight)
    (m, _), (n, _) = x.shape, weight.shape
    bias, bias_code = _bias("linear_e4m3", bias, n)
    _on_device("linear_e4m3", bias)
    code = ops._code(out_dtype)
    y = torch.empty_strided((m, n), (n, 1), dtype=out_dtype, device=x.device)
    pitch = x.values.shape[1]
    scratch, floats = _scratch("gemm_e4m3", "fms_e4m3_scratch", x.device, m, n, pitch, 0)
    ops._call("gemm_e4m3", "fms_linear_e4m3", x.values, x.scales, weight.rows.values, weight.rows.scales, bias, bias_code, y, code, m, n,
              pitch, scratch, floats, ops.error_flag(x.device), ops._stream())
    return y


def gated_linear_e4m3(x, weight: E4M3Weight, bias: Optional[torch.Tensor], activation: int) -> torch.Tensor:
    """act(x Wg^T) * (x Wu^T) in bfloat16 for weight = [Wg; Wu], the activation in the product's epilogue."""
    x = _rows_for("gated_linear_e4m3", x, weight)
    (m, _), (n, _) = x.shape, weight.shape
    if n % 2:
        raise ops.KernelError(f"gated_linear_e4m3: {n} rows are no gate and up matrix")
    bias, bias_code = _bias("gated_linear_e4m3", bias, n)
    _on_device("gated_linear_e4m3", bias)
    y = torch.empty((m, n // 2), dtype=torch.bfloat16, device=x.device)
    pitch = x.values.shape[1]
    scratch, floats = _scratch("gemm_e4m3", "fms_e4m3_scratch", x.device, m, n, pitch, 1)
    ops._call("gemm_e4m3", "fms_glu_e4m3", x.values, x.scales, weight.rows.values, weight.rows.scales, bias, bias_code, y, m, n // 2,
              pitch, int(activation), scratch, floats, ops.error_flag(x.device), ops._stream())
    return y


def _int4_checked(what: str, x: torch.Tensor, weight: Int4Weight, bias: Optional[torch.Tensor]):
    if not isinstance(weight, Int4Weight):
        raise ops.KernelError(f"{what}: the weight is an Int4Weight, not {type(weight).__name__}")
    if not isinstance(x, torch.Tensor) or x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != weight.shape[1]:
        got = f"{x.dtype} {tuple(x.shape)}" if isinstance(x, torch.Tensor) else type(x).__name__
        raise ops.KernelError(f"{what}: x is bfloat16 [rows, {weight.shape[1]}], not {got}")
    if x.data_ptr() % 16:
        raise ops.KernelError(f"{what}: x must be 16-byte aligned")
    bias, code = _bias(what, bias, weight.shape[0])
    _on_device(what, x, weight.blocks, bias)
    return bias, code


def linear_int4(x: torch.Tensor, weight: Int4Weight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows ``x`` [rows, in] bfloat16 times weight [out, in] transposed (+ bias, bfloat16 or float32), summed in float32, in
    bfloat16.  Up to 8 rows the weights are multiplied as they stand; more rows meet them rounded to bfloat16."""
    bias, bias_code = _int4_checked("linear_int4", x, weight, bias)
    (n, k), blocks = weight.shape, weight.blocks
    y = torch.empty_strided((x.shape[0], n), (n, 1), dtype=torch.bfloat16, device=x.device)
    scratch, floats = _scratch("gemm_int4", "fms_linear_int4_scratch", x.device, x.shape[0], n, k)
    ops._call("gemm_int4", "fms_linear_int4", x, blocks, bias, bias_code, y, x.shape[0], n, k, blocks.shape[1], weight.per, scratch, floats,
              ops.error_flag(x.device), ops._stream())
    return y


def gated_linear_int4(x: torch.Tensor, weight: Int4Weight, bias: Optional[torch.Tensor], activation: int) -> torch.Tensor:
    """act(x Wg^T) * (x Wu^T) in bfloat16 for weight = [Wg; Wu]: one kernel for few rows (and a hidden size that is a
    multiple of 16), else the product and ``gated_activation``."""
    bias, bias_code = _int4_checked("gated_linear_int4", x, weight, bias)
    (n, k), blocks = weight.shape, weight.blocks
    if n % 2:
        raise ops.KernelError(f"gated_linear_int4: {n} rows are no gate and up matrix")
    if x.shape[0] > INT4_FEW_ROWS or n % 32:
        return ops.gated_activation(linear_int4(x, weight, bias), activation)
    y = torch.empty((x.shape[0], n // 2), dtype=torch.bfloat16, device=x.device)
    ops._call("gemm_int4", "fms_glu_int4", x, blocks, bias, bias_code, y, x.shape[0], n // 2, k, blocks.shape[1], weight.per, int(activation),
              ops._stream())
    return y


def linear(x, weight, bias: Optional[torch.Tensor], out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    """What ``ops.linear`` does with a quantised weight."""
    if isinstance(weight, E4M3Weight):
        return linear_e4m3(x, weight, bias, out_dtype or torch.bfloat16)
    if out_dtype not in (None, torch.bfloat16):
        raise ops.KernelError(f"linear: the product with 4-bit weights is bfloat16, not {out_dtype}")
    return linear_int4(x, weight, bias)


def gated_linear(x, weight, bias: Optional[torch.Tensor], activation: int) -> torch.Tensor:
    """What ``ops.gated_linear`` does with a quantised weight."""
    return (gated_linear_e4m3 if isinstance(weight, E4M3Weight) else gated_linear_int4)(x, weight, bias, activation)


QUANTIZED_WEIGHTS = (E4M3Weight, Int4Weight)
