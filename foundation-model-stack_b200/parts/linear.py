"""A linear map y = x W^T (+ b) with W stored [out, in] as checkpoints store it
(the reference's ``get_linear`` default, fms/modules/linear.py:119-156), or quantised when it is loaded.

Option ``linear_type`` (the reference's ``linear_config["linear_type"]``, fms/modules/linear.py:11-156):

    "torch_linear"   W as it is stored
    "fp8"            W in e4m3 with one scale an output channel, and the rows of x in e4m3 with one scale each
    "int4"           W in 4 bits with a scale and a zero point for every ``group_size`` (128) input channels, x in bfloat16

The last two compute in bfloat16 models only.  What the checkpoint stores is rounded to the nearest as each matrix is loaded
(``ops.quantize_e4m3``, ``ops.quantize_int4``)."""
from __future__ import annotations

import torch

from ..kernels import ops
from .base import Part

LINEAR_TYPES = ("torch_linear", "fp8", "int4")


def linear_options(linear_config) -> tuple:
    """A configuration's ``linear_config`` as options of the specs; () for layers as they are stored."""
    values = dict(linear_config or {})
    kind = values.pop("linear_type", "torch_linear")
    if kind not in LINEAR_TYPES:
        raise ValueError(f"linear_type {kind!r} is not supported; supported: {list(LINEAR_TYPES)}")
    group = values.pop("group_size", 128) if kind == "int4" else 128
    if values or isinstance(group, bool) or not isinstance(group, int) or group <= 0 or group % 32:
        raise ValueError(f"linear_config {dict(linear_config)}: \"int4\" takes a group_size that is a multiple of 32, and nothing else is taken")
    return () if kind == "torch_linear" else (("linear_type", kind), ("group_size", group))


class Linear(Part):
    def __init__(self, in_features: int, out_features: int, bias: bool = False, options=()) -> None:
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.linear_type = dict(options).get("linear_type", "torch_linear")
        self.group_size = int(dict(options).get("group_size", 128))
        if self.linear_type not in LINEAR_TYPES:
            raise ValueError(f"linear_type {self.linear_type!r} is not supported; supported: {list(LINEAR_TYPES)}")
        if self.linear_type == "int4" and in_features % 8:
            raise ValueError(f"linear_type 'int4' needs input channels in a multiple of 8, not {in_features}")
        self.declare("weight", (out_features, in_features), role="matrix")
        if bias:
            self.declare("bias", (out_features,), role="vector")

    def set_tensor(self, name, value) -> None:
        super().set_tensor(name, value)
        if name == "weight" and self.linear_type == "fp8":
            self._tensors[name] = ops.quantize_e4m3(value)
        elif name == "weight" and self.linear_type == "int4":
            self._tensors[name] = ops.quantize_int4(value, self.group_size)

    def finalize(self, device, dtype) -> None:
        super().finalize(device, dtype)
        if self.linear_type != "torch_linear" and dtype != torch.bfloat16:
            raise ValueError(f"linear_type {self.linear_type!r} computes in bfloat16, not {dtype}")

    @property
    def takes_quantized_rows(self) -> bool:
        """Whether x may come as ``ops.QuantizedRows``."""
        return self.linear_type == "fp8"

    def by_sequence(self) -> bool:
        """Whether the product chooses its kernel by the sequences that its rows belong to (large float32 matrices)."""
        w = self.tensor("weight")
        return self.linear_type == "torch_linear" and w.dtype == torch.float32 and ops.f32_split_tokens(w) > 0

    def forward(self, x, out_dtype=None, sequences=None):
        """``sequences``: the rows' ``Batch`` or how many rows each sequence has, one behind the other; None: every row stands alone."""
        if sequences is not None and self.by_sequence():
            return ops.linear(x, self.tensor("weight"), self.tensor("bias"), out_dtype, sequences)
        return ops.linear(x, self.tensor("weight"), self.tensor("bias"), out_dtype)

    def kernel_libraries(self, dtype):
        if self.linear_type != "torch_linear":
            return ["quantize_rows", "gemm_e4m3"] if self.linear_type == "fp8" else ["gemm_int4"]
        w = self.tensor("weight")
        if dtype == torch.float32 or (w is not None and w.dtype == torch.float32):
            return ["gemm_f32"] + (["gemm_f32_tc"] if w is None or ops.f32_split_tokens(w) else [])
        return ["gemm_bf16_skinny", "gemm_bf16_tc"] + (["gemm_bf16_mid"] if ops.USE_MID_GEMM else [])
