"""A bias-free linear map y = a W^T with W stored [outputs, inputs]
(crates/forward/src/loader/shard.rs:81-83)."""
from __future__ import annotations

import torch

from ..kernels import ops


class Linear:
    """`weight`: a tensor, or a weight in a layout of its own (kernels.ops.PackedWeight)."""

    def __init__(self, weight):
        if weight.dim() != 2:
            raise ValueError("a linear weight is 2-d [outputs, inputs]")
        self.weight = weight
        self.packed = isinstance(weight, ops.PackedWeight)
        self.out_features, self.in_features = weight.shape

    def __call__(self, ctx, a: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        ops.linear(a, self.weight, out, ctx)
        return out

    def slabs(self, ctx, a: torch.Tensor, slabs: torch.Tensor) -> int:
        """The product as a sum of float32 slabs (split-K shares that the next kernel adds); returns how many."""
        return ops.linear_slabs(a, self.weight, slabs, ctx)

    def add_into(self, ctx, a: torch.Tensor, acc: torch.Tensor) -> bool:
        """acc += a W^T where the product's own epilogue can do the add (see ops.gemm_tc_add); False, with nothing
        done, where it cannot."""
        return ops.linear_add(a, self.weight, acc, ctx, ctx.max_slabs)


def held(runtime, weight: torch.Tensor):
    """A map's weight ([outputs, inputs] or [groups, outputs, inputs]) as the runtime holds the large maps' weights
    (Runtime.weight_format): as it is, or in four bits; in the 32-bit mode four-bit weights are held as the float32 numbers
    that they stand for."""
    if getattr(runtime, "weight_format", "stored") != "mxfp4":
        return weight
    if runtime.full_precision:
        return ops.dequantize_mxfp4(*ops.quantize_mxfp4(weight.contiguous()), weight.shape[-1], torch.float32)
    return ops.Mxfp4Weight.from_dense(weight)


def held_groups(runtime, weights):
    """`held` of the stacked weights of equal sizes, made one after the other."""
    if getattr(runtime, "weight_format", "stored") == "mxfp4" and not runtime.full_precision:
        rows = [ops.quantize_mxfp4(w.contiguous()) for w in weights]
        return ops.Mxfp4Weight(torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows]), weights[0].shape[-1])
    return torch.stack([held(runtime, w) for w in weights]).contiguous()


def interleave_rows(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Rows a_0, b_0, a_1, b_1, ...: two maps of one input whose outputs are wanted side by side."""
    if a.shape != b.shape or a.dtype != b.dtype:
        raise ValueError("interleaved weights must share shape and dtype")
    return torch.stack([a, b], dim=1).reshape(2 * a.shape[0], a.shape[1]).contiguous()


def concat_rows(tensors) -> torch.Tensor:
    """Stack weights that share their input so one product serves them all."""
    dts = {t.dtype for t in tensors}
    if len(dts) != 1:
        raise ValueError(f"fused weights must share a dtype, got {dts}")
    return torch.cat(list(tensors), dim=0).contiguous()
