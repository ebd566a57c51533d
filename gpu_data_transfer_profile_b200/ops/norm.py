"""Root-mean-square norm in front of a block, with the residual's addition (csrc/norm).

h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight  over the last dimension, in f32; h and y are rounded once, where
they are stored (y is that of the sum before its rounding). Rows are bf16, f16 or f32, of 1 to 32768 elements, any number of
leading dimensions; weights are of the rows' type or f32 (others are taken to f32 first). Two-dimensional inputs may have
rows further apart than their length; other strides are copied. A row's result does not depend on the rows beside it; where
rows are no multiple of 16 bytes long, it may be a rounding apart with the place within 16 bytes at which the row begins.

Calls can be captured into CUDA graphs, with their gradients too; as with every torch operation, let go of eager graphs of
the same leaves before a backward pass is captured.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _ext


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """y, or (y, h) with a residual (shape and type of x): h is the residual of the next block.

    Differentiable once in x, residual and weight. Gradients are computed in f32 and rounded once; the weight's is summed in a
    fixed order. Of 16-bit rows with a residual the backward reads x and residual again where the weight needs a gradient,
    and keeps both until then; else it reads h as it was stored, a rounding of h in the second term of x's gradient. No
    forward-mode derivatives, no function transforms, no tracing (refused)."""
    y, h = _ext.load().rms_norm(x, weight, residual, eps)
    return y if residual is None else (y, h)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 keep: bool = False) -> Tuple[Tuple[torch.Tensor, torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """-> ((q e4m3 [..., H], scales f32 [..., H/128]), y, h): what `Buffer.dispatch` takes in place of rows and
    `ops.gemm.grouped_gemm_fp8` multiplies; scale = max(amax, 1e-4) / 448 of 128 channels of y, as in the cast of an fp8
    dispatch, here of y before its rounding. y in the type of x if `keep` (for a router beside the experts), else None; h is
    None without a residual. H is a multiple of 128. NaN stays NaN in q and takes no part in its block's scale; a block with
    an infinite y has an infinite scale. For inference: refuses inputs that require a gradient."""
    q, scales, y, h = _ext.load().rms_norm_fp8(x, weight, residual, eps, keep)
    return (q, scales), y, h
