"""Layer norm of any row width, forward and backward, on sm_100a.

``fused.ln_shift_mix`` covers the blocks' LayerNorm together with the token shift
(float32 rows of 128 to 1024 channels, bf16 outputs). ``layer_norm`` is the plain
one, for any width up to 16384, float32, bfloat16 and float16 rows, float32
statistics and parameters: ``y = (x - mean) * rstd * weight + bias``. The backward
sums the parameters' gradients over the rows in a fixed order, and a row's result
does not depend on the pitch or alignment it lies at.
"""

from __future__ import annotations

from torch import Tensor

from ._native import ops


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """Layer norm of ``x`` [..., C] (CUDA, float32 / bfloat16 / float16, C <= 16384)
    over its last dimension, in x's dtype; weight and bias [C] (used in float32)
    or None. Differentiable in x, weight and bias. Rows need unit stride of the
    last index (others are copied); any row pitch is read in place. Raises
    ValueError for shapes and dtypes it does not take and NotImplementedError for
    tensors that are not on CUDA."""
    return ops.layer_norm(x, weight, bias, eps)
