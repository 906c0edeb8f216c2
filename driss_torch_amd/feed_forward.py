"""The operators of a gated feed-forward block between two norms, trained in bf16 and served with 8-bit integer
products.  A weight has a linear layer's layout, one row per output channel.  ``gated_linear`` and the norms have
gradients (of first order, in reverse mode); everything runs on the current stream of its inputs' device."""
from typing import Optional, Tuple

import torch

_ops = torch.ops.DrissTorch
Tensor = torch.Tensor

__all__ = ["int8_quantize", "int8_bf16", "gated_linear", "pre_norm", "post_norm", "post_pre_norm"]


def int8_quantize(input: Tensor) -> Tuple[Tensor, Tensor]:
    """Symmetric 8-bit integers with one scale per row: ``(q int8 [R, C], scale fp32 [R, 1])`` for bf16 or fp32
    ``input`` [R, C], contiguous.  ``c = max(amax, 1e-12)``, ``scale = c / 127``, ``q = round(input * (127 / c))`` in
    fp32, so that ``input`` is about ``q * scale``.  A row with an infinity or a NaN gets an infinite or NaN scale and
    zero codes: products with it are NaN.  Rows are tokens of activations, or output channels of a weight."""
    return _ops.int8_quantize(input)


def int8_bf16(a: Tensor, b: Tensor, a_scale: Tensor, b_scale: Tensor) -> Tensor:
    """bf16 ``(a @ b) * a_scale * b_scale`` for int8 operands with an fp32 scale per row of ``a`` and per column of
    ``b``, the sums taken in 32-bit integers (K < 131072).

    a: [M, K] row-major; b: [K, N] with stride(0) == 1 (an [N, K] weight transposed).  Rows may lie further apart than
    K.  a_scale and b_scale have M and N elements."""
    return _ops.int8_bf16(a, b, a_scale, b_scale)


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, activation: str = "silu") -> Tensor:
    """``act(x @ w_gate.t()) * (x @ w_up.t())`` in bf16, with sums, activation and product in fp32 and one rounding.

    x: [..., D]; w_gate, w_up: [F, D]; ``activation``: "silu", "gelu" or "gelu_tanh".  For the gradients both
    products are kept in fp32, 8 bytes an element of the result; their own gradients are rounded to bf16 before they are
    multiplied with x and the weights."""
    return _ops.gated_linear(x, w_gate, w_up, activation)


def pre_norm(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    """The RMS norm before a block: ``weight * x / sqrt(mean(x^2) + eps)`` over the last dimension, in fp32 and
    rounded once to x's dtype, bf16 or fp32, which ``weight`` shares."""
    return _ops.pre_norm(x, weight, eps)


def post_norm(residual: Tensor, branch: Tensor, weight: Tensor, gate: Optional[Tensor] = None, residual_scale: float = 1.0,
              eps: float = 1e-6) -> Tensor:
    """The RMS norm after a block and its way into the residual stream:
    ``residual + residual_scale * gate * (weight * branch / sqrt(mean(branch^2) + eps))``.

    residual, branch: [..., C]; gate: [C] or [..., C], whose rows are taken by equal shares of the residual's rows in
    turn: one for all rows, one per sequence (``[B, C]``, of whatever T, or ``[B, 1, C]`` with residual [B, T, C]), or one
    per row.  A shape that broadcasts to the residual's in another way (``[T, C]`` or ``[1, T, C]``, a row per
    position) is refused: expand it."""
    return _ops.post_norm(residual, branch, weight, gate, residual_scale, eps)


def post_pre_norm(residual: Tensor, branch: Tensor, post_weight: Tensor, pre_weight: Tensor, gate: Optional[Tensor] = None,
                  residual_scale: float = 1.0, eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    """Between two blocks: ``r = post_norm(residual, branch, post_weight, gate, residual_scale, eps)`` and
    ``pre_norm(r, pre_weight, eps)`` from one pass over the rows, the second from r before its rounding, as
    the gradients take it too.  For those ``residual`` (bf16) or r (fp32) is kept and may not change in place meanwhile."""
    return _ops.post_pre_norm(residual, branch, post_weight, pre_weight, gate, residual_scale, eps)
