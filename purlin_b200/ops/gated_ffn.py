"""The gated feed-forward block with its backward pass (csrc/src/gated_ffn.cu, csrc/src/torch_ops.cpp).

    h = act(x @ w_gate.T) * (x @ w_up.T)        one kernel: both projections, the activation and the product
    y = h @ w_down.T

``gated_ffn(x, w_gu, w_down)`` is differentiable in all three arguments; ``w_gu = interleave_gate_up(w_gate, w_up)`` is the weight
that ``gemm_swiglu`` takes, and its gradient has the same order of rows (``split_gate_up`` gives the two parts).
bf16 tensors, fp32 accumulation in tensor memory. Between forward and backward the block keeps ``h`` (bf16) and the pre-activations in
24 bits, together 8 bytes per token and intermediate column. Waits inside the kernels are bounded: see ``ops.waits``.
"""
from __future__ import annotations

from typing import Tuple

import torch

from .. import _native

ACTIVATIONS = {"silu": 0, "gelu": 1}     # gelu: 0.5 g (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3)))


def _check(x: torch.Tensor, w_gu: torch.Tensor, w_down: torch.Tensor, activation: str):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}")
    if x.dtype != torch.bfloat16 or w_gu.dtype != torch.bfloat16 or w_down.dtype != torch.bfloat16:
        raise TypeError("the gated feed-forward block takes bf16 operands")
    if w_gu.dim() != 2 or w_down.dim() != 2 or x.dim() < 1:
        raise ValueError("x is [..., hidden], w_gu is [2 * intermediate, hidden] and w_down is [hidden, intermediate]")
    hidden, intermediate = w_down.shape
    if x.shape[-1] != hidden or tuple(w_gu.shape) != (2 * intermediate, hidden):
        raise ValueError("x is [..., hidden], w_gu is [2 * intermediate, hidden] and w_down is [hidden, intermediate]")
    if hidden == 0 or intermediate == 0 or hidden % 8 or intermediate % 16:
        raise ValueError("hidden must be a multiple of 8 and intermediate of 16")
    if max(x.numel() // hidden, hidden, intermediate) >= 2 ** 29:
        raise ValueError("tokens, hidden and intermediate must be below 2^29")
    if not (x.is_cuda and w_gu.device == x.device and w_down.device == x.device):
        raise ValueError("operands must be CUDA tensors on one device")
    if not (x.is_contiguous() and w_gu.is_contiguous() and w_down.is_contiguous()):
        raise ValueError("operands must be contiguous")
    if (x.data_ptr() | w_gu.data_ptr() | w_down.data_ptr()) % 16:
        raise ValueError("operands must start on a 16-byte boundary")


def gated_ffn(x: torch.Tensor, w_gu: torch.Tensor, w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` for bf16 ``x [..., hidden]``, ``w_gu = interleave_gate_up(w_gate, w_up)``
    ``[2 * intermediate, hidden]`` and ``w_down [hidden, intermediate]``; differentiable once, in reverse mode (a forward-mode derivative is refused). ``activation``: "silu" or "gelu" (the form
    with the tanh). Where no gradient is asked for, nothing is kept. All tensors contiguous and on one device; hidden a multiple of 8,
    intermediate of 16; any number of tokens below 2^29, none included. Forward and backward can be captured into a
    CUDA graph; there use ``torch.autograd.grad``, because ``backward()`` accumulates on the stream on which an earlier graph of the same leaves,
    if it is still alive, was made."""
    _check(x, w_gu, w_down, activation)
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    y = _native.torch_ops().gated_ffn(rows, w_gu, w_down, ACTIVATIONS[activation])
    return y if x.dim() == 2 else y.view(x.shape)


def split_gate_up(w_gu: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gate and up parts, [I, K] each, of a weight that ``interleave_gate_up`` made, or of its gradient."""
    if w_gu.dim() != 2 or w_gu.shape[0] % 32:
        raise ValueError("w_gu is [2 * intermediate, hidden], its rows alternating 16 of gate and 16 of up")
    rows, k = w_gu.shape
    v = w_gu.reshape(rows // 32, 2, 16, k)
    return v[:, 0].reshape(rows // 2, k), v[:, 1].reshape(rows // 2, k)
