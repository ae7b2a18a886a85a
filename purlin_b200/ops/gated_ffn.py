"""The gated feed-forward block with its backward pass (csrc/src/gated_ffn.cu).

    h = act(x @ w_gate.T) * (x @ w_up.T)        one kernel: both projections, the activation and the product
    y = h @ w_down.T

``gated_ffn(x, w_gu, w_down)`` is differentiable in all three arguments; ``w_gu = interleave_gate_up(w_gate, w_up)`` is the weight
that ``gemm_swiglu`` takes, and its gradient has the same order of rows (``split_gate_up`` gives the two parts).
bf16 tensors, fp32 accumulation in tensor memory. Between forward and backward the block keeps ``h`` (bf16) and the pre-activations in
24 bits, together 8 bytes per token and intermediate column.
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext
from typing import Tuple

import torch

from .. import _native, _stream

ACTIVATIONS = {"silu": 0, "gelu": 1}     # gelu: 0.5 g (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3)))
_declared = False


def _lib():
    global _declared
    lib = _native.cuda()
    if not _declared:
        vp, i = C.c_void_p, C.c_int
        lib.purlin_ffn_saved_bytes.argtypes = [i, i]
        lib.purlin_ffn_saved_bytes.restype = C.c_size_t
        lib.purlin_ffn_forward.argtypes = [vp] * 6 + [i] * 4 + [vp, vp]
        lib.purlin_ffn_backward.argtypes = [vp] * 10 + [i] * 4 + [vp, vp]
        _declared = True
    return lib


def _on(device: torch.device):
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


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
    if not (x.is_cuda and w_gu.device == x.device and w_down.device == x.device):
        raise ValueError("operands must be CUDA tensors on one device")
    if not (x.is_contiguous() and w_gu.is_contiguous() and w_down.is_contiguous()):
        raise ValueError("operands must be contiguous")
    if (x.data_ptr() | w_gu.data_ptr() | w_down.data_ptr()) % 16:
        raise ValueError("operands must start on a 16-byte boundary")


def _forward(x, w_gu, w_down, activation, keep):
    """y, h and, where the backward will want them, the pre-activations; x is [tokens, hidden]."""
    tokens, (hidden, intermediate) = x.shape[0], w_down.shape
    y = torch.empty_like(x)
    h = torch.empty(tokens, intermediate, dtype=torch.bfloat16, device=x.device)
    lib = _lib()
    saved = torch.empty(lib.purlin_ffn_saved_bytes(tokens, intermediate), dtype=torch.uint8, device=x.device) if keep else None
    if tokens:
        with _on(x.device):
            rc = lib.purlin_ffn_forward(x.data_ptr(), w_gu.data_ptr(), w_down.data_ptr(), h.data_ptr(), saved.data_ptr() if keep else None,
                                        y.data_ptr(), tokens, hidden, intermediate, ACTIVATIONS[activation], None, _stream(None))
            _native.check(lib, rc)
    return y, h, saved


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gu, w_down, activation):
        need_x, need_gu, need_down = ctx.needs_input_grad[:3]
        y, h, saved = _forward(x, w_gu, w_down, activation, need_x or need_gu)
        ctx.activation = activation
        ctx.save_for_backward(x, w_gu, w_down, h if need_down else None, saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_gu, w_down, h, saved = ctx.saved_tensors
        need_x, need_gu, need_down = ctx.needs_input_grad[:3]
        tokens, (hidden, intermediate) = x.shape[0], w_down.shape
        dx = torch.empty_like(x) if need_x else None
        d_gu = torch.empty_like(w_gu) if need_gu else None
        d_down = torch.empty_like(w_down) if need_down else None
        if tokens == 0:
            return dx, d_gu.zero_() if need_gu else None, d_down.zero_() if need_down else None, None
        dy = dy.contiguous()
        if dy.data_ptr() % 16:
            dy = dy.clone()
        dz = torch.empty(tokens, 2 * intermediate, dtype=torch.bfloat16, device=x.device) if need_x or need_gu else None

        def ptr(t):
            return None if t is None else t.data_ptr()

        lib = _lib()
        with _on(x.device):
            rc = lib.purlin_ffn_backward(x.data_ptr(), w_gu.data_ptr(), w_down.data_ptr(), ptr(h), ptr(saved), dy.data_ptr(), ptr(dz), ptr(dx), ptr(d_gu),
                                         ptr(d_down), tokens, hidden, intermediate, ACTIVATIONS[ctx.activation], None, _stream(None))
            _native.check(lib, rc)
        return dx, d_gu, d_down, None


def gated_ffn(x: torch.Tensor, w_gu: torch.Tensor, w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` for bf16 ``x [..., hidden]``, ``w_gu = interleave_gate_up(w_gate, w_up)``
    ``[2 * intermediate, hidden]`` and ``w_down [hidden, intermediate]``; differentiable once. ``activation``: "silu" or "gelu" (the form
    with the tanh). Where no gradient is asked for, nothing is kept. All tensors contiguous and on one device; hidden a multiple of 8,
    intermediate of 16; any number of tokens, none included."""
    _check(x, w_gu, w_down, activation)
    rows = x.view(-1, x.shape[-1]) if x.numel() else x.reshape(0, x.shape[-1])
    if torch.is_grad_enabled() and (x.requires_grad or w_gu.requires_grad or w_down.requires_grad):
        y = _GatedFfn.apply(rows, w_gu, w_down, activation)
    else:
        y = _forward(rows, w_gu, w_down, activation, False)[0]
    return y.view(x.shape)


def split_gate_up(w_gu: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gate and up parts, [I, K] each, of a weight that ``interleave_gate_up`` made, or of its gradient."""
    if w_gu.dim() != 2 or w_gu.shape[0] % 32:
        raise ValueError("w_gu is [2 * intermediate, hidden], its rows alternating 16 of gate and 16 of up")
    rows, k = w_gu.shape
    v = w_gu.reshape(rows // 32, 2, 16, k)
    return v[:, 0].reshape(rows // 2, k), v[:, 1].reshape(rows // 2, k)
