"""The gated MLP block on one GPU: trained in bf16, served in 4 bits.

``GatedMLP`` is the block of ``models.tp_mlp`` (at a degree of one, or a rank's share of it) with gradients; ``GatedMLP.quantized()`` is the same
block with 4-bit microscaled weights and activations, for any number of tokens from one decoded token on.
"""
from __future__ import annotations

from typing import Optional

import torch

from ..ops.gated_ffn import gated_ffn
from ..ops.gemm import interleave_gate_up
from ..ops.mx4 import Mx4Tensor, mx4_gemm, mx4_gemm_swiglu, quantize_mx4


class GatedMLP(torch.nn.Module):
    """``(act(x Wg^T) * (x Wu^T)) Wd^T`` with ``w_gu`` (16 rows of gate and 16 of up in turn, see ``interleave_gate_up``) and ``w_down`` as parameters."""

    def __init__(self, hidden: int = 8192, intermediate: int = 28672, activation: str = "silu", device=None, seed: int = 3):
        super().__init__()
        self.hidden, self.intermediate, self.activation = hidden, intermediate, activation
        dev = torch.device(device if device is not None else "cuda")
        g = torch.Generator(device=dev).manual_seed(seed)

        def init(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=dev) * 0.02).to(torch.bfloat16)

        self.w_gu = torch.nn.Parameter(interleave_gate_up(init(intermediate, hidden), init(intermediate, hidden)))
        self.w_down = torch.nn.Parameter(init(hidden, intermediate))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_ffn(x, self.w_gu, self.w_down, self.activation)

    def quantized(self) -> "Mx4MLP":
        if self.activation != "silu":
            raise ValueError("the 4-bit block has the SwiGLU epilogue only")
        return Mx4MLP(quantize_mx4(self.w_gu.detach()), quantize_mx4(self.w_down.detach()))


class Mx4MLP:
    """The block with 4-bit weights: the activations of both products are quantised as they come, so ``hidden`` and the intermediate size are
    multiples of 32."""

    def __init__(self, w_gu: Mx4Tensor, w_down: Mx4Tensor):
        if w_gu.shape != (2 * w_down.shape[1], w_down.shape[0]):
            raise ValueError("w_gu is [2 * intermediate, hidden] and w_down is [hidden, intermediate]")
        self.w_gu, self.w_down = w_gu, w_down

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        return mx4_gemm(mx4_gemm_swiglu(x, self.w_gu), self.w_down, out)


def smoke_gated_mlp():
    """A tiny training step on one GPU against fp32 autograd, then the block in 4 bits."""
    from ..ops.gated_ffn import split_gate_up
    mlp = GatedMLP(hidden=512, intermediate=1024, device="cuda:0")
    g = torch.Generator(device="cuda:0").manual_seed(3)
    x = torch.randn(200, 512, generator=g, device="cuda:0").to(torch.bfloat16)
    y = mlp(x)
    y.backward(torch.ones_like(y))
    gate, up = (w.detach().float().requires_grad_() for w in split_gate_up(mlp.w_gu))
    down = mlp.w_down.detach().float().requires_grad_()
    ref = (torch.nn.functional.silu(x.float() @ gate.t()) * (x.float() @ up.t())) @ down.t()
    ref.backward(torch.ones_like(ref))
    d_gate, d_up = split_gate_up(mlp.w_gu.grad)
    served = mlp.quantized()(x)
    torch.cuda.synchronize()
    for got, want in ((y, ref), (d_gate, gate.grad), (d_up, up.grad), (mlp.w_down.grad, down.grad)):
        err = ((got.float() - want).norm() / want.norm()).item()
        assert err < 1e-2, f"gated MLP smoke mismatch: {err}"
    assert torch.isfinite(served).all()
