"""A training step of the gated MLP block, then the same block served in 4 bits: python examples/gated_mlp.py [tokens hidden intermediate]

Prints how far the gradients are from fp32 ones and how far the 4-bit block is from the bf16 one (relative 2-norms)."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from purlin_b200.models.gated_mlp import GatedMLP  # noqa: E402
from purlin_b200.ops.gated_ffn import split_gate_up  # noqa: E402

tokens, hidden, intermediate = (int(v) for v in sys.argv[1:4]) if len(sys.argv) >= 4 else (1000, 2048, 4096)
mlp = GatedMLP(hidden, intermediate, device="cuda")
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16)
target = torch.randn(tokens, hidden, generator=g, device="cuda")


def off(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


loss = (mlp(x).float() - target).square().mean()
loss.backward()

gate, up = (w.detach().float().requires_grad_() for w in split_gate_up(mlp.w_gu))
down = mlp.w_down.detach().float().requires_grad_()
reference = ((torch.nn.functional.silu(x.float() @ gate.t()) * (x.float() @ up.t())) @ down.t() - target).square().mean()
reference.backward()
d_gate, d_up = split_gate_up(mlp.w_gu.grad)
errors = [off(d_gate, gate.grad), off(d_up, up.grad), off(mlp.w_down.grad, down.grad)]
print("loss %.6f (fp32 %.6f)" % (float(loss.detach()), float(reference.detach())))
print("gradients off by " + " ".join("%.4f" % e for e in errors))

torch.optim.SGD(mlp.parameters(), lr=0.1).step()
served = mlp.quantized()
with torch.no_grad():
    whole = mlp(x)
    for rows in (1, tokens):
        print("4 bits, %d tokens: off by %.3f" % (rows, off(served(x[:rows]), whole[:rows])))
torch.cuda.synchronize()
assert max(errors) < 0.02
print("ok")
