"""Operators of the gated feed-forward block beyond its bf16 inference form, as they are used and in plain form.

Three kinds of work, each over the range it is used in:

  ffn        a training step of the gated block: ``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` and, from ``dy``, the gradients of the
             input and of both weights (hidden 8192, intermediate 28672 or the share of a rank, or an expert of 7168 / 2048)
  quantize   rows of activations or weights to microscaled 4-bit values (32 values of two bits of exponent and one of mantissa
             share a power of two), and back to the values that those stand for
  product    activations, quantised in the call, times weights that were quantised before, with or without the gate and
             the product of its epilogue: the projections of the block when it serves

``run`` with ``own`` false computes them with elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a handful of tokens through a small block: launches and latency
        {"name": "ffn_step_40", "kind": "ffn", "tokens": 40, "hidden": 264, "intermediate": 176, "activation": "silu"},
        # a micro-batch that is no multiple of a tile on the share of one rank at TP = 8
        {"name": "ffn_step_1000_tp8", "kind": "ffn", "tokens": 1000, "hidden": 8192, "intermediate": 3584, "activation": "silu"},
        # the rows of one expert of the MoE layer, an odd number of them, with the other activation
        {"name": "ffn_step_4099_expert", "kind": "ffn", "tokens": 4099, "hidden": 7168, "intermediate": 2048, "activation": "gelu"},
        # the whole block of bench.py as a training step
        {"name": "ffn_step_8192_block", "kind": "ffn", "tokens": 8192, "hidden": 8192, "intermediate": 28672, "activation": "silu"},
        # one decoded token's activations
        {"name": "quantize_1x8192", "kind": "quantize", "rows": 1, "cols": 8192, "dtype": "bf16"},
        # an odd decode batch of half-precision activations
        {"name": "quantize_333x7168_fp16", "kind": "quantize", "rows": 333, "cols": 7168, "dtype": "fp16"},
        # the activations of a prefill
        {"name": "quantize_8192x8192", "kind": "quantize", "rows": 8192, "cols": 8192, "dtype": "bf16"},
        # master weights of a rank's gate and up projections
        {"name": "quantize_14336x8192_fp32", "kind": "quantize", "rows": 14336, "cols": 8192, "dtype": "fp32"},
        # one decoded token through gate and up of one rank at TP = 8: bound by reading the weights
        {"name": "product_1_gated_tp8", "kind": "product", "tokens": 1, "n": 7168, "k": 8192, "gated": True},
        # a decode batch through the whole down projection
        {"name": "product_64_down", "kind": "product", "tokens": 64, "n": 8192, "k": 28672, "gated": False},
        # a chunk of a prompt that is no multiple of a tile, gate and up at TP = 4
        {"name": "product_1000_gated_tp4", "kind": "product", "tokens": 1000, "n": 14336, "k": 8192, "gated": True},
        # a prefill through gate and up of the whole block
        {"name": "product_8192_gated", "kind": "product", "tokens": 8192, "n": 57344, "k": 8192, "gated": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "quantize", "product", "product"])
    if kind == "ffn":
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "hidden": 8 * _log(rng, 16, 1024), "intermediate": 16 * _log(rng, 8, 1792),
                "activation": rng.choice(["silu", "gelu"])}
    if kind == "quantize":
        return {"kind": kind, "rows": _log(rng, 1, 14336), "cols": 32 * _log(rng, 8, 256), "dtype": rng.choice(sorted(DTYPES))}
    return {"kind": kind, "tokens": _log(rng, 1, 8192), "n": 32 * _log(rng, 8, 1792), "k": 32 * _log(rng, 8, 256), "gated": rng.random() < 0.5}


def _inputs(case, seed):
    """The tensors a program holds before the call, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(rows, cols, scale, dtype=torch.bfloat16):
        return torch.randn(rows, cols, generator=g, device="cuda").mul_(scale).to(dtype)

    def activations(rows, cols, dtype):
        """N(0, 1), with a few channels that are tens of times larger, as hidden states have them."""
        x = torch.randn(rows, cols, generator=g, device="cuda")
        loud = torch.rand(cols, generator=g, device="cuda") < 0.005
        return torch.where(loud, x * 30, x).to(dtype)

    if case["kind"] == "ffn":
        t, h, i = case["tokens"], case["hidden"], case["intermediate"]
        return {"x": normal(t, h, 1.0), "w_gu": normal(2 * i, h, h ** -0.5), "w_down": normal(h, i, i ** -0.5), "dy": normal(t, h, 1.0)}
    if case["kind"] == "quantize":
        x = normal(case["rows"], case["cols"], 0.02, torch.float32) if case["dtype"] == "fp32" else activations(case["rows"], case["cols"], DTYPES[case["dtype"]])
        return {"x": x}
    return {"x": activations(case["tokens"], case["k"], torch.bfloat16), "w": normal(case["n"], case["k"], case["k"] ** -0.5)}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["kind"] == "ffn" and own:
        for name in ("x", "w_gu", "w_down"):
            state[name].requires_grad_()
    if case["kind"] == "product":
        # a server quantises its weights once
        w = state.pop("w")
        if own:
            from purlin_b200.ops.mx4 import quantize_mx4
            state["w"] = quantize_mx4(w)
        else:
            state["w"] = _mx4_values(w)
    return state


def run(state):
    case = state["case"]
    if case["kind"] == "ffn":
        return (_ffn_own if own else _ffn_plain)(state["x"], state["w_gu"], state["w_down"], state["dy"], case["activation"])
    if case["kind"] == "quantize":
        if own:
            from purlin_b200.ops.mx4 import quantize_mx4
            return quantize_mx4(state["x"]).dequantize()
        return _mx4_values(state["x"]).to(torch.bfloat16)
    if own:
        from purlin_b200.ops.mx4 import mx4_gemm, mx4_gemm_swiglu
        return (mx4_gemm_swiglu if case["gated"] else mx4_gemm)(state["x"], state["w"])
    y = _mx4_values(state["x"]) @ state["w"].t()
    if case["gated"]:
        gate, up = _halves(y)
        y = (gate / (1 + torch.exp(-gate)) * up).flatten(1)
    return y.to(torch.bfloat16)


def _ffn_own(x, w_gu, w_down, dy, activation):
    from purlin_b200.ops.gated_ffn import gated_ffn
    y = gated_ffn(x, w_gu, w_down, activation)
    return (y.detach(), *torch.autograd.grad(y, (x, w_gu, w_down), dy))


def _halves(z):
    """Gate and up columns of ``z [rows, 2 I]`` whose columns alternate 16 of gate and 16 of up, as [rows, I / 16, 16] each."""
    z = z.view(z.shape[0], -1, 2, 16)
    return z[:, :, 0], z[:, :, 1]


def _ffn_plain(x, w_gu, w_down, dy, activation):
    x, w_gu, w_down, dy = x.float(), w_gu.float(), w_down.float(), dy.float()
    gate, up = _halves(x @ w_gu.t())
    if activation == "silu":
        s, ds = gate, 1.0
    else:                      # gelu with the tanh: g (1 + tanh(v)) / 2 = g sigmoid(2 v)
        c = 2 * math.sqrt(2 / math.pi)
        s, ds = c * (gate + 0.044715 * gate ** 3), c * (1 + 3 * 0.044715 * gate ** 2)
    sig = 1 / (1 + torch.exp(-s))
    act = gate * sig
    h = (act * up).flatten(1)
    y = h @ w_down.t()
    dh = (dy @ w_down).view_as(gate)
    dz = torch.stack([dh * up * (sig + act * (1 - sig) * ds), dh * act], 2).flatten(1)
    return tuple(v.to(torch.bfloat16) for v in (y, dz @ w_gu, dz.t() @ x, dy.t() @ h))


def _mx4_values(x):
    """What 32 values to a block, with a shared power of two and four bits each, hold of ``x``, in fp32. The power is that of the
    block's largest magnitude over 4 (the power of the format's largest value, 6), at least 2^-127; a value becomes the
    nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even code. In 64 bits, where the division is exact."""
    b = x.double().view(x.shape[0], -1, 32)
    exponent = torch.frexp(b.abs().amax(2, keepdim=True))[1].long() - 1 - 2
    scale = ((exponent.clamp(min=-127) + 1023) << 52).view(torch.float64)
    m = b.abs() / scale
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp(max=6.0)
    return torch.copysign(m * scale, b).float().flatten(1)


def work(case):
    if case["kind"] == "ffn":
        t, h, i = case["tokens"], case["hidden"], case["intermediate"]
        # x, dy, y, dx; the weights read and their gradients written
        return {"bytes": 2 * (4 * t * h + 6 * h * i), "flops": 18 * t * h * i}
    if case["kind"] == "quantize":
        n = case["rows"] * case["cols"]
        # the values read, 4 bits and a 32nd of a byte each written, the bf16 values written
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + n * 17 // 32 + 2 * n, "flops": 4 * n}
    t, n, k = case["tokens"], case["n"], case["k"]
    return {"bytes": 2 * t * k + n * k * 17 // 32 + 2 * t * (n // 2 if case["gated"] else n), "flops": 2 * t * n * k}


def _mx4_exact(x):
    """The same blocks from the list of the values: the nearest one in 64 bits, the even code where two are as near."""
    x = x.double()
    rows, cols = x.shape
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    between = (grid[1:] + grid[:-1]) / 2
    powers = torch.tensor([2.0 ** e for e in range(-127, 129)], dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for r in range(0, rows, 1024):
        b = x[r:r + 1024].view(-1, cols // 32, 32)
        # the largest power of two that is not above a quarter of the peak, or the smallest one of the format
        quarter = b.abs().max(2, keepdim=True).values / 4
        unit = powers[(torch.searchsorted(powers, quarter, right=True) - 1).clamp(min=0)]
        m = b.abs() / unit
        low, high = torch.bucketize(m, between), torch.bucketize(m, between, right=True)   # they differ where two values are as near
        code = torch.where(low % 2 == 0, low, high)
        out[r:r + 1024] = (torch.sign(b) * grid[code] * unit).view(-1, cols)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "quantize":
        return _mx4_exact(s["x"])
    if case["kind"] == "product":
        y = _mx4_exact(s["x"]) @ _mx4_exact(s["w"]).t()
        if case["gated"]:
            y = y.view(y.shape[0], -1, 32)
            y = (torch.nn.functional.silu(y[..., :16]) * y[..., 16:]).reshape(y.shape[0], -1)
        return y
    leaves = [s[name].double().requires_grad_() for name in ("x", "w_gu", "w_down")]
    x, w_gu, w_down = leaves
    w = w_gu.view(-1, 2, 16, w_gu.shape[1])
    gate, up = x @ w[:, 0].reshape(-1, w_gu.shape[1]).t(), x @ w[:, 1].reshape(-1, w_gu.shape[1]).t()
    act = torch.nn.functional.silu(gate) if case["activation"] == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
    y = (act * up) @ w_down.t()
    return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double()))
