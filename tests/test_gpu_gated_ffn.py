"""The gated feed-forward block and its gradients against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -8      # half a step of bf16, relative to the value


def _inputs(t, h, i, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(rows, cols, s):
        return (torch.randn(rows, cols, generator=g, device="cuda") * s).to(torch.bfloat16)

    return normal(t, h, scale), normal(2 * i, h, h ** -0.5), normal(h, i, i ** -0.5), normal(t, h, 1.0)


def _parts(x, w_gu, activation):
    z = (x @ w_gu.t()).view(x.shape[0], -1, 2, 16)
    g, u = z[:, :, 0], z[:, :, 1]
    if activation == "silu":
        s, ds = g, torch.ones_like(g)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        s, ds = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
    sig = torch.sigmoid(s)
    return g, u, g * sig, sig + g * sig * (1 - sig) * ds


def _oracle(x, w_gu, w_down, dy, activation):
    """y, dx, dw_gu, dw_down by the formulas in 64 bits, and for each the sum of the magnitudes of its terms."""
    x, w_gu, w_down, dy = (v.double() for v in (x, w_gu, w_down, dy))
    g, u, act, dact = _parts(x, w_gu, activation)
    h = (act * u).flatten(1)
    dh = (dy @ w_down).view_as(g)
    dz = torch.stack([dh * u * dact, dh * act], 2).flatten(1)
    # what dz and h may be off by before their own rounding: the fp32 sums of z and dh (relative to the terms' magnitudes), z's 24 bits
    # and the fast exponential and division; 2^-16 of these magnitudes is above all of them together for sums of up to 2^15 terms
    zmag = (x.abs() @ w_gu.abs().t()).view(x.shape[0], -1, 2, 16)
    gm, um = zmag[:, :, 0], zmag[:, :, 1]
    dhm = (dy.abs() @ w_down.abs()).view_as(g)
    # |act'| <= 1.2 and |act''| <= 1 for both activations; |act(g)| <= |g|
    loose_h = 2.0 ** -15 * (1.2 * gm * u.abs() + act.abs() * um + (act * u).abs())
    loose_dz = 2.0 ** -15 * torch.stack([dhm * (u.abs() * 1.2) + dh.abs() * (1.2 * um + u.abs() * gm), dhm * act.abs() + dh.abs() * 1.2 * gm], 2)
    h_off = STEP * h.abs() + loose_h.flatten(1)
    dz_off = STEP * dz.abs() + loose_dz.flatten(1)
    y, dx, dgu, dd = h @ w_down.t(), dz @ w_gu, dz.t() @ x, dy.t() @ h
    off = (h_off @ w_down.abs().t(), dz_off @ w_gu.abs(), dz_off.t() @ x.abs(), dy.abs().t() @ h_off)
    # the products' own fp32 sums and the result's rounding
    mags = (h.abs() @ w_down.abs().t(), dz.abs() @ w_gu.abs(), dz.abs().t() @ x.abs(), dy.abs().t() @ h.abs())
    out = (y, dx, dgu, dd)
    return out, [a + STEP * (v.abs() + a) + 2.0 ** -17 * m + 1e-30 for v, a, m in zip(out, off, mags)]


def _run(x, w_gu, w_down, dy, activation):
    from purlin_b200.ops.gated_ffn import gated_ffn
    leaves = [v.clone().requires_grad_() for v in (x, w_gu, w_down)]
    y = gated_ffn(*leaves, activation)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


NAMES = ("y", "dx", "dw_gu", "dw_down")


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("t,h,i", [(1, 8, 16), (1, 264, 176), (7, 72, 48), (40, 264, 176), (64, 1024, 512), (127, 200, 144), (128, 136, 272), (129, 520, 1040),
                                   (333, 776, 336), (513, 1000, 528), (1100, 2048, 784), (2051, 264, 1296),
                                   (1, 1024, 4096), (100, 1024, 2048), (300, 424, 8192), (700, 136, 10000), (1500, 264, 4096)])   # few tiles, long sums: dx in parts
def test_outputs_and_gradients_against_64_bits(t, h, i, activation):
    args = _inputs(t, h, i, seed=t + h + i)
    want, off = _oracle(*args, activation)
    for name, got, ref, tol in zip(NAMES, _run(*args, activation), want, off):
        err = (got.double() - ref).abs()
        assert (err <= tol).all(), f"{name}: {(err / tol).max().item()} of what rounding allows"


@pytest.mark.parametrize("t,h,i", [(40, 2048, 1024), (513, 2048, 4096), (2100, 4096, 1024), (4099, 2048, 2048), (9000, 1024, 4096)])
def test_gradients_on_small_integers_are_the_products(t, h, i):
    # Every product of the block, in every order of its operands, exact: with a gate of 128 the sigmoid is 1 (act = g, act' = 1), all values
    # are small whole numbers that bf16 holds, and all sums are exact in fp32.
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.zeros(t, h, device="cuda")
    x[:, :8] = torch.randint(0, 2, (t, 8), generator=g, device="cuda").float()
    x[:, 0] = 1
    w_gu = torch.zeros(2 * i // 32, 2, 16, h, device="cuda")
    w_gu[:, 0, :, 0] = 128.0                                     # the gate: 128 and whole numbers
    w_gu[:, 1, :, :8] = torch.randint(-1, 2, (2 * i // 32, 16, 8), generator=g, device="cuda").float()
    w_gu = w_gu.view(2 * i, h)
    w_down = torch.randint(-1, 2, (h, i), generator=g, device="cuda").float() * (torch.rand(h, i, generator=g, device="cuda") < 0.01)
    dy = torch.randint(-1, 2, (t, h), generator=g, device="cuda").float() * (torch.rand(t, h, generator=g, device="cuda") < 0.02)
    args = [v.to(torch.bfloat16) for v in (x, w_gu, w_down, dy)]
    xd, wd, dd, dyd = (v.double() for v in args)
    z = (xd @ wd.t()).view(t, -1, 2, 16)
    gate, up = z[:, :, 0], z[:, :, 1]
    h_ = (gate * up).flatten(1)
    dh = (dyd @ dd).view_as(gate)
    dz = torch.stack([dh * up, dh * gate], 2).flatten(1)
    assert dz.abs().max() < 2 ** 15 and (dz.to(torch.bfloat16).double() == dz).all() and (h_.to(torch.bfloat16).double() == h_).all()
    want = (h_ @ dd.t(), dz @ wd, dz.t() @ xd, dyd.t() @ h_)
    for name, got, ref in zip(NAMES, _run(*args, "silu"), want):
        assert torch.equal(got.double(), ref.to(torch.bfloat16).double()), name
