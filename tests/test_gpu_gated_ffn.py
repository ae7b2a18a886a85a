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


def test_gradients_against_differences():
    # The formula's gradient (64 bits) against central differences of the definition, and the kernels' against the same: the derivative along a
    # direction of all three arguments, whose bf16 gradients are off by what the first test allows.
    from purlin_b200.ops.gated_ffn import gated_ffn
    for activation in ("silu", "gelu"):
        x, w_gu, w_down, dy = _inputs(33, 72, 48, seed=9)
        args = [v.double() for v in (x, w_gu, w_down)]
        g = torch.Generator(device="cuda").manual_seed(1)
        way = [torch.randn(v.shape, generator=g, device="cuda", dtype=torch.float64) for v in args]

        def loss(step):
            a, b, c = (v + step * d for v, d in zip(args, way))
            z = (a @ b.t()).view(a.shape[0], -1, 2, 16)
            act = torch.nn.functional.silu(z[:, :, 0]) if activation == "silu" else torch.nn.functional.gelu(z[:, :, 0], approximate="tanh")
            return (((act * z[:, :, 1]).flatten(1) @ c.t()) * dy.double()).sum()

        e = 2.0 ** -12
        slope = (loss(e) - loss(-e)) / (2 * e)
        want, off = _oracle(x, w_gu, w_down, dy, activation)
        along = sum((v * d).sum() for v, d in zip(want[1:], way))
        assert abs(along - slope) <= 1e-4 * abs(slope) + 1e-3          # the differences' error is of the order of e^2
        got = _run(x, w_gu, w_down, dy, activation)
        mine = sum((v.double() * d).sum() for v, d in zip(got[1:], way))
        assert abs(mine - along) <= sum((t * d.abs()).sum() for t, d in zip(off[1:], way))


@pytest.mark.parametrize("mask", range(1, 8))
@pytest.mark.parametrize("t,h,i", [(100, 264, 2048), (700, 520, 272)])
def test_only_the_gradients_that_are_asked_for(t, h, i, mask):
    from purlin_b200.ops.gated_ffn import gated_ffn
    args = _inputs(t, h, i, seed=4)
    want, off = _oracle(*args, "silu")
    leaves = [v.clone().requires_grad_(bool(mask >> n & 1)) for n, v in enumerate(args[:3])]
    y = gated_ffn(*leaves)
    y.backward(args[3])
    for n, leaf in enumerate(leaves):
        if mask >> n & 1:
            assert ((leaf.grad.double() - want[n + 1]).abs() <= off[n + 1]).all()
        else:
            assert leaf.grad is None


def test_some_of_the_gradients_and_a_second_pass_over_a_kept_graph():
    from purlin_b200.ops.gated_ffn import gated_ffn
    args = _inputs(300, 264, 528, seed=14)
    want, off = _oracle(*args, "silu")
    leaves = [v.clone().requires_grad_() for v in args[:3]]
    y = gated_ffn(*leaves)
    first = torch.autograd.grad(y, leaves, args[3], retain_graph=True)
    for n in range(3):
        (one,) = torch.autograd.grad(y, leaves[n], args[3], retain_graph=True)
        assert ((one.double() - want[n + 1]).abs() <= off[n + 1]).all()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, args[3]), first))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, args[3])


def test_under_checkpointing_and_from_threads():
    # the forward runs again in the backward's thread; two host threads call at once, each on a stream of its own
    import threading

    from torch.utils.checkpoint import checkpoint

    from purlin_b200.ops.gated_ffn import gated_ffn
    args = _inputs(300, 264, 528, seed=15)
    want = _run(*args, "silu")
    for reentrant in (False, True):
        leaves = [v.clone().requires_grad_() for v in args[:3]]
        y = checkpoint(gated_ffn, *leaves, use_reentrant=reentrant)
        y.backward(args[3])
        assert all(torch.equal(p.grad, q) for p, q in zip(leaves, want[1:]))
    others = [_inputs(100 + 50 * n, 264, 272, seed=16 + n) for n in range(2)]
    wants = [_run(*a, "gelu") for a in others]
    torch.cuda.synchronize()
    right = [0, 0]

    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _run(*others[n], "gelu")
                torch.cuda.current_stream().synchronize()
                right[n] += all(torch.equal(p, q) for p, q in zip(got, wants[n]))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert right == [20, 20]


def test_without_gradients_nothing_is_kept_and_the_values_are_the_same_operator():
    from purlin_b200.ops.gated_ffn import gated_ffn
    for activation in ("silu", "gelu"):
        for t in (1, 100, 700):
            args = _inputs(t, 264, 272, seed=t)
            want, off = _oracle(*args, activation)
            leaves = [v.clone().requires_grad_() for v in args[:3]]
            with torch.no_grad():
                y = gated_ffn(*leaves, activation)
            assert not y.requires_grad and ((y.double() - want[0]).abs() <= off[0]).all()


def test_shapes_of_batches_one_token_and_none():
    from purlin_b200.ops.gated_ffn import gated_ffn
    x, w_gu, w_down, dy = _inputs(30, 72, 48, seed=2)
    want = _run(x, w_gu, w_down, dy, "silu")
    b = x.view(2, 5, 3, 72).clone().requires_grad_()
    w = [v.clone().requires_grad_() for v in (w_gu, w_down)]
    y = gated_ffn(b, *w)
    assert y.shape == b.shape and torch.equal(y.flatten(0, 2), want[0])
    grads = torch.autograd.grad(y, (b, *w), dy.view(2, 5, 3, 72))
    assert grads[0].shape == b.shape and all(torch.equal(p.reshape(q.shape), q) for p, q in zip(grads, want[1:]))
    one = x[7].clone().requires_grad_()                  # a vector
    assert gated_ffn(one, w_gu, w_down).shape == (72,)
    for shape in ((0, 72), (4, 0, 72)):
        empty = torch.empty(shape, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = gated_ffn(empty, *w)
        assert y.shape == shape
        dx, d_gu, d_down = torch.autograd.grad(y, (empty, *w), torch.empty_like(y))
        assert dx.shape == shape and not d_gu.any() and not d_down.any()


def test_gradients_of_any_strides_and_alignment_and_a_shared_weight():
    from purlin_b200.ops.gated_ffn import gated_ffn
    x, w_gu, w_down, _ = _inputs(40, 72, 48, seed=3)
    ones = torch.ones_like(x)
    want = _run(x, w_gu, w_down, ones, "silu")
    leaves = [v.clone().requires_grad_() for v in (x, w_gu, w_down)]
    gated_ffn(*leaves).sum().backward()                   # an expanded gradient: all strides zero
    assert all(torch.equal(v.grad, w) for v, w in zip(leaves, want[1:]))
    odd = torch.ones(40 * 72 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(40, 72)          # starts two bytes off
    leaves = [v.clone().requires_grad_() for v in (x, w_gu, w_down)]
    y = gated_ffn(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, odd), want[1:]))
    turned = torch.ones(72, 40, dtype=torch.bfloat16, device="cuda").t()
    y = gated_ffn(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, turned), want[1:]))
    # the same weights twice in one graph: their gradients add up
    a, b = x.clone(), (x * 2).clone()
    w = [v.clone().requires_grad_() for v in (w_gu, w_down)]
    (gated_ffn(a, *w).sum() + gated_ffn(b, *w).sum()).backward()
    parts = [_run(v, w_gu, w_down, ones, "silu")[2:] for v in (a, b)]
    for n in range(2):
        s = parts[0][n].double() + parts[1][n].double()
        assert ((w[n].grad.double() - s).abs() <= STEP * s.abs() + 2.0 ** -133).all()


def test_differentiable_once():
    from purlin_b200.ops.gated_ffn import gated_ffn
    x, w_gu, w_down, dy = _inputs(16, 72, 48)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(gated_ffn(x, w_gu, w_down), x, dy, create_graph=True)
    assert torch.equal(dx.detach(), _run(x.detach(), w_gu, w_down, dy, "silu")[1])
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(dx.float().sum(), x)


def test_a_weight_that_changed_before_the_backward_is_noticed():
    from purlin_b200.ops.gated_ffn import gated_ffn
    x, w_gu, w_down, dy = _inputs(16, 72, 48)
    x.requires_grad_()
    y = gated_ffn(x, w_gu, w_down)
    w_down.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_bits_do_not_change_from_call_to_call():
    for t, h, i in ((100, 1024, 2048), (2100, 1024, 784)):
        args = _inputs(t, h, i, seed=6)
        first = _run(*args, "silu")
        for _ in range(4):
            assert all(torch.equal(p, q) for p, q in zip(_run(*args, "silu"), first))


def test_values_out_of_the_ordinary():
    # tokens with huge, infinite and NaN activations next to ordinary ones: only their own rows of y and dx are affected, and the sigmoid's
    # ends are exact
    from purlin_b200.ops.gated_ffn import gated_ffn
    for activation in ("silu", "gelu"):
        x, w_gu, w_down, dy = _inputs(200, 136, 144, seed=8)
        clean = _run(x, w_gu, w_down, dy, activation)
        bad = x.clone()
        bad[3] = float("nan")
        bad[50, 5] = float("inf")
        bad[77] *= 2.0 ** 20
        bad[199] = 0
        leaves = [v.clone().requires_grad_() for v in (bad, w_gu, w_down)]
        y = gated_ffn(*leaves, activation)
        (dx,) = torch.autograd.grad(y, leaves[:1], dy)
        keep = torch.ones(200, dtype=torch.bool)
        keep[[3, 50, 77, 199]] = False
        assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
        assert y[3].isnan().all() and dx[3].isnan().all() and not y[199].any()
        want, off = _oracle(bad[77:78], w_gu, w_down, dy[77:78], activation)
        assert ((y[77].double() - want[0][0]).abs() <= off[0][0]).all() and ((dx[77].double() - want[1][0]).abs() <= off[1][0]).all()


def test_on_a_stream_of_its_own_and_in_a_graph():
    from purlin_b200.ops.gated_ffn import gated_ffn
    args = _inputs(300, 264, 528, seed=11)
    want = _run(*args, "silu")
    leaves = [v.clone().requires_grad_() for v in args[:3]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = gated_ffn(*leaves)
        got = (y.detach(), *torch.autograd.grad(y, leaves, args[3]))
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    # captured while an eager graph of the same leaves is alive; two graphs of two sizes replayed in turn, with new inputs
    alive = gated_ffn(*leaves)
    other = _inputs(100, 264, 2048, seed=12)
    _run(*other, "silu")
    graphs = []
    for a in (args, other):
        static = [v.clone().requires_grad_() for v in a[:3]] + [a[3].clone()]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = gated_ffn(*static[:3])
            out = (y.detach(), *torch.autograd.grad(y, static[:3], static[3]))
        graphs.append((g, static, out))
    for seed in (21, 22):
        for (g, static, out), (t, h, i) in zip(graphs, ((300, 264, 528), (100, 264, 2048))):
            new = _inputs(t, h, i, seed=seed)
            with torch.no_grad():
                for s, v in zip(static, new):
                    s.copy_(v)
            g.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, _run(*new, "silu")))
    assert torch.equal(alive.detach(), want[0])


def test_a_training_step_through_the_model_then_4_bits():
    from purlin_b200.models.gated_mlp import GatedMLP
    from purlin_b200.ops.gated_ffn import split_gate_up
    mlp = GatedMLP(hidden=512, intermediate=1024, seed=7)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(200, 512, generator=g, device="cuda").to(torch.bfloat16)
    optimizer = torch.optim.SGD(mlp.parameters(), lr=0.125)
    before = [p.detach().clone() for p in mlp.parameters()]
    y = mlp(x)
    (0.5 * y.float().square().sum() / 256).backward()
    want, off = _oracle(x, *before, (y.detach().float() / 256).to(torch.bfloat16), "silu")
    for p, ref, tol in zip(mlp.parameters(), want[2:], off[2:]):
        assert ((p.grad.double() - ref).abs() <= tol).all()
    optimizer.step()
    for p, b in zip(mlp.parameters(), before):
        assert torch.equal(p.detach(), b.add(p.grad, alpha=-0.125))
    served = mlp.quantized()
    w_gu, w_down = served.w_gu.dequantize(torch.float32).double(), served.w_down.dequantize(torch.float32).double()
    from purlin_b200.ops.mx4 import quantize_mx4
    for rows in (1, 64, 200):
        got = served(x[:rows].clone())
        gate, up = split_gate_up(w_gu)
        q = quantize_mx4(x[:rows].clone()).dequantize(torch.float32).double()
        h = torch.nn.functional.silu(q @ gate.t()) * (q @ up.t())
        # h is rounded to bf16 and then to 4 bits; a value next to a border may fall on its other side, so the product is checked against the
        # kernels' own h, which is checked against the formula (2^-8 of the value and the fp32 sums)
        from purlin_b200.ops.mx4 import mx4_gemm_swiglu
        mine = mx4_gemm_swiglu(x[:rows].clone(), served.w_gu)
        mag = (q.abs() @ gate.abs().t()) * (q.abs() @ up.abs().t())
        assert ((mine.double() - h).abs() <= STEP * h.abs() + 2.0 ** -14 * mag + 1e-30).all()
        hq = quantize_mx4(mine).dequantize(torch.float32).double()
        ref, m = hq @ w_down.t(), hq.abs() @ w_down.abs().t()
        assert ((got.double() - ref).abs() <= STEP * ref.abs() + 2.0 ** -16 * m + 1e-30).all()


def test_example():
    import pathlib
    import subprocess
    import sys
    example = pathlib.Path(__file__).resolve().parent.parent / "examples" / "gated_mlp.py"
    done = subprocess.run([sys.executable, str(example), "200", "512", "1024"], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout + done.stderr      # it checks its own gradients


def test_offsets_past_32_bits():
    # 6.9 GB of saved pre-activations, 4.6 GB of dZ: the last tokens against the formula on them alone
    from purlin_b200.ops.gated_ffn import gated_ffn
    t, h, i = 20000, 64, 57344
    x, w_gu, w_down, dy = _inputs(t, h, i, seed=20)
    x.requires_grad_()
    y = gated_ffn(x, w_gu, w_down)
    (dx,) = torch.autograd.grad(y, x, dy)
    for rows in (slice(0, 24), slice(12340, 12364), slice(t - 24, t)):
        want, off = _oracle(x.detach()[rows], w_gu, w_down, dy[rows], "silu")
        assert ((y.detach()[rows].double() - want[0]).abs() <= off[0]).all() and ((dx[rows].double() - want[1]).abs() <= off[1]).all()
