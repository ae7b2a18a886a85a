"""The operators of the gated block at the edges of what their documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(rows, cols, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, cols, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 64, 65, 300])
def test_a_product_in_place_of_its_activations(m):
    # on both sides of every border between the kernels: the output is the activations' own memory, all of it or a part
    from purlin_b200.ops.mx4 import mx4_gemm, mx4_gemm_swiglu, quantize_mx4
    k = 8192 if m < 5 else 1024
    x, w = _rand(m, k, m), quantize_mx4(_rand(k, k, 1))
    want, gated = mx4_gemm(x, w), mx4_gemm_swiglu(x, w)
    for _ in range(3):
        y = x.clone()
        assert mx4_gemm(y, w, out=y) is y and torch.equal(y, want)
        y = x.clone()
        half = y.flatten()[:m * k // 2].view(m, k // 2)
        assert torch.equal(mx4_gemm_swiglu(y, w, out=half), gated)
        room = torch.zeros(m * k + 64, dtype=torch.bfloat16, device="cuda")
        room[:m * k] = x.flatten()
        assert torch.equal(mx4_gemm(room[:m * k].view(m, k), w, out=room[64:].view(m, k)), want) and torch.equal(room[:64], x.flatten()[:64])


@pytest.mark.parametrize("m", [2, 300])
def test_a_product_over_a_quantised_operand_is_refused(m):
    from purlin_b200.ops.mx4 import Mx4Tensor, mx4_gemm, quantize_mx4
    x = _rand(m, 256, 1)
    room = torch.zeros(m * 256 * 2 + 2 ** 16, dtype=torch.uint8, device="cuda")
    out = room[:m * 512].view(torch.bfloat16).view(m, 256)
    q, w = quantize_mx4(x), quantize_mx4(_rand(256, 256, 2))
    inside = Mx4Tensor(room[:m * 128].view(m, 128), q.scales)
    with pytest.raises(ValueError, match="overlaps"):
        mx4_gemm(inside, w, out=out)
    tail = Mx4Tensor(w.data, room[m * 512 - 16:][:w.scales.numel()])
    for a in (x, q):
        with pytest.raises(ValueError, match="overlaps"):
            mx4_gemm(a, tail, out=out)


def test_producer_quantisation_and_the_way_back_over_the_same_buffers():
    # each kernel is set up while the one before it writes what it will read; the values change from pass to pass, the buffers stay, in a graph too
    from purlin_b200.ops.mx4 import mx4_gemm_swiglu, quantize_mx4
    w = quantize_mx4(_rand(2 * 2048, 256, 3))
    x, h = torch.empty(700, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(700, 2048, dtype=torch.bfloat16, device="cuda")

    def work():
        mx4_gemm_swiglu(x, w, out=h)
        return quantize_mx4(h).dequantize()

    news = [_rand(700, 256, 50 + n) for n in range(8)]
    wants = []
    for new in news:                                # one kernel at a time
        f = mx4_gemm_swiglu(new, w)
        torch.cuda.synchronize()
        q = quantize_mx4(f)
        torch.cuda.synchronize()
        wants.append(q.dequantize())
        torch.cuda.synchronize()
    x.copy_(news[0])
    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    got = []
    for _ in range(5):
        for new in news:
            x.copy_(new)
            got.append(work())
            graph.replay()
            got.append(out.clone())
    assert all(torch.equal(v, wants[n // 2 % 8]) for n, v in enumerate(got))


def test_forward_mode_derivatives_of_the_block_are_refused():
    from purlin_b200.ops.gated_ffn import gated_ffn
    args = [_rand(16, 64, 1), _rand(64, 64, 2), _rand(64, 32, 3)]
    with torch.autograd.forward_ad.dual_level():
        for k in range(3):
            called = list(args)
            called[k] = torch.autograd.forward_ad.make_dual(args[k], torch.ones_like(args[k]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                    gated_ffn(*called)
        assert gated_ffn(*args).shape == (16, 64)            # a dual level alone is no reason
        leaves = [v.clone().requires_grad_() for v in args]
        y = gated_ffn(*leaves)
        with pytest.raises(RuntimeError, match="forward-mode"):                                      # of the backward pass
            torch.autograd.grad(y, leaves, torch.autograd.forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_differentiating_a_4_bit_product_raises():
    from purlin_b200.models.gated_mlp import GatedMLP
    from purlin_b200.ops.mx4 import mx4_gemm, mx4_gemm_swiglu, quantize_mx4
    w = quantize_mx4(_rand(256, 256, 1))
    for m in (2, 300):
        plain = _rand(m, 256, 2)
        x = plain.clone().requires_grad_()
        for f in (mx4_gemm, mx4_gemm_swiglu):
            y = f(x, w)
            assert y.requires_grad and torch.equal(y.detach(), f(plain, w))
            with pytest.raises(RuntimeError, match="not differentiable"):
                y.float().sum().backward()
            with torch.no_grad():
                assert not f(x, w).requires_grad
            assert not f(plain, w).requires_grad and not f(quantize_mx4(x), w).requires_grad
            out = torch.empty_like(y)
            with pytest.raises(RuntimeError, match="not differentiable"):
                f(x, w, out=out)
            with torch.no_grad():
                assert torch.equal(f(x, w, out=out), y.detach())
        served = GatedMLP(256, 512, seed=1).quantized()
        with pytest.raises(RuntimeError, match="not differentiable"):
            served(x).float().sum().backward()


def test_an_output_that_a_graph_keeps_is_noticed():
    from purlin_b200.ops.gated_ffn import gated_ffn
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    h, w = _rand(16, 64, 1), quantize_mx4(_rand(64, 64, 4))
    w_gu = _rand(64, 64, 2).requires_grad_()
    y = gated_ffn(h, w_gu, _rand(64, 32, 3))
    mx4_gemm(_rand(16, 64, 5), w, out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))
    with torch.inference_mode():
        kept = torch.empty(16, 64, dtype=torch.bfloat16, device="cuda")
        mx4_gemm(h, w, out=kept)
    assert torch.equal(mx4_gemm(h, w, out=kept), mx4_gemm(h, w))


def _plant(words):
    """What a kernel whose wait gave up writes, from the host."""
    import ctypes
    from purlin_b200 import _native
    at = (ctypes.c_uint32 * 4).from_address(_native.torch_ops().wait_words(torch.cuda.current_device()))
    at[:] = words


def test_a_wait_that_gave_up_is_told_to_the_next_call():
    from purlin_b200.ops.gated_ffn import gated_ffn
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    from purlin_b200.ops.waits import check_waits
    leaves = [v.requires_grad_() for v in (_rand(16, 64, 1), _rand(64, 64, 2), _rand(64, 32, 3))]
    q, w = quantize_mx4(_rand(300, 64, 5)), quantize_mx4(_rand(64, 64, 4))
    few = _rand(2, 64, 6)
    y = gated_ffn(*leaves)
    check_waits()
    for call in (lambda: gated_ffn(*leaves), lambda: torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True), lambda: mx4_gemm(q, w), lambda: mx4_gemm(few, w)):
        want = call()
        _plant((5, 3, 17, 2))
        with pytest.raises(RuntimeError, match="gave up.*where 3, 17, 2"):
            call()
        got = call()                              # told once
        assert all(torch.equal(a, b) for a, b in zip(want, got)) if isinstance(got, tuple) else torch.equal(want, got)
    for device in (None, 0, "cuda", "cuda:0", torch.device("cuda", 0)):
        _plant((5, 1, 2, 3))
        with pytest.raises(TimeoutError, match="where 1, 2, 3"):
            check_waits(device)
        check_waits(device)


def test_the_words_of_waits_when_the_first_call_is_captured():
    # a process of its own: nothing has been called before
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
x, w = torch.ones(300, 64, device="cuda", dtype=torch.bfloat16), quantize_mx4(torch.ones(64, 64, device="cuda", dtype=torch.bfloat16))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = mx4_gemm(x, w)
g.replay()
assert (y == 64).all()
from purlin_b200.ops.waits import check_waits
check_waits()
print("ok")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=str(Path(__file__).resolve().parent.parent))
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout + done.stderr


@pytest.mark.parametrize("m", [1, 31, 32, 33, 65, 66, 72, 79, 80, 81, 127, 128])
@pytest.mark.parametrize("n,k", [(384, 2048), (1024, 28672), (8160, 4096), (8192, 4096)])
def test_products_around_the_borders_of_the_kernel_for_few_rows(m, n, k):
    # below 8192 columns it takes up to 80 rows, whose partial tiles and scales are the most that it holds, else up to 64; sums of whole numbers that
    # fp32 holds exactly, so that a wrong column, row or scale cannot hide in a tolerance: the magnitudes of a block's terms add up to at most
    # 16 * 32 + 31 * 8 * 16 = 4480, and those of 896 blocks to less than 2^24
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    g = torch.Generator(device="cuda").manual_seed(m + n)

    def whole(rows, most):                          # small whole numbers, a power of two to each block of 32 of a row, each block's largest is 4 times it
        v = torch.randint(-2, 3, (rows, k), generator=g, device="cuda").float()
        v.view(rows, -1, 32)[:, :, 0] = 4
        power = torch.exp2(torch.randint(0, most + 1, (rows, k // 32, 1), generator=g, device="cuda").float())
        return (v.view(rows, -1, 32) * power).view(rows, k)

    a, w = whole(m, 2), whole(n, 3)
    y = a.double() @ w.double().t()
    assert (a.abs().double() @ w.abs().double().t()).max() < 2 ** 24
    for x in (a, a.to(torch.bfloat16)):
        assert torch.equal(mx4_gemm(quantize_mx4(x), quantize_mx4(w)).double(), y.to(torch.bfloat16).double())
        assert torch.equal(mx4_gemm(x, quantize_mx4(w)).double(), y.to(torch.bfloat16).double())


def test_every_code_with_every_scale_byte_that_a_caller_may_build():
    # exact up to byte 252, NaNs at 255; between, what is past the largest number becomes an infinity
    from purlin_b200.ops.mx4 import Mx4Tensor, scale_bytes
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    codes = torch.arange(32, dtype=torch.uint8).view(1, 32).expand(256, 32) % 16
    data = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous().cuda()
    scales = torch.zeros(scale_bytes(256, 32), dtype=torch.uint8)
    row = torch.arange(256)
    scales[row // 128 * 512 + row % 32 * 16 + row // 32 % 4 * 4] = row.to(torch.uint8)
    q = Mx4Tensor(data, scales.cuda())
    assert torch.equal(q.scale_matrix().cpu().flatten(), row.to(torch.uint8))
    values = torch.where(codes < 8, 1.0, -1.0).double() * grid[codes.long() % 8] * torch.pow(torch.tensor(2.0, dtype=torch.float64), row.double() - 127)[:, None]
    values[255] = float("nan")
    assert (values[:253].abs() < 2.0 ** 128).all()
    for dtype in (torch.bfloat16, torch.float32):
        got = q.dequantize(dtype).cpu()
        want = torch.where(values.abs() >= 2.0 ** 128, values.sign() * float("inf"), values)
        assert torch.equal(got.double().nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), want.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
        assert got[:253].isfinite().all()
