"""4-bit microscaled quantisation and products against the format's definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _definition(x):
    """Codes, scale bytes and values of [rows, cols] from the definition, on the CPU in 64 bits."""
    x = x.double().cpu()
    rows, cols = x.shape
    b = x.view(rows, cols // 32, 32)
    peak = b.abs().amax(2)
    fine = torch.isfinite(peak) & ~torch.isnan(b).any(2)
    exponent = torch.frexp(torch.where(fine, peak, 1.0))[1].to(torch.int64) - 3
    byte = torch.where(fine, torch.where(peak > 0, (exponent + 127).clamp(min=0), 0), 255)      # zeros alone: the least power
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64), (byte - 127).double())
    m = torch.where(fine[..., None], b.abs() / power[..., None], 0.0)
    grid = torch.tensor(GRID, dtype=torch.float64)
    d = (m[..., None] - grid).abs()
    nearest = d.amin(-1, keepdim=True)
    # of two values that are as near, the one with the even code
    code = (torch.where(d == nearest, torch.tensor([0, 1, 0, 1, 0, 1, 0, 1]), 9)).argmin(-1)
    sign = torch.signbit(b) & fine[..., None]
    values = torch.where(fine[..., None], torch.where(sign, -1.0, 1.0) * grid[code] * power[..., None], float("nan"))
    return (code + 8 * sign.long()).view(rows, cols), byte, values.view(rows, cols)


def _codes(q):
    d = q.data.cpu().long()
    return torch.stack([d & 15, d >> 4], 2).flatten(1)


def _rand(rows, cols, seed, dtype=torch.bfloat16, spread=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    if spread:
        x = x * torch.exp2(torch.randn(rows, 1, generator=g, device="cuda") * spread)
    return x.to(dtype)


def _same(q, x):
    codes, byte, values = _definition(x)
    assert torch.equal(q.scale_matrix().cpu().long(), byte)
    assert torch.equal(_codes(q), codes)
    for dtype in (torch.bfloat16, torch.float32):
        assert torch.equal(q.dequantize(dtype).cpu().double().nan_to_num(nan=7.0), values.nan_to_num(nan=7.0))
    # what lies past the edges is zero
    rows, cols = q.shape
    v = q.scales.view(-(-rows // 128), -(-cols // 128), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)
    assert (v[rows:] == 0).all() and (v[:, cols // 32:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 96), (3, 128), (31, 160), (33, 1024), (127, 288), (128, 256), (129, 544), (700, 4096), (2, 28672)])
def test_quantisation_is_the_definition(rows, cols, dtype):
    from purlin_b200.ops.mx4 import quantize_mx4
    x = _rand(rows, cols, rows + cols, dtype, spread=3.0)
    _same(quantize_mx4(x), x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantisation_at_the_borders(dtype):
    # every tie between neighbouring values, both signs, at the smallest and largest powers, zero blocks, subnormal blocks, saturation, -0
    from purlin_b200.ops.mx4 import quantize_mx4
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 7.5, 0.5, 4.0, 0.0, -0.0, 3.0, 1.5])
    block = torch.cat([ties, -ties])
    lowest, highest = {torch.bfloat16: (-133, 125), torch.float16: (-24, 13), torch.float32: (-149, 125)}[dtype]
    rows = [block * 2.0 ** e for e in range(max(lowest, -120), highest + 1, 7)] + [torch.zeros(32), -torch.zeros(32)]
    tiny = torch.finfo(dtype).smallest_normal
    for m in (1.0, 0.5, 2.0 ** -6 if dtype != torch.float16 else 2.0 ** -9):     # around and below the smallest normal number
        rows.append(torch.full((32,), tiny * m))
    rows.append(torch.full((32,), torch.finfo(dtype).max))
    rows.append(torch.full((32,), -torch.finfo(dtype).max) * torch.linspace(0, 1, 32))
    x = torch.stack(rows).to(dtype).cuda()
    _same(quantize_mx4(x), x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_block_with_an_infinity_or_a_nan_stands_for_nans(dtype):
    from purlin_b200.ops.mx4 import quantize_mx4
    x = _rand(5, 128, 1, dtype)
    x[0, 3], x[1, 40], x[2, 127], x[3, 0], x[3, 5] = float("inf"), float("-inf"), float("nan"), float("inf"), float("nan")
    q = quantize_mx4(x)
    _same(q, x)
    assert (q.scale_matrix() == 255).sum() == 4


def _product_oracle(a, w, swiglu):
    """The product of the values that both operands stand for, and the sum of the magnitudes of its terms, in 64 bits."""
    a, w = a.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    y, mag = a @ w.t(), a.abs() @ w.abs().t()
    if not swiglu:
        return y, mag, None
    v, m = y.view(y.shape[0], -1, 2, 16), mag.view(y.shape[0], -1, 2, 16)
    return v, m, (torch.nn.functional.silu(v[:, :, 0]) * v[:, :, 1]).flatten(1)


def _check_product(got, a, w, swiglu):
    y, mag, gated = _product_oracle(a, w, swiglu)
    # products of 4-bit values and powers of two are exact; the fp32 sums of up to 2^15 terms are within 2^-17 of the terms' magnitudes; one
    # rounding to bf16 is 2^-8 of the value (2^-133 in its subnormal numbers)
    if not swiglu:
        tol = 2.0 ** -8 * y.abs() + 2.0 ** -16 * mag + 2.0 ** -133
        err = (got.double() - y).abs()
    else:
        g, u = y[:, :, 0], y[:, :, 1]
        loose = 2.0 ** -16 * (1.2 * mag[:, :, 0] * u.abs() + g.abs() * mag[:, :, 1] + 2.0 ** -3 * (g * u).abs())     # |silu'| <= 1.2, the fast exponential and division
        tol = 2.0 ** -8 * gated.abs() + (1 + 2.0 ** -8) * loose.flatten(1) + 2.0 ** -133
        err = (got.double() - gated).abs()
    assert (err <= tol).all(), f"{(err / tol).max().item()} of what rounding allows"


@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 136, 96), (2, 128, 64), (15, 264, 160), (16, 1024, 256), (17, 120, 544), (33, 640, 1024), (64, 4096, 4096), (65, 2048, 1120),
                                    (127, 384, 2048), (128, 1024, 4096), (3, 8192, 14336)])
def test_few_rows(m, n, k):
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    a, w = quantize_mx4(_rand(m, k, 1, spread=2.0)), quantize_mx4(_rand(n, k, 2, spread=2.0))
    _check_product(mx4_gemm(a, w), a, w, False)


@pytest.mark.parametrize("m,n,k", [(129, 8, 32), (129, 264, 96), (256, 256, 256), (257, 128, 64), (300, 520, 544), (511, 1000, 288), (1000, 1024, 1120), (513, 14336, 256), (2049, 4104, 96),
                                    (4096, 2048, 2048)])
def test_many_rows(m, n, k):
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    a, w = quantize_mx4(_rand(m, k, 3, spread=2.0)), quantize_mx4(_rand(n, k, 4, spread=2.0))
    _check_product(mx4_gemm(a, w), a, w, False)


@pytest.mark.parametrize("m,i,k", [(1, 16, 32), (1, 3584, 1024), (7, 80, 96), (100, 528, 544), (128, 1024, 512), (129, 16, 64), (300, 528, 224), (1000, 1040, 512), (777, 7168, 256)])
def test_gated_product(m, i, k):
    from purlin_b200.ops.mx4 import mx4_gemm_swiglu, quantize_mx4
    a, w = quantize_mx4(_rand(m, k, 5)), quantize_mx4(_rand(2 * i, k, 6) * (4 * k ** -0.5))
    _check_product(mx4_gemm_swiglu(a, w), a, w, True)
