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


@pytest.mark.parametrize("m,n,k", [(129, 8, 32), (129, 264, 96), (256, 256, 256), (257, 128, 64), (300, 520, 544), (511, 1000, 288), (1000, 1024, 1120), (513, 14336, 256), (2049, 4104, 96), (200, 14208, 256), (500, 7104, 288), (1000, 14336, 96), (4096, 4864, 160),
                                    (4096, 2048, 2048)])
def test_many_rows(m, n, k):
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    a, w = quantize_mx4(_rand(m, k, 3, spread=2.0)), quantize_mx4(_rand(n, k, 4, spread=2.0))
    _check_product(mx4_gemm(a, w), a, w, False)


@pytest.mark.parametrize("m,i,k", [(1, 16, 32), (1, 3584, 1024), (7, 80, 96), (100, 528, 544), (128, 1024, 512), (129, 16, 64), (300, 528, 224), (1000, 1040, 512), (777, 7168, 256), (200, 7104, 256), (1000, 7168, 96)])      # the last ones: widths of 192 columns, tiles of the last wave in quarters
def test_gated_product(m, i, k):
    from purlin_b200.ops.mx4 import mx4_gemm_swiglu, quantize_mx4
    a, w = quantize_mx4(_rand(m, k, 5)), quantize_mx4(_rand(2 * i, k, 6) * (4 * k ** -0.5))
    _check_product(mx4_gemm_swiglu(a, w), a, w, True)


@pytest.mark.parametrize("m", [1, 63, 64, 65, 80, 81, 128, 129])
@pytest.mark.parametrize("n", [8160, 8192])
def test_both_kernels_at_their_border(m, n):
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    a, w = quantize_mx4(_rand(m, 288, 7, spread=2.0)), quantize_mx4(_rand(n, 288, 8, spread=2.0))
    _check_product(mx4_gemm(a, w), a, w, False)


@pytest.mark.parametrize("m", [2, 90, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_activations_quantised_in_the_call_and_given_outputs(m, dtype):
    from purlin_b200.ops.mx4 import mx4_gemm, mx4_gemm_swiglu, quantize_mx4
    x, w = _rand(m, 224, 9, dtype), quantize_mx4(_rand(544, 224, 10))
    q = quantize_mx4(x)
    for f, cols in ((mx4_gemm, 544), (mx4_gemm_swiglu, 272)):
        want = f(q, w)
        assert torch.equal(f(x, w), want)
        out = torch.full((m + 2, cols), 7.0, dtype=torch.bfloat16, device="cuda")
        assert f(x, w, out[1:-1]) .data_ptr() == out[1:-1].data_ptr()
        assert torch.equal(out[1:-1], want) and (out[0] == 7).all() and (out[-1] == 7).all()
        assert torch.equal(f(q, w, out[1:-1]), want)
        assert torch.equal(f(x.view(1, m, 224), w), want.view(1, m, cols))
        assert f(x[0], w).shape == (cols,)
        assert f(x[:0], w).shape == (0, cols) and f(x[:0].view(3, 0, 224), w).shape == (3, 0, cols)
    assert quantize_mx4(x[:0]).shape == (0, 224) and quantize_mx4(x[:0]).dequantize().shape == (0, 224)


@pytest.mark.parametrize("m", [3, 70, 200])
def test_nans_stay_in_their_rows_and_columns(m):
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    x, w = _rand(m, 288, 11), _rand(264, 288, 12)
    clean = mx4_gemm(quantize_mx4(x), quantize_mx4(w))
    bad_x, bad_w = x.clone(), w.clone()
    bad_x[1, 280], bad_w[130, 3] = float("nan"), float("inf")
    got = mx4_gemm(quantize_mx4(bad_x), quantize_mx4(bad_w))
    rows, cols = torch.arange(m) != 1, torch.arange(264) != 130
    assert got[1].isnan().all() and got[:, 130].isnan().all()
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


@pytest.mark.parametrize("m,n,k", [(5, 264, 544), (300, 520, 544)])
def test_scales_at_the_ends_of_their_range(m, n, k):
    # powers of two from 2^-127 to 2^125 on one side and their inverses on the other: products and sums that fp32 holds exactly
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    g = torch.Generator(device="cuda").manual_seed(13)
    e = torch.tensor([-100.0, -60.0, 0.0, 60.0, 100.0], device="cuda")[torch.randint(0, 5, (k // 32,), generator=g, device="cuda")]
    power = torch.exp2(e).repeat_interleave(32)
    a = torch.randint(-4, 5, (m, k), generator=g, device="cuda").float() * power
    w = torch.randint(-1, 2, (n, k), generator=g, device="cuda").float() / power
    a[:, ::32], w[:, ::32] = 4 * power[::32], 4 / power[::32]          # so that every block's largest magnitude is 4: whole numbers are exact
    got = mx4_gemm(quantize_mx4(a), quantize_mx4(w))
    ref = quantize_mx4(a).dequantize(torch.float32).double() @ quantize_mx4(w).dequantize(torch.float32).double().t()
    assert torch.equal(got.double(), ref.to(torch.bfloat16).double())


def test_bits_do_not_change_from_call_to_call():
    from purlin_b200.ops.mx4 import mx4_gemm_swiglu, quantize_mx4
    w = quantize_mx4(_rand(2048, 4096, 14))
    for m in (1, 50, 500):
        x = _rand(m, 4096, 15)
        first = mx4_gemm_swiglu(x, w)
        for _ in range(4):
            assert torch.equal(mx4_gemm_swiglu(x, w), first)


def test_on_a_stream_of_its_own_and_in_graphs():
    from purlin_b200.ops.mx4 import mx4_gemm, mx4_gemm_swiglu, quantize_mx4
    wg, wd = quantize_mx4(_rand(1024, 288, 16) * 0.1), quantize_mx4(_rand(288, 512, 17) * 0.1)

    def block(x):
        return mx4_gemm(mx4_gemm_swiglu(x, wg), wd)

    xs = {m: _rand(m, 288, 18 + m) for m in (1, 300)}
    want = {m: block(x) for m, x in xs.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = {m: block(x) for m, x in xs.items()}
    side.synchronize()
    assert all(torch.equal(got[m], want[m]) for m in xs)
    graphs = {}
    for m, x in xs.items():
        static, g = x.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = block(static)
        graphs[m] = (g, static, y)
    for seed in (1, 2):
        for m, (g, static, y) in graphs.items():
            static.copy_(_rand(m, 288, seed))
            g.replay()
            assert torch.equal(y, block(_rand(m, 288, seed)))


def test_a_tensor_of_more_than_4_gib():
    from purlin_b200.ops.mx4 import quantize_mx4
    rows, cols = 140003, 16416                                # 4.6 GB of bf16, codes of more than 2^31 values
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for r in range(0, rows, 20000):
        x[r:r + 20000] = _rand(min(20000, rows - r), cols, r)
    q = quantize_mx4(x)
    v = q.dequantize()
    scales = q.scale_matrix()
    for r in (0, 65535, 130999, rows - 40):
        part = quantize_mx4(x[r:r + 40].clone())
        assert torch.equal(q.data[r:r + 40], part.data) and torch.equal(v[r:r + 40], part.dequantize()) and torch.equal(scales[r:r + 40], part.scale_matrix())


def test_refusals_of_tensors_on_the_gpu():
    from purlin_b200.ops.gated_ffn import gated_ffn
    from purlin_b200.ops.mx4 import Mx4Tensor, mx4_gemm, mx4_gemm_swiglu, quantize_mx4
    x, w = _rand(4, 64, 1), quantize_mx4(_rand(48, 64, 2))
    flat = torch.zeros(4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    for bad in (x.t().contiguous().t(), x[:, ::2], flat[1:257].view(4, 64)):
        for f in (quantize_mx4, lambda v: mx4_gemm(v, w)):
            with pytest.raises(ValueError):
                f(bad)
    with pytest.raises(TypeError):
        mx4_gemm(x, x)
    with pytest.raises(TypeError):
        quantize_mx4(x.long())
    with pytest.raises(ValueError):
        mx4_gemm(x[:, :32].contiguous(), w)
    with pytest.raises(ValueError):
        mx4_gemm_swiglu(x, w)                                  # 48 rows are no whole groups of gate and up
    with pytest.raises(ValueError):
        mx4_gemm(x, quantize_mx4(_rand(4, 64, 2)))
    with pytest.raises(TypeError):
        mx4_gemm(x, w, torch.empty(4, 48, device="cuda"))
    for out in (torch.empty(4, 40, device="cuda", dtype=torch.bfloat16), torch.empty(48, 4, device="cuda", dtype=torch.bfloat16).t()):
        with pytest.raises(ValueError):
            mx4_gemm(x, w, out)
    with pytest.raises(ValueError):
        Mx4Tensor(w.data, w.scales[:-1])
    with pytest.raises(ValueError):
        Mx4Tensor(w.data.t(), w.scales)
    with pytest.raises(TypeError):
        Mx4Tensor(w.data.int(), w.scales)
    with pytest.raises(TypeError):
        w.dequantize(torch.float16)
    same = Mx4Tensor(w.data.clone(), w.scales.clone())          # what a checkpoint gives back
    assert torch.equal(mx4_gemm(x, same), mx4_gemm(x, w))
    g = torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        gated_ffn(x.t().contiguous().t(), g, torch.zeros(64, 32, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        gated_ffn(flat[1:257].view(4, 64), g, torch.zeros(64, 32, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        gated_ffn(x.cpu(), g, torch.zeros(64, 32, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("m", [1, 3, 4, 5, 8, 15, 16, 17])
@pytest.mark.parametrize("n,k", [(64, 32), (264, 96), (160, 288), (4096, 4096), (544, 14336), (20000, 512)])
def test_a_few_tokens_quantised_inside_the_product(m, n, k):
    # the same bits as from the quantised activations, gated or not, with blocks of zeros, huge values and NaNs among them
    from purlin_b200.ops.mx4 import mx4_gemm, mx4_gemm_swiglu, quantize_mx4
    x = _rand(m, k, 30 + m, spread=8.0)
    x[m - 1, :32] = 0
    x[0, k - 1] = 3e38
    w = quantize_mx4(_rand(n, k, 31))
    q = quantize_mx4(x)
    assert torch.equal(mx4_gemm(x, w), mx4_gemm(q, w))
    if n % 32 == 0:
        assert torch.equal(mx4_gemm_swiglu(x, w).nan_to_num(nan=7.0), mx4_gemm_swiglu(q, w).nan_to_num(nan=7.0))
    x[m // 2, k // 2] = float("nan")
    got, want = mx4_gemm(x, w), mx4_gemm(quantize_mx4(x), w)
    assert got[m // 2].isnan().all() and torch.equal(got.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


def test_a_product_of_more_than_2_to_the_31_values():
    from purlin_b200.ops.mx4 import mx4_gemm, quantize_mx4
    x, w = _rand(70001, 64, 40), quantize_mx4(_rand(32776, 64, 41))
    y = mx4_gemm(x, w)
    for r in (0, 65530, 70001 - 300):
        assert torch.equal(y[r:r + 300], mx4_gemm(x[r:r + 300].clone(), w))
