"""What the operators refuse before anything reaches a GPU."""
import pytest
import torch


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_gated_ffn_refuses():
    from purlin_b200.ops.gated_ffn import gated_ffn
    ok = (_t(4, 64), _t(96, 64), _t(64, 48))
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(*ok, "relu")
    for n in range(3):
        args = list(ok)
        args[n] = args[n].float()
        with pytest.raises(TypeError):
            gated_ffn(*args)
    for bad in ((_t(4, 56), ok[1], ok[2]), (ok[0], _t(64, 64), ok[2]), (ok[0], ok[1], _t(64, 32)), (ok[0], ok[1].view(2, 48, 64), ok[2]),
                (_t(4, 60), _t(96, 60), _t(60, 48)), (ok[0], _t(80, 64), _t(64, 40)), (_t(4, 0), _t(96, 0), _t(0, 48)), (_t(4, 64), _t(0, 64), _t(64, 0)),
                (torch.zeros((), dtype=torch.bfloat16), ok[1], ok[2])):
        with pytest.raises(ValueError):
            gated_ffn(*bad)
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn(*ok)


def test_quantisation_and_products_refuse():
    from purlin_b200.ops.mx4 import Mx4Tensor, mx4_gemm, quantize_mx4, scale_bytes
    for dtype in (torch.float64, torch.int8):
        with pytest.raises(TypeError):
            quantize_mx4(_t(4, 64, dtype=dtype))
    for bad in (_t(4, 48), _t(4, 0), torch.zeros((), dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            quantize_mx4(bad)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_mx4(_t(4, 64))
    with pytest.raises(TypeError, match="Mx4Tensor"):
        mx4_gemm(_t(4, 64), _t(8, 64))
    data, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(scale_bytes(4, 64), dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        Mx4Tensor(data, scales)
    with pytest.raises(ValueError):
        Mx4Tensor(data, scales[1:])
    with pytest.raises(ValueError):
        Mx4Tensor(data[:, :8], scales)
    with pytest.raises(TypeError):
        Mx4Tensor(data.float(), scales)


@pytest.mark.parametrize("rows,cols,want", [(1, 32, 512), (128, 128, 512), (129, 128, 1024), (128, 160, 1024), (300, 288, 3 * 3 * 512), (0, 64, 0)])
def test_scale_bytes(rows, cols, want):
    from purlin_b200 import _native
    from purlin_b200.ops.mx4 import scale_bytes
    assert scale_bytes(rows, cols) == want
    lib = _native.cuda()
    lib.purlin_mx4_scale_bytes.restype = __import__("ctypes").c_size_t
    assert lib.purlin_mx4_scale_bytes(rows, cols) == want


def test_split_gate_up_is_the_inverse_of_the_interleaving():
    from purlin_b200.ops.gated_ffn import split_gate_up
    from purlin_b200.ops.gemm import interleave_gate_up
    gate, up = torch.randn(48, 8), torch.randn(48, 8)
    g, u = split_gate_up(interleave_gate_up(gate, up))
    assert torch.equal(g, gate) and torch.equal(u, up)
    with pytest.raises(ValueError):
        split_gate_up(torch.zeros(48, 8))


def test_c_entries_refuse_without_a_launch():
    # null operands, sizes that do not fit, unknown types: an error text and no launch
    import ctypes as C

    from purlin_b200 import _native
    lib = _native.cuda()
    p = C.c_void_p(4096)                     # never followed: every call is refused by its sizes or a missing operand

    def refused(rc):
        assert rc != 0 and _native.last_error(lib)

    i, n = C.c_int, None
    for sizes in ((0, 64, 32), (4, 60, 32), (4, 64, 24), (4, -8, 32), (4, 64, 0)):
        refused(lib.purlin_ffn_forward(p, p, p, p, n, p, *map(i, sizes), i(0), n, n))
        refused(lib.purlin_ffn_backward(p, p, p, p, p, p, p, p, p, p, n, C.c_size_t(0), *map(i, sizes), i(0), n, n))
    refused(lib.purlin_ffn_forward(p, p, p, p, n, p, i(4), i(64), i(32), i(2), n, n))
    refused(lib.purlin_ffn_forward(n, p, p, p, n, p, i(4), i(64), i(32), i(0), n, n))
    for missing in (3, 4, 5, 6):             # h, saved, dy, dz
        args = [p] * 10
        args[missing] = n
        refused(lib.purlin_ffn_backward(*args, n, C.c_size_t(0), i(4), i(64), i(32), i(0), n, n))
    refused(lib.purlin_mx4_quantize(p, i(0), p, p, i(4), i(48), n))
    refused(lib.purlin_mx4_quantize(p, i(0), n, p, i(4), i(64), n))
    refused(lib.purlin_mx4_quantize(C.c_void_p(4098), i(0), p, p, i(4), i(64), n))
    refused(lib.purlin_mx4_dequantize(p, p, n, i(0), i(4), i(64), n))
    refused(lib.purlin_mx4_gemm(p, p, p, p, p, i(4), i(12), i(64), i(0), n, n))
    refused(lib.purlin_mx4_gemm(p, p, p, p, p, i(4), i(48), i(64), i(1), n, n))
    refused(lib.purlin_mx4_gemm(p, p, p, p, p, i(4), i(64), i(64), i(2), n, n))
    refused(lib.purlin_mx4_gemm(p, p, p, n, p, i(4), i(64), i(64), i(0), n, n))
    refused(lib.purlin_mx4_linear(n, i(0), n, p, p, p, i(4), i(64), i(64), i(0), n, n))
    refused(lib.purlin_mx4_linear(C.c_void_p(4098), i(0), n, p, p, p, i(4), i(64), i(64), i(0), n, n))
    refused(lib.purlin_mx4_linear(p, i(0), n, p, p, p, i(400), i(64), i(64), i(0), n, n))      # no workspace
    refused(lib.purlin_mx4_linear(p, i(0), n, p, p, p, i(4), i(60), i(64), i(0), n, n))
