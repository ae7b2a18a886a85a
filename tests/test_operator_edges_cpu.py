"""What the operators of the gated block refuse, or have to have in their source, at the edges of what they take; no GPU."""
import ctypes as C

import pytest
import torch

i, p, n = C.c_int, C.c_void_p, None


def _refusal(rc):
    from purlin_b200 import _native
    assert rc != 0
    return _native.last_error(_native.cuda())


def test_products_refuse_an_output_over_their_operands():
    # addresses that no call follows: the refusal comes before anything is launched
    from purlin_b200 import _native
    lib = _native.cuda()
    a, sa, w, sw, c = (p(v << 20) for v in range(1, 6))
    m, cols, k = 4, 64, 64
    for at in ((1 << 20) + 32, (2 << 20) + 496, (3 << 20) + 2032, (4 << 20), (1 << 20) - 496, (3 << 20) - 496):     # C: 512 bytes; a 128, w 2048, scales 512
        assert "overlaps" in _refusal(lib.purlin_mx4_gemm(a, sa, w, sw, p(at), i(m), i(cols), i(k), i(0), n, n)), at
        if at > 2.5 * 2 ** 20:
            assert "overlaps" in _refusal(lib.purlin_mx4_linear(c, i(0), n, w, sw, p(at), i(m), i(cols), i(k), i(0), n, n)), at
    # x itself: quantised by a launch of its own, for which there is no workspace here
    for at in (5 << 20, (5 << 20) - 496, (5 << 20) + 496):
        assert "overlaps x" in _refusal(lib.purlin_mx4_linear(c, i(0), n, w, sw, p(at), i(m), i(cols), i(k), i(0), n, n)), at


def test_no_load_of_the_kernels_takes_the_non_coherent_path():
    # Kernels here are set up while the one before them still runs, and wait for it inside. The non-coherent path is defined for memory that nobody
    # writes during a kernel's whole life, set-up included; no run shows a stale line reliably, so the source is read: no such load, and no
    # kernel's pointer that is const and restrict, which lets the compiler choose one.
    import re
    from pathlib import Path
    csrc = Path(__file__).resolve().parent.parent / "csrc"
    for path in sorted([*csrc.glob("src/*.cu"), *csrc.glob("include/purlin/*.cuh")]):
        text = path.read_text()
        assert not re.search(r"\bld\.global[\w.:]*\.nc\b|__ldg\(", text), path.name
        for head in re.findall(r"__global__[^{;]*", text):
            assert not re.search(r"\bconst\s+[\w:]+\s*\*\s*__restrict__", head), (path.name, head[:200])


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_rows_of_2_to_the_31_values_are_refused():
    # the kernels count columns in 32 bits; 2^32 + 64 of them would be 64
    from purlin_b200 import _native
    from purlin_b200.ops.mx4 import Mx4Tensor, mx4_gemm, quantize_mx4, scale_bytes
    for cols in (2 ** 31 - 1024, 2 ** 31, 2 ** 32 + 64):
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            with pytest.raises(ValueError, match="columns"):
                quantize_mx4(_meta(1, cols, dtype=dtype))
        with pytest.raises(ValueError, match="columns"):
            Mx4Tensor(_meta(1, cols // 2, dtype=torch.uint8), _meta(scale_bytes(1, cols), dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):               # the widest that fits: refused for its device alone
        quantize_mx4(_meta(1, 2 ** 31 - 1056))
    lib = _native.cuda()
    assert "large" in _refusal(lib.purlin_mx4_quantize(p(4096), i(0), p(4096), p(4096), i(1), i(2 ** 31 - 1024), n))


def test_the_block_refuses_2_to_the_29_tokens_in_python_as_in_c():
    from purlin_b200 import _native
    from purlin_b200.ops.gated_ffn import gated_ffn
    most = 2 ** 29
    for tokens, hidden, intermediate in ((most, 64, 32), (most + 5, 64, 32), (4, most, 16), (4, 8, most), (1, 2 ** 32 + 8, 16), (1, 8, 2 ** 32 + 16)):
        with pytest.raises(ValueError, match=r"below 2\^29"):
            gated_ffn(_meta(tokens, hidden), _meta(2 * intermediate, hidden), _meta(hidden, intermediate))
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn(_meta(most - 1, 64), _meta(64, 64), _meta(64, 32))
    lib = _native.cuda()
    for sizes in ((most, 64, 32), (4, most, 16), (4, 8, most)):
        assert "below 2^29" in _refusal(lib.purlin_ffn_forward(p(4096), p(4096), p(4096), p(4096), n, p(4096), *map(i, sizes), i(0), n, n))


def _dual(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


def test_forward_mode_derivatives_are_refused():
    # below the checks of the device, so that it needs none: a tangent on any argument, with and without gradients asked for
    from purlin_b200 import _native
    ops = _native.torch_ops()
    args = [torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16), torch.zeros(64, 32, dtype=torch.bfloat16)]
    with torch.autograd.forward_ad.dual_level():
        for k in range(3):
            for needs in (False, True):
                called = [v.clone().requires_grad_(needs) for v in args]
                called[k] = _dual(called[k])
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                        ops.gated_ffn(*called, 0)


def test_a_product_with_an_output_refuses_gradients_and_any_product_tangents():
    from purlin_b200 import _native
    ops = _native.torch_ops()
    x, data, scales = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    out = torch.zeros(4, 64, dtype=torch.bfloat16)
    for a, o in ((x.clone().requires_grad_(), out), (x, out.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="not differentiable"):
            ops.mx4_product(a, 0, None, data, scales, o, 4, 0)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.mx4_product(_dual(x), 0, None, data, scales, out, 4, 0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.mx4_new_product(_dual(x), 0, None, data, scales, [4, 64], 4, 0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.mx4_quantize(_dual(x), 0, 4, 64)


def test_no_wait_of_the_operators_has_a_fixed_limit():
    # an epilogue waits for sums of up to 2^29 tokens, which may take longer than any limit that does not know of them
    from pathlib import Path
    src = Path(__file__).resolve().parent.parent / "csrc" / "src"
    for name, launches in (("gated_ffn.cu", 1), ("mx4.cu", 2)):
        limits = [line.split("timeoutNs =")[1] for line in (src / name).read_text().splitlines() if "timeoutNs =" in line]
        assert len(limits) == launches and all("waitLimitNs(" in v for v in limits), name
