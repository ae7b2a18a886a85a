"""4-bit microscaled tensors and products of them (csrc/src/mx4.cu, csrc/src/torch_ops.cpp).

32 neighbouring values of a row share a power of two (a byte, e8m0); each is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, with a sign (e2m1): 4.25
bits a value. ``quantize_mx4`` makes such a tensor, ``mx4_gemm`` and ``mx4_gemm_swiglu`` multiply activations with a weight that was quantised once;
both operands go to the block-scaled tensor cores as they are, sums are fp32. For inference: nothing here is differentiable. A quantised tensor
knows of no gradient; a product of a dense tensor that requires one gives a result whose differentiation raises, and is refused with ``out``.
Waits inside the kernels are bounded: see ``ops.waits``.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _native

EPI_STORE, EPI_SWIGLU = 0, 1
MAX_ROWS = 2 ** 30
MAX_COLS = 2 ** 31 - 1056        # a step of the quantisation past them still counts in 32 bits
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def scale_bytes(rows: int, cols: int) -> int:
    """Bytes of the scales of a [rows, cols] tensor: 512 for every 128 rows x 128 columns, the last ones filled up."""
    return -(-rows // 128) * -(-cols // 128) * 512


def _refuse_sizes(rows: int):
    raise ValueError("at most 2^30 rows" if rows > MAX_ROWS else "at most 2^31 - 1056 columns")


class Mx4Tensor:
    """A [rows, cols] tensor in 4-bit microscaled form. ``data``: uint8 [rows, cols / 2], the even column in a byte's low half. ``scales``: uint8, a
    byte b per 32 columns of a row for 2^(b - 127) (255: the block stands for NaNs), in the tensor cores' order: blocks of 512 bytes for
    128 rows x 128 columns, [rows / 128][cols / 128][row % 32][row / 32 % 4][col / 32 % 4], zeros past the edges."""
    __slots__ = ("data", "scales", "shape", "device")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        if data.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("data and scales are uint8 tensors")
        if data.dim() != 2 or data.shape[1] == 0 or data.shape[1] % 16 or scales.numel() != scale_bytes(data.shape[0], 2 * data.shape[1]):
            raise ValueError("data is [rows, cols / 2] with cols a multiple of 32, and scales has 512 bytes for every 128 rows x 128 columns")
        if data.shape[0] > MAX_ROWS or 2 * data.shape[1] > MAX_COLS:
            _refuse_sizes(data.shape[0])
        if not (data.is_cuda and scales.device == data.device and data.is_contiguous() and scales.is_contiguous()):
            raise ValueError("data and scales must be contiguous CUDA tensors on one device")
        if (data.data_ptr() | scales.data_ptr()) % 16:
            raise ValueError("data and scales must start on a 16-byte boundary")
        self.data, self.scales, self.shape, self.device = data, scales, (data.shape[0], 2 * data.shape[1]), data.device

    @classmethod
    def _of(cls, data: torch.Tensor, scales: torch.Tensor, rows: int, cols: int) -> "Mx4Tensor":
        q = cls.__new__(cls)                 # (what the quantisation made needs no check)
        q.data, q.scales, q.shape, q.device = data, scales, (rows, cols), data.device
        return q

    def scale_matrix(self) -> torch.Tensor:
        """The scales' bytes in the order of the values, uint8 [rows, cols / 32]."""
        rows, cols = self.shape
        v = self.scales.view(-(-rows // 128), -(-cols // 128), 32, 4, 4).permute(0, 3, 2, 1, 4)
        return v.reshape(-(-rows // 128) * 128, -1)[:rows, :cols // 32].contiguous()

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the tensor stands for in ``dtype`` (bf16 or fp32); they carry no gradient. Exact for what ``quantize_mx4`` makes; of
        scale bytes of 253 and 254, which it never makes, the largest values are past the types' range and become infinities."""
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("values come back in bf16 or fp32")
        return _native.torch_ops().mx4_dequantize(self.data, self.scales, TYPES[dtype])


def _check_dense(x: torch.Tensor) -> Tuple[int, int, int]:
    """Rows, columns and type number of a dense operand."""
    kind = TYPES.get(x.dtype)
    if kind is None:
        raise TypeError("quantisation takes bf16, fp16 or fp32 values")
    shape = x.shape
    cols = shape[-1] if shape else 0
    if cols == 0 or cols % 32:
        raise ValueError("the last dimension must be a multiple of 32")
    rows = x.numel() // cols
    if rows > MAX_ROWS or cols > MAX_COLS:
        _refuse_sizes(rows)
    if not (x.is_cuda and x.is_contiguous()):
        raise ValueError("operands must be contiguous CUDA tensors")
    if x.data_ptr() % 16:
        raise ValueError("operands must start on a 16-byte boundary")
    return rows, cols, kind


def quantize_mx4(x: torch.Tensor) -> Mx4Tensor:
    """``x [..., cols]`` (bf16, fp16 or fp32, contiguous, cols a multiple of 32) as an ``Mx4Tensor`` of its rows. A block's power of two is that of its
    largest magnitude over 4, at least 2^-127; values are rounded to the nearest of the format, ties to the even code, and above 6 times the power
    to 6. A block that holds an infinity or a NaN stands for NaNs. Not differentiable: the result, and what it is dequantised to, has no gradient."""
    rows, cols, kind = _check_dense(x)
    return Mx4Tensor._of(*_native.torch_ops().mx4_quantize(x, kind, rows, cols), rows, cols)


def _product(a: Union[torch.Tensor, Mx4Tensor], w: Mx4Tensor, out: Optional[torch.Tensor], epilogue: int) -> torch.Tensor:
    if not isinstance(w, Mx4Tensor):
        raise TypeError("w is an Mx4Tensor (quantize_mx4)")
    n, k = w.shape
    if isinstance(a, Mx4Tensor):
        rows, cols = a.shape
        operand = (a.data, 0, a.scales)
    else:
        rows, cols, kind = _check_dense(a)
        operand = (a, kind, None)
    if cols != k or a.device != w.device:
        raise ValueError("a is [..., K] and w is [N, K], on one device")
    if n == 0 or n % (32 if epilogue == EPI_SWIGLU else 8):
        raise ValueError("the SwiGLU epilogue needs N to be a multiple of 32 (16 rows of gate and 16 of up in turn)" if epilogue == EPI_SWIGLU
                         else "N must be a multiple of 8")
    shape = (*a.shape[:-1], n // 2 if epilogue == EPI_SWIGLU else n)
    if out is None:
        return _native.torch_ops().mx4_new_product(*operand, w.data, w.scales, shape, rows, epilogue)
    if out.dtype != torch.bfloat16:
        raise TypeError("out is a bf16 tensor")
    if out.shape != shape or out.device != w.device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out is a contiguous tensor of {shape} on the operands' device")
    _native.torch_ops().mx4_product(*operand, w.data, w.scales, out, rows, epilogue)
    return out


def mx4_gemm(a: Union[torch.Tensor, Mx4Tensor], w: Mx4Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ w.T`` in bf16 for ``a [..., K]``, an ``Mx4Tensor`` or a bf16, fp16 or fp32 tensor that is quantised in the call, and ``w [N, K]``; N a multiple of
    8. One token or many. ``out`` may be (or overlap) a dense ``a``; it may not overlap a quantised operand.
    Not differentiable: where ``a`` requires a gradient, differentiating the result raises, and a call with ``out`` is refused."""
    return _product(a, w, out, EPI_STORE)


def mx4_gemm_swiglu(a: Union[torch.Tensor, Mx4Tensor], w_gu: Mx4Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``silu(a @ w_gate.T) * (a @ w_up.T)`` for ``w_gu = quantize_mx4(interleave_gate_up(w_gate, w_up))``; ``a`` and ``out`` as in ``mx4_gemm``."""
    return _product(a, w_gu, out, EPI_SWIGLU)
