"""Waits inside the kernels of ``ops.gated_ffn`` and ``ops.mx4``.

Every wait of these kernels is bounded. One that gives up leaves its outputs incomplete; the next call of any of these operators on the device
raises then (a backward pass too), and ``check_waits`` asks without a call, after the last step or a graph's replay.
"""
from __future__ import annotations

import torch

from .. import _native


def check_waits(device=None) -> None:
    """Synchronises the device (the current one by default) and raises if a wait inside an earlier kernel of these operators gave up."""
    torch.cuda.synchronize(device)
    device = torch.device("cuda" if device is None else device) if not isinstance(device, int) else torch.device("cuda", device)
    code, where, tile, k_block = _native.torch_ops().take_wait_report(torch.cuda.current_device() if device.index is None else device.index)
    if code:
        raise TimeoutError(f"purlin: a wait inside a kernel of the operators gave up (where {where}, {tile}, {k_block}): what it computed is not complete")
