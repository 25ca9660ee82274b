"""What the training passes (forward, backward, optimizer) share: operands as
tensors, their checks, and the device that launches go to.

Operands are GPUBuffers or contiguous device tensors. Everything is checked
before any launch: a rejected call changes nothing.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence, Union

import torch

from .. import _lib
from .gpu_types import GPUBuffer1D, GPUBuffer2D, GPUContext

Operand = Union[GPUBuffer1D, GPUBuffer2D, torch.Tensor]

FLOATS = (torch.float32, torch.bfloat16)
F32 = (torch.float32,)
I32 = (torch.int32,)

_HERE = contextlib.nullcontext()


def on(dev: torch.device):
    """Launches go to the current device: make it the operands'."""
    if torch._C._cuda_getDevice() == (dev.index or 0):
        return _HERE
    return torch.cuda.device(dev)


def operand(ctx: GPUContext, buf: Operand, name: str, shape: Optional[Sequence[int]],
            dtypes: Sequence[torch.dtype], align: int = 16) -> torch.Tensor:
    """The operand's tensor: of `shape` (None: any), one of `dtypes`, contiguous and
    aligned, on the context's device."""
    t = buf if isinstance(buf, torch.Tensor) else getattr(buf, "buffer", None)
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a GPUBuffer or a tensor, got {type(buf).__name__}")
    if shape is not None and t.shape != torch.Size(shape):
        raise ValueError(f"{name} shape mismatch: got {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    dev = ctx.device
    if not t.is_cuda or t.get_device() != (dev.index or 0):
        raise ValueError(f"{name} must live on {dev}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.data_ptr() % align:
        raise ValueError(f"{name} must be {align}-byte aligned")
    return t


def rows_of(ctx: GPUContext, buf: Operand, name: str, dtypes: Sequence[torch.dtype],
            align: int = 16) -> torch.Tensor:
    """A 2-D operand of any shape that holds elements."""
    t = operand(ctx, buf, name, None, dtypes, align)
    if t.dim() != 2 or t.numel() == 0:
        raise ValueError(f"{name} must be 2-D and hold elements, got shape {tuple(t.shape)}")
    if max(t.shape) >= 1 << 31:
        raise ValueError(f"{name} is too large: {tuple(t.shape)}")
    return t


def apart(outputs: Sequence[tuple], inputs: Sequence[tuple]) -> None:
    """ValueError if an output (tensor, name) overlaps another output or an input."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), name)
             for t, name in (*outputs, *inputs) if t is not None]
    n_out = sum(t is not None for t, _ in outputs)
    for i in range(n_out):
        for j in range(i + 1, len(spans)):
            if spans[i][0] < spans[j][1] and spans[j][0] < spans[i][1]:
                raise ValueError(f"{spans[i][2]} overlaps {spans[j][2]}")


def workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    """Workspace of one call, from torch's caching allocator in stream order: calls on
    different streams, and captured calls, do not share one."""
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=dev)


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def stream(dev: torch.device) -> int:
    return _lib.stream_handle(dev)
