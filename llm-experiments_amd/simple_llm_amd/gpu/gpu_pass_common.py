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


def operand(ctx: GPUContext, buf: Operand, name: str, shape: Optional[tuple],
            dtypes: Sequence[torch.dtype], align: int = 16) -> torch.Tensor:
    """The operand's tensor: of `shape` (None: any), one of `dtypes`, contiguous and
    aligned, on the context's device."""
    t = buf if isinstance(buf, torch.Tensor) else getattr(buf, "buffer", None)
    dev = ctx.device
    # Fast path first: every check again below, to say what is wrong.
    if (isinstance(t, torch.Tensor) and (shape is None or t.shape == shape) and t.dtype in dtypes
            and t.is_cuda and t.get_device() == (dev.index or 0) and t.is_contiguous()
            and not t.data_ptr() % align):
        return t
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a GPUBuffer or a tensor, got {type(buf).__name__}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} shape mismatch: got {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if not t.is_cuda or t.get_device() != (dev.index or 0):
        raise ValueError(f"{name} must live on {dev}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    raise ValueError(f"{name} must be {align}-byte aligned")


def rows_of(ctx: GPUContext, buf: Operand, name: str, dtypes: Sequence[torch.dtype],
            align: int = 16) -> torch.Tensor:
    """A 2-D operand of any shape that holds elements."""
    t = operand(ctx, buf, name, None, dtypes, align)
    shape = t.shape
    if len(shape) != 2 or not shape[0] or not shape[1]:
        raise ValueError(f"{name} must be 2-D and hold elements, got shape {tuple(shape)}")
    if shape[0] >= 1 << 31 or shape[1] >= 1 << 31:
        raise ValueError(f"{name} is too large: {tuple(shape)}")
    return t


_WS_BYTES: dict = {}


def workspace(query: str, dev: torch.device, *sizes: int) -> torch.Tensor:
    """Workspace of one call, of the bytes that the C function `query` asks for, from torch's
    caching allocator in stream order: calls on different streams, and captured calls, do not
    share one."""
    key = (query, *sizes)
    need = _WS_BYTES.get(key)
    if need is None:
        if len(_WS_BYTES) > 4096:
            _WS_BYTES.clear()
        need = _WS_BYTES[key] = max(int(getattr(_lib.lib(), query)(*sizes)), 16)
    return torch.empty(need, dtype=torch.uint8, device=dev)


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def stream(dev: torch.device) -> int:
    return _lib.stream_handle(dev)
