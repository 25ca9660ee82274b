"""What the training passes (forward, backward, optimizer) share: operands as
tensors, their checks, and the device that launches go to.

Operands are GPUBuffers or contiguous device tensors. Everything is checked
before any launch: a rejected call changes nothing.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from .. import _lib
from .gpu_ops import batch_count
from .gpu_types import GPUBuffer1D, GPUBuffer2D, GPUContext

Operand = Union[GPUBuffer1D, GPUBuffer2D, torch.Tensor]

FLOATS = (torch.float32, torch.bfloat16)
F32 = (torch.float32,)
I32 = (torch.int32,)


def device_of(ctx: GPUContext) -> int:
    """The number of the device that a context's operands live on."""
    return ctx.device.index or 0


def tensor_of(buf: Operand) -> Optional[torch.Tensor]:
    return buf if isinstance(buf, torch.Tensor) else getattr(buf, "buffer", None)


def required(dev: int, buf: Operand, name: str, shape: Optional[tuple],
             dtypes: Sequence[torch.dtype], align: int = 16) -> int:
    """The address of an operand: of `shape` (None: any), one of `dtypes`, contiguous and
    aligned, on device number `dev`."""
    t = buf if isinstance(buf, torch.Tensor) else getattr(buf, "buffer", None)
    # All checks at once first: every one again below, to say what is wrong.
    if (isinstance(t, torch.Tensor) and (shape is None or t.shape == shape) and t.dtype in dtypes
            and t.get_device() == dev and t.is_contiguous()):
        p = t.data_ptr()
        if not p % align:
            return p
        raise ValueError(f"{name} must be {align}-byte aligned")
    if not isinstance(t, torch.Tensor):
        got = None if buf is None else type(buf).__name__
        raise ValueError(f"{name} must be a GPUBuffer or a tensor, got {got}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} shape mismatch: got {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} must live on cuda:{dev}, got {t.device}")
    raise ValueError(f"{name} must be contiguous")


def operand(dev: int, buf: Optional[Operand], name: str, shape: Optional[tuple],
            dtypes: Sequence[torch.dtype], align: int = 16) -> Optional[int]:
    """required() of an operand that may be None: its address then."""
    return None if buf is None else required(dev, buf, name, shape, dtypes, align)


def rows_of(dev: int, buf: Operand, name: str, dtypes: Sequence[torch.dtype],
            cols: Optional[int] = None) -> tuple:
    """(address, rows, columns, dtype) of a 2-D operand that holds elements; cols: how many
    columns it has to have."""
    p = required(dev, buf, name, None, dtypes)
    t = tensor_of(buf)
    shape = t.shape
    if len(shape) != 2 or not 0 < shape[0] < 1 << 31 or not 0 < shape[1] < 1 << 31:
        raise ValueError(f"{name} must be 2-D with 1 to 2^31 - 1 rows and columns, got shape "
                         f"{tuple(shape)}")
    rows, d = shape
    if cols is not None and d != cols:
        raise ValueError(f"{name} shape mismatch: got {tuple(shape)}, expected (*, {cols})")
    return p, rows, d, t.dtype


_LAUNCH_DEVICE = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def launch(ctx: GPUContext, dev: int, name: str, *args) -> None:
    """The C function `name` of these arguments and torch's current stream of device number
    `dev` (where the operands are), which launches go to."""
    fn = getattr(_lib.lib(), name)
    batch_count(ctx)
    if _LAUNCH_DEVICE() == dev:
        rc = fn(*args, _lib.stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.stream_handle(dev))
    if rc:
        _lib.check(rc, name)


_WS_BYTES: dict = {}


def workspace(dev: int, query: str, *sizes: int) -> torch.Tensor:
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
