"""The optimizer of a training step on gfx950: AdamW over all tensors of a model in
one launch, with moments in 32 or 8 bits.

The work of adamw in simple-llm/src/gpu/gpu_pass_optimizer.py:28-393 (one tensor a
launch, fp32 moments), with this package's own arguments.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Union

import numpy as np
import torch

from .. import _lib
from .gpu_pass_common import F32, FLOATS, Operand, device_of, launch, required, tensor_of
from .gpu_types import GPUContext

_CHUNK = 4096  # elements of a tensor that a workgroup takes at a time
_BLOCK = 128  # moments that share a scale; a tensor's begin a block
_ZERO_SCALE = 127 - 90  # the scale byte of a block of zeros
_LEAST = 2.0 ** -126  # the least normal float32


class AdamWState:
    """The optimizer of a list of tensors: what adamw_create returns.

    m, v: the moments of all tensors end to end, tensor i's from offsets[i] on (a
    multiple of 128; the places in between hold zeros): float32, or uint8 codes with
    m_scale, v_scale, a byte for 128 moments (include/skv.h has the formats).
    step: int32 device tensor [1], the steps taken, advanced on the device by every
    adamw_update, also when a captured one is replayed.
    seed: of the 8-bit moments' rounding; a number, read by adamw_update.

    m, v, the scales, step and seed are all there is to save. A program that resumes copies
    the saved tensors into those of a new state (state.m.copy_(saved), ...): the attributes
    themselves cannot be replaced. The parameters, gradients and copies are held, and used
    where they were when the state was made.
    """

    def __init__(self, params: List[torch.Tensor], grads: List[torch.Tensor],
                 copies: Optional[List[torch.Tensor]], bits: int, offsets: List[int], seed: int,
                 m: torch.Tensor, v: torch.Tensor, m_scale: Optional[torch.Tensor],
                 v_scale: Optional[torch.Tensor], count: torch.Tensor, tensors: torch.Tensor,
                 chunks: torch.Tensor):
        self.params = params
        self.grads = grads
        self.copies = copies
        self.offsets = offsets
        self.seed = seed
        self._bits = bits
        self._m = m
        self._v = v
        self._m_scale = m_scale
        self._v_scale = v_scale
        self._step = count[:1]
        self._count = count
        self._tensors = tensors
        self._chunks = chunks
        self._grad_dtype = grads[0].dtype
        # Every tensor that the kernel reaches by its address: it has to be there still, and
        # a second reference keeps the memory from being given away in any case.
        self._held = [*params, *grads, *(copies or []), m, v, self._step]
        if bits == 8:
            self._held += [m_scale, v_scale]
        self._at = [t.data_ptr() for t in self._held]
        self._memory = [t.detach() for t in self._held]

    bits = property(lambda self: self._bits)
    m = property(lambda self: self._m)
    v = property(lambda self: self._v)
    m_scale = property(lambda self: self._m_scale)
    v_scale = property(lambda self: self._v_scale)
    step = property(lambda self: self._step)

    @property
    def seed(self) -> int:
        return self._seed

    @seed.setter
    def seed(self, seed: int) -> None:
        if not 0 <= int(seed) < 1 << 32:
            raise ValueError(f"seed must lie in [0, 2^32), got {seed}")
        self._seed = int(seed)

    def _scales(self) -> tuple:
        if self.bits == 32:
            return None, None
        return self.m_scale.data_ptr(), self.v_scale.data_ptr()

    def __repr__(self) -> str:
        return (f"AdamWState(tensors={len(self.params)}, elements={self.m.numel()}, "
                f"bits={self.bits})")


def adamw_create(ctx: GPUContext, params: Sequence[Operand], grads: Sequence[Operand],
                 bits: int = 32, copies: Optional[Sequence[Operand]] = None,
                 decay: Optional[Sequence[bool]] = None, seed: int = 0) -> AdamWState:
    """The AdamW state of params, zero moments and zero steps.

    params: float32, any shapes; grads: their gradients' buffers, like params, all float32
    or all bfloat16; copies: bfloat16 buffers like params that every step writes the new
    weights to as well, or None. decay: whether weight decay applies, by tensor (default:
    to all). bits: 32, or 8 (moments in blocks of 128 with a shared power-of-two scale, each
    rounded up or down at random; seed: of that rounding).
    """
    if bits not in (32, 8):
        raise ValueError(f"bits must be 32 or 8, got {bits}")
    if not 0 <= int(seed) < 1 << 32:
        raise ValueError(f"seed must lie in [0, 2^32), got {seed}")
    n = len(params)
    if n == 0:
        raise ValueError("params holds no tensors")
    for name, given in (("grads", grads), ("copies", copies), ("decay", decay)):
        if given is not None and len(given) != n:
            raise ValueError(f"{name} must have an entry for each of the {n} params, got "
                             f"{len(given)}")
    if grads is None:
        raise ValueError("grads must have an entry for each of the params")
    dev = device_of(ctx)
    ps, gs, cs = [], [], []
    for i in range(n):
        required(dev, params[i], f"params[{i}]", None, F32, 4)
        p = tensor_of(params[i])
        if p.numel() == 0:
            raise ValueError(f"params[{i}] holds no elements")
        ps.append(p)
        required(dev, grads[i], f"grads[{i}]", p.shape, FLOATS if i == 0 else (gs[0].dtype,), 2)
        gs.append(tensor_of(grads[i]))
        if copies is not None:
            required(dev, copies[i], f"copies[{i}]", p.shape, (torch.bfloat16,), 2)
            cs.append(tensor_of(copies[i]))
    _disjoint([(p, f"params[{i}]", True) for i, p in enumerate(ps)]
              + [(c, f"copies[{i}]", True) for i, c in enumerate(cs)]
              + [(g, f"grads[{i}]", False) for i, g in enumerate(gs)])

    sizes = np.array([p.numel() for p in ps], np.int64)
    ends = np.cumsum(-(-sizes // _BLOCK) * _BLOCK)
    offsets = np.concatenate([[0], ends[:-1]]).astype(np.int64)
    total = int(ends[-1])
    counts = -(-sizes // _CHUNK)
    if int(counts.sum()) >= 1 << 31:
        raise ValueError("params holds too many elements")
    table = np.zeros((n, 6), np.int64)  # skv_adamw_tensor
    table[:, 0] = [p.data_ptr() for p in ps]
    table[:, 1] = [g.data_ptr() for g in gs]
    table[:, 2] = [c.data_ptr() for c in cs] if cs else 0
    table[:, 3] = sizes
    table[:, 4] = offsets
    table[:, 5] = 1 if decay is None else [1 if d else 0 for d in decay]
    which = np.repeat(np.arange(n), counts)
    inside = np.arange(int(counts.sum())) - np.repeat(np.cumsum(counts) - counts, counts)
    chunks = np.stack([which, inside], -1).astype(np.int32)

    def zeros(size: int, dtype: torch.dtype) -> torch.Tensor:
        return torch.zeros(size, dtype=dtype, device=dev)

    scales = [None, None]
    if bits == 8:
        scales = [torch.full((total // _BLOCK,), _ZERO_SCALE, dtype=torch.uint8, device=dev)
                  for _ in range(2)]
    kind = torch.float32 if bits == 32 else torch.uint8
    return AdamWState(ps, gs, cs or None, bits, [int(o) for o in offsets], int(seed),
                      zeros(total, kind), zeros(total, kind), *scales, zeros(2, torch.int32),
                      torch.from_numpy(table).to(dev), torch.from_numpy(chunks).to(dev))


def _disjoint(tensors: Sequence[tuple]) -> None:
    """ValueError if a written tensor overlaps any other; (tensor, name, written)."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w, name)
                   for t, name, w in tensors)
    reach = written = None  # the furthest ends so far: of all, of written ones
    for lo, hi, w, name in spans:
        over = reach if w else written
        if over is not None and lo < over[0]:
            raise ValueError(f"{name} overlaps {over[1]}")
        if reach is None or hi > reach[0]:
            reach = (hi, name)
        if w and (written is None or hi > written[0]):
            written = (hi, name)


def _number(dev: int, x: Union[float, Operand], name: str) -> tuple:
    """(value, None) of a number, (0, its address) of one in device memory."""
    if isinstance(x, (int, float)):
        if not math.isfinite(x):
            raise ValueError(f"{name} must be finite, got {x}")
        return float(x), None
    return 0.0, required(dev, x, name, (1,), F32, 4)


def adamw_update(ctx: GPUContext, state: AdamWState, lr: Union[float, Operand],
                 beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                 weight_decay: float = 0.01,
                 grad_scale: Union[float, Operand] = 1.0) -> None:
    """One step of every tensor, with t the steps taken after it:

        m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,  g = grad_scale * grad
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

    lr, grad_scale: numbers, or float32 device tensors [1], which a captured step reads anew
    when it is replayed. eps: 0 or at least 2^-126. With 8-bit moments the step uses them before
    they are rounded.
    """
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError(f"beta1 and beta2 must lie in [0, 1), got {beta1} and {beta2}")
    if not ((eps == 0 or _LEAST <= eps < math.inf) and math.isfinite(weight_decay)):
        raise ValueError(f"eps must be 0, or at least 2^-126 and finite, and weight_decay finite, "
                         f"got {eps} and {weight_decay}")
    dev = device_of(ctx)
    lr, lr_dev = _number(dev, lr, "lr")
    grad_scale, scale_dev = _number(dev, grad_scale, "grad_scale")
    _check_state(ctx, state)
    launch(ctx, dev, "skv_adamw", state._tensors.data_ptr(), state._chunks.data_ptr(),
           state._chunks.shape[0], state.m.data_ptr(), state.v.data_ptr(), *state._scales(),
           state._count.data_ptr(), state.bits, _lib.dtype_code(state._grad_dtype), lr, lr_dev,
           float(beta1), float(beta2), float(eps), float(weight_decay), grad_scale, scale_dev,
           state.seed)


def _check_state(ctx: GPUContext, state: AdamWState) -> None:
    if [t.data_ptr() for t in state._held] != state._at:
        raise ValueError("a parameter, gradient, copy or tensor of the state is no longer where it "
                         "was when the state was made: write into their buffers, or make a new state")
    if state.m.get_device() != device_of(ctx):
        raise ValueError(f"the state lives on {state.m.device}, the context on {ctx.device}")


def adamw_read(ctx: GPUContext, state: AdamWState, m: Operand, v: Operand) -> None:
    """The moments of an 8-bit state as values: m, v float32 or bfloat16 (both the same;
    exact in either), of the state's elements in the state's order (AdamWState.offsets)."""
    if state.bits != 8:
        raise ValueError("adamw_read reads 8-bit moments; a 32-bit state holds them in m and v")
    dev = device_of(ctx)
    n = state.m.numel()
    mo = required(dev, m, "m", (n,), FLOATS)
    dtype = tensor_of(m).dtype
    vo = required(dev, v, "v", (n,), (dtype,))
    _check_state(ctx, state)
    launch(ctx, dev, "skv_adamw_read", mo, vo, state.m.data_ptr(), state.v.data_ptr(),
           *state._scales(), n, _lib.dtype_code(dtype))


__all__ = ["AdamWState", "adamw_create", "adamw_read", "adamw_update"]
