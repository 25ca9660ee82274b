"""Forward passes of a training step on gfx950: the embedding, LayerNorm, causal
FlashAttention and the cross-entropy loss.

embedding, layernorm and cross_entropy_loss have the work of their namesakes in
simple-llm/src/gpu/gpu_pass_forward.py (:84-137, :140-176, :331-416); their arguments
are this package's own: they take fp32 and bf16 activations, and GPUBuffers or
contiguous device tensors.

flash_attention: causal FlashAttention with its row statistics, fp32.

Drop-in for flash_attention of simple-llm/src/gpu/gpu_pass_forward.py:497-588:
same arguments, checks and error messages. The reference's WGSL kernel
(gpu/gpu_kernels.py:499-770) runs one workgroup per (query block, head,
sequence) with an online softmax over key blocks; skv_flash_fwd runs the same
computation on MFMA tiles (fp32 products, up to head_dim 128 as six partial
products of operands split into three bf16 parts) and writes O, L (softmax sums) and M (row
maxima of the scaled scores), which flash_attention_backward consumes.
"""
from __future__ import annotations

from typing import Optional

import numpy as np
import torch

from .. import _lib
from .gpu_pass_common import (F32, FLOATS, I32, Operand, device_of, launch, operand, required,
                              rows_of, tensor_of, workspace)
from .gpu_ops import batch_count, validate_buffer_shape_1d, validate_buffer_shape_2d
from .gpu_types import GPUBuffer1D, GPUBuffer2D, GPUContext


def _f32(buf, name: str) -> torch.Tensor:
    t = buf.buffer
    if t.dtype != torch.float32 or not t.is_contiguous() or t.device.type != "cuda":
        raise ValueError(f"{name} must be a contiguous float32 device buffer")
    return t


def flash_attention(
    ctx: GPUContext,
    Q: GPUBuffer2D,
    K: GPUBuffer2D,
    V: GPUBuffer2D,
    O: GPUBuffer2D,
    L: GPUBuffer1D,
    M: GPUBuffer1D,
    batch_size: int,
    seq_len: int,
    n_heads: int,
    head_dim: int,
) -> None:
    """Causal attention forward (reference: gpu_pass_forward.py:497-588).

    Q, K, V, O: [batch_size*seq_len, n_heads*head_dim]; L, M:
    [batch_size*seq_len*n_heads], indexed (b*seq_len + t)*n_heads + h.
    Raises ValueError on a bad shape or dimension, as the reference does.
    """
    if head_dim > ctx.config.flash_attn_max_head_dim:
        raise ValueError(
            f"head_dim {head_dim} exceeds maximum supported by config: "
            f"{ctx.config.flash_attn_max_head_dim}. "
            f"Increase flash_attn_max_head_dim in GPUConfig or use smaller head_dim.")
    if batch_size <= 0 or seq_len <= 0 or n_heads <= 0 or head_dim <= 0:
        raise ValueError(
            f"Invalid dimensions: batch_size={batch_size}, seq_len={seq_len}, "
            f"n_heads={n_heads}, head_dim={head_dim}")
    embedding_dim = n_heads * head_dim
    total_tokens = batch_size * seq_len
    validate_buffer_shape_2d(Q, (total_tokens, embedding_dim), "Q")
    validate_buffer_shape_2d(K, (total_tokens, embedding_dim), "K")
    validate_buffer_shape_2d(V, (total_tokens, embedding_dim), "V")
    validate_buffer_shape_2d(O, (total_tokens, embedding_dim), "O")
    stats_size = batch_size * seq_len * n_heads
    validate_buffer_shape_1d(L, stats_size, "L")
    validate_buffer_shape_1d(M, stats_size, "M")
    q, k, v, o, lt, mt = (_f32(b, n) for b, n in zip((Q, K, V, O, L, M),
                                                     ("Q", "K", "V", "O", "L", "M")))
    lib = _lib.lib()
    batch_count(ctx)
    rc = lib.skv_flash_fwd(o.data_ptr(), lt.data_ptr(), mt.data_ptr(), q.data_ptr(),
                           k.data_ptr(), v.data_ptr(), batch_size, seq_len, n_heads, head_dim,
                           float(1.0 / np.sqrt(head_dim)), _lib.stream_handle(q.device))
    _lib.check(rc, "skv_flash_fwd")


def embedding(ctx: GPUContext, tokens: Operand, table: Operand, output: Operand,
              scale: float = 1.0, pos_table: Optional[Operand] = None) -> None:
    """output[i] = scale * table[tokens[i]] + pos_table[i % len(pos_table)].

    tokens: int32 [n], a batch's sequences end to end; table: [vocab, d], output: [n, d],
    each float32 or bfloat16; pos_table: float32 [context, d] or None (positions of sequences
    of exactly `context` tokens). A token outside [0, vocab) is padding: its table row counts
    as zeros.
    """
    dev = device_of(ctx)
    w, vocab, d, w_dtype = rows_of(dev, table, "table", FLOATS)
    ids = required(dev, tokens, "tokens", None, I32, 4)
    shape = tensor_of(tokens).shape
    if len(shape) != 1 or not 0 < shape[0] < 1 << 31:
        raise ValueError(f"tokens must be 1-D and hold elements, got shape {tuple(shape)}")
    n = shape[0]
    out = required(dev, output, "output", (n, d), FLOATS)
    pos, n_pos = None, 0
    if pos_table is not None:
        pos, n_pos, _, _ = rows_of(dev, pos_table, "pos_table", F32, d)
    launch(ctx, dev, "skv_embedding_fwd", out, ids, w, pos, n, vocab, d, n_pos, float(scale),
           _lib.dtype_code(w_dtype), _lib.dtype_code(tensor_of(output).dtype))


def layernorm(ctx: GPUContext, input: Operand, gamma: Operand, beta: Operand, output: Operand,
              mean: Optional[Operand] = None, rstd: Optional[Operand] = None,
              eps: float = 1e-5) -> None:
    """output = (input - mean) * rstd * gamma + beta of every row.

    input, output: [rows, d], both float32 or both bfloat16, d up to 16384; output may be
    input. gamma, beta: float32 [d]. mean, rstd: float32 [rows], the rows' statistics for
    layernorm_backward (rstd = 1 / sqrt(var + eps)), or None.
    """
    dev = device_of(ctx)
    x, rows, d, dtype = rows_of(dev, input, "input", FLOATS)
    y = required(dev, output, "output", (rows, d), (dtype,))
    g = required(dev, gamma, "gamma", (d,), F32)
    b = required(dev, beta, "beta", (d,), F32)
    mu = operand(dev, mean, "mean", (rows,), F32, 4)
    rs = operand(dev, rstd, "rstd", (rows,), F32, 4)
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    launch(ctx, dev, "skv_layernorm_fwd", y, mu, rs, x, g, b, rows, d, float(eps),
           _lib.dtype_code(dtype))


def cross_entropy_loss(ctx: GPUContext, logits: Operand, targets: Operand, loss: Operand,
                       grad_logits: Optional[Operand] = None,
                       row_losses: Optional[Operand] = None, grad_scale: float = 1.0) -> None:
    """loss[0] = the mean of logsumexp(logits[i]) - logits[i, targets[i]] over the rows with a
    target in [0, vocab); the other rows are ignored. 0 if there are none.

    logits: [rows, vocab], float32 or bfloat16; targets: int32 [rows]; loss: float32 [1].
    grad_logits: the loss's gradient times grad_scale, like logits and possibly the same
    buffer, or None. row_losses: float32 [rows], 0 where ignored, or None.
    """
    dev = device_of(ctx)
    x, rows, vocab, dtype = rows_of(dev, logits, "logits", FLOATS)
    t = required(dev, targets, "targets", (rows,), I32, 4)
    out = required(dev, loss, "loss", (1,), F32, 4)
    dx = operand(dev, grad_logits, "grad_logits", (rows, vocab), (dtype,))
    row = operand(dev, row_losses, "row_losses", (rows,), F32, 4)
    ws = workspace(dev, "skv_cross_entropy_workspace_bytes", rows)
    launch(ctx, dev, "skv_cross_entropy", out, row, dx, x, t, rows, vocab, float(grad_scale),
           ws.data_ptr(), ws.numel(), _lib.dtype_code(dtype))


__all__ = ["cross_entropy_loss", "embedding", "flash_attention", "layernorm"]
