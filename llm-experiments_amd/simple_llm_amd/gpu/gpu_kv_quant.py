"""Block-scaled KV caches (torch.float4_e2m1fn_x2 and torch.float8_e4m3fn): the
launches behind the functions of gpu_kv_cache, which have checked the
arguments. The formats and layouts are in include/skv.h (skv_q_*).

The split workspaces are allocated per call from torch's caching allocator,
in stream order: calls on different streams, and captured calls, do not share
one.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import threading
from typing import Optional

import numpy as np
import torch

from .. import _lib
from .gpu_types import GPUBuffer2D, GPUContext, KVCache, KVCacheLayer

GROUP = 32  # elements that share a scale
MAX_HEAD_DIM = 256
MAX_GROUPS = 16  # query heads per kv head
MAX_TOKENS = 1 << 30  # of a sequence

_BITS = {torch.float4_e2m1fn_x2: 4, torch.float8_e4m3fn: 8}


def check_sizes(batch_size: int, n_heads: int, n_kv_heads: int, head_dim: int,
                tokens: int) -> None:
    """tokens: what a sequence can hold."""
    if head_dim % GROUP or head_dim > MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of {GROUP} up to {MAX_HEAD_DIM} in a "
                         f"block-scaled cache, got {head_dim}")
    if n_heads // n_kv_heads > MAX_GROUPS:
        raise ValueError(f"a block-scaled cache takes up to {MAX_GROUPS} query heads per kv head, "
                         f"got {n_heads // n_kv_heads}")
    if batch_size > 65535 or n_kv_heads > 65535:
        raise ValueError("a block-scaled cache takes up to 65535 sequences and kv heads, got "
                         f"{batch_size} and {n_kv_heads}")
    if tokens > MAX_TOKENS:
        raise ValueError("a block-scaled cache takes sequences of up to 2^30 tokens, got "
                         f"{tokens}")


def create_layer(ctx: GPUContext, batch_size: int, rows: int, head_dim: int,
                 dtype: torch.dtype) -> KVCacheLayer:
    """rows: head rows, [sequences or pages, kv heads, positions] flattened."""
    def buf(width: int) -> GPUBuffer2D:
        t = torch.zeros((rows, width), dtype=torch.uint8, device=ctx.device)
        return GPUBuffer2D(buffer=t, shape=(rows, width), size=rows * width)

    codes, scales = head_dim * _BITS[dtype] // 8, head_dim // GROUP
    return KVCacheLayer(k_cache=buf(codes), v_cache=buf(codes),
                        lens=torch.zeros(batch_size, dtype=torch.int32, device=ctx.device),
                        host_lens=np.zeros(batch_size, dtype=np.int64),
                        k_scale=buf(scales), v_scale=buf(scales))


_HERE = contextlib.nullcontext()


def _on(dev: torch.device):
    """Launches go to the current device: make it the cache's."""
    if torch._C._cuda_getDevice() == (dev.index or 0):
        return _HERE
    return torch.cuda.device(dev)


def _storage(layer: KVCacheLayer) -> tuple:
    return (layer.k_cache.buffer.data_ptr(), layer.k_scale.buffer.data_ptr(),
            layer.v_cache.buffer.data_ptr(), layer.v_scale.buffer.data_ptr())


def _pages(cache: KVCache) -> tuple:
    """(block table, pages a sequence, page size)."""
    if not cache.paged:
        return None, 0, 0
    return cache.block_table.data_ptr(), cache.block_table.shape[1], cache.block_size


def append(cache: KVCache, layer: KVCacheLayer, k: torch.Tensor, v: torch.Tensor) -> None:
    dev = layer.lens.device
    with _on(dev):
        rc = _lib.lib().skv_q_append(*_storage(layer), k.data_ptr(), v.data_ptr(),
                                     layer.lens.data_ptr(), *_pages(cache), cache.batch_size,
                                     cache.n_kv_heads, cache.head_dim, cache.max_seq_len,
                                     _lib.QUANT_FORMATS[cache.dtype], _lib.dtype_code(k.dtype),
                                     _lib.stream_handle(dev))
    _lib.check(rc, "skv_q_append")


def read(cache: KVCache, layer: KVCacheLayer, k_out: torch.Tensor, v_out: torch.Tensor,
         start: np.ndarray) -> None:
    """start: first positions (int32), one for every sequence or one for all."""
    dev = layer.lens.device
    with _on(dev):
        rc = _lib.lib().skv_q_read(k_out.data_ptr(), v_out.data_ptr(), *_storage(layer),
                                   layer.lens.data_ptr(), _lib.host_ptr(start), start.size,
                                   *_pages(cache), cache.batch_size, k_out.shape[1],
                                   cache.n_kv_heads, cache.head_dim, cache.max_seq_len,
                                   _lib.QUANT_FORMATS[cache.dtype], _lib.dtype_code(k_out.dtype),
                                   _lib.stream_handle(dev))
    _lib.check(rc, "skv_q_read")


_PLAN_OUT = threading.local()


def plan(cache: KVCache, q_dt: int, out_dt: int, max_len: int, total_len: int, covering: bool,
         hint: int = 0) -> tuple[int, int, int]:
    """(chunk_tokens, n_chunks, n_wg) of skv_q_decode_plan."""
    out = getattr(_PLAN_OUT, "refs", None)
    if out is None:  # per thread: the call releases the GIL while it fills them
        v = tuple(ctypes.c_int() for _ in range(3))
        out = _PLAN_OUT.refs = v + tuple(ctypes.byref(x) for x in v)
    rc = _lib.lib().skv_q_decode_plan(cache.batch_size, cache.n_heads, cache.n_kv_heads,
                                      cache.head_dim, _lib.QUANT_FORMATS[cache.dtype], q_dt,
                                      out_dt, max(max_len, 1), total_len, covering, hint, out[3],
                                      out[4], out[5])
    if rc:
        _lib.check(rc, "skv_q_decode_plan")
    return out[0].value, out[1].value, out[2].value


def attend(ctx: GPUContext, cache: KVCache, layer: KVCacheLayer, q: torch.Tensor,
           out: torch.Tensor, scale: Optional[float], max_len: int, total: int, covering: bool,
           new_k: Optional[torch.Tensor] = None, new_v: Optional[torch.Tensor] = None) -> None:
    """decode_attention, after the append of new_k and new_v if given. total: the
    fills' sum; covering: the call serves any fills up to max_len, not only those
    that sum to it. A captured call does: it may be replayed with others."""
    dev = layer.lens.device
    max_len = min(int(max_len), cache.block_table.shape[1] * cache.block_size if cache.paged
                  else cache.max_seq_len)  # more is workspace that no fill reaches
    L = _lib.lib()
    B, Hq, Hkv, D = cache.batch_size, cache.n_heads, cache.n_kv_heads, cache.head_dim
    qdt, odt = _lib.dtype_code(q.dtype), _lib.dtype_code(out.dtype)
    sc = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    nk = nv = None
    idt = 0
    if new_k is not None:
        nk, nv, idt = new_k.data_ptr(), new_v.data_ptr(), _lib.dtype_code(new_k.dtype)
    with _on(dev):
        chunk, n, n_wg = plan(cache, qdt, odt, max_len, total,
                              covering or torch.cuda.is_current_stream_capturing(),
                              int(ctx.config.decode_chunk_tokens))
        ws, need = None, 0
        if n > 1:
            need = int(L.skv_q_decode_workspace_bytes(B, Hq, D, n))
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        rc = L.skv_q_decode_attn(out.data_ptr(), q.data_ptr(), *_storage(layer), nk, nv,
                                 layer.lens.data_ptr(), *_pages(cache), B, Hq, Hkv, D,
                                 cache.max_seq_len, sc, chunk, n, n_wg,
                                 ws.data_ptr() if ws is not None else None, need,
                                 _lib.QUANT_FORMATS[cache.dtype], idt, qdt, odt,
                                 _lib.stream_handle(dev))
    _lib.check(rc, "skv_q_decode_attn")


def prefill(ctx: GPUContext, cache: KVCache, layer: KVCacheLayer, new_k: torch.Tensor,
            new_v: torch.Tensor, q: Optional[torch.Tensor], out: Optional[torch.Tensor],
            counts: Optional[np.ndarray], scale: Optional[float], n_splits: int) -> None:
    """kv_cache_prefill; counts: tokens per sequence, or None for whole chunks."""
    dev = layer.lens.device
    L = _lib.lib()
    B, Hq, Hkv, D = cache.batch_size, cache.n_heads, cache.n_kv_heads, cache.head_dim
    C = int(new_k.shape[1])
    fmt, idt = _lib.QUANT_FORMATS[cache.dtype], _lib.dtype_code(new_k.dtype)
    n_host = None if counts is None else np.ascontiguousarray(counts, np.int32)
    n_ptr = None if counts is None else _lib.host_ptr(n_host)
    with _on(dev):
        stream = _lib.stream_handle(dev)
        if q is None:
            rc = L.skv_q_append_chunk(*_storage(layer), new_k.data_ptr(), new_v.data_ptr(),
                                      layer.lens.data_ptr(), None, n_ptr, 1, *_pages(cache), B, C,
                                      Hkv, D, cache.max_seq_len, fmt, idt, stream)
            _lib.check(rc, "skv_q_append_chunk")
            return
        ns = ctypes.c_int(int(n_splits))
        if n_splits <= 0:
            fills = np.ascontiguousarray(layer.host_lens, np.int32)
            _lib.check(L.skv_q_prefill_plan(B, C, Hq, Hkv, D, _lib.host_ptr(fills), n_ptr,
                                            ctypes.byref(ns)), "skv_q_prefill_plan")
        need = int(L.skv_prefill_workspace_bytes(B, C, Hq, D, ns.value)) + 8 * B
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        sc = float(scale) if scale is not None else 1.0 / math.sqrt(D)
        rc = L.skv_q_append_prefill_attn(out.data_ptr(), q.data_ptr(), *_storage(layer),
                                         new_k.data_ptr(), new_v.data_ptr(),
                                         layer.lens.data_ptr(), None, n_ptr, *_pages(cache), B, C,
                                         Hq, Hkv, D, cache.max_seq_len, sc, ns.value,
                                         ws.data_ptr(), need, fmt, idt, _lib.dtype_code(q.dtype),
                                         _lib.dtype_code(out.dtype), stream)
        _lib.check(rc, "skv_q_append_prefill_attn")
