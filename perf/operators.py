"""The block-scaled 4-bit and 8-bit KV cache as measurable cases: writing it,
reading it back, and the attention over it.

Cache rows are cut into groups of 32 consecutive elements of a head. A group
holds 32 elements (E2M1 in 4 bits: 0, .5, 1, 1.5, 2, 3, 4, 6; or E4M3 in 8 bits)
and one scale 2^e in a byte, e + 127:

  e  = the smallest integer with max|x| <= top 2^e, top = 7 (E2M1) or 464 (E4M3),
       the largest element plus half a step of its binade; clamped to [-100, 125]
       (E2M1) or [-100, 119] (E4M3)
  c  = x 2^-e rounded to the nearest element (ties to the even code), saturating
  a group with a NaN or an infinity: scale byte 255, codes 0; it reads back as NaN

A cache is [batch, kv_heads, capacity, head_dim] (paged: [pages, kv_heads,
page, head_dim]); two 4-bit codes share a byte, the even element in the low half.

  append   tokens quantised into the cache at each sequence's fill, and read back:
           kv_cache_append (one token) or kv_cache_prefill (a chunk), kv_cache_read
  read     a window of positions back as rows: kv_cache_read
  decode   one query a sequence over its fill: decode_attention
  step     a decode step, append and attention: kv_cache_append_attend
  prefill  a chunk of a prompt with its causal attention: kv_cache_prefill
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "llm-experiments_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False  # True: run() makes the framework's calls; False: the plain forms

DEV = "cuda:0"
_IO = {"fp32": torch.float32, "bf16": torch.bfloat16}
_IO_BYTES = {"fp32": 4, "bf16": 2}
_BITS = {"fp4": 4, "fp8": 8}
_GROUP = 32


def listed():
    return [
        # Loading a stored prefix: 2048 tokens of four sequences at once.
        {"name": "append_long", "kind": "append", "fmt": "fp4", "batch": 4, "kv_heads": 16,
         "groups": 1, "head_dim": 128, "fill": 30000, "lens": "equal", "page": 0, "chunk": 2048,
         "ragged": False, "io": "bf16"},
        # Ragged chunks of prompts that are still being admitted, fp32 activations.
        {"name": "append_ragged", "kind": "append", "fmt": "fp8", "batch": 6, "kv_heads": 8,
         "groups": 4, "head_dim": 128, "fill": 1900, "lens": "uniform", "page": 0, "chunk": 333,
         "ragged": True, "io": "fp32"},
        # One token of each of 64 sequences into a paged cache: the smallest call.
        {"name": "append_token", "kind": "append", "fmt": "fp4", "batch": 64, "kv_heads": 8,
         "groups": 4, "head_dim": 128, "fill": 8192, "lens": "lognormal", "page": 16, "chunk": 1,
         "ragged": False, "io": "bf16"},
        # Handing a long prefix to a program that wants it as bf16 rows.
        {"name": "read_long", "kind": "read", "fmt": "fp4", "batch": 4, "kv_heads": 16,
         "groups": 1, "head_dim": 128, "fill": 32000, "lens": "equal", "page": 0, "start": 16000,
         "chunk": 8192, "io": "bf16"},
        # The last positions of a few short sequences of a paged cache, head_dim 64.
        {"name": "read_short", "kind": "read", "fmt": "fp8", "batch": 3, "kv_heads": 12,
         "groups": 1, "head_dim": 64, "fill": 1000, "lens": "uniform", "page": 16, "start": 200,
         "chunk": 77, "io": "fp32"},
        # Long-context serving: the repository's headline decode shape.
        {"name": "decode_long", "kind": "decode", "fmt": "fp4", "batch": 4, "kv_heads": 16,
         "groups": 1, "head_dim": 128, "fill": 32000, "lens": "equal", "page": 0, "io": "bf16"},
        # Batched serving of a grouped-query model from a paged cache, ragged fills.
        {"name": "decode_paged_gqa", "kind": "decode", "fmt": "fp4", "batch": 64, "kv_heads": 8,
         "groups": 4, "head_dim": 128, "fill": 8192, "lens": "lognormal", "page": 16,
         "io": "bf16"},
        # A small cache with fills of every length, fp32 queries and outputs.
        {"name": "decode_small", "kind": "decode", "fmt": "fp8", "batch": 8, "kv_heads": 8,
         "groups": 1, "head_dim": 64, "fill": 2040, "lens": "uniform", "page": 0, "io": "fp32"},
        # A decode step of one layer of a 12-head model, 16 sequences, fp32 activations.
        {"name": "step_small", "kind": "step", "fmt": "fp4", "batch": 16, "kv_heads": 12,
         "groups": 1, "head_dim": 64, "fill": 700, "lens": "uniform", "page": 0, "io": "fp32"},
        # The same of a grouped-query model, 64 paged sequences.
        {"name": "step_paged_gqa", "kind": "step", "fmt": "fp8", "batch": 64, "kv_heads": 8,
         "groups": 4, "head_dim": 128, "fill": 8192, "lens": "lognormal", "page": 16,
         "io": "bf16"},
        # A 512-token chunk of four long prompts onto a 32K prefix.
        {"name": "prefill_long", "kind": "prefill", "fmt": "fp4", "batch": 4, "kv_heads": 16,
         "groups": 1, "head_dim": 128, "fill": 32256, "lens": "equal", "page": 0, "chunk": 512,
         "ragged": False, "io": "bf16"},
        # Short ragged prompts of a grouped-query model, as a server admits them.
        {"name": "prefill_ragged", "kind": "prefill", "fmt": "fp8", "batch": 6, "kv_heads": 8,
         "groups": 4, "head_dim": 128, "fill": 1900, "lens": "uniform", "page": 0, "chunk": 333,
         "ragged": True, "io": "bf16"},
    ]


# ---------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode", "step", "step",
                       "prefill", "prefill"])
    while True:
        c = {"kind": kind, "fmt": rng.choice(["fp4", "fp8"]),
             "batch": _log(rng, 1, 64 if kind != "prefill" else 8),
             "kv_heads": rng.choice([1, 2, 3, 4, 8, 8, 12, 16]),
             "groups": rng.choice([1, 1, 2, 4, 8]),
             "head_dim": rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256]),
             "fill": _log(rng, 30, 32000), "lens": rng.choice(["equal", "uniform", "lognormal"]),
             "page": rng.choice([0, 0, 16, 64]), "io": rng.choice(["fp32", "bf16"])}
        if kind in ("decode", "step"):
            c["groups"] = rng.choice([c["groups"], 3, 5, 16])
        if kind == "append":
            c["chunk"] = rng.choice([1, _log(rng, 2, 2048)])
            c["ragged"] = c["chunk"] > 1 and rng.choice([True, False])
        if kind == "read":
            c["chunk"] = _log(rng, 1, 8192)
            c["start"] = rng.choice([0, int(rng.uniform(0, c["fill"]))])
        if kind == "prefill":
            c["chunk"] = _log(rng, 9, 1024)
            c["ragged"] = rng.choice([True, False])
            c["io"] = "bf16"  # its products take bf16 operands
        w = work(c)
        most = _MOST[kind]
        # the cache itself and its rows in 32 bits stay within the listed cases'
        cells = c["batch"] * c["kv_heads"] * (c["fill"] + c.get("chunk", 1)) * c["head_dim"]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and cells <= 5.4e8:
            return c


#: The most bytes and flops of a drawn case, by kind (the largest listed ones').
_MOST = {"append": (1.9e8, 1.0), "read": (3.5e8, 1.0), "decode": (2.9e8, 2.2e9),
         "step": (3e8, 2.3e9), "prefill": (3.3e8, 5.5e11)}


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------

def _lengths(kind, n, top, salt):
    """n fills in [0, top], the case's own: equal ones, or ragged ones of which
    the longest is top (and, of several uniform ones, one is empty)."""
    r = np.random.default_rng(1000003 * n + 7 * top + salt)
    if kind == "equal":
        return np.full(n, top, np.int64)
    if kind == "uniform":
        lens = r.integers(0, top + 1, n)
        lens[int(r.integers(n))] = 0
    else:  # lognormal around 1500 of 8192, in proportion
        lens = np.clip(np.exp(r.normal(math.log(max(top * 1500 / 8192, 1)), 0.8, n)),
                       min(16, top), top)
    lens = lens.astype(np.int64)
    lens[int(r.integers(n))] = top
    return lens


def _fills(c):
    return _lengths(c["lens"], c["batch"], c["fill"], 1)


def _counts(c):
    if c.get("ragged"):
        return _lengths("uniform", c["batch"], c["chunk"], 2)
    return np.full(c["batch"], c.get("chunk", 1), np.int64)


def work(c):
    d, hkv = c["head_dim"], c["kv_heads"]
    hq = hkv * c["groups"]
    row = 2 * hkv * (d * _BITS[c["fmt"]] // 8 + d // _GROUP)  # K and V of a token, stored
    io = _IO_BYTES[c["io"]]
    fills, n = _fills(c), int(_counts(c).sum())
    if c["kind"] == "append":  # rows in, codes out, codes in, rows out
        out = c["batch"] * c["chunk"]
        return {"bytes": int(2 * n * hkv * d * io + 2 * n * row + 2 * out * hkv * d * io),
                "flops": 0}
    if c["kind"] == "read":
        got = int(np.clip(fills - c["start"], 0, c["chunk"]).sum())
        return {"bytes": int(got * row + 2 * c["batch"] * c["chunk"] * hkv * d * io), "flops": 0}
    if c["kind"] == "decode":
        total = int(fills.sum())
        return {"bytes": int(total * row + 2 * c["batch"] * hq * d * io),
                "flops": int(4 * total * hq * d)}
    if c["kind"] == "step":
        b, total = c["batch"], int(fills.sum()) + c["batch"]
        return {"bytes": int(total * row + b * row + 2 * b * hq * d * io + 4 * b * hkv * d * io),
                "flops": int(4 * total * hq * d)}
    counts = _counts(c)
    rows = c["batch"] * c["chunk"]
    pairs = int((counts * fills + counts * (counts + 1) // 2).sum())
    return {"bytes": int((fills.sum() + 2 * n) * row + 2 * n * hkv * d * io + 2 * rows * hq * d * io
                         + 2 * rows * hkv * d * io),
            "flops": int(4 * pairs * hq * d)}


# ---------------------------------------------------------------------------
# The plain form of the cache
# ---------------------------------------------------------------------------

def _two_to(e):
    """2^e of int32 exponents in [-126, 127], exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x, fmt):
    """(codes, scale bytes) of rows x [..., head_dim]: codes one to a byte."""
    g = x.float().reshape(*x.shape[:-1], x.shape[-1] // _GROUP, _GROUP)
    amax = g.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, torch.ones_like(amax), amax)
    m, p = torch.frexp(amax)  # amax = m 2^p, m in [1/2, 1)
    if fmt == "fp4":
        e = (p - 3 + (m > 0.875).int()).clamp(-100, 125)
    else:
        e = (p - 9 + (m > 0.90625).int()).clamp(-100, 119)
    e = torch.where(amax == 0, torch.full_like(e, -100), e).int()
    y = g * _two_to(-e)[..., None]
    if fmt == "fp4":
        a = y.abs().clamp(max=6.0)
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        r = torch.round(a / step) * step
        code = torch.where(r < 2, 2 * r, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8)
        code = code | (torch.signbit(y).to(torch.uint8) << 3)
    else:
        a = y.abs().clamp(max=448.0)
        _, q = torch.frexp(a)  # steps of 2^(q - 4), at least 2^-9
        step = _two_to(q.int().clamp(min=-5) - 4)
        r = torch.copysign(torch.round(a / step) * step, y)
        code = r.to(torch.float8_e4m3fn).view(torch.uint8)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code.reshape(x.shape), byte


def _pack(code, fmt):
    return code if fmt == "fp8" else code[..., 0::2] | (code[..., 1::2] << 4)


def _unpack(packed, fmt):
    if fmt == "fp8":
        return packed
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def _tables(fmt):
    if fmt == "fp4":
        mag = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        values = torch.tensor(mag + [-v for v in mag], device=DEV)
    else:
        values = torch.arange(256, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn).float()
    scales = torch.full((256,), float("nan"), device=DEV)
    scales[1:255] = _two_to(torch.arange(-126, 128, device=DEV, dtype=torch.int32))
    return values, scales


def _values(code, byte, tables):
    """The fp32 values of codes [..., d] under scale bytes [..., d / 32]."""
    values, scales = tables
    v = values[code.int()].reshape(*byte.shape, _GROUP) * scales[byte.int()][..., None]
    return v.reshape(code.shape)


def _rows(s, which, top):
    """Positions [0, top) of every sequence in fp32: [batch, kv_heads, top, d]."""
    packed, byte = s[which], s[which + "s"]
    if s["table"] is not None:
        pages = s["table"][:, :-(-top // s["case"]["page"])].long()
        packed, byte = (t[pages].transpose(1, 2).flatten(2, 3) for t in (packed, byte))
    packed, byte = packed[:, :, :top], byte[:, :, :top]
    return _values(_unpack(packed, s["case"]["fmt"]), byte, s["tables"])


def _softmax_rows(sc, hide):
    """softmax of sc over its last axis where not hidden; rows that see nothing are 0."""
    sc = sc.masked_fill_(hide, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    top = torch.where(torch.isneginf(top), torch.zeros_like(top), top)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, torch.ones_like(total), total))


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _keys(g, *shape):
    """Rows as attention keys are: channels of unlike size and offset."""
    d = shape[-1]
    return _randn(g, *shape) * torch.exp(0.5 * _randn(g, d)) + 0.5 * _randn(g, d)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    fmt, kind, page = c["fmt"], c["kind"], c["page"]
    b, hkv, hq, d = c["batch"], c["kv_heads"], c["kv_heads"] * c["groups"], c["head_dim"]
    chunk = c.get("chunk", 1)
    cap = c["fill"] + (chunk if kind != "read" else 0)
    io = _IO[c["io"]]
    lens = _fills(c)
    s = {"case": c, "host": lens, "lens": torch.from_numpy(lens).to(DEV), "cap": cap,
         "tables": _tables(fmt), "table": None, "top": int(lens.max())}
    if page:
        per = -(-cap // page)
        perm = np.random.default_rng(int(seed) + 1).permutation(b * per)
        s["table"] = torch.from_numpy(perm.reshape(b, per).astype(np.int32)).to(DEV)
        shape = (b * per, hkv, page, d)
    else:
        shape = (b, hkv, cap, d)
    if kind == "append":  # what earlier tokens left is not read
        s["k"], s["v"] = (torch.zeros(*shape[:-1], d * _BITS[fmt] // 8, dtype=torch.uint8,
                                      device=DEV) for _ in range(2))
        s["ks"], s["vs"] = (torch.zeros(*shape[:-1], d // _GROUP, dtype=torch.uint8, device=DEV)
                            for _ in range(2))
    else:
        code, s["ks"] = _quantise(_keys(g, *shape), fmt)
        s["k"] = _pack(code, fmt)
        code, s["vs"] = _quantise(_randn(g, *shape), fmt)
        s["v"] = _pack(code, fmt)
    if kind in ("append", "step", "prefill"):
        s["nk"] = _keys(g, b, chunk, hkv, d).to(io)
        s["nv"] = _randn(g, b, chunk, hkv, d).to(io)
        counts = _counts(c)
        s["count"] = counts
        s["counts"] = torch.from_numpy(counts).to(DEV)
    if kind in ("decode", "step"):
        s["q"] = _randn(g, b, hq, d).to(io)
        s["out"] = torch.empty_like(s["q"])
    if kind == "prefill":
        s["q"] = _randn(g, b, chunk, hq, d).to(io)
        s["out"] = torch.empty_like(s["q"])
    if kind != "decode":
        s["ko"], s["vo"] = (torch.empty((b, chunk, hkv, d), dtype=io, device=DEV)
                            for _ in range(2))
    if own:
        _handle(s)
    return s


def _handle(s):
    """The framework's cache over these rows, as a serving program holds it."""
    from simple_llm_amd.gpu import gpu

    c = s["case"]
    dtype = {"fp4": torch.float4_e2m1fn_x2, "fp8": torch.float8_e4m3fn}[c["fmt"]]
    ctx = gpu.context_create()
    cache = gpu.kv_cache_create(ctx, gpu.KVCacheConfig(
        c["batch"], s["cap"], 1, c["kv_heads"] * c["groups"], c["head_dim"],
        n_kv_heads=c["kv_heads"], dtype=dtype, block_size=c["page"]))
    if c["page"]:
        gpu.kv_cache_set_block_table(cache, s["table"])
    layer = cache.layers[0]
    for buf, t in ((layer.k_cache, s["k"]), (layer.v_cache, s["v"]), (layer.k_scale, s["ks"]),
                   (layer.v_scale, s["vs"])):
        buf.buffer.copy_(t.reshape(buf.shape))
    s.update(gpu=gpu, ctx=ctx, cache=cache, lens32=s["lens"].int())
    _rewind(s)


def _rewind(s):
    """The fills as the pass finds them (a pass that appends advances them)."""
    layer = s["cache"].layers[0]
    layer.lens.copy_(s["lens32"])
    layer.host_lens = s["host"].copy()


# ---------------------------------------------------------------------------
# run: one pass
# ---------------------------------------------------------------------------

def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["kind"]](s)


def _own_append(s):
    gpu, ctx, cache, c = s["gpu"], s["ctx"], s["cache"], s["case"]
    _rewind(s)
    if c["chunk"] == 1:
        gpu.kv_cache_append(ctx, cache, 0, s["nk"], s["nv"])
    else:
        gpu.kv_cache_prefill(ctx, cache, 0, s["nk"], s["nv"],
                             n_new=s["count"] if c["ragged"] else None)
    gpu.kv_cache_read(ctx, cache, 0, s["ko"], s["vo"], start=s["host"])
    return s["ko"], s["vo"]


def _own_read(s):
    s["gpu"].kv_cache_read(s["ctx"], s["cache"], 0, s["ko"], s["vo"], start=s["case"]["start"])
    return s["ko"], s["vo"]


def _own_decode(s):
    s["gpu"].decode_attention(s["ctx"], s["cache"], 0, s["q"], s["out"])
    return s["out"]


def _own_step(s):
    _rewind(s)
    s["gpu"].kv_cache_append_attend(s["ctx"], s["cache"], 0, s["nk"], s["nv"], s["q"], s["out"])
    s["gpu"].kv_cache_read(s["ctx"], s["cache"], 0, s["ko"], s["vo"], start=s["host"])
    return s["out"], s["ko"], s["vo"]


def _own_prefill(s):
    _rewind(s)
    s["gpu"].kv_cache_prefill(s["ctx"], s["cache"], 0, s["nk"], s["nv"], s["q"], s["out"],
                              n_new=s["count"] if s["case"]["ragged"] else None)
    s["gpu"].kv_cache_read(s["ctx"], s["cache"], 0, s["ko"], s["vo"], start=s["host"])
    return s["out"], s["ko"], s["vo"]


def _stored(s, which):
    """The new rows [batch, chunk, kv_heads, d] as the cache holds them, in fp32, and
    where a row is one (its index is below the sequence's count)."""
    code, byte = _quantise(s[which], s["case"]["fmt"])
    x = _values(code, byte, s["tables"])
    here = torch.arange(x.shape[1], device=DEV)[None, :] < s["counts"][:, None]
    return x, here


def _plain_append(s):
    io = _IO[s["case"]["io"]]
    k, here = _stored(s, "nk")
    v, _ = _stored(s, "nv")
    gone = ~here[:, :, None, None]
    return k.masked_fill_(gone, 0).to(io), v.masked_fill_(gone, 0).to(io)


def _plain_read(s):
    c = s["case"]
    io, at = _IO[c["io"]], torch.arange(c["chunk"], device=DEV) + c["start"]
    top = min(c["start"] + c["chunk"], s["cap"])
    gone = (at[None, :] >= s["lens"][:, None])[:, :, None, None]

    def rows(which):
        x = _window(s, which, c["start"], top)
        if x.shape[1] < c["chunk"]:
            x = torch.cat([x, x.new_zeros(x.shape[0], c["chunk"] - x.shape[1], *x.shape[2:])], 1)
        return x.masked_fill(gone, 0).to(io)

    return rows("k"), rows("v")


def _window(s, which, lo, hi):
    """Positions [lo, hi) as rows [batch, hi - lo, kv_heads, d] in fp32."""
    packed, byte = s[which], s[which + "s"]
    at = torch.arange(lo, hi, device=DEV)
    if s["table"] is not None:
        page = s["case"]["page"]
        pages = s["table"].long()[:, at // page]  # [batch, positions]
        packed, byte = packed[pages, :, at % page], byte[pages, :, at % page]
    else:
        packed, byte = packed[:, :, lo:hi].transpose(1, 2), byte[:, :, lo:hi].transpose(1, 2)
    return _values(_unpack(packed, s["case"]["fmt"]), byte.contiguous(), s["tables"])


def _attend_one(s, k, v, lens):
    """softmax(q k^T / sqrt(d)) v of one query a sequence and head, rounded to the output."""
    c = s["case"]
    b, hkv, d = c["batch"], c["kv_heads"], c["head_dim"]
    q = s["q"].float().reshape(b, hkv, c["groups"], d)
    sc = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    hide = torch.arange(k.shape[2], device=DEV)[None, :] >= lens[:, None]
    p = _softmax_rows(sc, hide[:, None, None, :])
    v = v.masked_fill(hide[:, None, :, None], 0)
    return torch.matmul(p, v).reshape(s["q"].shape).to(_IO[c["io"]])


def _plain_decode(s):
    return _attend_one(s, _rows(s, "k", s["top"]), _rows(s, "v", s["top"]), s["lens"])


def _with_new(s, which, new, here, top):
    """Positions [0, top) with the new rows at each sequence's fill."""
    x = _rows(s, which, top)
    seq, i = torch.nonzero(here, as_tuple=True)
    x[seq, :, s["lens"][seq] + i] = new[seq, i]
    return x


def _plain_step(s):
    io = _IO[s["case"]["io"]]
    nk, here = _stored(s, "nk")
    nv, _ = _stored(s, "nv")
    top = s["top"] + 1
    out = _attend_one(s, _with_new(s, "k", nk, here, top), _with_new(s, "v", nv, here, top),
                      s["lens"] + 1)
    return out, nk.to(io), nv.to(io)


def _plain_prefill(s):
    c = s["case"]
    b, hkv, grp, d, n = c["batch"], c["kv_heads"], c["groups"], c["head_dim"], c["chunk"]
    io = _IO[c["io"]]
    nk, here = _stored(s, "nk")
    nv, _ = _stored(s, "nv")
    top = int((s["host"] + s["count"]).max())
    k, v = _with_new(s, "k", nk, here, top), _with_new(s, "v", nv, here, top)
    q = s["q"].float().reshape(b, n, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(
        b, hkv, grp * n, d)
    sc = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    t = torch.arange(top, device=DEV)
    last = s["lens"][:, None] + torch.arange(n, device=DEV)  # what row i sees, its own included
    hide = t[None, None, :] > torch.where(here, last, torch.full_like(last, -1))[:, :, None]
    sc = sc.reshape(b, hkv, grp, n, top)
    p = _softmax_rows(sc, hide[:, None, None]).reshape(b, hkv, grp * n, top)
    o = torch.matmul(p, v).reshape(b, hkv, grp, n, d).permute(0, 3, 1, 2, 4)
    gone = ~here[:, :, None, None]
    return (o.reshape(s["q"].shape).to(io), nk.masked_fill_(gone, 0).to(io),
            nv.masked_fill_(gone, 0).to(io))


_OWN = {"append": _own_append, "read": _own_read, "decode": _own_decode, "step": _own_step,
        "prefill": _own_prefill}
_PLAIN = {"append": _plain_append, "read": _plain_read, "decode": _plain_decode,
          "step": _plain_step, "prefill": _plain_prefill}


# ---------------------------------------------------------------------------
# exact: from the definition, in 64 bits
# ---------------------------------------------------------------------------

def _grid(fmt):
    """The non-negative elements in code order, in 64 bits."""
    bits, bias = (1, 1) if fmt == "fp4" else (3, 7)
    out = []
    for code in range(8 if fmt == "fp4" else 127):
        e, m = code >> bits, code & ((1 << bits) - 1)
        out.append(math.ldexp(m, 1 - bias - bits) if e == 0
                   else math.ldexp((1 << bits) + m, e - bias - bits))
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _exact_round_trip(x, fmt):
    """x [..., d] after one trip through the cache, in 64 bits."""
    grid = _grid(fmt)
    top = float(grid[-1] + (grid[-1] - grid[-2]) / 2)
    x = x.double()
    g = x.unflatten(-1, (-1, _GROUP))
    amax = g.abs().amax(-1, keepdim=True)
    usable = torch.isfinite(amax) & (amax > 0)
    e = torch.ceil(torch.log2(torch.where(usable, amax, torch.ones_like(amax)) / top))
    # the logarithm may be a rounding off next to a power of two: settle it by comparison
    e = torch.where(amax > top * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= top * torch.exp2(e - 1), e - 1, e)
    e = torch.where(amax == 0, torch.full_like(e, -100), e)
    scale = torch.exp2(e.clamp(-100, 125 if fmt == "fp4" else 119))
    y = g / scale
    mid = (grid[1:] + grid[:-1]) / 2
    a = y.abs().clamp(max=float(grid[-1])).contiguous()
    below = torch.bucketize(a, mid)  # nearest code; a tie counts as the lower one
    above = torch.bucketize(a, mid, right=True)  # and here as the upper one
    code = torch.where(below % 2 == 0, below, above)
    r = torch.copysign(grid[code], y) * scale
    r = torch.where(torch.isfinite(amax), r, torch.full_like(r, float("nan")))
    return r.reshape(x.shape)


def _exact_cache(s, which, b, lo, hi):
    """Positions [lo, hi) of sequence b in 64 bits: [kv_heads, hi - lo, d]."""
    c = s["case"]
    packed, byte = s[which], s[which + "s"]
    if s["table"] is not None:
        at = torch.arange(lo, hi, device=DEV)
        row = s["table"][b].long()[at // c["page"]]
        packed = packed[row, :, at % c["page"]].transpose(0, 1)
        byte = byte[row, :, at % c["page"]].transpose(0, 1)
    else:
        packed, byte = packed[b, :, lo:hi], byte[b, :, lo:hi]
    grid = _grid(c["fmt"])
    if c["fmt"] == "fp4":
        code = torch.empty(*packed.shape[:-1], c["head_dim"], dtype=torch.long, device=DEV)
        code[..., 0::2] = packed & 15
        code[..., 1::2] = packed >> 4
        half = 8
    else:
        code, half = packed.long(), 128
    v = grid[(code % half).clamp(max=len(grid) - 1)]
    v = torch.where(code >= half, -v, v)
    return v * torch.exp2(byte.double() - 127).repeat_interleave(_GROUP, -1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    b, hkv, grp, d = c["batch"], c["kv_heads"], c["groups"], c["head_dim"]
    fills = [int(n) for n in s["host"]]
    if c["kind"] == "read":
        ko = torch.zeros(b, c["chunk"], hkv, d, dtype=torch.float64, device=DEV)
        vo = torch.zeros_like(ko)
        for i, n in enumerate(fills):
            hi = min(n, c["start"] + c["chunk"])
            if hi > c["start"]:
                ko[i, :hi - c["start"]] = _exact_cache(s, "k", i, c["start"], hi).transpose(0, 1)
                vo[i, :hi - c["start"]] = _exact_cache(s, "v", i, c["start"], hi).transpose(0, 1)
        return ko, vo
    if c["kind"] != "decode":
        nk, nv = _exact_round_trip(s["nk"], c["fmt"]), _exact_round_trip(s["nv"], c["fmt"])
        for i, n in enumerate(s["count"]):
            nk[i, int(n):] = 0
            nv[i, int(n):] = 0
        if c["kind"] == "append":
            return nk, nv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, n in enumerate(fills):
        k, v = _exact_cache(s, "k", i, 0, n), _exact_cache(s, "v", i, 0, n)
        rows = 1
        if c["kind"] != "decode":
            rows = int(s["count"][i])
            k = torch.cat([k, nk[i, :rows].transpose(0, 1)], 1)
            v = torch.cat([v, nv[i, :rows].transpose(0, 1)], 1)
        if k.shape[1] == 0 or rows == 0:
            continue
        q = s["q"][i].double().reshape(-1, hkv, grp, d)[:rows]  # [rows, kv_heads, groups, d]
        sees = k.shape[1] - rows + torch.arange(rows, device=DEV)  # the last position of a row
        late = torch.arange(k.shape[1], device=DEV)[None, :] > sees[:, None]
        for h in range(hkv):
            sc = torch.einsum("rgd,td->grt", q[:, h], k[h]) / math.sqrt(d)
            sc = sc.masked_fill(late, float("-inf"))
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            o = torch.einsum("grt,td->rgd", w / w.sum(-1, keepdim=True), v[h])
            if c["kind"] == "prefill":
                out[i, :rows, h * grp:(h + 1) * grp] = o
            else:
                out[i, h * grp:(h + 1) * grp] = o[0]
    return out if c["kind"] == "decode" else (out, nk, nv)
