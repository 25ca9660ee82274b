"""Block-scaled caches on the GPU: the stored values against the oracle's bit
for bit, attention against float64 over the stored values.

Error bounds, by arithmetic (u = 2^-24, half an fp32 step). A score is a sum of
D products, each rounding at most u of the running magnitude A = scale * sum
|q k|, then scaled and shifted (three roundings): off by at most (D + 8) u A.
Its exponential is off by that much (natural units) plus one step of the
exponential unit, weights and their sum by twice it, and the sums over n tokens
by u for each sequential addition (at most n / 16 + 64 with four lanes, four
wavefronts and chunks in parallel). All of it multiplies sum p |v|. With bf16
in and out the probabilities carry 17 bits (2^-17) in decode and 8 (2^-8) in
prefill, fp32 queries of a prefill are rounded to bf16 (2^-8 A on a score), and
a bf16 output rounds by 2^-8 of itself.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import banner
from oracle import quant_oracle as qo

pytestmark = pytest.mark.gpu

DT = {"fp4": torch.float4_e2m1fn_x2, "fp8": torch.float8_e4m3fn}
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _rows(rng, *shape):
    """Key-like rows: channels of unlike size, some groups all zero."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-1])) * 0.7
    x[..., :qo.GROUP] *= rng.random(shape[:-1] + (1,)) > 0.1
    return x.astype(np.float32)


def _dev(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda:0").to(dtype)


class Model:
    """What the cache should hold: float64 values [B, T, Hkv, D] and fills."""

    def __init__(self, B, T, H, D, fmt):
        self.k = np.zeros((B, T, H, D))
        self.v = np.zeros((B, T, H, D))
        self.lens = np.zeros(B, np.int64)
        self.fmt, self.cap = fmt, T

    def append(self, k, v, n=None):
        """k, v [B, C, H, D]; n: rows of each sequence."""
        n = np.full(len(self.lens), k.shape[1]) if n is None else n
        k, v = qo.round_trip(k, self.fmt), qo.round_trip(v, self.fmt)
        for b, m in enumerate(n):
            at = self.lens[b]
            m = int(min(m, self.cap - at))
            self.k[b, at:at + m] = k[b, :m]
            self.v[b, at:at + m] = v[b, :m]
            self.lens[b] = at + m


def _make(ctx, B, T, Hkv, G, D, fmt, page=0, seed=0):
    from simple_llm_amd.gpu import gpu

    cache = gpu.kv_cache_create(ctx, gpu.KVCacheConfig(B, T, 1, Hkv * G, D, n_kv_heads=Hkv,
                                                       dtype=DT[fmt], block_size=page))
    cap = T
    if page:
        per = -(-T // page)
        perm = np.random.default_rng(seed + 77).permutation(B * per).astype(np.int32)
        gpu.kv_cache_set_block_table(cache, torch.from_numpy(perm.reshape(B, per)))
        cap = per * page
    return gpu, cache, Model(B, cap, Hkv, D, fmt)


def _fill(gpu, ctx, cache, m, rng, counts, dtype=F32):
    """counts[b] tokens of each sequence, as one ragged chunk."""
    counts = np.asarray(counts)
    C = int(counts.max())
    if C == 0:
        return
    B, _, H, D = m.k.shape
    k, v = (_dev(_rows(rng, B, C, H, D), dtype) for _ in range(2))
    gpu.kv_cache_prefill(ctx, cache, 0, k, v, n_new=counts)
    m.append(_np(k), _np(v), counts)


def _check_stored(gpu, ctx, cache, m, start=0, C=None, dtype=F32):
    B, T, H, D = m.k.shape
    C = T - start if C is None else C
    ko = torch.full((B, C, H, D), 7.0, dtype=dtype, device="cuda:0")
    vo = torch.full_like(ko, 7.0)
    gpu.kv_cache_read(ctx, cache, 0, ko, vo, start=start)
    for got, want in ((ko, m.k), (vo, m.v)):
        w = np.zeros((B, C, H, D))
        for b, n in enumerate(m.lens):
            hi = min(int(n), start + C)
            if hi > start:
                w[b, :hi - start] = want[b, start:hi]
        np.testing.assert_array_equal(_np(got), w)
    assert cache.layers[0].lens.cpu().tolist() == m.lens.tolist()
    assert cache.seq_lens().tolist() == m.lens.tolist()


def _check_attention(got, q, m, G, scale, exact32, out_bf16, rows=None, prefill=False, q_f32=False):
    """got, q [B, rows, Hq, D]; the last row of sequence b sees its whole fill."""
    got, q = _np(got), _np(q)
    B, R, Hq, D = q.shape
    n_rows = np.full(B, R) if rows is None else rows
    for b in range(B):
        n, r = int(m.lens[b]), int(n_rows[b])
        assert not got[b, r:].any(), f"rows past the count of sequence {b} are not zeros"
        last = n - r + np.arange(r)
        for h in range(Hq):
            want, mag, big = qo.attention(q[b, :r, h], m.k[b, :n, h // G], m.v[b, :n, h // G],
                                          scale, last)
            tol = 2 * (D + 8) * U * big + (n / 16 + 64) * U
            if prefill:
                tol = tol + 2.0 ** -8 + (2 * 2.0 ** -8 * big if q_f32 else 0.0)
            elif not exact32:
                tol = tol + 2.0 ** -17
            bound = tol[:, None] * mag + (2.0 ** -8 * (np.abs(want) + tol[:, None] * mag)
                                          if out_bf16 else 0.0) + 1e-37
            err = np.abs(got[b, :r, h] - want)
            assert not np.isnan(got[b, :r, h]).any()
            assert (err <= bound).all(), (
                f"sequence {b} head {h}: off by {(err / bound).max():.2f} of the bound")


# ---- writing and reading ---------------------------------------------------

@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("B,H,D,C,page,dtype", [
    (1, 1, 32, 1, 0, F32), (3, 5, 64, 7, 0, BF16), (2, 3, 96, 45, 4, F32), (4, 2, 128, 33, 16, BF16),
    (2, 1, 160, 17, 1, F32), (1, 7, 224, 5, 0, BF16), (2, 2, 256, 40, 32, F32)])
def test_chunk_append_and_read(gpu_ctx, fmt, B, H, D, C, page, dtype):
    banner(f"quant chunk append {fmt} B={B} H={H} D={D} C={C} page={page} {dtype}")
    rng = np.random.default_rng(D * 7 + C)
    gpu, cache, m = _make(gpu_ctx, B, 2 * C + 3, H, 1, D, fmt, page)
    counts = rng.integers(0, C + 1, B)
    counts[0] = C
    _fill(gpu, gpu_ctx, cache, m, rng, counts, dtype)
    _fill(gpu, gpu_ctx, cache, m, rng, rng.integers(0, C + 1, B), dtype)
    _check_stored(gpu, gpu_ctx, cache, m)
    _check_stored(gpu, gpu_ctx, cache, m, start=C // 2, C=C, dtype=BF16)
    at = rng.integers(0, C, B)  # a start of its own for each sequence
    ko = torch.empty((B, 3, H, D), device="cuda:0")
    vo = torch.empty_like(ko)
    gpu.kv_cache_read(gpu_ctx, cache, 0, ko, vo, start=at)
    for b in range(B):
        n = max(0, min(3, int(m.lens[b] - at[b])))
        np.testing.assert_array_equal(_np(ko)[b, :n], m.k[b, at[b]:at[b] + n])
        assert not _np(ko)[b, n:].any() and not _np(vo)[b, n:].any()


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("B,H,D,page", [(1, 1, 32, 0), (5, 3, 64, 8), (3, 16, 128, 0), (2, 9, 256, 2)])
def test_token_append_until_full(gpu_ctx, fmt, B, H, D, page):
    banner(f"quant token append {fmt} B={B} H={H} D={D} page={page}")
    rng = np.random.default_rng(D + B)
    gpu, cache, m = _make(gpu_ctx, B, 6, H, 1, D, fmt, page)
    _fill(gpu, gpu_ctx, cache, m, rng, rng.integers(0, 5, B))
    for i in range(9):  # past the capacity: full sequences stay as they are
        k, v = (_dev(_rows(rng, B, H, D), BF16 if i % 2 else F32) for _ in range(2))
        gpu.kv_cache_append(gpu_ctx, cache, 0, k, v)
        m.append(_np(k)[:, None], _np(v)[:, None])
    _check_stored(gpu, gpu_ctx, cache, m)
    assert (m.lens == m.cap).all()


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_stored_bytes_at_the_edges(gpu_ctx, fmt):
    """Group maxima at, just below and just above every border of the scale rule,
    ties, both clamps, subnormals, zeros of both signs: codes and scale bytes."""
    banner(f"quant edges {fmt}")
    top = 7.0 if fmt == "fp4" else 464.0
    rng = np.random.default_rng(5)
    peaks = []
    for e in (-149, -140, -127, -126, -110, -103, -102, -101, -100, -50, -1, 0, 1, 60, 118, 119,
              120, 124, 125, 126):
        for base in (1.0, 1.5, 1.75, 1.8125, 1.99999988):
            with np.errstate(over="ignore"):
                p = np.float32(np.ldexp(base, e))
            if np.isfinite(p):
                peaks += [p, np.nextafter(p, np.float32(0)), np.nextafter(p, np.float32(np.inf))]
    peaks += [np.float32(0), np.finfo(np.float32).max, np.float32(top), np.float32(top / 2)]
    peaks = np.array([p for p in peaks if np.isfinite(p)], np.float32)
    n = -(-len(peaks) // 8) * 8
    x = rng.uniform(-1, 1, (n, 32)).astype(np.float32)
    x[:len(peaks)] *= peaks[:, None]
    x[np.arange(len(peaks)), rng.integers(0, 32, len(peaks))] = peaks
    # exact midpoints of the grid under scale 1, both signs
    g = qo.grid(fmt)
    mids = np.concatenate([(g[1:] + g[:-1]) / 2, g])
    ties = np.zeros((-(-len(mids) // 31), 32), np.float32)
    for i, t in enumerate(mids):
        ties[i // 31, i % 31] = t if i % 2 else -t
    ties[:, 31] = g[-1]
    x = np.concatenate([x, ties, -np.zeros((1, 32), np.float32)])
    x = np.concatenate([x, np.zeros((-len(x) % 4, 32), np.float32)]).reshape(1, -1, 1, 128)
    gpu, cache, m = _make(gpu_ctx, 1, x.shape[1], 1, 1, 128, fmt)
    k = _dev(x, F32)
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, -k)
    code, byte = qo.quantise(x[0, :, 0], fmt)
    lay = cache.layers[0]
    np.testing.assert_array_equal(lay.k_scale.buffer.cpu().numpy(), byte)
    np.testing.assert_array_equal(lay.v_scale.buffer.cpu().numpy(), byte)
    np.testing.assert_array_equal(lay.k_cache.buffer.cpu().numpy(), qo.pack(code, fmt))
    np.testing.assert_array_equal(lay.v_cache.buffer.cpu().numpy(),
                                  qo.pack(code ^ (8 if fmt == "fp4" else 128), fmt))


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_groups_that_are_not_finite(gpu_ctx, fmt):
    banner(f"quant not finite {fmt}")
    rng = np.random.default_rng(8)
    x = _rows(rng, 1, 5, 2, 64)
    x[0, 1, 0, 3] = np.nan
    x[0, 2, 1, 40] = np.inf
    x[0, 3, 0, 63] = -np.inf
    x[0, 4, 1, 0], x[0, 4, 1, 1] = np.inf, np.nan
    gpu, cache, m = _make(gpu_ctx, 1, 5, 2, 1, 64, fmt)
    for dtype in (F32, BF16):
        gpu.kv_cache_reset(cache)
        m.lens[:] = 0
        k = _dev(x, dtype)
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, k)
        m.append(_np(k), _np(k))
        _check_stored(gpu, gpu_ctx, cache, m)
        _check_stored(gpu, gpu_ctx, cache, m, dtype=BF16)


# ---- decode ----------------------------------------------------------------

DECODE = [
    # B, Hkv, G, D, lens, page, io
    (1, 1, 1, 32, [1], 0, F32), (3, 2, 1, 64, [0, 31, 33], 0, F32),
    (2, 3, 2, 64, [127, 129], 0, BF16), (4, 1, 3, 96, [5, 0, 200, 64], 8, F32),
    (2, 2, 4, 128, [300, 17], 16, BF16), (3, 4, 1, 128, [511, 512, 513], 0, F32),
    (2, 1, 5, 160, [90, 257], 1, F32), (1, 2, 8, 128, [1000], 64, F32),
    (2, 1, 16, 256, [140, 31], 0, F32), (1, 1, 16, 64, [77], 2, BF16),
    (2, 2, 1, 224, [65, 128], 0, BF16), (1, 3, 7, 192, [150], 32, F32),
    (5, 12, 1, 64, [700, 1, 0, 350, 699], 0, F32), (2, 8, 4, 128, [2100, 900], 16, F32),
    (1, 2, 1, 256, [400], 4, BF16),
]


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("B,Hkv,G,D,lens,page,io", DECODE)
def test_decode_attention(gpu_ctx, fmt, B, Hkv, G, D, lens, page, io):
    banner(f"quant decode {fmt} B={B} Hkv={Hkv} G={G} D={D} lens={lens} page={page} {io}")
    rng = np.random.default_rng(B * 100 + D + G)
    gpu, cache, m = _make(gpu_ctx, B, max(lens) + 2, Hkv, G, D, fmt, page)
    _fill(gpu, gpu_ctx, cache, m, rng, lens)
    q = _dev(rng.standard_normal((B, Hkv * G, D)).astype(np.float32), io)
    outs = []
    for hint in (0, 128, 4096):  # several chunks a row, and one
        gpu_ctx.config.decode_chunk_tokens = hint
        out = torch.full_like(q, 9.0)
        gpu.decode_attention(gpu_ctx, cache, 0, q, out)
        _check_attention(out[:, None], q[:, None], m, G, D ** -0.5, io == F32, io == BF16)
        outs.append(out)
    gpu_ctx.config.decode_chunk_tokens = 0
    again = torch.empty_like(q)
    gpu.decode_attention(gpu_ctx, cache, 0, q, again)
    assert torch.equal(again, outs[0])
    # types of their own for q and out, another scale
    mixed = torch.empty(q.shape, dtype=BF16 if io == F32 else F32, device="cuda:0")
    gpu.decode_attention(gpu_ctx, cache, 0, q, mixed, scale=0.05)
    _check_attention(mixed[:, None], q[:, None], m, G, 0.05, True, io == F32)


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("B,Hkv,G,D,lens,page,io", [
    (1, 1, 1, 32, [0], 0, F32), (3, 2, 2, 64, [0, 127, 128], 0, F32),
    (2, 4, 4, 128, [255, 40], 16, BF16), (2, 1, 8, 256, [3, 130], 4, F32),
    (4, 12, 1, 64, [700, 0, 31, 352], 0, F32), (2, 3, 3, 96, [64, 9], 1, BF16)])
def test_append_attend(gpu_ctx, fmt, B, Hkv, G, D, lens, page, io):
    """The one call against append and attention apart, several steps, up to full
    sequences: the same bytes, fills and bits."""
    banner(f"quant append_attend {fmt} B={B} Hkv={Hkv} G={G} D={D} lens={lens} page={page} {io}")
    rng = np.random.default_rng(D + G)
    T = max(lens) + 3
    gpu, cache, m = _make(gpu_ctx, B, T, Hkv, G, D, fmt, page)
    _, twin, m2 = _make(gpu_ctx, B, T, Hkv, G, D, fmt, page)
    if max(lens):
        k, v = (_dev(_rows(rng, B, max(lens), Hkv, D), F32) for _ in range(2))
        for c in (cache, twin):
            gpu.kv_cache_prefill(gpu_ctx, c, 0, k, v, n_new=lens)
        m.append(_np(k), _np(v), lens)
    for _ in range(5):
        k, v = (_dev(_rows(rng, B, Hkv, D), io) for _ in range(2))
        q = _dev(rng.standard_normal((B, Hkv * G, D)).astype(np.float32), io)
        out, want = torch.empty_like(q), torch.empty_like(q)
        fills = gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q, out)
        gpu.kv_cache_append(gpu_ctx, twin, 0, k, v)
        gpu.decode_attention(gpu_ctx, twin, 0, q, want)
        m.append(_np(k)[:, None], _np(v)[:, None])
        assert fills.tolist() == m.lens.tolist()
        assert torch.equal(out, want)
        _check_attention(out[:, None], q[:, None], m, G, D ** -0.5, io == F32, io == BF16)
    _check_stored(gpu, gpu_ctx, cache, m)


def test_update_and_attention_of_the_reference(gpu_ctx):
    """The reference's pair, kv_cache_update and attention_with_kv_cache, 2-D buffers."""
    banner("quant reference pair")
    rng = np.random.default_rng(3)
    B, H, D = 2, 4, 64
    gpu, cache, m = _make(gpu_ctx, B, 40, H, 1, D, "fp8")
    for _ in range(40):
        k, v = _rows(rng, B, H, D), _rows(rng, B, H, D)
        bk, bv = (gpu.gpu_buffer_2d_create(gpu_ctx, B, H * D, x.reshape(B, -1)) for x in (k, v))
        gpu.kv_cache_update(gpu_ctx, cache, 0, bk, bv)
        m.append(k[:, None], v[:, None])
    q = rng.standard_normal((B, H * D)).astype(np.float32)
    bq, out = gpu.gpu_buffer_2d_create(gpu_ctx, B, H * D, q), gpu.gpu_buffer_2d_create(gpu_ctx, B, H * D)
    gpu.attention_with_kv_cache(gpu_ctx, cache, 0, bq, out)
    _check_attention(out.buffer.reshape(B, 1, H, D), bq.buffer.reshape(B, 1, H, D), m, 1, D ** -0.5,
                     True, False)
    with pytest.raises(ValueError, match="Cache is full"):
        gpu.kv_cache_update(gpu_ctx, cache, 0, bk, bv)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_of_any_sign(gpu_ctx, scale):
    banner(f"quant decode scale {scale}")
    rng = np.random.default_rng(17)
    B, H, G, D = 2, 2, 2, 64
    gpu, cache, m = _make(gpu_ctx, B, 260, H, G, D, "fp8")
    _fill(gpu, gpu_ctx, cache, m, rng, [257, 40])
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    out = torch.empty_like(q)
    gpu.decode_attention(gpu_ctx, cache, 0, q, out, scale=scale)
    got = _np(out)
    for b in range(B):
        n = int(m.lens[b])
        for h in range(H * G):
            want, mag, big = qo.attention(_np(q)[b, h][None], m.k[b, :n, h // G],
                                          m.v[b, :n, h // G], scale, np.array([n - 1]))
            big = abs(big[0])  # (the oracle's bound carries the scale's sign)
            tol = 2 * (D + 8) * U * max(big, 0.0) + (n / 16 + 64) * U
            assert (np.abs(got[b, h] - want[0]) <= tol * mag[0] + 1e-37).all()


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("G", [1, 6, 12])
def test_tiny_queries_of_large_keys(gpu_ctx, G, io):
    """Scores of ordinary size from queries whose last bits bf16 cannot hold unscaled."""
    banner(f"quant tiny queries G={G} {io}")
    rng = np.random.default_rng(19)
    B, H, D, n = 2, 2, 96, 140
    gpu, cache, m = _make(gpu_ctx, B, n, H, G, D, "fp8")
    k = _rows(rng, B, n, H, D).astype(np.float64) * 2.0 ** 118
    k, v = _dev(k.astype(np.float32), F32), _dev(_rows(rng, B, n, H, D), F32)
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v)
    m.append(_np(k), _np(v))
    x = rng.standard_normal((B, H * G, D)) * 2.0 ** -122
    q = _dev(x.astype(np.float32), io)
    out = torch.empty_like(q)
    scale = 16 * D ** -0.5
    gpu.decode_attention(gpu_ctx, cache, 0, q, out, scale=scale)
    _check_attention(out[:, None], q[:, None], m, G, scale, io == F32, io == BF16)


def test_empty_cache_gives_zeros(gpu_ctx):
    banner("quant decode of nothing")
    for page in (0, 16):
        gpu, cache, m = _make(gpu_ctx, 3, 300, 2, 4, 128, "fp4", page)
        for kw in ({}, {"max_len": 300}):
            out = torch.full((3, 8, 128), 5.0, device="cuda:0")
            gpu.decode_attention(gpu_ctx, cache, 0, torch.ones_like(out), out, **kw)
            assert not out.any()
        out = torch.full((3, 4, 8, 128), 5.0, device="cuda:0")
        new = torch.ones((3, 4, 2, 128), device="cuda:0")
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, new, new, torch.ones_like(out), out, n_new=[0, 0, 0])
        assert not out.any() and cache.current_len == 0


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("page", [0, 8])
def test_other_rows_stay_as_they_were(gpu_ctx, fmt, page):
    """Appends write the bytes of their rows and no others; reading and attention none."""
    banner(f"quant other rows {fmt} page={page}")
    rng = np.random.default_rng(23)
    B, T, H, G, D, C = 3, 40, 3, 2, 96, 9
    gpu, cache, m = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    lay = cache.layers[0]
    bufs = (lay.k_cache, lay.v_cache, lay.k_scale, lay.v_scale)
    for t in bufs:
        t.buffer.fill_(0xA5)
    written = np.zeros((B, m.cap), bool)
    lens = np.array([0, 7, T - 3])
    lay.lens.copy_(torch.from_numpy(lens.astype(np.int32)))
    lay.host_lens = lens.astype(np.int64)

    def rows(n):
        return [_dev(_rows(rng, B, n, H, D), F32) for _ in range(2)]

    k, v = rows(C)
    counts = [C, 4, 2]
    q, out = (torch.zeros((B, C, H * G, D), dtype=BF16, device="cuda:0") for _ in range(2))
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts)
    for b, n in enumerate(counts):
        written[b, lens[b]:lens[b] + n] = True
    lens = lens + counts
    k, v = rows(1)
    gpu.kv_cache_append(gpu_ctx, cache, 0, k, v)
    q1, out1 = (torch.zeros((B, H * G, D), device="cuda:0") for _ in range(2))
    k, v = rows(1)
    gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q1, out1)
    for _ in range(2):
        for b in range(B):
            if lens[b] < m.cap:
                written[b, lens[b]] = True
                lens[b] += 1
    gpu.decode_attention(gpu_ctx, cache, 0, q1, out1)
    gpu.kv_cache_read(gpu_ctx, cache, 0, *(torch.empty((B, T, H, D), device="cuda:0") for _ in "kv"))
    assert cache.layers[0].lens.cpu().tolist() == lens.tolist()
    for t in bufs:
        x = t.buffer.cpu().numpy().reshape(-1, H, page or m.cap, t.shape[1])
        if page:
            x = x[cache.block_table.cpu().numpy()].transpose(0, 2, 1, 3, 4)
            x = x.reshape(B, H, m.cap, -1)
        untouched = (x == 0xA5).all(-1)  # [B, H, T]
        assert untouched[~np.repeat(written[:, None], H, 1)].all()
        assert not untouched[np.repeat(written[:, None], H, 1)].any()


def test_refused_calls_change_nothing(gpu_ctx):
    banner("quant refused calls")
    gpu, cache, m = _make(gpu_ctx, 2, 20, 1, 3, 64, "fp4")
    _fill(gpu, gpu_ctx, cache, m, np.random.default_rng(1), [5, 9])
    kv, q = torch.ones((2, 3, 1, 64), device="cuda:0"), torch.ones((2, 3, 3, 64), device="cuda:0")
    row, q1 = torch.ones((2, 1, 64), device="cuda:0"), torch.ones((2, 3, 64), device="cuda:0")
    half = row.half()
    for call, match in (
            (lambda: gpu.kv_cache_prefill(gpu_ctx, cache, 0, kv, kv, q, q.clone()), "query heads"),
            (lambda: gpu.kv_cache_prefill(gpu_ctx, cache, 0, kv, kv, n_new=[1, 4]), "n_new"),
            (lambda: gpu.kv_cache_prefill(gpu_ctx, cache, 0, kv.repeat(1, 5, 1, 1),
                                          kv.repeat(1, 5, 1, 1)), "Cache is full"),
            (lambda: gpu.kv_cache_append(gpu_ctx, cache, 0, half, half), "dtype"),
            (lambda: gpu.kv_cache_append_attend(gpu_ctx, cache, 0, half, half, q1, q1.clone()), "dtype"),
            (lambda: gpu.kv_cache_append_attend(gpu_ctx, cache, 0, row, row, q1, q1.clone(),
                                                max_len=9), "max_len"),
            (lambda: gpu.decode_attention(gpu_ctx, cache, 0, q1, q1.clone(), max_len=8), "max_len"),
            (lambda: gpu.decode_attention(gpu_ctx, cache, 0, q1.half(), q1.clone()), "dtype"),
            (lambda: gpu.kv_cache_read(gpu_ctx, cache, 0, kv, kv.clone(), start=[0, 1, 2]), "start")):
        with pytest.raises(ValueError, match=match):
            call()
    _check_stored(gpu, gpu_ctx, cache, m)


def test_page_layout_does_not_change_the_bits(gpu_ctx):
    banner("quant paged against contiguous")
    rng = np.random.default_rng(4)
    B, H, G, D, lens = 3, 2, 4, 128, [333, 64, 1]
    k, v = (_dev(_rows(rng, B, 333, H, D), F32) for _ in range(2))
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    outs = []
    for page in (0, 1, 16, 256):
        gpu, cache, _ = _make(gpu_ctx, B, 340, H, G, D, "fp4", page)
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, n_new=lens)
        out = torch.empty_like(q)
        gpu.decode_attention(gpu_ctx, cache, 0, q, out)
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_nan_group_reaches_its_heads_only(gpu_ctx):
    banner("quant decode NaN")
    rng = np.random.default_rng(6)
    B, H, G, D = 2, 2, 2, 64
    gpu, cache, m = _make(gpu_ctx, B, 200, H, G, D, "fp4")
    k, v = _rows(rng, B, 200, H, D), _rows(rng, B, 200, H, D)
    k[0, 50, 0, 3] = np.nan   # sequence 0, kv head 0: every element of its heads
    v[1, 120, 1, 40] = np.inf  # sequence 1, kv head 1: elements 32..63 of its heads
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, _dev(k, F32), _dev(v, F32))
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    out = torch.empty_like(q)
    gpu.decode_attention(gpu_ctx, cache, 0, q, out)
    nan = torch.isnan(out).cpu().numpy()
    want = np.zeros((B, H * G, D), bool)
    want[0, :G] = True
    want[1, G:, 32:] = True
    np.testing.assert_array_equal(nan, want)


def test_plan_that_does_not_cover_a_fill_gives_nan(gpu_ctx):
    """A captured plan that a sequence outgrew: NaN rows, the others right, the
    token of a fused append still stored."""
    banner("quant outgrown plan")
    rng = np.random.default_rng(9)
    B, H, D = 2, 2, 64
    gpu, cache, m = _make(gpu_ctx, B, 600, H, 1, D, "fp8")
    _fill(gpu, gpu_ctx, cache, m, rng, [500, 100])
    from simple_llm_amd.gpu import gpu_kv_quant as gq

    layer = cache.layers[0]
    q = _dev(rng.standard_normal((B, H, D)).astype(np.float32), F32)
    k, v = (_dev(_rows(rng, B, H, D), F32) for _ in range(2))
    for chunk in (128, 512):  # two chunks; one (no merge)
        gpu_ctx.config.decode_chunk_tokens = chunk
        out = torch.empty_like(q)
        gq.attend(gpu_ctx, cache, layer, q, out, None, 150, 300, True, k, v)
        m.append(_np(k)[:, None], _np(v)[:, None])
        layer.host_lens = m.lens.copy()
        tokens, n, _ = gq.plan(cache, 0, 0, 150, 300, True, chunk)
        assert n == (2 if chunk == 128 else 1) and m.lens[1] <= tokens * n < m.lens[0]
        assert torch.isnan(out[0]).all()
        assert not torch.isnan(out[1]).any()
    gpu_ctx.config.decode_chunk_tokens = 0
    _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("page", [0, 16])
def test_grid_that_does_not_cover_the_batch_gives_nan(gpu_ctx, page):
    """Fills that grew behind the host's back: the sequences whose chunks do not
    fit in the planned workgroups are NaN, the others right, every token of a
    fused append stored, every fill advanced."""
    banner(f"quant cut grid page={page}")
    rng = np.random.default_rng(10)
    B, H, G, D = 6, 2, 4, 64
    gpu, cache, m = _make(gpu_ctx, B, 600, H, G, D, "fp4", page)
    _fill(gpu, gpu_ctx, cache, m, rng, [130, 300, 0, 500, 1, 257])
    from simple_llm_amd.gpu import gpu_kv_quant as gq

    layer = cache.layers[0]
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    gpu_ctx.config.decode_chunk_tokens = 128
    for fused in (False, True):
        new = [_dev(_rows(rng, B, H, D), F32) for _ in range(2)] if fused else []
        out = torch.empty_like(q)
        # planned for fills that sum to 200: 1 + 6 workgroups of 2 + 3 + 1 + 4 + 1 + 3
        assert gq.plan(cache, 0, 0, 512, 200, False, 128) == (128, 4, 7)
        gq.attend(gpu_ctx, cache, layer, q, out, None, 512, 200, False, *new)
        if fused:
            m.append(_np(new[0])[:, None], _np(new[1])[:, None])
            layer.host_lens = m.lens.copy()
        assert torch.isnan(out[3:]).all() and not torch.isnan(out[:3]).any()
        keep = Model(3, m.cap, H, D, "fp4")
        keep.k, keep.v, keep.lens = m.k[:3], m.v[:3], m.lens[:3]
        _check_attention(out[:3, None], q[:3, None], keep, G, D ** -0.5, True, False)
    gpu_ctx.config.decode_chunk_tokens = 0
    _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("B", [65, 200, 300])
def test_large_ragged_batches(gpu_ctx, B):
    """Batches past one scan step, and past the scan."""
    banner(f"quant ragged batch {B}")
    rng = np.random.default_rng(B)
    H, G, D = 1, 2, 32
    lens = rng.integers(0, 400, B)
    gpu, cache, m = _make(gpu_ctx, B, 402, H, G, D, "fp4")
    _fill(gpu, gpu_ctx, cache, m, rng, lens, BF16)
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    for hint in (0, 128):
        gpu_ctx.config.decode_chunk_tokens = hint
        k, v = (_dev(_rows(rng, B, H, D), F32) for _ in range(2))
        out = torch.empty_like(q)
        gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q, out)
        m.append(_np(k)[:, None], _np(v)[:, None])
        _check_attention(out[:, None], q[:, None], m, G, D ** -0.5, True, False)
    gpu_ctx.config.decode_chunk_tokens = 0
    _check_stored(gpu, gpu_ctx, cache, m)


# ---- prefill ---------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("B,Hkv,G,D,lens,C,counts,page,io", [
    (1, 1, 1, 32, [0], 1, None, 0, BF16), (2, 2, 1, 64, [0, 70], 33, [33, 5], 0, F32),
    (2, 1, 2, 96, [129, 3], 40, None, 8, BF16), (3, 2, 4, 128, [0, 64, 200], 50, [50, 0, 17], 16, BF16),
    (1, 4, 8, 128, [30], 70, None, 0, BF16), (2, 1, 1, 128, [1000, 40], 130, [7, 130], 64, F32),
    (1, 2, 1, 160, [65], 31, None, 1, BF16), (2, 1, 2, 256, [100, 0], 66, None, 0, BF16),
    (1, 1, 8, 256, [5], 20, [11], 4, F32), (1, 12, 1, 64, [300], 257, None, 0, BF16),
    (4, 8, 8, 32, [60, 61, 62, 63], 90, None, 0, BF16)])
def test_prefill(gpu_ctx, fmt, B, Hkv, G, D, lens, C, counts, page, io):
    banner(f"quant prefill {fmt} B={B} Hkv={Hkv} G={G} D={D} lens={lens} C={C} {counts} page={page}")
    rng = np.random.default_rng(C + D)
    for splits in (0, 1, 3):
        gpu, cache, m = _make(gpu_ctx, B, max(lens) + C + 1, Hkv, G, D, fmt, page)
        _fill(gpu, gpu_ctx, cache, m, rng, lens)
        k, v = (_dev(_rows(rng, B, C, Hkv, D), io) for _ in range(2))
        q = _dev(rng.standard_normal((B, C, Hkv * G, D)).astype(np.float32), io)
        out = torch.full_like(q, 9.0)
        fills = gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts, n_splits=splits)
        m.append(_np(k), _np(v), counts)
        assert fills.tolist() == m.lens.tolist()
        _check_attention(out, q, m, G, D ** -0.5, False, io == BF16,
                         np.asarray(counts) if counts else None, True, io == F32)
        _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("B,Hkv,splits", [(70, 2, 0), (70, 8, 1), (33, 8, 2), (33, 8, 1), (64, 1, 8),
                                          (13, 5, 3), (300, 1, 0), (300, 1, 2)])
def test_prefill_of_ragged_batches(gpu_ctx, B, Hkv, splits):
    """More (sequence, head, split) groups than the 512 that are ordered by their rows, and
    as many; sequences without rows among them."""
    banner(f"quant ragged prefill B={B} Hkv={Hkv} splits={splits}")
    rng = np.random.default_rng(B * Hkv + splits)
    G, D, C = 2, 32, 300  # three tiles of 256 rows a group
    gpu, cache, m = _make(gpu_ctx, B, C + 150, Hkv, G, D, "fp8")
    _fill(gpu, gpu_ctx, cache, m, rng, rng.integers(0, 150, B))
    counts = rng.integers(0, 20, B)
    counts[::5] = 0
    counts[[3, B - 2]] = C, 129
    k, v = (_dev(_rows(rng, B, C, Hkv, D), BF16) for _ in range(2))
    q = _dev(rng.standard_normal((B, C, Hkv * G, D)).astype(np.float32), BF16)
    out = torch.full_like(q, 9.0)
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts, n_splits=splits)
    m.append(_np(k), _np(v), counts)
    _check_attention(out, q, m, G, D ** -0.5, False, True, counts, True, False)
    _check_stored(gpu, gpu_ctx, cache, m)


def test_prefill_equals_a_bf16_cache_of_the_same_values(gpu_ctx):
    """K and V enter as a bf16 cache holding the stored values would give them."""
    banner("quant prefill against bf16 cache")
    from simple_llm_amd.gpu import gpu as g

    rng = np.random.default_rng(12)
    B, H, G, D, C = 2, 2, 4, 128, 100
    for fmt in ("fp4", "fp8"):
        gpu, cache, m = _make(gpu_ctx, B, 400, H, G, D, fmt)
        plain = g.kv_cache_create(gpu_ctx, g.KVCacheConfig(B, 400, 1, H * G, D, n_kv_heads=H,
                                                           dtype=BF16))
        for n in (250, C):
            k, v = (_dev(_rows(rng, B, n, H, D), BF16) for _ in range(2))
            sk, sv = (_dev(qo.round_trip(_np(x), fmt).astype(np.float32), BF16) for x in (k, v))
            q = _dev(rng.standard_normal((B, n, H * G, D)).astype(np.float32), BF16)
            out, want = torch.empty_like(q), torch.empty_like(q)
            gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out)
            g.kv_cache_prefill(gpu_ctx, plain, 0, sk, sv, q, want)
            assert torch.equal(out, want)


@pytest.mark.parametrize("splits", [1, 2])
def test_prefill_nan_stays_behind_the_mask(gpu_ctx, splits):
    """A NaN group reaches the queries that attend its token, not earlier ones of
    the same tile: K all elements, V its group's."""
    banner(f"quant prefill NaN splits={splits}")
    rng = np.random.default_rng(14)
    B, H, D, C = 1, 2, 64, 150
    gpu, cache, m = _make(gpu_ctx, B, 300, H, 1, D, "fp4")
    _fill(gpu, gpu_ctx, cache, m, rng, [70])
    k, v = _rows(rng, B, C, H, D), _rows(rng, B, C, H, D)
    k[0, 60, 0, 3] = np.nan
    v[0, 100, 1, 40] = np.nan
    q = _dev(rng.standard_normal((B, C, H, D)).astype(np.float32), BF16)
    out = torch.empty_like(q)
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, _dev(k, BF16), _dev(v, BF16), q, out, n_splits=splits)
    want = np.zeros((B, C, H, D), bool)
    want[0, 60:, 0] = True
    want[0, 100:, 1, 32:] = True
    np.testing.assert_array_equal(torch.isnan(out).cpu().numpy(), want)


# ---- together, streams, graphs, far offsets --------------------------------

@pytest.mark.parametrize("fmt,page", [("fp4", 0), ("fp8", 16)])
def test_serving_run(gpu_ctx, fmt, page):
    """A server's use: ragged prompts prefilled in two chunks, decode steps, a
    finished sequence replaced, more steps."""
    banner(f"quant serving run {fmt} page={page}")
    rng = np.random.default_rng(21)
    B, H, G, D, T = 3, 2, 2, 64, 160
    gpu, cache, m = _make(gpu_ctx, B, T, H, G, D, fmt, page)

    def prefill(C, counts):
        k, v = (_dev(_rows(rng, B, C, H, D), BF16) for _ in range(2))
        q = _dev(rng.standard_normal((B, C, H * G, D)).astype(np.float32), BF16)
        out = torch.empty_like(q)
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts)
        m.append(_np(k), _np(v), counts)
        _check_attention(out, q, m, G, D ** -0.5, False, True, np.asarray(counts), True)

    def steps(n):
        for _ in range(n):
            k, v = (_dev(_rows(rng, B, H, D), F32) for _ in range(2))
            q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
            out = torch.empty_like(q)
            gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q, out)
            m.append(_np(k)[:, None], _np(v)[:, None])
            _check_attention(out[:, None], q[:, None], m, G, D ** -0.5, True, False)

    prefill(40, [40, 0, 13])
    prefill(64, [20, 64, 1])
    steps(6)
    lay = cache.layers[0]
    lay.lens[1] = 0  # sequence 1 is done; another takes its place
    lay.host_lens[1] = 0
    m.lens[1] = 0
    prefill(30, [0, 30, 0])
    steps(4)
    _check_stored(gpu, gpu_ctx, cache, m)


def test_captured_steps(gpu_ctx):
    """Decode steps in a captured graph, replayed between eager calls of the same
    cache: every replay equals the eager step."""
    banner("quant captured steps")
    rng = np.random.default_rng(31)
    B, H, G, D, T = 2, 2, 4, 128, 700
    gpu, cache, _ = _make(gpu_ctx, B, T, H, G, D, "fp4", 16)
    _, twin, m = _make(gpu_ctx, B, T, H, G, D, "fp4", 16)
    k0, v0 = (_dev(_rows(rng, B, 300, H, D), F32) for _ in range(2))
    for c in (cache, twin):
        gpu.kv_cache_prefill(gpu_ctx, c, 0, k0, v0, n_new=[300, 120])
    k, v = (torch.zeros(B, H, D, device="cuda:0") for _ in range(2))
    q = torch.zeros(B, H * G, D, device="cuda:0")
    out = torch.empty_like(q)
    lay = cache.layers[0]
    lens0, host0 = lay.lens.clone(), lay.host_lens.copy()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # a step before the capture, undone
        gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q, out, max_len=600)
    side.synchronize()
    lay.lens.copy_(lens0)
    lay.host_lens = host0.copy()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q, out, max_len=600)
    lay.host_lens = host0.copy()
    for i in range(6):
        k.copy_(_dev(_rows(rng, B, H, D), F32))
        v.copy_(_dev(_rows(rng, B, H, D), F32))
        q.copy_(_dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32))
        want = torch.empty_like(q)
        gpu.kv_cache_append_attend(gpu_ctx, twin, 0, k, v, q, want, max_len=600)
        graph.replay()
        torch.cuda.synchronize()
        lay.host_lens += 1
        assert torch.allclose(out, want, rtol=0, atol=2e-5 * float(want.abs().max()))
        assert lay.lens.cpu().tolist() == twin.layers[0].lens.cpu().tolist()
        eager = torch.empty_like(q)  # over the graph's cache, its plan, between the replays
        gpu.decode_attention(gpu_ctx, cache, 0, q, eager)
        assert torch.allclose(out, eager, rtol=0, atol=2e-5 * float(want.abs().max()))
    for a, b in ((lay.k_cache, twin.layers[0].k_cache), (lay.v_scale, twin.layers[0].v_scale)):
        assert torch.equal(a.buffer, b.buffer)


def test_captured_call_without_a_bound(gpu_ctx):
    """Replayed with fills that sum to more than at the capture, none past its longest."""
    banner("quant captured without a bound")
    rng = np.random.default_rng(37)
    B, H, G, D = 3, 2, 2, 64
    gpu, cache, m = _make(gpu_ctx, B, 2200, H, G, D, "fp8")
    _fill(gpu, gpu_ctx, cache, m, rng, [2100, 5, 0])
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    out, want = torch.empty_like(q), torch.empty_like(q)
    gpu.decode_attention(gpu_ctx, cache, 0, q, out)  # eager before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.decode_attention(gpu_ctx, cache, 0, q, out)
    for counts in ([0, 1000, 1], [0, 1095, 2099]):
        _fill(gpu, gpu_ctx, cache, m, rng, counts)
        gpu.decode_attention(gpu_ctx, cache, 0, q, want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
        assert torch.allclose(out, want, rtol=0, atol=2e-5 * float(want.abs().max()))


@pytest.mark.parametrize("fmt,page,splits", [("fp4", 0, 1), ("fp8", 16, 2), ("fp4", 8, 0)])
def test_captured_chunk(gpu_ctx, fmt, page, splits):
    """A ragged chunk with attention, one without and a read in a captured graph: replays
    go on from the fills they find, with the counts and starts of the capture."""
    banner(f"quant captured chunk {fmt} page={page} splits={splits}")
    rng = np.random.default_rng(43)
    B, H, G, D, C, T = 3, 2, 4, 64, 30, 400
    gpu, cache, m = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    _, twin, _ = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    counts, more = [C, 0, 7], [1, 12, 0]
    k, v = (torch.zeros(B, C, H, D, device="cuda:0") for _ in range(2))
    q = torch.zeros(B, C, H * G, D, dtype=BF16, device="cuda:0")
    outs = [torch.empty_like(q), *(torch.empty(B, 50, H, D, device="cuda:0") for _ in "kv")]
    want = [torch.empty_like(x) for x in outs]

    def calls(c, o):
        gpu.kv_cache_prefill(gpu_ctx, c, 0, k, v, q, o[0], n_new=counts, n_splits=splits)
        gpu.kv_cache_prefill(gpu_ctx, c, 0, k, v, n_new=more)
        gpu.kv_cache_read(gpu_ctx, c, 0, o[1], o[2], start=[10, 0, 3])

    lay = cache.layers[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # before the capture, undone
        calls(cache, outs)
    side.synchronize()
    lay.lens.zero_()
    lay.host_lens[:] = 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(cache, outs)
    lay.host_lens[:] = 0
    for _ in range(4):
        k.copy_(_dev(_rows(rng, B, C, H, D), F32))
        v.copy_(_dev(_rows(rng, B, C, H, D), F32))
        q.copy_(_dev(rng.standard_normal((B, C, H * G, D)).astype(np.float32), BF16))
        calls(twin, want)
        graph.replay()
        torch.cuda.synchronize()
        lay.host_lens += np.array(counts) + more
        assert lay.lens.cpu().tolist() == twin.layers[0].lens.cpu().tolist() == lay.host_lens.tolist()
        for a, b in zip(outs[1:], want[1:]):
            assert torch.equal(a, b)
        # (the splits of the eager call follow its fills: each side rounds p by 2^-8)
        assert torch.allclose(outs[0].float(), want[0].float(), rtol=2.0 ** -7,
                              atol=2.0 ** -6 * float(v.abs().max()))


def test_bound_past_the_capacity(gpu_ctx):
    """A max_len of any size plans for what the cache can hold."""
    banner("quant bound past the capacity")
    rng = np.random.default_rng(38)
    for page in (0, 16):
        gpu, cache, m = _make(gpu_ctx, 2, 300, 2, 2, 64, "fp4", page)
        _fill(gpu, gpu_ctx, cache, m, rng, [300, 17])
        q = _dev(rng.standard_normal((2, 4, 64)).astype(np.float32), F32)
        a, b = torch.empty_like(q), torch.empty_like(q)
        gpu.decode_attention(gpu_ctx, cache, 0, q, a, max_len=m.cap)
        gpu.decode_attention(gpu_ctx, cache, 0, q, b, max_len=10**12)
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_chunk_beside_a_sequence_past_max_seq_len(gpu_ctx):
    """Appends fill a paged sequence's last page; others go on taking chunks."""
    banner("quant chunk beside a full sequence")
    rng = np.random.default_rng(39)
    gpu, cache, m = _make(gpu_ctx, 2, 20, 2, 1, 32, "fp8", 16)
    _fill(gpu, gpu_ctx, cache, m, rng, [20, 3])
    for _ in range(2):
        k, v = (_dev(_rows(rng, 2, 1, 2, 32), F32) for _ in range(2))
        gpu.kv_cache_append(gpu_ctx, cache, 0, k, v)
        m.append(_np(k), _np(v))
    _fill(gpu, gpu_ctx, cache, m, rng, [0, 15])
    with pytest.raises(ValueError, match="Cache is full"):
        _fill(gpu, gpu_ctx, cache, m, rng, [1, 0])
    with pytest.raises(ValueError, match="Cache is full"):
        _fill(gpu, gpu_ctx, cache, m, rng, [0, 1])
    _check_stored(gpu, gpu_ctx, cache, m)


def test_two_streams_at_once(gpu_ctx):
    """Calls of one context on two streams share no workspace."""
    banner("quant two streams")
    rng = np.random.default_rng(41)
    runs = []
    for fmt in ("fp4", "fp8"):
        gpu, cache, m = _make(gpu_ctx, 2, 3000, 4, 1, 128, fmt)
        _fill(gpu, gpu_ctx, cache, m, rng, [2900, 1500])
        q = _dev(rng.standard_normal((2, 4, 128)).astype(np.float32), F32)
        want = torch.empty_like(q)
        gpu.decode_attention(gpu_ctx, cache, 0, q, want)
        runs.append((cache, q, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for cache, q, want, s in runs:
            with torch.cuda.stream(s):
                out = torch.empty_like(q)
                gpu.decode_attention(gpu_ctx, cache, 0, q, out)
                outs.append((out, want))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in outs)


def test_offsets_past_32_bits(gpu_ctx):
    """The last sequence's rows lie past 4 GiB of codes."""
    banner("quant far offsets")
    rng = np.random.default_rng(51)
    B, H, G, D, T = 3, 16, 2, 128, 1 << 21
    gpu, cache, _ = _make(gpu_ctx, B, T, H, G, D, "fp4")
    assert cache.layers[0].k_cache.buffer.numel() > 2 ** 32
    m = Model(B, 400, H, D, "fp4")
    _fill(gpu, gpu_ctx, cache, m, rng, [3, 0, 300])
    k, v = (_dev(_rows(rng, B, H, D), F32) for _ in range(2))
    q = _dev(rng.standard_normal((B, H * G, D)).astype(np.float32), F32)
    out = torch.empty_like(q)
    gpu.kv_cache_append_attend(gpu_ctx, cache, 0, k, v, q, out)
    m.append(_np(k)[:, None], _np(v)[:, None])
    _check_attention(out[:, None], q[:, None], m, G, D ** -0.5, True, False)
    C = 20
    k, v = (_dev(_rows(rng, B, C, H, D), BF16) for _ in range(2))
    q = _dev(rng.standard_normal((B, C, H * G, D)).astype(np.float32), BF16)
    out = torch.empty_like(q)
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out)
    m.append(_np(k), _np(v))
    _check_attention(out, q, m, G, D ** -0.5, False, True, None, True)
    _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("splits", [1, 2, 3, 5])
def test_prefill_keeps_nan_keys_of_any_split(gpu_ctx, fmt, page, splits):
    """Queries whose every token in one split has a NaN key are NaN, as with one
    split: the first position of a later split, a whole split, every split. The
    rows that attend none of them keep the bits of a call without NaN."""
    banner(f"quant prefill NaN split {fmt} page={page} splits={splits}")
    rng = np.random.default_rng(15)
    B, H, G, D, P, C = 2, 3, 2, 64, 70, 150  # 220 positions; splits of 128 (2, 3) or 64 tokens
    prefix = [_rows(rng, B, P, H, D) for _ in range(2)]
    k, v = _rows(rng, B, C, H, D), _rows(rng, B, C, H, D)
    q = _dev(rng.standard_normal((B, C, H * G, D)).astype(np.float32), BF16)
    want = np.zeros((B, C, H, D), bool)
    bad_prefix, bad = prefix[0].copy(), k.copy()
    for at, h in ((128, 0), (192, 1)):  # the first position of a split
        bad[0, at - P, h, 3] = np.nan
        want[0, at - P:, h] = True
    bad[0, 128 - P:, 2, 40] = np.nan  # every position past 127
    want[0, 128 - P:, 2] = True
    bad_prefix[1, :, 1, 7] = np.nan  # every key of a head
    bad[1, :, 1, 7] = np.nan
    want[1, :, 1] = True
    outs = []
    for first, keys in ((prefix[0], k), (bad_prefix, bad)):
        gpu, cache, _ = _make(gpu_ctx, B, P + C, H, G, D, fmt, page)
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, _dev(first, F32), _dev(prefix[1], F32))
        out = torch.empty_like(q)
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, _dev(keys, F32), _dev(v, F32), q, out,
                             n_splits=splits)
        outs.append(out)
    want = torch.from_numpy(np.repeat(want, G, 2)).to("cuda:0")
    assert torch.equal(torch.isnan(outs[1]), want)
    assert torch.equal(outs[1][~want], outs[0][~want])


def _check_prefill_fp32(got, q, m, G, scale, rows, out_bf16):
    """Prefill with fp32 q or out, got, q [B, C, Hq, D]. The bounds at the top of the
    file, with what this kernel does otherwise: a score is 3 D / 16 products of 16
    elements (the second and third parts of q are 2^-8 and 2^-16 of it): (D + 3 D / 16
    + 8) u A, within 2 (D + 8) u A. A lane sums its column's tokens alone: of each 16,
    three products and one more rounding inside them, so n / 4 steps, 64 for the
    rescalings, the sum of p, the merge and the division. Three parts hold all of p."""
    got, q = _np(got), _np(q)
    B, C, Hq, D = q.shape
    for b in range(B):
        n, r = int(m.lens[b]), int(rows[b])
        assert not got[b, r:].any(), f"rows past the count of sequence {b} are not zeros"
        last = n - r + np.arange(r)
        for h in range(Hq):
            want, mag, big = qo.attention(q[b, :r, h], m.k[b, :n, h // G], m.v[b, :n, h // G],
                                          scale, last)
            tol = (2 * (D + 8) * U * big + (n / 4 + 64) * U)[:, None] * mag
            bound = tol + (2.0 ** -8 * (np.abs(want) + tol) if out_bf16 else 0.0) + 1e-37
            err = np.abs(got[b, :r, h] - want)
            assert not np.isnan(got[b, :r, h]).any()
            assert (err <= bound).all(), (
                f"sequence {b} head {h}: off by {(err / bound).max():.2f} of the bound")


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("B,Hkv,G,D,lens,C,counts,page", [
    (1, 1, 1, 32, [0], 1, None, 0), (2, 2, 8, 32, [3, 200], 47, [47, 9], 16),
    (2, 2, 1, 64, [0, 70], 33, [33, 5], 0), (1, 3, 4, 64, [300], 257, None, 8),
    (2, 1, 2, 96, [129, 3], 40, None, 8), (3, 2, 4, 128, [0, 64, 200], 50, [50, 0, 17], 16),
    (2, 1, 1, 128, [1000, 40], 130, [7, 130], 0), (1, 1, 8, 128, [63], 65, None, 1),
    (1, 2, 1, 160, [65], 31, None, 1), (2, 1, 2, 256, [100, 0], 66, None, 0),
    (1, 1, 8, 256, [5], 20, [11], 4), (1, 2, 4, 224, [500], 70, None, 0)])
def test_prefill_of_fp32_keeps_fp32(gpu_ctx, fmt, B, Hkv, G, D, lens, C, counts, page):
    """fp32 q or output: products of fp32 accuracy, as in decode over the same cache."""
    banner(f"quant prefill fp32 {fmt} B={B} Hkv={Hkv} G={G} D={D} lens={lens} C={C} {counts} {page}")
    rng = np.random.default_rng(C + D)
    rows = np.full(B, C) if counts is None else np.asarray(counts)
    for splits, qt, ot in ((0, F32, F32), (1, F32, F32), (3, F32, F32), (1, BF16, F32),
                           (2, F32, BF16)):
        gpu, cache, m = _make(gpu_ctx, B, max(lens) + C + 1, Hkv, G, D, fmt, page)
        _fill(gpu, gpu_ctx, cache, m, rng, lens)
        k, v = (_dev(_rows(rng, B, C, Hkv, D), F32) for _ in range(2))
        q = _dev(rng.standard_normal((B, C, Hkv * G, D)).astype(np.float32), qt)
        out = torch.full(q.shape, 9.0, dtype=ot, device="cuda:0")
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts, n_splits=splits)
        m.append(_np(k), _np(v), counts)
        _check_prefill_fp32(out, q, m, G, D ** -0.5, rows, ot == BF16)
        _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("G,D", [(1, 64), (2, 96), (4, 256)])
def test_prefill_of_tiny_queries(gpu_ctx, G, D):
    """Scores of ordinary size from queries whose last bits bf16 cannot hold unscaled."""
    banner(f"quant prefill tiny queries G={G} D={D}")
    rng = np.random.default_rng(29)
    B, H, C = 1, 2, 130
    gpu, cache, m = _make(gpu_ctx, B, C, H, G, D, "fp8")
    k = _dev(_rows(rng, B, C, H, D).astype(np.float64) * 2.0 ** 118, F32)
    v = _dev(_rows(rng, B, C, H, D), F32)
    q = _dev((rng.standard_normal((B, C, H * G, D)) * 2.0 ** -122).astype(np.float32), F32)
    out = torch.empty_like(q)
    scale = 16 * D ** -0.5
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, scale=scale)
    m.append(_np(k), _np(v))
    _check_prefill_fp32(out, q, m, G, scale, [C], False)


def test_prefill_of_fp32_nan_groups(gpu_ctx):
    """NaN groups of K and V reach the queries that attend their tokens, no others."""
    banner("quant prefill fp32 NaN")
    rng = np.random.default_rng(14)
    B, H, D, C = 1, 2, 64, 150
    for splits in (1, 2):
        gpu, cache, m = _make(gpu_ctx, B, 300, H, 1, D, "fp8")
        _fill(gpu, gpu_ctx, cache, m, rng, [70])
        k, v = _rows(rng, B, C, H, D), _rows(rng, B, C, H, D)
        k[0, 60, 0, 3] = np.nan
        v[0, 100, 1, 40] = np.nan
        q = _dev(rng.standard_normal((B, C, H, D)).astype(np.float32), F32)
        out = torch.empty_like(q)
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, _dev(k, F32), _dev(v, F32), q, out,
                             n_splits=splits)
        want = np.zeros((B, C, H, D), bool)
        want[0, 60:, 0] = True
        want[0, 100:, 1, 32:] = True
        np.testing.assert_array_equal(torch.isnan(out).cpu().numpy(), want)


@pytest.mark.parametrize("fmt,page,splits,io", [("fp4", 0, 1, BF16), ("fp8", 16, 2, BF16),
                                                ("fp8", 0, 3, F32), ("fp4", 8, 1, F32)])
def test_c_counts_on_the_device(gpu_ctx, fmt, page, splits, io):
    """The C entry points with the counts in device memory, and an append that does
    not advance: the bytes, fills and outputs of counts on the host."""
    banner(f"quant device counts {fmt} page={page} splits={splits} {io}")
    from simple_llm_amd import _lib
    from simple_llm_amd.gpu import gpu_kv_quant as gq

    rng = np.random.default_rng(47)
    B, H, G, D, C, T = 4, 2, 4, 96, 37, 300
    gpu, cache, m = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    _, twin, _ = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    lay, L = cache.layers[0], _lib.lib()
    code = _lib.dtype_code(io)
    q = _dev(rng.standard_normal((B, C, H * G, D)).astype(np.float32), io)
    ws = torch.empty(L.skv_prefill_workspace_bytes(B, C, H * G, D, splits) + 8 * B,
                     dtype=torch.uint8, device="cuda:0")
    for counts in ([C, 0, 5, 36], [0, 1, C, 2], None):
        n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda:0")
        n_ptr = None if n is None else n.data_ptr()
        k, v = (_dev(_rows(rng, B, C, H, D), io) for _ in range(2))
        sizes = (*gq._pages(cache), B, C, H, D, T, _lib.QUANT_FORMATS[cache.dtype], code,
                 _lib.stream_handle(lay.lens.device))
        chunk = (*gq._storage(lay), k.data_ptr(), v.data_ptr(), lay.lens.data_ptr(), n_ptr, None)
        fills = lay.lens.clone()
        assert L.skv_q_append_chunk(*chunk, 0, *sizes) == 0  # the rows alone
        assert torch.equal(lay.lens, fills)
        assert L.skv_q_append_chunk(*chunk, 1, *sizes) == 0  # the same rows again, and the fills
        gpu.kv_cache_prefill(gpu_ctx, twin, 0, k, v, n_new=counts)
        m.append(_np(k), _np(v), counts)
        assert torch.equal(lay.lens, twin.layers[0].lens)
        k, v = (_dev(_rows(rng, B, C, H, D), io) for _ in range(2))
        out, want = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
        rc = L.skv_q_append_prefill_attn(
            out.data_ptr(), q.data_ptr(), *gq._storage(lay), k.data_ptr(), v.data_ptr(),
            lay.lens.data_ptr(), n_ptr, None, *gq._pages(cache), B, C, H * G, H, D, T, D ** -0.5,
            splits, ws.data_ptr(), ws.numel(), _lib.QUANT_FORMATS[cache.dtype], code, code, code,
            _lib.stream_handle(lay.lens.device))
        assert rc == 0
        gpu.kv_cache_prefill(gpu_ctx, twin, 0, k, v, q, want, n_new=counts, n_splits=splits)
        m.append(_np(k), _np(v), counts)
        assert torch.equal(out, want)
        for x in ("k_cache", "k_scale", "v_cache", "v_scale"):
            assert torch.equal(getattr(lay, x).buffer, getattr(twin.layers[0], x).buffer)
    lay.host_lens = m.lens.copy()
    _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("fmt,page,splits,io", [("fp4", 0, 1, BF16), ("fp8", 16, 2, BF16),
                                                ("fp4", 8, 0, BF16), ("fp8", 0, 0, F32),
                                                ("fp4", 16, 3, F32)])
def test_captured_chunk_outputs(gpu_ctx, fmt, page, splits, io):
    """A captured ragged chunk, replayed: the eager call's bits where both take the same
    splits, else within the bounds of float64 over the stored values."""
    banner(f"quant captured chunk outputs {fmt} page={page} splits={splits} {io}")
    rng = np.random.default_rng(53)
    B, H, G, D, C, T = 3, 2, 4, 64, 30, 400
    gpu, cache, m = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    _, twin, _ = _make(gpu_ctx, B, T, H, G, D, fmt, page)
    counts = np.array([C, 0, 7])
    k, v = (torch.zeros(B, C, H, D, device="cuda:0") for _ in range(2))
    q = torch.zeros(B, C, H * G, D, dtype=io, device="cuda:0")
    out, want = torch.empty_like(q), torch.empty_like(q)
    lay = cache.layers[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # before the capture, undone
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts, n_splits=splits)
    side.synchronize()
    lay.lens.zero_()
    lay.host_lens[:] = 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts, n_splits=splits)
    lay.host_lens[:] = 0
    for _ in range(4):
        k.copy_(_dev(_rows(rng, B, C, H, D), F32))
        v.copy_(_dev(_rows(rng, B, C, H, D), F32))
        q.copy_(_dev(rng.standard_normal((B, C, H * G, D)).astype(np.float32), io))
        out.fill_(9.0)
        gpu.kv_cache_prefill(gpu_ctx, twin, 0, k, v, q, want, n_new=counts, n_splits=splits)
        graph.replay()
        torch.cuda.synchronize()
        lay.host_lens += counts
        m.append(_np(k), _np(v), counts)
        if splits:
            assert torch.equal(out, want)
        if io == F32:
            _check_prefill_fp32(out, q, m, G, D ** -0.5, counts, False)
        else:
            _check_attention(out, q, m, G, D ** -0.5, False, True, counts, True)
    _check_stored(gpu, gpu_ctx, cache, m)


@pytest.mark.parametrize("B,Hkv,D,splits", [(70, 2, 32, 0), (33, 8, 32, 2), (33, 8, 64, 1),
                                            (13, 5, 128, 3), (300, 1, 32, 2)])
def test_prefill_of_fp32_ragged_batches(gpu_ctx, B, Hkv, D, splits):
    """Tiles of 128 rows, several a group: groups that are ordered by their rows and, past
    512 of them, not; sequences without rows among them."""
    banner(f"quant ragged prefill fp32 B={B} Hkv={Hkv} D={D} splits={splits}")
    rng = np.random.default_rng(B * Hkv + splits)
    G, C = 2, 300
    gpu, cache, m = _make(gpu_ctx, B, C + 150, Hkv, G, D, "fp4")
    _fill(gpu, gpu_ctx, cache, m, rng, rng.integers(0, 150, B))
    counts = rng.integers(0, 20, B)
    counts[::5] = 0
    counts[[3, B - 2]] = C, 129
    k, v = (_dev(_rows(rng, B, C, Hkv, D), F32) for _ in range(2))
    q = _dev(rng.standard_normal((B, C, Hkv * G, D)).astype(np.float32), F32)
    out = torch.full_like(q, 9.0)
    gpu.kv_cache_prefill(gpu_ctx, cache, 0, k, v, q, out, n_new=counts, n_splits=splits)
    m.append(_np(k), _np(v), counts)
    _check_prefill_fp32(out, q, m, G, D ** -0.5, counts, False)
    _check_stored(gpu, gpu_ctx, cache, m)
