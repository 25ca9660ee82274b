"""Block-scaled caches on the CPU: the oracle against torch's own 8-bit type and
by hand, and every refusal, in Python and at the C entry points (no call here
reaches a launch)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import quant_oracle as qo
from simple_llm_amd import _lib
from simple_llm_amd.gpu import gpu
from simple_llm_amd.gpu.gpu_types import GPUConfig, GPUContext, PipelineCache

FP4, FP8 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn


def _ctx():
    return GPUContext(device=torch.device("cpu"), config=GPUConfig(), batch_state=None,
                      pipeline_cache=PipelineCache())


# ---- the oracle ------------------------------------------------------------

def test_grids():
    assert qo.grid("fp4").tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    want = torch.arange(127).to(torch.uint8).view(FP8).double().numpy()
    np.testing.assert_array_equal(qo.grid("fp8"), want)


def test_rounding_equals_torch_float8():
    """Under scale 1 (a group maximum of 448) the codes are torch's conversion."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((500, 32)) * np.exp(rng.uniform(-8, 5, (500, 1)))).astype(np.float32)
    x = np.clip(x, -448, 448)
    x[:, 0] = 448
    code, byte = qo.quantise(x, "fp8")
    assert (byte == 127).all()
    np.testing.assert_array_equal(code, torch.from_numpy(x).to(FP8).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt,peak,e", [
    ("fp4", 7.0, 0), ("fp4", 7.0000005, 1), ("fp4", 3.5, -1), ("fp4", 3.5000002, 0),
    ("fp4", 6.0, 0), ("fp4", 4.0, 0), ("fp4", 0.0, -100), ("fp4", 1e-38, -100),
    ("fp4", 3.4e38, 125), ("fp8", 464.0, 0), ("fp8", 464.00003, 1), ("fp8", 448.0, 0),
    ("fp8", 232.0, -1), ("fp8", 3.4e38, 119), ("fp8", 1e-45, -100)])
def test_scale_rule(fmt, peak, e):
    x = np.zeros((1, 32), np.float32)
    x[0, 7] = -peak
    _, byte = qo.quantise(x, fmt)
    assert int(byte[0, 0]) - 127 == e


def test_values_round_to_the_nearest_and_fit_bf16():
    rng = np.random.default_rng(1)
    for fmt in ("fp4", "fp8"):
        x = rng.standard_normal((64, 64)).astype(np.float32)
        y = qo.round_trip(x, fmt)
        g = np.abs(x.reshape(64, 2, 32)).max(-1).repeat(32, -1)
        # half a step of the binade, and of the smallest scale whose top reaches the maximum
        rel, tiny = (0.25, 2.0 / 3.5 / 8) if fmt == "fp4" else (2.0 ** -4, 2.0 ** -10 / 232)
        assert (np.abs(y - x) <= np.maximum(rel * np.abs(x), tiny * g) + 1e-30).all()
        bf = torch.from_numpy(y).to(torch.bfloat16).double().numpy()
        np.testing.assert_array_equal(bf, y)


def test_groups_that_are_not_finite_read_as_nan():
    x = np.ones((3, 64), np.float32)
    x[0, 5], x[1, 40] = np.nan, -np.inf
    y = qo.round_trip(x, "fp4")
    assert np.isnan(y[0, :32]).all() and np.isnan(y[1, 32:]).all()
    assert np.isfinite(y[0, 32:]).all() and np.isfinite(y[1, :32]).all()
    assert np.isfinite(y[2]).all()


# ---- Python refusals -------------------------------------------------------

@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=48), "multiple of 32"), (dict(head_dim=288), "up to 256"),
    (dict(n_heads=34, n_kv_heads=2), "up to 16 query heads"),
    (dict(dtype=torch.float16), "dtype must be"), (dict(dtype=torch.float8_e5m2), "dtype must be"),
    (dict(max_seq_len=2**30 + 1), "2\\^30"), (dict(max_seq_len=2**30 + 1, block_size=16), "2\\^30"),
    (dict(block_size=12), "power of two"), (dict(batch_size=70000, max_seq_len=1), "65535")])
def test_create_refuses(kw, match):
    args = dict(batch_size=2, max_seq_len=8, n_layers=1, n_heads=4, head_dim=64, dtype=FP4)
    with pytest.raises(ValueError, match=match):
        gpu.kv_cache_create(_ctx(), gpu.KVCacheConfig(**{**args, **kw}))


@pytest.mark.parametrize("dtype,width", [(FP4, 32), (FP8, 64)])
@pytest.mark.parametrize("page", [0, 4])
def test_layout(dtype, width, page):
    cache = gpu.kv_cache_create(_ctx(), gpu.KVCacheConfig(3, 10, 2, 4, 64, n_kv_heads=2,
                                                          dtype=dtype, block_size=page))
    rows = 3 * 3 * 4 * 2 if page else 3 * 10 * 2
    assert cache.quantized and cache.current_len == 0
    for lay in cache.layers:
        assert lay.k_cache.shape == lay.v_cache.shape == (rows, width)
        assert lay.k_scale.shape == lay.v_scale.shape == (rows, 2)
        assert lay.k_cache.buffer.dtype == lay.k_scale.buffer.dtype == torch.uint8
    plain = gpu.kv_cache_create(_ctx(), gpu.KVCacheConfig(3, 10, 1, 4, 64))
    assert not plain.quantized and plain.layers[0].k_scale is None


def test_calls_refuse_before_any_device_work():
    ctx = _ctx()
    cache = gpu.kv_cache_create(ctx, gpu.KVCacheConfig(2, 8, 1, 4, 64, dtype=FP8))
    row, q = torch.zeros(2, 4, 64), torch.zeros(2, 4, 64)
    chunk = torch.zeros(2, 3, 4, 64)
    for call in (lambda: gpu.kv_cache_append(ctx, cache, 0, row, row),
                 lambda: gpu.decode_attention(ctx, cache, 0, q, torch.zeros_like(q)),
                 lambda: gpu.kv_cache_append_attend(ctx, cache, 0, row, row, q, torch.zeros_like(q)),
                 lambda: gpu.kv_cache_prefill(ctx, cache, 0, chunk, chunk),
                 lambda: gpu.kv_cache_read(ctx, cache, 0, chunk, chunk)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="must hold"):
        gpu.kv_cache_append(ctx, cache, 0, torch.zeros(2, 4, 32), row)
    with pytest.raises(ValueError, match="out of range"):
        gpu.kv_cache_read(ctx, cache, 1, chunk, chunk)
    assert cache.current_len == 0
    plain = gpu.kv_cache_create(ctx, gpu.KVCacheConfig(2, 8, 1, 4, 64))
    with pytest.raises(ValueError, match="not block-scaled"):
        gpu.kv_cache_read(ctx, plain, 0, chunk, chunk)


def test_model_refuses_a_block_scaled_cache():
    from simple_llm_amd.model import TransformerModel, TransformerModelParams

    with pytest.raises(ValueError, match="float32 or bfloat16"):
        TransformerModel(_ctx(), TransformerModelParams(32, 64, 16, 2, 1), kv_dtype=FP4)


# ---- C refusals ------------------------------------------------------------

START = (ctypes.c_int * 2)()
TOO_MANY, NEGATIVE = (ctypes.c_int * 2)(1, 4), (ctypes.c_int * 2)(-1, 2)
FAKE = 4096  # never dereferenced: each call below fails validation first
BASE = dict(k=FAKE, ks=FAKE, v=FAKE, vs=FAKE, bt=None, mb=0, bs=0, B=2, Hq=8, H=4, D=64, T=128,
            fmt=_lib.MXFP4, idt=0, qdt=0, odt=0, C=3, new=FAKE, lens=FAKE, q=FAKE, out=FAKE,
            chunk=128, n=2, wg=4, ws=FAKE, nb=None, splits=1, scale=0.125)


def _call(which, **kw):
    a = {**BASE, **kw}
    L = _lib.lib()
    st = (a["k"], a["ks"], a["v"], a["vs"])
    pg = (a["bt"], a["mb"], a["bs"])
    nb = a["nb"]
    if which == "append":
        return L.skv_q_append(*st, a["new"], a["new"], a["lens"], *pg, a["B"], a["H"], a["D"],
                              a["T"], a["fmt"], a["idt"], None)
    if which == "chunk":
        return L.skv_q_append_chunk(*st, a["new"], a["new"], a["lens"], kw.get("n_new"),
                                    kw.get("n_host"), 1, *pg, a["B"], a["C"], a["H"], a["D"],
                                    a["T"], a["fmt"], a["idt"], None)
    if which == "read":
        return L.skv_q_read(a["out"], a["out"], *st, a["lens"], kw.get("start", START),
                            a.get("n_start", 2), *pg, a["B"], a["C"], a["H"], a["D"], a["T"],
                            a["fmt"], a["odt"], None)
    if which == "decode":
        if nb is None:
            nb = L.skv_q_decode_workspace_bytes(a["B"], a["Hq"], a["D"], a["n"])
        return L.skv_q_decode_attn(a["out"], a["q"], *st, a["new"], kw.get("new_v", a["new"]),
                                   a["lens"], *pg, a["B"], a["Hq"], a["H"], a["D"], a["T"],
                                   a["scale"], a["chunk"], a["n"], a["wg"], a["ws"], nb, a["fmt"],
                                   a["idt"], a["qdt"], a["odt"], None)
    if nb is None:
        nb = L.skv_prefill_workspace_bytes(a["B"], a["C"], a["Hq"], a["D"], a["splits"])
    return L.skv_q_append_prefill_attn(a["out"], a["q"], *st, a["new"], a["new"], a["lens"],
                                       kw.get("n_new"), kw.get("n_host"), *pg, a["B"], a["C"],
                                       a["Hq"], a["H"], a["D"], a["T"], a["scale"], a["splits"],
                                       a["ws"], nb, a["fmt"], a["idt"], a["qdt"], a["odt"], None)


INV, UNS, WSP = _lib.SKV_E_INVALID, _lib.SKV_E_UNSUPPORTED, _lib.SKV_E_WORKSPACE


@pytest.mark.parametrize("which", ["append", "chunk", "read", "decode", "prefill"])
@pytest.mark.parametrize("kw,rc", [
    (dict(k=None), INV), (dict(ks=None), INV), (dict(v=None), INV), (dict(vs=None), INV),
    (dict(lens=None), INV), (dict(fmt=0), INV), (dict(fmt=1), INV), (dict(fmt=4), INV),
    (dict(D=0), INV), (dict(D=48), UNS), (dict(D=288), UNS), (dict(B=0), INV), (dict(H=0), INV),
    (dict(B=65536), UNS), (dict(T=0), INV), (dict(k=FAKE + 8), INV),
    (dict(bt=FAKE, mb=4, bs=12), INV), (dict(bt=FAKE, mb=0, bs=16), INV),
    (dict(bt=FAKE, mb=1 << 28, bs=16), INV), (dict(bt=FAKE, mb=(1 << 26) + 1, bs=16), UNS),
    (dict(T=(1 << 30) + 1), UNS)])
def test_cache_arguments_refused(which, kw, rc):
    assert _call(which, **kw) == rc
    assert _lib.lib().skv_last_error()


@pytest.mark.parametrize("which,kw,rc", [
    ("append", dict(new=None), INV), ("append", dict(new=FAKE + 4), INV),
    ("append", dict(idt=2), INV), ("chunk", dict(C=0), INV), ("chunk", dict(new=None), INV),
    ("chunk", dict(idt=3), INV), ("chunk", dict(new=FAKE + 8), INV), ("read", dict(C=0), INV),
    ("read", dict(start=None), INV), ("read", dict(n_start=3), INV),
    ("read", dict(out=None), INV), ("read", dict(odt=2), INV), ("read", dict(out=FAKE + 4), INV),
    ("decode", dict(q=None), INV), ("decode", dict(out=None), INV),
    ("decode", dict(new_v=None), INV), ("decode", dict(qdt=2), INV), ("decode", dict(odt=5), INV),
    ("decode", dict(idt=2), INV), ("decode", dict(q=FAKE + 4), INV), ("decode", dict(Hq=10), INV),
    ("decode", dict(Hq=0), INV), ("decode", dict(Hq=68), UNS), ("decode", dict(chunk=96), INV),
    ("decode", dict(chunk=0), INV), ("decode", dict(n=0), INV), ("decode", dict(nb=16), WSP),
    ("decode", dict(ws=None), WSP), ("decode", dict(chunk=1 << 30, n=4), UNS),
    ("decode", dict(scale=float("inf")), INV), ("decode", dict(scale=float("nan")), INV),
    ("decode", dict(chunk=(1 << 30) + 128, n=1, wg=2), UNS), ("decode", dict(wg=1), INV),
    ("decode", dict(wg=5), INV), ("decode", dict(B=300, wg=599), INV),
    ("decode", dict(B=300, n=300, wg=90000), UNS),
    ("chunk", dict(n_host=TOO_MANY), INV), ("chunk", dict(n_host=NEGATIVE), INV),
    ("chunk", dict(n_host=START, n_new=FAKE), INV), ("prefill", dict(n_host=TOO_MANY), INV),
    ("prefill", dict(n_host=START, n_new=FAKE), INV), ("prefill", dict(n_host=START, nb=4), WSP),
    ("prefill", dict(new=None), INV), ("prefill", dict(new=FAKE + 8), INV),
    ("prefill", dict(idt=2), INV), ("prefill", dict(C=0), INV), ("prefill", dict(q=None), INV),
    ("prefill", dict(Hq=12), UNS),
    ("prefill", dict(Hq=10), INV), ("prefill", dict(qdt=2), INV), ("prefill", dict(scale=0.0), INV),
    ("prefill", dict(splits=0), INV), ("prefill", dict(splits=33), INV),
    ("prefill", dict(splits=2, nb=16), WSP)])
def test_arguments_refused(which, kw, rc):
    assert _call(which, **kw) == rc
    assert _lib.lib().skv_last_error()


@pytest.mark.parametrize("covering", [0, 1])
@pytest.mark.parametrize("B,H,top,total,hint", [
    (1, 1, 1, 0, 0), (257, 2, 5000, 70000, 0), (60000, 1, 4000, 0, 0), (256, 1, 300, 300, 0),
    (4, 16, 32000, 0, 0), (64, 8, 8192, 100000, 0), (3, 5, 130, 131, 0), (65535, 1, 1, 0, 0),
    (1, 1, 2**31 - 1, 0, 0), (1, 900, 2**31 - 1, 0, 0), (2, 2, 1000, 0, 100), (2, 2, 1000, 0, 5000)])
def test_decode_plan_covers_every_length(B, H, top, total, hint, covering):
    c, n, wg = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    assert _lib.lib().skv_q_decode_plan(B, 2 * H, H, 128, _lib.MXFP4, 0, 0, top, total, covering,
                                        hint, ctypes.byref(c), ctypes.byref(n),
                                        ctypes.byref(wg)) == 0
    assert c.value > 0 and c.value % 128 == 0 and n.value >= 1
    assert (n.value - 1) * c.value < top <= n.value * c.value
    assert B <= wg.value <= 65535
    if covering or B > 256:
        assert wg.value == B * n.value
    elif total:  # any lengths up to top that sum to total: the most chunks they can have
        rng = np.random.default_rng(B)
        for _ in range(20):
            lens = rng.multinomial(total, rng.dirichlet(np.full(B, 0.3)))
            if lens.max() <= top:
                assert np.maximum(-(-lens // c.value), 1).sum() <= wg.value


def test_decode_plan_refuses():
    c, n, wg = (ctypes.c_int() for _ in range(3))
    L = _lib.lib()
    out = tuple(ctypes.byref(x) for x in (c, n, wg))
    for a in ((0, 2, 1, 64), (65536, 2, 1, 64), (1, 2, 0, 64), (1, 0, 1, 64), (1, 3, 2, 64),
              (1, 2, 1, 0)):
        assert L.skv_q_decode_plan(*a, _lib.MXFP4, 0, 0, 10, 0, 0, 0, *out) == INV
    assert L.skv_q_decode_plan(1, 2, 1, 64, _lib.MXFP4, 0, 0, 0, 0, 0, 0, *out) == INV
    assert L.skv_q_decode_plan(1, 2, 1, 64, _lib.MXFP4, 0, 0, 9, 0, 0, 0, None, *out[1:]) == INV
    assert L.skv_q_decode_workspace_bytes(2, 8, 64, 3) == 2 * 8 * 3 * 68 * 4
    assert L.skv_q_decode_workspace_bytes(0, 8, 64, 3) == 0


def _prefill_plan(B, C, Hq, H, D, lens, n):
    a, b = (np.asarray(0 if x is None else x, np.int32) for x in (lens, n))
    ns = ctypes.c_int(-1)
    rc = _lib.lib().skv_q_prefill_plan(B, C, Hq, H, D, _lib.host_ptr(a),
                                       None if n is None else _lib.host_ptr(b), ctypes.byref(ns))
    return rc, ns.value


def test_prefill_plan():
    rng = np.random.default_rng(3)
    for _ in range(300):
        B, H, G, C = (int(rng.integers(1, m)) for m in (40, 17, 9, 700))
        lens, n = rng.integers(0, 1 << int(rng.integers(1, 28)), B), rng.integers(0, C + 1, B)
        rc, ns = _prefill_plan(B, C, H * G, H, int(rng.choice([32, 64, 96, 128, 256])), lens, n)
        assert rc == 0 and 1 <= ns <= 32
        assert ns == 1 or (ns - 1) * 256 < (lens + n)[n > 0].max()
    # a few rows after long prefixes are split, many after short ones are not,
    # and sequences without a chunk do not count
    assert _prefill_plan(2, 64, 16, 2, 128, [20000, 9000], [64, 5])[1] > 8
    assert _prefill_plan(16, 400, 32, 8, 128, [500] * 16, [399] * 16)[1] == 1
    assert _prefill_plan(2, 8, 8, 8, 64, [2**30, 10], [0, 8])[1] == 1
    assert (_prefill_plan(4, 512, 16, 16, 128, [32256] * 4, None)
            == _prefill_plan(4, 512, 16, 16, 128, [32256] * 4, [512] * 4) == (0, 2))
    assert _prefill_plan(2, 8, 8, 8, 64, [2**30, 10], [0, 0])[1] == 1


def test_prefill_plan_refuses():
    ok = (2, 8, 8, 4, 64)
    for i, bad in ((0, 0), (1, 0), (2, 0), (2, 6), (3, 0), (4, 0), (4, 288)):
        assert _prefill_plan(*ok[:i], bad, *ok[i + 1:], [1, 1], [1, 1])[0] == INV
    for lens, n in (([-1, 0], [1, 1]), ([1, 1], [1, 9]), ([1, 1], [-1, 1])):
        assert _prefill_plan(*ok, lens, n)[0] == INV
    f = _lib.lib().skv_q_prefill_plan
    ns = ctypes.c_int()
    assert f(*ok, None, FAKE, ctypes.byref(ns)) == INV
    assert f(*ok, FAKE, FAKE, None) == INV


def test_read_refuses_bad_starts(monkeypatch):
    """Before any device work; the tensor checks are stubbed out (no GPU here)."""
    from simple_llm_amd.gpu import gpu_kv_cache as gk

    ctx = _ctx()
    cache = gpu.kv_cache_create(ctx, gpu.KVCacheConfig(2, 8, 1, 4, 64, dtype=FP8))
    rows = torch.zeros(2, 3, 4, 64)
    monkeypatch.setattr(gk, "_check_tensor", lambda *a: None)
    seen = []
    monkeypatch.setattr(gk.gpu_kv_quant, "read", lambda c, l, k, v, at: seen.append(at.tolist()))
    for bad in (-1, 2**31, [0, -1], np.array([2**31, 0]), [1, 2, 3], np.zeros((2, 1))):
        with pytest.raises(ValueError, match="start must"):
            gpu.kv_cache_read(ctx, cache, 0, rows, rows, start=bad)
    for good in (None, 5, np.int64(5), [1, 2], np.array([3, 4]), [7]):
        gpu.kv_cache_read(ctx, cache, 0, rows, rows, start=good)
    assert seen == [[0], [5], [5], [1, 2], [3, 4], [7]]
    with pytest.raises(ValueError, match="at least one row"):
        gpu.kv_cache_read(ctx, cache, 0, rows[:, :0], rows[:, :0])


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -0.125])
def test_prefill_refuses_a_scale_that_is_not_positive_and_finite(scale):
    assert _call("prefill", scale=scale) == INV
    assert b"scale" in _lib.lib().skv_last_error()
