"""The training operators on the CPU: the oracle against autograd in 64 bits and
against differences, the 8-bit moments' format, and every refusal, in Python and at
the C entry points (no call here reaches a launch)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import train_oracle as to
from simple_llm_amd import _lib
from simple_llm_amd.gpu import gpu
from simple_llm_amd.gpu.gpu_pass_optimizer import _disjoint
from simple_llm_amd.gpu.gpu_types import GPUConfig, GPUContext, PipelineCache


def _ctx():
    return GPUContext(device=torch.device("cpu"), config=GPUConfig(), batch_state=None,
                      pipeline_cache=PipelineCache())


# ---- the oracle ------------------------------------------------------------

def test_layernorm_gradients():
    rng = np.random.default_rng(0)
    x, dy, res = (rng.standard_normal((7, 20)) for _ in range(3))
    x = x * 3 + 5
    g, b = rng.standard_normal((2, 20))
    xt, gt, bt = (torch.from_numpy(t).requires_grad_() for t in (x, g, b))
    yt = torch.nn.functional.layer_norm(xt, (20,), gt, bt, 1e-5)
    yt.backward(torch.from_numpy(dy))
    y, mean, rstd = to.layernorm(x, g, b)
    np.testing.assert_allclose(y, yt.detach().numpy(), rtol=1e-12, atol=1e-12)
    dx, dg, db = to.layernorm_backward(dy, x, g, mean, rstd, res)
    np.testing.assert_allclose(dx - res, xt.grad.numpy(), rtol=1e-9, atol=1e-12)
    np.testing.assert_allclose(dg, gt.grad.numpy(), rtol=1e-9, atol=1e-12)
    np.testing.assert_allclose(db, bt.grad.numpy(), rtol=1e-12)
    # and against differences: f(x + h e) - f(x - h e), h = 1e-5, error of order h^2
    h = 1e-5
    for i, j in ((0, 0), (3, 11), (6, 19)):
        lo, hi = x.copy(), x.copy()
        lo[i, j] -= h
        hi[i, j] += h
        slope = ((to.layernorm(hi, g, b)[0] - to.layernorm(lo, g, b)[0]) * dy).sum() / (2 * h)
        assert abs(slope - (dx - res)[i, j]) < 1e-8


def test_cross_entropy_gradients():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((9, 33)) * 4
    x[2, 5:9] = -np.inf
    t = rng.integers(0, 33, 9)
    t[2] = 20
    t[[1, 4]] = -100
    t[7] = 33
    xt = torch.from_numpy(x).requires_grad_()
    lt = torch.nn.functional.cross_entropy(xt, torch.from_numpy(np.where(t == 33, -100, t)))
    lt.backward()
    loss, row, dx = to.cross_entropy(x, t, 2.5)
    assert abs(loss - lt.item()) < 1e-13
    assert (row[[1, 4, 7]] == 0).all() and (dx[[1, 4, 7]] == 0).all()
    np.testing.assert_allclose(dx, 2.5 * xt.grad.numpy(), rtol=1e-10, atol=1e-15)


def test_embedding_gradients():
    rng = np.random.default_rng(2)
    w, pos = rng.standard_normal((11, 6)), rng.standard_normal((4, 6))
    ids = np.array([3, 10, 3, -1, 11, 0, 3])
    dy = rng.standard_normal((7, 6))
    out = to.embedding(ids, w, 2.0, pos)
    assert (out[3] == pos[3]).all() and (out[4] == pos[0]).all()
    wt = torch.from_numpy(w).requires_grad_()
    real = (ids >= 0) & (ids < 11)
    got = 2.0 * wt[torch.from_numpy(ids[real])]
    np.testing.assert_allclose(out[real], got.detach().numpy() + pos[np.arange(7)[real] % 4])
    got.backward(torch.from_numpy(dy[real]))
    np.testing.assert_allclose(to.embedding_backward(dy, ids, 11, 2.0), wt.grad.numpy())


def test_adamw_follows_torch():
    rng = np.random.default_rng(3)
    p = rng.standard_normal(50)
    pt = torch.from_numpy(p.copy()).requires_grad_()
    opt = torch.optim.AdamW([pt], lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    m = v = np.zeros(50, np.float32)
    for t in range(1, 6):
        g = rng.standard_normal(50)
        pt.grad = torch.from_numpy(g)
        opt.step()
        m, v = to.moments(m, v, g, 0.9, 0.99)
        p = to.stepped(p, m, v, t, 1e-2, 0.9, 0.99, 1e-8, 0.1)
    # moments of 32 bits: each a few roundings of 2^-24 off
    np.testing.assert_allclose(p, pt.detach().numpy(), atol=1e-2 * 5 * 20 * 2.0 ** -24)


# ---- the 8-bit moments -----------------------------------------------------

def test_moment_grids():
    """m's codes are those of torch's float8_e4m3fn; v's have twice its range."""
    want = torch.arange(127).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(to.grid(False), want)
    v = to.grid(True)
    assert v[0] == 0 and v[1] == 2.0 ** -32 and v[8] == 2.0 ** -29 and v[240] == 1
    assert (np.diff(v) > 0).all() and v[255] == 3.75


@pytest.mark.parametrize("unsigned", [False, True])
def test_moments_are_rounded_without_bias(unsigned):
    """Every value is rounded to a neighbour, and the mean over all random bits is the
    value but for half of the 2^-16 of a step that 16 bits resolve."""
    rng = np.random.default_rng(4)
    x = np.exp(rng.uniform(-30 if unsigned else -14, 0, 128)).astype(np.float32)
    x[:3] = 1.5, 0, 2.0 ** -31 if unsigned else 2.0 ** -16
    x = x if unsigned else x * rng.choice([-1, 1], 128).astype(np.float32)
    step = np.zeros(128)
    total = np.zeros(128)
    n = 1 << 10
    for r in range(0, 1 << 16, 1 << 6):
        code, byte = to.store(x, np.full(128, r + 32), unsigned)
        y = to.values(code, byte, unsigned)
        total += y
        step = np.maximum(step, np.abs(y - x))
    gr = np.append(to.grid(unsigned), np.inf) * (1.0 if unsigned else 2.0 ** -7)
    gap = gr[np.searchsorted(gr, np.abs(x), "right")] - gr[np.searchsorted(gr, np.abs(x), "right") - 1]
    assert (step <= gap).all()
    low = (np.abs(x) > 0) & (np.abs(x) < gr[1]) if unsigned else np.zeros(128, bool)
    assert (np.abs(total / n - x)[~low] <= gap[~low] * 2.0 ** -9).all()


def test_moment_blocks():
    x = np.zeros((7, 128), np.float32)
    x[1, 3] = 1e-30
    x[1, 4] = 1e-44  # above zero: never the code 0
    x[2, 5] = 3e38
    x[3, 6] = np.inf
    x[4, 7] = np.nan
    x[5] = 2.0 ** -100
    x[6, 0] = 1.9999999
    for bits in (0, 0xffff):
        code, byte = to.store(x.reshape(-1), np.full(x.size, bits), True)
        code = code.reshape(x.shape)
        assert byte.tolist() == [37, 37, 253, 255, 255, 37, 127]
        assert (code[0] == 0).all() and code[1, 4] == 1 and code[2, 5] >= 0xf8
        assert (code[3] == 0).all() and (code[5] > 0).all()
        back = to.values(code.reshape(-1), byte, True).reshape(x.shape)
        assert np.isnan(back[3:5]).all() and np.isfinite(back[[0, 1, 2, 5, 6]]).all()
        code, byte = to.store(-x.reshape(-1), np.full(x.size, bits), False)
        code = code.reshape(x.shape)
        assert byte.tolist() == [37, 37, 253, 255, 255, 37, 127]
        assert (code[2, 5] & 127) <= 126 and code[2, 5] >= 128
        assert to.values(code.reshape(-1), byte, False).reshape(x.shape)[6, 0] <= -1.875


def test_hash_is_even():
    """16 low and 16 high bits of a million places: each bit set half the time (within 5
    deviations of 500), neither following the other, another at the next step."""
    h, h2 = to.hashed(7, 100, 1 << 20), to.hashed(7, 101, 1 << 20)
    for b in range(32):
        for word in (h >> b & 1, (h ^ h2) >> b & 1, (h ^ (h >> 16)) >> (b % 16) & 1):
            assert abs(int(word.sum()) - (1 << 19)) < 5 * 512


# ---- refusals --------------------------------------------------------------

def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_python_refusals_name_the_operand():
    c = _ctx()
    bf = torch.bfloat16
    x, g, r, i = t(6, 8), t(8), t(6), t(6, dtype=torch.int32)
    cases = [
        (lambda: gpu.layernorm(c, t(6), g, g, x), "input must be 2-D|input must live"),
        (lambda: gpu.layernorm(c, x.half(), g, g, x), "input must be torch.float32 or"),
        (lambda: gpu.layernorm(c, [1.0], g, g, x), "input must be a GPUBuffer or a tensor"),
        (lambda: gpu.embedding(c, i, x, x), "must live on"),
        (lambda: gpu.embedding_backward(c, x, i, x.to(bf)), "must live on|must be"),
        (lambda: gpu.cross_entropy_loss(c, x.int(), i, t(1)), "logits must be"),
        (lambda: gpu.layernorm_backward(c, x, x.double(), g, r, r, x, g, g), "input must be"),
    ]
    for call, match in cases:
        with pytest.raises(ValueError, match=match):
            call()


def test_adamw_create_refusals():
    c = _ctx()
    p = [t(4, 4)]
    for kw, match in ((dict(bits=16), "bits must be"), (dict(seed=-1), "seed must"),
                      (dict(seed=1 << 32), "seed must"), (dict(decay=[True, False]), "decay must"),
                      (dict(copies=[]), "copies must")):
        with pytest.raises(ValueError, match=match):
            gpu.adamw_create(c, p, p, **kw)
    with pytest.raises(ValueError, match="holds no tensors"):
        gpu.adamw_create(c, [], [])
    with pytest.raises(ValueError, match="grads must"):
        gpu.adamw_create(c, p, [])
    with pytest.raises(ValueError, match=r"params\[0\] must be torch.float32"):
        gpu.adamw_create(c, [t(4, dtype=torch.bfloat16)], p)


def test_disjoint():
    a = t(100)
    _disjoint([(a[:50], "a", True), (a[50:], "b", True), (t(8), "g", False)])
    g = t(64)
    _disjoint([(a, "a", True), (g[:40], "g", False), (g[10:], "h", False)])  # read only
    for x, y, w in ((a[:51], a[50:], False), (a[50:], a[:51], False), (a, a[3:9], False)):
        with pytest.raises(ValueError, match="overlaps"):
            _disjoint([(x, "x", True), (y, "y", w), (g, "g", False)])
    with pytest.raises(ValueError, match="overlaps"):  # past a longer read-only one
        _disjoint([(a[0:90], "x", False), (a[5:9], "y", False), (a[60:], "z", True)])


FAKE = 4096  # never dereferenced: each call below fails validation first


def test_c_entry_points_refuse():
    L = _lib.lib()
    inv, uns, wsp = _lib.SKV_E_INVALID, _lib.SKV_E_UNSUPPORTED, _lib.SKV_E_WORKSPACE

    def fwd(y=FAKE, x=FAKE, g=FAKE, M=4, d=8, dt=0):
        return L.skv_layernorm_fwd(y, None, None, x, g, FAKE, M, d, 1e-5, dt, None)

    assert fwd(y=None) == inv and fwd(M=0) == inv and fwd(d=-1) == inv and fwd(dt=2) == inv
    assert fwd(x=FAKE + 4) == inv and b"aligned" in L.skv_last_error()
    assert fwd(d=16385) == uns and b"16384" in L.skv_last_error()

    need = L.skv_layernorm_bwd_workspace_bytes(1000, 768)
    assert need >= 2 * 768 * 4 and L.skv_layernorm_bwd_workspace_bytes(0, 768) == 0

    def bwd(dx=FAKE, ws=FAKE, nb=need, res=None, M=1000, d=768):
        return L.skv_layernorm_bwd(dx, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, res, M, d, 0, ws, nb,
                                   0, None)

    assert bwd(dx=None) == inv and bwd(ws=None) == inv and bwd(nb=need - 1) == wsp
    assert bwd(res=FAKE + 8) == inv and bwd(d=20000) == uns

    def emb(out=FAKE, T=4, n_pos=0, pos=None, dt=0):
        return L.skv_embedding_fwd(out, FAKE, FAKE, pos, T, 10, 8, n_pos, 1.0, dt, 0, None)

    assert emb(out=None) == inv and emb(T=0) == inv and emb(pos=FAKE) == inv and emb(dt=3) == inv
    assert emb(out=FAKE + 2) == inv
    need = L.skv_embedding_bwd_workspace_bytes(100, 1000, 64)

    def embb(grad=FAKE, T=100, V=1000, nb=need, dt=0):
        return L.skv_embedding_bwd(grad, FAKE, FAKE, T, V, 64, 1.0, 0, FAKE, nb, dt, None)

    assert embb(grad=None) == inv and embb(T=-1) == inv and embb(dt=9) == inv
    assert embb(nb=need - 1) == wsp and embb(V=(1 << 30) + 1) == uns

    need = L.skv_cross_entropy_workspace_bytes(10)

    def ce(loss=FAKE, x=FAKE, M=10, V=20, nb=need, dt=1):
        return L.skv_cross_entropy(loss, None, None, x, FAKE, M, V, 1.0, FAKE, nb, dt, None)

    assert ce(loss=None) == inv and ce(V=0) == inv and ce(dt=2) == inv and ce(x=FAKE + 2) == inv
    assert ce(nb=need - 1) == wsp

    def adamw(tensors=FAKE, n=3, ms=None, bits=32, dt=0, b1=0.9, b2=0.999, m=FAKE):
        return L.skv_adamw(tensors, FAKE, n, m, FAKE, ms, ms, FAKE, bits, dt, 1e-3, None, b1, b2, 1e-8,
                           0.1, 1.0, None, 0, None)

    assert adamw(tensors=None) == inv and adamw(n=0) == inv and adamw(bits=16) == inv
    assert adamw(bits=8) == inv  # no scales
    assert adamw(b1=1.0) == inv and adamw(b2=-0.1) == inv and adamw(dt=2) == inv
    assert adamw(m=FAKE + 4) == inv and adamw(b1=float("nan")) == inv
    assert L.skv_adamw_read(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 100, 0, None) == inv
    assert L.skv_adamw_read(FAKE, None, FAKE, FAKE, FAKE, FAKE, 128, 0, None) == inv
    assert L.skv_adamw_read(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 41, 0, None) == uns


def test_c_entry_points_refuse_too_many_rows():
    """More than a launch or a kernel's 32-bit loops can have, on either side of the limits
    that are refused before memory is looked at."""
    L = _lib.lib()
    uns = _lib.SKV_E_UNSUPPORTED
    big = (1 << 31) - 1

    def fwd(M, d):
        return L.skv_layernorm_fwd(FAKE, None, None, FAKE, FAKE, FAKE, M, d, 1e-5, 1, None)

    # lanes of a row: 16, 32, 64, 256 and 1024
    for d, lanes in ((1, 16), (256, 16), (257, 32), (512, 32), (513, 64), (2048, 64), (2049, 256),
                     (8192, 256), (8193, 1024)):
        most = ((1 << 32) - 1) // lanes
        for M in (min(most + 1, big), big):
            assert fwd(M, d) == uns, (M, d)
        assert fwd(most // 1024 * 1024, d) == _lib.SKV_E_INVALID  # gets as far as the overlaps
    assert L.skv_layernorm_bwd_workspace_bytes(big, 8) == 0
    assert L.skv_layernorm_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, big, 8, 0, FAKE,
                               1 << 40, 0, None) == uns
    for T, d in (((1 << 26) + 1, 8), (big, 8), (4, (1 << 22) + 1)):
        assert L.skv_embedding_fwd(FAKE, FAKE, FAKE, None, T, 10, d, 0, 1.0, 0, 0, None) == uns
    for T, V, d in ((big, 10, 8), (1 << 30, 10, 257), (4, big, 8), (4, 10, big), (1 << 20, 10, 1 << 20)):
        assert L.skv_embedding_bwd_workspace_bytes(T, V, d) > 0
        assert L.skv_embedding_bwd(FAKE, FAKE, FAKE, T, V, d, 1.0, 0, FAKE, 1 << 62, 0, None) == uns
    for M, V in ((big, 1), ((1 << 26) + 1, 2048), (1 << 24, 2049), (1 << 23, 16385), (1 << 22, 40000)):
        assert L.skv_cross_entropy(FAKE, None, FAKE, FAKE, FAKE, M, V, 1.0, FAKE, 1 << 62, 1, None) == uns
    assert L.skv_adamw(FAKE, FAKE, big, FAKE, FAKE, None, None, FAKE, 32, 0, 1e-3, None, 0.9, 0.99,
                       1e-8, 0.1, 1.0, None, 0, None) == uns
