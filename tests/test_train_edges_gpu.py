"""The training operators at the ends of their number ranges and sizes, on the MI355X
against oracle/train_oracle.py (float64). u = 2^-24 is half a step of fp32."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import banner
from oracle import train_oracle as to
from test_train_gpu import BF, F32, HYPER, U, dev, g64, half_step, norm_inputs, p_tol, within

pytestmark = pytest.mark.gpu


# ---- cross-entropy: large finite logits --------------------------------------

# A vocabulary for every number of wavefronts a row (1, 4, 8, 16), and two that are read
# twice: of whole vectors, and ending inside one.
VOCABS = [(v, F32) for v in (1000, 5003, 16001, 50257, 70000, 70001)] + [
    (v, BF) for v in (2001, 10007, 30001, 100003, 140000, 140001)]


def loss_bounds(x, t, scale):
    """(bound of dx, of the rows' losses, of the loss), absolute.

    An exponential e^-r: the difference from the maximum is rounded, log2(e) is, and their
    product: 2.3 r u; the instruction 2 u. A logit reaches its row's sum by at most three
    such factors (to its lane's, its wavefront's and the row's maximum, whose r add up): 6 u
    and a product's rounding each, 3 u. The sum: at most 129 additions in a lane, or a row's
    1024th part and a vector and an edge; 6 over a wavefront, 4 over the wavefronts. Then
    1 / count, 1 / sum and two products: 4 u."""
    x = g64(x)
    rows = np.arange(len(x))
    real = (t >= 0) & (t < x.shape[1])
    at = np.where(real, t, 0)
    top = x.max(-1, keepdims=True)
    r = top - x
    with np.errstate(under="ignore"):
        p = np.exp(-r)
    total = p.sum(-1, keepdims=True)
    p /= total
    of_sum = 2.3 * (p * r).sum(-1) + 9 + max(129, x.shape[1] / 1024 + 9) + 10
    inv = scale / max(1, int(real.sum()))
    dx = U * inv * p * (2.3 * r + 2 + of_sum[:, None] + 4)
    dx[rows, at] += U * inv  # p inv - inv: the latter's rounding, and that of the difference
    dx += U * inv * np.abs(p - (np.arange(x.shape[1]) == at[:, None]))
    dx[~real] = 0
    picked = top[:, 0] - x[rows, at]
    row = U * (picked + of_sum + 2 * np.log(total[:, 0]) + (picked + np.log(total[:, 0])))
    row[~real] = 0
    return dx, row, row.sum() / max(1, int(real.sum()))


def masked_rows(rng, vocab, mask):
    """Logits with masked places of one large value, and targets: an allowed part of 300 at
    either end and inside, an unused end, one allowed place, a masked target, a row of
    nothing but the mask, one of nothing but its opposite, and an ignored row."""
    x = 3 * rng.standard_normal((9, vocab))
    n = min(300, vocab // 3)
    mid = vocab // 2 + 5
    x[0, n:] = x[1, :-n] = mask
    x[2, :mid] = x[2, mid + n:] = mask
    x[3, -(vocab // 20):] = mask
    x[4, :] = mask
    x[4, vocab // 3] = 1.5
    x[5, ::2] = mask
    x[6, :] = mask
    x[7, :] = -mask
    t = np.array([n - 1, vocab - n, mid, 7, vocab // 3, 2, vocab - 1, 3, -100], np.int32)
    return x, t


@pytest.mark.parametrize("vocab,dtype", VOCABS)
def test_cross_entropy_of_finite_masks(gpu_ctx, vocab, dtype):
    from simple_llm_amd.gpu import gpu
    rng = np.random.default_rng(vocab)
    most = torch.finfo(dtype).max
    for mask in (-1e9, -1e10, -2e10, -1e30, -0.7 * most, -most):
        banner(f"cross_entropy {vocab} {dtype} mask {mask:.3g}")
        x, t = masked_rows(rng, vocab, mask)
        x, td = dev(x, dtype), dev(t, torch.int32)
        loss, row, dx = torch.empty(1).cuda(), torch.empty(9).cuda(), torch.empty_like(x)
        gpu.cross_entropy_loss(gpu_ctx, x, td, loss, dx, row, grad_scale=0.5)
        wl, wr, wx = to.cross_entropy(g64(x), t, 0.5)
        assert np.isfinite(wx).all() and np.isfinite(wr).all()
        tx, tr, tl = loss_bounds(x, t, 0.5)
        within(dx, wx, tx + half_step(dtype) * (np.abs(wx) + tx), f"mask {mask:.3g} dx")
        within(row, wr, tr, f"mask {mask:.3g} rows")
        within(loss, np.array([wl]), tl + U * abs(wl), f"mask {mask:.3g} loss")
        only, into = torch.empty(1).cuda(), x.clone()
        gpu.cross_entropy_loss(gpu_ctx, x, td, only)
        gpu.cross_entropy_loss(gpu_ctx, into, td, loss, into, grad_scale=0.5)
        assert torch.equal(only, loss) and torch.equal(into, dx)


def test_cross_entropy_of_finite_masks_past_the_caches(gpu_ctx):
    """More than 256 MB of gradients: the rows of a small call, bit by bit."""
    from simple_llm_amd.gpu import gpu
    rng = np.random.default_rng(0)
    x, t = masked_rows(rng, 50304, torch.finfo(F32).min)
    x, t = dev(x[:8]).repeat(256, 1), dev(t[:8], torch.int32).repeat(256)
    dx, part = torch.empty_like(x), torch.empty(8, 50304, device="cuda")
    loss, one = torch.empty(1).cuda(), torch.empty(1).cuda()
    gpu.cross_entropy_loss(gpu_ctx, x, t, loss, dx)
    gpu.cross_entropy_loss(gpu_ctx, x[:8].clone(), t[:8].clone(), one, part, grad_scale=8 / 2048)
    assert part.isfinite().all() and torch.equal(loss, one)
    assert torch.equal(dx, part.repeat(256, 1))


@pytest.mark.parametrize("vocab,dtype", VOCABS)
def test_cross_entropy_bits_do_not_depend_on_addresses(gpu_ctx, vocab, dtype):
    """The same logits at every 16-byte granule of a cache line."""
    from simple_llm_amd.gpu import gpu
    x = torch.randn(9, vocab, device="cuda").to(dtype)
    t = torch.arange(9, device="cuda").int()
    want = None
    for k in range(8):
        banner(f"cross_entropy {vocab} {dtype} {16 * k} bytes on")
        at = 16 * k // x.element_size()
        here = torch.empty(9 * vocab + at, dtype=dtype, device="cuda")[at:].view(9, vocab).copy_(x)
        loss, row, dx = torch.empty(1).cuda(), torch.empty(9).cuda(), torch.empty_like(x)
        gpu.cross_entropy_loss(gpu_ctx, here, t, loss, dx, row)
        gpu.cross_entropy_loss(gpu_ctx, here, t, loss, here)
        got = (loss, row, dx, here.clone())
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- LayerNorm: bad rows, rows that end inside a vector ------------------------

@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_layernorm_of_a_bad_row(gpu_ctx, bad, dtype):
    """One NaN or infinity: the row's output and rstd are NaN, and no other row changes."""
    from simple_llm_amd.gpu import gpu
    for d in (3, 300, 2000, 6000, 16384):
        banner(f"layernorm 9 x {d} {dtype} with {bad}")
        _, x, gamma, beta = norm_inputs(9, d, dtype)
        (y, mean, rstd), clean = ((torch.empty_like(x), torch.empty(9).cuda(), torch.empty(9).cuda())
                                  for _ in range(2))
        gpu.layernorm(gpu_ctx, x, gamma, beta, *clean)
        x[4, d // 2] = bad
        gpu.layernorm(gpu_ctx, x, gamma, beta, y, mean, rstd)
        assert y[4].isnan().all() and rstd[4].isnan()
        keep = torch.arange(9) != 4
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip((y, mean, rstd), clean))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_layernorm_mean_of_a_bad_row(gpu_ctx, dtype):
    """The mean of a row with an infinity is that infinity, of one with a NaN, or with
    infinities of both signs, NaN."""
    from simple_llm_amd.gpu import gpu
    inf, nan = float("inf"), float("nan")
    for d in (3, 300, 2000, 6000):
        _, x, gamma, beta = norm_inputs(4, d, dtype)
        x[0, d - 1], x[1, 0], x[2, d // 2] = inf, -inf, nan
        x[3, 0], x[3, 1] = inf, -inf
        y, mean, rstd = torch.empty_like(x), torch.empty(4).cuda(), torch.empty(4).cuda()
        gpu.layernorm(gpu_ctx, x, gamma, beta, y, mean, rstd)
        np.testing.assert_array_equal(g64(mean), [inf, -inf, nan, nan])
        assert rstd.isnan().all() and y.isnan().all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [2, 7, 30, 257, 1027, 4099])
def test_layernorm_backward_of_constant_rows_far_out(gpu_ctx, d, dtype):
    """Rows of one value whose product with rstd overflows: xh is 0 in every column, so dx =
    rstd (g - mean(g)), and dgamma gets nothing from them; also where rows end inside a
    vector."""
    from simple_llm_amd.gpu import gpu
    banner(f"layernorm_backward of constant rows, {d} {dtype}")
    rng = np.random.default_rng(d)
    x = torch.full((5, d), 2.0 ** 121, dtype=dtype, device="cuda")
    gamma = dev(1 + 0.3 * rng.standard_normal(d))
    dy = dev(rng.standard_normal((5, d)), dtype)
    mean, rstd = torch.full((5,), 2.0 ** 121).cuda(), torch.full((5,), 256.0).cuda()
    dx, dg, db = torch.empty_like(x), torch.empty(d).cuda(), torch.empty(d).cuda()
    gpu.layernorm_backward(gpu_ctx, dy, x, gamma, mean, rstd, dx, dg, db)
    g = g64(dy) * g64(gamma)
    want = 256 * (g - g.mean(-1, keepdims=True))
    # g is rounded; its mean has a path of at most 16 + 10 + 17 additions and 2 more; then two
    # differences and a product
    tol = 256 * U * (3 * np.abs(g) + 47 * np.abs(g).mean(-1, keepdims=True)) + U * 2 * np.abs(want)
    within(dx, want, tol + half_step(dtype) * (np.abs(want) + tol), "dx")
    assert not dg.any()
    # five rows on up to 32 places: at most 1 + 10, 4 + 2 + 16 additions, none of them long
    within(db, g64(dy).sum(0), 33 * U * np.abs(g64(dy)).sum(0), "dbeta")


# ---- AdamW: the smallest moments -----------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_adamw_of_subnormal_moments(gpu_ctx, eps, bits):
    """Gradients whose v is below 2^-126, with an eps that does not hide it."""
    from simple_llm_amd.gpu import gpu
    banner(f"adamw subnormal v, eps {eps} bits {bits}")
    rng = np.random.default_rng(0)
    n = 1152
    g = np.exp(rng.uniform(np.log(1e-21), np.log(1e-16), n)) * rng.choice([-1, 1], n)
    g = g.astype(np.float32)
    pd, gd = dev(rng.standard_normal(n)), dev(g)
    opt = gpu.adamw_create(gpu_ctx, [pd], [gd], bits=bits, seed=5)
    h = {**HYPER, "eps": eps}
    m, v = np.zeros(n, np.float32), np.zeros(n, np.float32)
    for t in (1, 2):
        old = g64(pd)
        gpu.adamw_update(gpu_ctx, opt, **h)
        m, v = to.moments(m, v, g, h["beta1"], h["beta2"])
        assert (v > 0).all() and (t == 2 or (v < 2.0 ** -126).sum() > n // 2)
        want = to.stepped(old, m, v, t, **h)
        within(pd, want, p_tol(old, m.astype(float), v.astype(float), t, h, want), f"step {t}")
        if bits == 32:
            np.testing.assert_array_equal(opt.v.cpu().numpy(), v)
        else:
            m = to.values(opt.m.cpu().numpy(), opt.m_scale.cpu().numpy(), False).astype(np.float32)
            v = to.values(opt.v.cpu().numpy(), opt.v_scale.cpu().numpy(), True).astype(np.float32)


def test_adamw_of_the_least_eps(gpu_ctx):
    """Weights without gradients stay where they are, up to their decay."""
    from simple_llm_amd.gpu import gpu
    p, g = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda")
    opt = gpu.adamw_create(gpu_ctx, [p], [g])
    gpu.adamw_update(gpu_ctx, opt, 2.0 ** -10, eps=2.0 ** -126, weight_decay=0.5)
    assert (p == 1 - 2.0 ** -11).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_resumes(gpu_ctx, bits):
    """A saved state copied into a new one goes on bit by bit; one that was replaced is refused
    before anything is launched."""
    from simple_llm_amd.gpu import gpu
    torch.manual_seed(bits)
    p, g = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")
    opt = gpu.adamw_create(gpu_ctx, [p], [g], bits=bits, seed=11)
    for _ in range(3):
        gpu.adamw_update(gpu_ctx, opt, 1e-2)
    names = ["m", "v", "step"] + (["m_scale", "v_scale"] if bits == 8 else [])
    saved = {n: getattr(opt, n).cpu() for n in names}
    q = p.clone()
    new = gpu.adamw_create(gpu_ctx, [q], [g], bits=bits, seed=opt.seed)
    for n in names:
        getattr(new, n).copy_(saved[n])
    for _ in range(2):
        gpu.adamw_update(gpu_ctx, opt, 1e-2)
        gpu.adamw_update(gpu_ctx, new, 1e-2)
    assert torch.equal(p, q) and all(torch.equal(getattr(opt, n), getattr(new, n)) for n in names)
    before = p.clone()
    for n in names:
        at = getattr(opt, n).data
        getattr(opt, n).data = saved[n].cuda()
        with pytest.raises(ValueError, match="no longer where it was"):
            gpu.adamw_update(gpu_ctx, opt, 1e-2)
        getattr(opt, n).data = at
    assert torch.equal(p, before) and opt.step.item() == 5
    gpu.adamw_update(gpu_ctx, opt, 1e-2)
    assert opt.step.item() == 6 and not torch.equal(p, before)
