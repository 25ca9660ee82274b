"""The training operators on the MI355X against oracle/train_oracle.py (float64).

Tolerances are counted in roundings: u = 2^-24 is half a step of fp32, 2^-8 of bf16,
each relative to the value rounded. A sum of fp32 terms over a path of k additions is
off by at most k u times the sum of magnitudes; the paths' lengths follow from the
kernels' lanes (at most 16 columns of a row a lane, at most 128 logits) and trees.
Moments of AdamW are equal bit by bit.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import banner
from oracle import train_oracle as to

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def g64(t):
    return t.detach().double().cpu().numpy()


def dev(a, dtype=F32):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().to(dtype)


def half_step(dtype):
    """Of an output's rounding, relative."""
    return 2.0 ** -8 if dtype == BF else 0.0


def within(got, want, tol, what):
    got, want = g64(got) if isinstance(got, torch.Tensor) else got, np.asarray(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    ok = np.isfinite(want)
    np.testing.assert_array_equal(got[~ok], want[~ok], err_msg=what)
    off = np.abs(got[ok] - want[ok]) / np.maximum(np.broadcast_to(tol, want.shape)[ok], 1e-300)
    worst = float(off.max()) if off.size else 0.0
    print(f"{what}: {worst:.3f} of the bound")
    assert worst <= 1, what


def ids_of(rng, n, vocab, padded=True):
    p = 1 / (np.arange(vocab) + 2.7)
    ids = rng.permutation(vocab)[rng.choice(vocab, n, p=p / p.sum())].astype(np.int32)
    if padded and n > 3:
        ids[-(n // 4):] = -1
        ids[0] = vocab
    return ids


# ---- LayerNorm -------------------------------------------------------------

NORM = [(1, 1), (1, 8), (3, 2), (5, 7), (4, 64), (130, 390), (33, 513), (257, 768), (9, 1000),
        (64, 1024), (17, 1025), (6, 1536), (70, 2048), (5, 4095), (3, 4096), (7, 4098), (2, 5000),
        (600, 8192), (3, 16383), (2, 16384), (2049, 256)]
# Rows on 16, 32 and 64 lanes, and on both sides of where their number or width changes that.
MANY = [(5000, 96), (8191, 129), (8193, 200), (8192, 256), (4095, 257), (4097, 300), (4096, 511),
        (4100, 512), (4100, 513), (9000, 7), (2047, 1500), (2048, 1025), (2050, 1500), (2049, 2047),
        (2048, 2048), (511, 5000), (512, 5003), (513, 8192), (2047, 1280), (2048, 1280), (2060, 1279),
        (2048, 1281)]


def norm_inputs(rows, d, dtype, offset=0.5):
    rng = np.random.default_rng(rows * 31 + d)
    x = dev(rng.standard_normal((rows, d)) * np.exp(0.5 * rng.standard_normal(d))
            + offset * rng.standard_normal(d), dtype)
    gamma, beta = dev(1 + 0.3 * rng.standard_normal(d)), dev(rng.standard_normal(d))
    return rng, x, gamma, beta


def check_norm(x, gamma, beta, y, mean, rstd, what):
    want, mu, rs = to.layernorm(g64(x), g64(gamma), g64(beta))
    sd = 1 / rs
    # the mean: rounded once, after a correction whose path is at most 16 + 10 + 4 (32 + 6 + 2 in
    # wide bf16 rows, held to the same: their roundings do not all add up)
    within(mean, mu, U * (np.abs(mu) + 30 * sd), f"{what} mean")
    # the variance's path is as long, its terms have two roundings each, then a quotient and a
    # root: 36 u of the variance and half of that of rstd; 3 more
    within(rstd, rs, 22 * U * rs, f"{what} rstd")
    xh = (g64(x) - mu[:, None]) * rs[:, None]
    tol = U * (np.abs(g64(gamma)) * (26 * np.abs(xh) + 31) + np.abs(g64(beta)) + np.abs(want))
    within(y, want, tol + half_step(x.dtype) * (np.abs(want) + tol), f"{what} y")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,d", NORM + MANY)
def test_layernorm(gpu_ctx, rows, d, dtype):
    from simple_llm_amd.gpu import gpu
    banner(f"layernorm {rows} x {d} {dtype}")
    _, x, gamma, beta = norm_inputs(rows, d, dtype)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows).cuda(), torch.empty(rows).cuda()
    gpu.layernorm(gpu_ctx, x, gamma, beta, y, mean, rstd)
    check_norm(x, gamma, beta, y, mean, rstd, "layernorm")
    again = x.clone()  # in place, statistics not asked for
    gpu.layernorm(gpu_ctx, again, gamma, beta, again)
    assert torch.equal(again, y)


def test_layernorm_far_from_zero(gpu_ctx):
    """Means of thousands of deviations: what a mean rounded to fp32 would lose comes back
    through the deviations' own mean; and constant rows."""
    from simple_llm_amd.gpu import gpu
    rng, x, gamma, beta = norm_inputs(40, 1000, F32)
    x += 3e4
    x[7] = 123.456
    y, mean, rstd = torch.empty_like(x), torch.empty(40).cuda(), torch.empty(40).cuda()
    gpu.layernorm(gpu_ctx, x, gamma, beta, y, mean, rstd)
    keep = np.arange(40) != 7
    check_norm(x[keep], gamma, beta, y[keep], mean[keep], rstd[keep], "far")
    # a constant row: its deviations are at most the mean's rounding, u |mean|, and rstd
    # 1 / sqrt(1e-5), twice that after the correction
    dv = 2 * U * 123.456 / np.sqrt(1e-5)
    within(y[7], g64(beta), np.abs(g64(gamma)) * dv + U * np.abs(g64(beta)), "constant")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_layernorm_rows_do_not_mix(gpu_ctx, bad):
    from simple_llm_amd.gpu import gpu
    for d in (300, 2000, 6000):
        _, x, gamma, beta = norm_inputs(9, d, F32)
        y, clean = torch.empty_like(x), torch.empty_like(x)
        gpu.layernorm(gpu_ctx, x, gamma, beta, clean)
        x[4, d // 2] = bad
        gpu.layernorm(gpu_ctx, x, gamma, beta, y)
        assert y[4].isnan().all()
        keep = torch.arange(9) != 4
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,d", NORM + MANY)
@pytest.mark.parametrize("residual,accumulate", [(False, True), (True, False)])
def test_layernorm_backward(gpu_ctx, rows, d, dtype, residual, accumulate):
    from simple_llm_amd.gpu import gpu
    banner(f"layernorm_backward {rows} x {d} {dtype} residual={residual}")
    rng, x, gamma, _ = norm_inputs(rows, d, dtype)
    dy = dev(rng.standard_normal((rows, d)), dtype)
    res = dev(rng.standard_normal((rows, d)), dtype) if residual else None
    _, mu, rs = to.layernorm(g64(x), g64(gamma), 0.0)
    mean, rstd = dev(mu), dev(rs)
    before = rng.standard_normal((2, d))
    dx, (dg, db) = torch.empty_like(x), dev(before).unbind(0)
    if d % 4:
        dg, db = dg.clone(), db.clone()
    old = (g64(dg), g64(db)) if accumulate else (0.0, 0.0)
    gpu.layernorm_backward(gpu_ctx, dy, x, gamma, mean, rstd, dx, dg, db, res, accumulate)
    want, wg, wb = to.layernorm_backward(g64(dy), g64(x), g64(gamma), g64(mean), g64(rstd),
                                         None if res is None else g64(res))
    mu, rs = g64(mean)[:, None], g64(rstd)[:, None]
    xh = np.abs((g64(x) - mu) * rs)
    g = np.abs(g64(dy) * g64(gamma))
    # xh: two roundings; g: one; the means: a path of at most 16 + 10 + 17 and 2, their terms 3;
    # then the differences and products: 6
    tol = U * rs * (8 * g + 50 * g.mean(-1, keepdims=True)
                    + 52 * xh * (g * xh).mean(-1, keepdims=True)) + 2 * U * np.abs(want)
    within(dx, want, tol + half_step(dtype) * (np.abs(want) + tol), "dx")
    # a lane's rows one after the other (of 4 x up to 512 wavefronts or 512 workgroups), four
    # wavefronts, then up to 8 + 6; the terms have 3 roundings
    path = -(-rows // (2048 if d <= 1024 else 512)) + 4 + 8 + 6 + 3
    s = np.abs(g64(dy))
    within(dg, wg + old[0], U * (path * (s * xh).sum(0) + 2 * np.abs(wg + old[0])), "dgamma")
    within(db, wb + old[1], U * (path * s.sum(0) + 2 * np.abs(wb + old[1])), "dbeta")
    # the same bits again, and in place of each of its inputs
    for into in (dy.clone(), x.clone()) + (() if res is None else (res.clone(),)):
        dg2, db2 = (dev(b) for b in before) if accumulate else (torch.empty_like(dg) for _ in "ab")
        which = 0 if torch.equal(into, dy) else 1 if torch.equal(into, x) else 2
        gpu.layernorm_backward(gpu_ctx, into if which == 0 else dy, into if which == 1 else x, gamma,
                               mean, rstd, into, dg2, db2, into if which == 2 else res, accumulate)
        assert torch.equal(into, dx) and torch.equal(dg2, dg) and torch.equal(db2, db)


def test_layernorm_gradient_by_differences(gpu_ctx):
    """f(x + h e) - f(x - h e) of the operator's own forward, f = sum of y * dy in 64 bits."""
    from simple_llm_amd.gpu import gpu
    rng, x, gamma, beta = norm_inputs(5, 40, F32)
    dy = dev(rng.standard_normal((5, 40)))
    y, mean, rstd = torch.empty_like(x), torch.empty(5).cuda(), torch.empty(5).cuda()
    gpu.layernorm(gpu_ctx, x, gamma, beta, y, mean, rstd)
    dx, dg, db = torch.empty_like(x), torch.empty(40).cuda(), torch.empty(40).cuda()
    gpu.layernorm_backward(gpu_ctx, dy, x, gamma, mean, rstd, dx, dg, db)

    def f():
        gpu.layernorm(gpu_ctx, x, gamma, beta, y)
        return float((y.double() * dy.double()).sum())

    h = 2.0 ** -6
    for t, grad, at in ((x, dx, (0, 3)), (x, dx, (4, 39)), (gamma, dg, (7,)), (beta, db, (11,))):
        old = float(t[at])
        t[at] = old + h
        hi = f()
        t[at] = old - h
        lo = f()
        t[at] = old
        # h^2 / 6 of a third derivative of order 10 / sd^3, sd >= 1/2; and two sums of 200 values
        # with 60 u each over 2 h
        assert abs((hi - lo) / (2 * h) - float(grad[at])) < h * h / 6 * 80 + 200 * 60 * U * 8 / h


# ---- embedding -------------------------------------------------------------

EMBED = [(1, 1, 1), (1, 5, 64), (7, 3, 2), (33, 100, 50), (64, 256, 256), (100, 50304, 768),
         (2331, 256, 390), (500, 17, 513), (4097, 40000, 96), (20000, 300, 64), (1000, 1, 100),
         (31, 200000, 8), (6000, 5000, 1024)]


@pytest.mark.parametrize("table_dt,out_dt", [(F32, F32), (BF, BF), (F32, BF), (BF, F32)])
@pytest.mark.parametrize("n,vocab,d", EMBED)
def test_embedding(gpu_ctx, n, vocab, d, table_dt, out_dt):
    from simple_llm_amd.gpu import gpu
    banner(f"embedding {n} of {vocab} x {d} {table_dt} {out_dt}")
    rng = np.random.default_rng(n + vocab + d)
    ids = ids_of(rng, n, vocab)
    table = dev(rng.standard_normal((vocab, d)), table_dt)
    pos = dev(rng.standard_normal((7, d)))
    for scale, p in ((1.0, None), (2.5, pos)):
        out = torch.full((n, d), float("nan"), dtype=out_dt, device="cuda")
        gpu.embedding(gpu_ctx, dev(ids, torch.int32), table, out, scale, p)
        want = to.embedding(ids, g64(table), scale, None if p is None else g64(p))
        tol = U * (np.abs(scale * to.embedding(ids, g64(table))) + np.abs(want))
        within(out, want, tol + half_step(out_dt) * (np.abs(want) + tol), "embedding")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,vocab,d", EMBED)
def test_embedding_backward(gpu_ctx, n, vocab, d, dtype):
    from simple_llm_amd.gpu import gpu
    banner(f"embedding_backward {n} of {vocab} x {d} {dtype}")
    rng = np.random.default_rng(n * 3 + vocab + d)
    ids = ids_of(rng, n, vocab)
    dy = dev(rng.standard_normal((n, d)), dtype)
    before = rng.standard_normal((vocab, d))
    want = to.embedding_backward(g64(dy), ids, vocab, 3.0)
    size = to.embedding_backward(np.abs(g64(dy)), ids, vocab, 3.0)
    count = np.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=vocab)[:, None]
    # a range's tokens one after the other, the ranges' parts over 8 wavefronts, the scale
    path = np.minimum(count, 32) + -(-count // 256) + 8 + 3
    for accumulate in (False, True):
        grad = dev(before)
        was = g64(grad)
        gpu.embedding_backward(gpu_ctx, dy, dev(ids, torch.int32), grad, 3.0, accumulate)
        w = want + (was if accumulate else 0)
        within(grad, w, U * (path * size + 2 * np.abs(w) * (count > 0)), f"accumulate={accumulate}")
        again = dev(before)
        gpu.embedding_backward(gpu_ctx, dy, dev(ids, torch.int32), again, 3.0, accumulate)
        assert torch.equal(again, grad)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 1023, 1024, 1025, 40000])
def test_embedding_backward_of_one_token(gpu_ctx, n):
    """All tokens the same, all padding, and all different: every way a row can lie in the
    sorted order's ranges."""
    from simple_llm_amd.gpu import gpu
    dy = torch.ones(n, 12, device="cuda")
    for vocab, v in ((1, 0), (3, 1), (70000, 69999)):
        grad = torch.full((vocab, 12), 7.0, device="cuda")
        gpu.embedding_backward(gpu_ctx, dy, torch.full((n,), v, dtype=torch.int32, device="cuda"), grad)
        want = torch.zeros(vocab, 12, device="cuda")
        want[v] = n
        assert torch.equal(grad, want)
        gpu.embedding_backward(gpu_ctx, dy, torch.full((n,), -1, dtype=torch.int32, device="cuda"), grad,
                               accumulate=True)
        assert torch.equal(grad, want)
        gpu.embedding_backward(gpu_ctx, dy, torch.full((n,), vocab, dtype=torch.int32, device="cuda"),
                               grad)
        assert not grad.any()
    ids = torch.randperm(n, device="cuda").int()
    dy = torch.randn(n, 12, device="cuda")
    grad = torch.empty(n, 12, device="cuda")
    gpu.embedding_backward(gpu_ctx, dy, ids, grad)
    assert torch.equal(grad[ids.long()], dy)


@pytest.mark.parametrize("n,vocab,often", [(65536, 256, 0.9), (65536, 50000, 0.3), (100003, 700, 0.5),
                                           (1048576, 3, 0.2), (1200007, 9000, 0.1)])
def test_embedding_backward_of_many_tokens(gpu_ctx, n, vocab, often):
    """Runs whose lists overflow, some only after others did not, and runs past 16-bit places.
    Small whole numbers: every sum is exact in any order below 2^24."""
    from simple_llm_amd.gpu import gpu
    rng = np.random.default_rng(n)
    ids = ids_of(rng, n, vocab)
    ids[rng.random(n) < often * np.arange(n) / n] = vocab // 2
    dy = rng.integers(-4, 5, (n, 3)).astype(np.float64)
    grad = torch.full((vocab, 3), 7.0, device="cuda")
    gpu.embedding_backward(gpu_ctx, dev(dy), dev(ids, torch.int32), grad)
    assert np.array_equal(g64(grad), to.embedding_backward(dy, ids, vocab, 1.0))


def test_embedding_backward_keeps_a_bad_row_to_itself(gpu_ctx):
    from simple_llm_amd.gpu import gpu
    rng = np.random.default_rng(5)
    ids = ids_of(rng, 3000, 50, False)
    dy = dev(rng.standard_normal((3000, 20)))
    clean, grad = torch.empty(50, 20).cuda(), torch.empty(50, 20).cuda()
    gpu.embedding_backward(gpu_ctx, dy, dev(ids, torch.int32), clean)
    dy[1234, 3] = float("nan")
    gpu.embedding_backward(gpu_ctx, dy, dev(ids, torch.int32), grad)
    clean[int(ids[1234]), 3] = float("nan")
    assert torch.equal(grad.nan_to_num(9e9), clean.nan_to_num(9e9))


# ---- cross-entropy ---------------------------------------------------------

LOSS = [(1, 1), (1, 2), (3, 7), (5, 15), (8, 64), (255, 257), (33, 256), (9, 1000), (7, 1025),
        (40, 4096), (5, 4099), (6, 8193), (3, 16389), (17, 32768), (20, 50257), (9, 50304), (3, 65536),
        (4, 65537), (2, 130001), (3, 200000)]


def check_loss(x, t, loss, row, dx, scale, what):
    wl, wr, wx = to.cross_entropy(g64(x), t, scale)
    x = g64(x)
    rows = np.arange(len(x))
    real = (t >= 0) & (t < x.shape[1])
    with np.errstate(all="ignore"):
        top = x.max(-1)
        r = np.where(np.isfinite(x), top[:, None] - x, 0.0)
        p = np.where(x == -np.inf, 0.0, np.exp(-r))
        mean_r = np.where(np.isfinite(top), (p * r).sum(-1) / p.sum(-1), 0)
    # an exponential: its argument's rounding, r log2(e) ln 2 u, the constant's, r u / 2, and the
    # instruction's ulp, 2 u; their sum: a path of at most 128 + 10 + 16 (streamed rows: 200000 /
    # 1024 + 26), weighted with the probabilities
    path = 128 + 26 + x.shape[1] / 1024 + 4
    rel = U * (1.6 * r + 1.6 * mean_r[:, None] + path)
    count = max(1, int(real.sum()))
    with np.errstate(all="ignore"):
        tol = np.where(real[:, None], rel * np.abs(np.where(np.isnan(wx), 1, wx)), 0)
    tol[rows[real], t[real]] += rel[rows[real], t[real]] * abs(scale) / count  # p - 1
    tol = tol + U * 3 * np.abs(wx)
    picked = x[rows, np.where(real, t, 0)]
    with np.errstate(all="ignore"):
        row_tol = np.where(real, U * (np.abs(top - picked) + 2 * np.abs(wr) + 1.6 * mean_r + path
                                      + np.abs(np.log(p.sum(-1))) * 3), 0)
    if dx is not None:
        within(dx, wx, tol + half_step(dx.dtype) * (np.abs(wx) + tol) + 1e-40, f"{what} dx")
    if row is not None:
        within(row, wr, row_tol, f"{what} rows")
    within(loss, np.array([wl]), np.nansum(row_tol) / count + U * abs(wl) * 2, f"{what} loss")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,vocab", LOSS)
def test_cross_entropy(gpu_ctx, rows, vocab, dtype):
    from simple_llm_amd.gpu import gpu
    banner(f"cross_entropy {rows} x {vocab} {dtype}")
    rng = np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)) * 3
    if vocab > 40:
        x[:, -vocab // 20:] = -np.inf  # an unused end
    x = dev(x, dtype)
    t = rng.integers(0, max(1, vocab - vocab // 20 - 1), rows).astype(np.int32)
    if rows > 2:
        t[rng.random(rows) < 0.2] = -100
        t[0], t[1], t[2] = 0, vocab - vocab // 20 - 2 if vocab > 40 else vocab - 1, vocab
    loss, row, dx = torch.empty(1).cuda(), torch.empty(rows).cuda(), torch.full_like(x, float("nan"))
    gpu.cross_entropy_loss(gpu_ctx, x, dev(t, torch.int32), loss, dx, row, grad_scale=0.5)
    check_loss(x, t, loss, row, dx, 0.5, "cross_entropy")
    only = torch.empty(1).cuda()  # without a gradient, and into the logits themselves
    gpu.cross_entropy_loss(gpu_ctx, x, dev(t, torch.int32), only)
    into = x.clone()
    again = torch.empty(1).cuda()
    gpu.cross_entropy_loss(gpu_ctx, into, dev(t, torch.int32), again, into, grad_scale=0.5)
    assert torch.equal(only, loss) and torch.equal(again, loss) and torch.equal(into, dx)


@pytest.mark.parametrize("vocab", [50, 3000, 50257, 70001])
def test_cross_entropy_hard_rows(gpu_ctx, vocab):
    """Logits of thousands, a target of -inf, rows of NaN, +inf and -inf only, an ignored row
    of NaN, and a batch in which no row counts."""
    from simple_llm_amd.gpu import gpu
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((8, vocab)).astype(np.float32)
    x[0] += 5000
    x[1, 3:] = -np.inf
    x[2, 9] = -np.inf
    x[3, vocab - 1] = np.nan
    x[4, 11] = np.inf
    x[5] = -np.inf
    x[6, 2] = np.nan
    x[7] *= 1e4
    t = np.array([1, 2, 9, 0, 5, 1, -1, int(x[7].argmax())], np.int32)
    for dtype in (F32, BF):
        xd = dev(x, dtype)
        loss, row, dx = torch.empty(1).cuda(), torch.empty(8).cuda(), torch.empty_like(xd)
        gpu.cross_entropy_loss(gpu_ctx, xd, dev(t, torch.int32), loss, dx, row)
        check_loss(xd, t, loss, row, dx, 1.0, f"hard {vocab}")
        gpu.cross_entropy_loss(gpu_ctx, xd, dev(-t - 1, torch.int32), loss, dx, row)
        t0 = -t - 1  # row 6 counts now, with target 0
        check_loss(xd, t0, loss, row, dx, 1.0, f"hard {vocab} others")
        gpu.cross_entropy_loss(gpu_ctx, xd, dev(np.full(8, -1), torch.int32), loss, dx, row)
        assert loss.item() == 0 and not dx.any() and not row.any()


@pytest.mark.parametrize("rows,vocab,dtype", [(4096, 50257, BF), (2048, 50304, F32), (65536, 4099, BF),
                                              (1 << 20, 100, F32), (1 << 17, 1001, BF),
                                              (16384, 9000, BF), (1024, 200000, BF), (512, 200001, F32)])
def test_cross_entropy_past_the_caches(gpu_ctx, rows, vocab, dtype):
    """Gradients of more than 256 MB have loads and stores of their own: 64 rows of them equal a
    call of those rows, bit by bit (row counts and scales are powers of two, and 64 rows on a
    row begins at the same place of a cache line, which decides the order of its sum)."""
    from simple_llm_amd.gpu import gpu
    banner(f"cross_entropy past the caches {rows} x {vocab} {dtype}")
    x = torch.empty(rows, vocab, dtype=dtype, device="cuda").normal_()
    t = torch.randint(0, vocab, (rows,), device="cuda").int()
    dx, loss, row = torch.empty_like(x), torch.empty(1).cuda(), torch.empty(rows).cuda()
    gpu.cross_entropy_loss(gpu_ctx, x, t, loss, dx, row)
    part = torch.empty(64, vocab, dtype=dtype, device="cuda")
    few, one = torch.empty(64).cuda(), torch.empty(1).cuda()
    for i in (0, rows // 2, rows - 64):
        gpu.cross_entropy_loss(gpu_ctx, x[i:i + 64].clone(), t[i:i + 64].clone(), one, part, few,
                               grad_scale=64 / rows)
        assert torch.equal(dx[i:i + 64], part) and torch.equal(row[i:i + 64], few)
    within(loss, row.double().mean().cpu().numpy()[None], 2 * U * abs(loss.item()), "loss")
    t[::3] = -1  # rows that are ignored, and in place
    want = torch.empty_like(x)
    gpu.cross_entropy_loss(gpu_ctx, x, t, loss, want)
    gpu.cross_entropy_loss(gpu_ctx, x, t, loss, x)
    assert torch.equal(x, want) and not x[::3].any()


# ---- AdamW -----------------------------------------------------------------

SIZES = [(3,), (128,), (127, 5), (1,), (2048,), (64, 100), (4096,), (4097,), (129,), (2, 8191)]
HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.98, eps=1e-8, weight_decay=0.1)


def p_tol(p, m, v, t, h, want):
    """The weight: its decay factor, product and difference, 3 u; the step: the coefficient's
    expm1 and quotient (its argument rounded once), the root's, both ulps, 16 u."""
    step = h["lr"] / (1 - h["beta1"] ** t) * np.abs(m) / (
        np.sqrt(v / (1 - h["beta2"] ** t)) + h["eps"])
    return U * (3 * np.abs(p) + np.abs(want) + 16 * step)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grads", [F32, BF])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw(gpu_ctx, bits, grads, offset):
    """Steps of tensors of every size, moments bit by bit; offset: tensors that begin at no
    multiple of 16 bytes."""
    from simple_llm_amd.gpu import gpu
    banner(f"adamw bits={bits} grads={grads} offset={offset}")
    rng = np.random.default_rng(bits + offset)

    def tensors(dtype, scale=1.0):
        out = []
        for s in SIZES:
            n = int(np.prod(s))
            flat = torch.zeros(n + offset, dtype=dtype, device="cuda")
            flat[offset:] = dev(scale * rng.standard_normal(n) * np.exp(2 * rng.standard_normal(n)),
                                dtype)
            out.append(flat[offset:].view(s))
        return out

    ps, gs, cs = tensors(F32), tensors(grads, 1e-2), tensors(BF)
    decay = [i % 2 == 0 for i in range(len(SIZES))]
    opt = gpu.adamw_create(gpu_ctx, ps, gs, bits=bits, copies=cs, decay=decay, seed=12345)
    n = opt.m.numel()
    assert opt.offsets[0] == 0 and all(o % 128 == 0 for o in opt.offsets)
    m, v = np.zeros(n, np.float32), np.zeros(n, np.float32)
    place = np.concatenate([o + np.arange(p.numel()) for o, p in zip(opt.offsets, ps)])
    for t in range(1, 4):
        for g in gs:
            g.mul_(0.5).add_(torch.randn_like(g) * 1e-3)
        old = np.concatenate([g64(p).ravel() for p in ps])
        g = np.zeros(n, np.float32)
        g[place] = np.concatenate([g64(x).ravel() for x in gs])
        g = g * np.float32(0.25)
        gpu.adamw_update(gpu_ctx, opt, grad_scale=0.25, **HYPER)
        m, v = to.moments(m, v, g, HYPER["beta1"], HYPER["beta2"])
        dec = np.concatenate([np.full(p.numel(), d) for p, d in zip(ps, decay)])
        h = dict(HYPER)
        want = np.where(dec, to.stepped(old, m[place], v[place], t, **h),
                        to.stepped(old, m[place], v[place], t, **{**h, "weight_decay": 0}))
        got = np.concatenate([g64(p).ravel() for p in ps])
        within(got, want, p_tol(old, m[place].astype(float), v[place].astype(float), t, h, want),
               f"step {t}")
        for p, c in zip(ps, cs):
            assert torch.equal(c, p.bfloat16())
        assert opt.step.item() == t and opt._count[1].item() == 0
        if bits == 32:
            np.testing.assert_array_equal(opt.m.cpu().numpy(), m)
            np.testing.assert_array_equal(opt.v.cpu().numpy(), v)
        else:
            r = to.hashed(12345, t, n)
            for x, name, shift, uns in ((m, "m", 0, False), (v, "v", 16, True)):
                code, byte = to.store(x, (r >> shift) & 0xffff, uns)
                np.testing.assert_array_equal(getattr(opt, name).cpu().numpy(), code)
                np.testing.assert_array_equal(getattr(opt, name + "_scale").cpu().numpy(), byte)
            for dt in (F32, BF):
                mo, vo = (torch.full((n,), 9.0, dtype=dt, device="cuda") for _ in range(2))
                gpu.adamw_read(gpu_ctx, opt, mo, vo)
                m = to.values(opt.m.cpu().numpy(), opt.m_scale.cpu().numpy(), False)
                v = to.values(opt.v.cpu().numpy(), opt.v_scale.cpu().numpy(), True)
                np.testing.assert_array_equal(g64(mo), m)
                np.testing.assert_array_equal(g64(vo), v)
            m, v = m.astype(np.float32), v.astype(np.float32)


def test_adamw_extreme_moments(gpu_ctx):
    """Blocks of zeros, of the smallest and the largest gradients, with NaN and infinity, and
    the first and the last values of the codes' range."""
    from simple_llm_amd.gpu import gpu
    rng = np.random.default_rng(0)
    g = np.zeros((9, 128), np.float32)
    g[1] = 1e-25
    g[2] = rng.standard_normal(128) * 1e-19
    g[3, 5] = 1e19
    g[4, 6] = np.nan
    g[5, 7] = np.inf
    g[6] = np.exp(rng.uniform(-60, 0, 128))
    g[7] = rng.standard_normal(128)
    g[8] = np.ldexp(1.0, rng.integers(-20, 20, 128))
    p = rng.standard_normal((9, 128)).astype(np.float32)
    for bits in (32, 8):
        pd, gd = dev(p), dev(g)
        opt = gpu.adamw_create(gpu_ctx, [pd], [gd], bits=bits, seed=3)
        m, v = np.zeros(1152, np.float32), np.zeros(1152, np.float32)
        want = p.astype(np.float64).ravel()
        for t in (1, 2):
            old = g64(pd).ravel()
            gpu.adamw_update(gpu_ctx, opt, **HYPER)
            m, v = to.moments(m, v, g.ravel(), HYPER["beta1"], HYPER["beta2"])
            want = to.stepped(old, m, v, t, **HYPER)
            with np.errstate(invalid="ignore"):
                fine = np.isfinite(want)
                got = g64(pd).ravel()
                np.testing.assert_array_equal(np.isfinite(got), fine)
                tol = p_tol(old, m.astype(float), v.astype(float), t, HYPER, want)
            within(got[fine], want[fine], tol[fine], f"bits {bits} step {t}")
            if bits == 8:
                r = to.hashed(3, t, 1152)
                back = []
                for x, name, shift, uns in ((m, "m", 0, False), (v, "v", 16, True)):
                    code, byte = to.store(x, (r >> shift) & 0xffff, uns)
                    np.testing.assert_array_equal(getattr(opt, name).cpu().numpy(), code)
                    np.testing.assert_array_equal(getattr(opt, name + "_scale").cpu().numpy(), byte)
                    back.append(to.values(code, byte, uns).astype(np.float32))
                m, v = back
            else:
                np.testing.assert_array_equal(opt.m.cpu().numpy(), m)
                np.testing.assert_array_equal(opt.v.cpu().numpy(), v)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured(gpu_ctx, bits):
    """A captured step counts on when replayed, with the learning rate and gradient scale of
    the moment, as eager steps do: bit by bit."""
    from simple_llm_amd.gpu import gpu
    torch.manual_seed(0)
    p0, g0 = torch.randn(3000, device="cuda"), torch.randn(3000, device="cuda")
    lrs, scales = [1e-2, 5e-3, 2e-3, 1e-3], [1.0, 0.5, 2.0, 0.1]
    ends = []
    for captured in (False, True):
        p, g = p0.clone(), g0.clone()
        lr, gs = torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")
        opt = gpu.adamw_create(gpu_ctx, [p], [g], bits=bits, seed=1)
        step = lambda: gpu.adamw_update(gpu_ctx, opt, lr, grad_scale=gs)
        if captured:
            s = torch.cuda.Stream()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
                step()
            step = graph.replay
        for i, (a, b) in enumerate(zip(lrs, scales)):
            lr.fill_(a)
            gs.fill_(b)
            g.copy_(g0 * (i + 1))
            step()
            torch.cuda.synchronize()
            assert opt.step.item() == i + 1
        ends.append((p.clone(), opt.m.clone(), opt.v.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*ends))
    q, h = p0.clone(), g0.clone()  # and as numbers
    opt = gpu.adamw_create(gpu_ctx, [q], [h], bits=bits, seed=1)
    for i, (a, b) in enumerate(zip(lrs, scales)):
        h.copy_(g0 * (i + 1))
        gpu.adamw_update(gpu_ctx, opt, a, grad_scale=b)
    assert torch.equal(q, ends[0][0]) and torch.equal(opt.v, ends[0][2])


def test_adamw8_moves_slow_moments(gpu_ctx):
    """beta2 = 0.999 over 2000 steps of constant gradients from zero: rounding to the nearest
    would stop v far below; at random it reaches (1 - 0.999^2000) g^2 on average, to 5
    deviations of the mean. A value's own deviation: a rounding adds at most a quarter of a
    squared step, at most (v / 8)^2, whenever one happens, and its part fades with 0.999 a
    step; the steps round up or down by 1 / 8 as often as the drift of v / 1000 needs, so the
    variances sum up to at most 500 (1 / 1000) (1 / 8) v^2: 0.25 v."""
    from simple_llm_amd.gpu import gpu
    n = 128 * 64
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.125, device="cuda")
    opt = gpu.adamw_create(gpu_ctx, [p], [g], bits=8, seed=9)
    for _ in range(2000):
        gpu.adamw_update(gpu_ctx, opt, 0.0)
    m, v = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    gpu.adamw_read(gpu_ctx, opt, m, v)
    want = (1 - 0.999 ** 2000) * 0.125 ** 2
    off, own = v.double().mean().item() / want - 1, v.double().std().item() / want
    print(f"mean {off:+.4f}, deviation {own:.3f}")
    assert abs(off) < 5 * 0.25 / np.sqrt(n) and own < 0.25
    assert abs(m.double().mean().item() / 0.125 - 1) < 0.02


def test_adamw_refuses(gpu_ctx):
    from simple_llm_amd.gpu import gpu
    p, g = torch.zeros(10, 4, device="cuda"), torch.zeros(10, 4, device="cuda")
    flat = torch.zeros(100, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        gpu.adamw_create(gpu_ctx, [flat[:60], flat[50:]], [flat[:60].clone(), flat[50:].clone()])
    with pytest.raises(ValueError, match="overlaps"):
        gpu.adamw_create(gpu_ctx, [p], [p])
    with pytest.raises(ValueError, match=r"grads\[0\] shape"):
        gpu.adamw_create(gpu_ctx, [p], [g.view(4, 10)])
    with pytest.raises(ValueError, match=r"params\[0\] must be contiguous"):
        gpu.adamw_create(gpu_ctx, [p.t()], [g.t()])
    with pytest.raises(ValueError, match=r"copies\[0\] must be torch.bfloat16"):
        gpu.adamw_create(gpu_ctx, [p], [g], copies=[g])
    opt = gpu.adamw_create(gpu_ctx, [p], [g])
    for kw, match in ((dict(lr=float("nan")), "lr must be finite"), (dict(lr=1.0, beta1=1.0), "beta1"),
                      (dict(lr=1.0, eps=-1.0), "eps"),
                      (dict(lr=torch.zeros(2, device="cuda")), "lr shape mismatch"),
                      (dict(lr=1.0, grad_scale=torch.zeros(1)), "grad_scale must live")):
        with pytest.raises(ValueError, match=match):
            gpu.adamw_update(gpu_ctx, opt, **kw)
    with pytest.raises(ValueError, match="a 32-bit state"):
        gpu.adamw_read(gpu_ctx, opt, p.view(-1), g.view(-1))
    g.data = torch.zeros(10, 4, device="cuda")
    with pytest.raises(ValueError, match="no longer where it was"):
        gpu.adamw_update(gpu_ctx, opt, 1e-3)
    assert opt.step.item() == 0


# ---- together --------------------------------------------------------------

def test_refusals_change_nothing(gpu_ctx):
    from simple_llm_amd.gpu import gpu
    x, g, r = torch.ones(6, 8).cuda(), torch.ones(8).cuda(), torch.ones(6).cuda()
    i = torch.zeros(6, dtype=torch.int32).cuda()
    big = torch.ones(14, 8).cuda()
    c = gpu_ctx
    for call, match in (
            (lambda: gpu.layernorm(c, x, g, g, big[:6].t()), "output shape"),
            (lambda: gpu.layernorm(c, big[::2][:6], g, g, x), "input must be contiguous"),
            (lambda: gpu.layernorm(c, big[:6], g, g, big[1:7]), "overlaps"),
            (lambda: gpu.layernorm(c, x, g[:4], g, x), "gamma shape"),
            (lambda: gpu.layernorm(c, x, g, g.cpu(), x), "beta must live"),
            (lambda: gpu.layernorm(c, x, g, g, x, eps=-1.0), "eps"),
            (lambda: gpu.layernorm(c, torch.ones(1, 20000).cuda(), torch.ones(20000).cuda(),
                                   torch.ones(20000).cuda(), torch.ones(1, 20000).cuda()), "16384"),
            (lambda: gpu.layernorm(c, torch.ones(49).cuda()[1:].view(6, 8), g, g, x), "16-byte"),
            (lambda: gpu.layernorm_backward(c, x, x, g, r, r, big[:6], g.clone(), g.clone(),
                                            residual=big[1:7]), "overlaps"),
            (lambda: gpu.layernorm_backward(c, x, x, g, r, r, x, g, g.clone()), "overlaps"),
            (lambda: gpu.layernorm_backward(c, x.bfloat16(), x, g, r, r, x, g, g), "grad_output must"),
            (lambda: gpu.embedding(c, i.long(), x, x.clone()), "tokens must be"),
            (lambda: gpu.embedding(c, i, x, x), "overlaps"),
            (lambda: gpu.embedding(c, i, x, x.clone(), pos_table=torch.ones(3, 4).cuda()), "pos_table"),
            (lambda: gpu.embedding_backward(c, x, i[:5], x.clone()), "tokens shape"),
            (lambda: gpu.embedding_backward(c, x, i, x), "overlaps"),
            (lambda: gpu.cross_entropy_loss(c, x, i, r), "loss shape"),
            (lambda: gpu.cross_entropy_loss(c, x, i, r[:1], x.bfloat16()), "grad_logits must"),
            (lambda: gpu.cross_entropy_loss(c, big[:6], i, r[:1], big[2:8]), "overlaps"),
            (lambda: gpu.cross_entropy_loss(c, x, i, r[:1], row_losses=r), "overlaps")):
        with pytest.raises(ValueError, match=match):
            call()
    torch.cuda.synchronize()
    assert (x == 1).all() and (g == 1).all() and (r == 1).all() and (big == 1).all()


def test_batch_limit_counts(gpu_ctx):
    from simple_llm_amd.gpu import gpu
    ctx = gpu.context_create(config=gpu.GPUConfig(max_batch_operations=2))
    x, g = gpu.gpu_buffer_2d_create(ctx, 4, 8), gpu.gpu_buffer_1d_create(ctx, 8)
    gpu.batch_begin(ctx)
    gpu.layernorm(ctx, x, g, g, x)
    gpu.layernorm(ctx, x, g, g, x)
    with pytest.raises(RuntimeError, match="Batch operation limit"):
        gpu.layernorm(ctx, x, g, g, x)
    gpu.batch_commit(ctx)


def _chain(gpu, ctx, n, vocab, d):
    """Embedding, LayerNorm, a loss over the channels and all of it back, then AdamW."""
    rng = np.random.default_rng(n)
    s = dict(ids=dev(ids_of(rng, n, vocab), torch.int32), table=dev(rng.standard_normal((vocab, d))),
             gamma=dev(1 + 0.1 * rng.standard_normal(d)), beta=dev(0.1 * rng.standard_normal(d)),
             targets=dev(rng.integers(-1, d, n), torch.int32))
    e = lambda *shape: torch.zeros(shape, device="cuda")
    s.update(x=e(n, d), y=e(n, d), mean=e(n), rstd=e(n), loss=e(1), dy=e(n, d), dx=e(n, d),
             dg=e(d), db=e(d), dt=e(vocab, d))
    s["opt"] = gpu.adamw_create(ctx, [s["table"], s["gamma"], s["beta"]], [s["dt"], s["dg"], s["db"]],
                                bits=8, decay=[True, False, False])

    def step():
        gpu.embedding(ctx, s["ids"], s["table"], s["x"], 2.0)
        gpu.layernorm(ctx, s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"])
        gpu.cross_entropy_loss(ctx, s["y"], s["targets"], s["loss"], s["dy"])
        gpu.layernorm_backward(ctx, s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], s["dx"],
                               s["dg"], s["db"])
        gpu.embedding_backward(ctx, s["dx"], s["ids"], s["dt"], 2.0)
        gpu.adamw_update(ctx, s["opt"], 1e-2)
    return s, step


def test_captured_steps_equal_eager_ones(gpu_ctx):
    """Whole steps as graphs, two of them in turn with eager work and waits between, each
    equal to its eager twin bit by bit; and on two streams at once."""
    from simple_llm_amd.gpu import gpu
    shapes = [(700, 300, 200), (90, 2000, 1030)]
    eager = [_chain(gpu, gpu_ctx, *sh) for sh in shapes]
    graphs, caught = [], [_chain(gpu, gpu_ctx, *sh) for sh in shapes]
    streams = [torch.cuda.Stream() for _ in shapes]
    torch.cuda.synchronize()
    for (_, step), s in zip(caught, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            step()
        graphs.append(g)
    for _ in range(4):
        for _, step in eager:
            step()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (a, _), (b, _) in zip(eager, caught):
            for k in ("loss", "dy", "dx", "dg", "db", "dt", "table", "gamma", "beta"):
                assert torch.equal(a[k], b[k]), k
            assert torch.equal(a["opt"].v, b["opt"].v)
    both = [_chain(gpu, gpu_ctx, *sh) for sh in shapes]
    torch.cuda.synchronize()
    for _ in range(4):
        for (_, step), s in zip(both, streams):
            with torch.cuda.stream(s):
                step()
    torch.cuda.synchronize()
    for (a, _), (b, _) in zip(eager, both):
        assert torch.equal(a["table"], b["table"]) and torch.equal(a["dt"], b["dt"])


def test_gradients_of_a_small_model(gpu_ctx):
    """One attention layer between an embedding and its tied logits, through this package's
    operators and torch's products, against autograd in 64 bits."""
    from simple_llm_amd.gpu import gpu
    B, N, H, D, V = 2, 37, 2, 32, 101
    d, n = H * D, B * N
    rng = np.random.default_rng(8)
    w = {k: dev(rng.standard_normal(s) * f) for k, s, f in (
        ("table", (V, d), 0.3), ("wq", (d, d), 0.15), ("wk", (d, d), 0.15), ("wv", (d, d), 0.15),
        ("wo", (d, d), 0.15), ("g1", (d,), 1.0), ("b1", (d,), 0.1), ("g2", (d,), 1.0),
        ("b2", (d,), 0.1))}
    pos = dev(rng.standard_normal((N, d)))
    ids = dev(rng.integers(0, V, n), torch.int32)
    targets = rng.integers(0, V, n).astype(np.int32)
    targets[5:9] = -100
    e = lambda *s: torch.empty(s, device="cuda")
    buf = gpu.gpu_buffer_from_tensor
    c = gpu_ctx

    x, h, mean1, rstd1 = e(n, d), e(n, d), e(n), e(n)
    gpu.embedding(c, ids, w["table"], x, 1.0, pos)
    gpu.layernorm(c, x, w["g1"], w["b1"], h, mean1, rstd1)
    q, k, v = (h @ w[i] for i in ("wq", "wk", "wv"))
    o, L, M = e(n, d), e(n * H), e(n * H)
    gpu.flash_attention(c, *map(buf, (q, k, v, o, L, M)), B, N, H, D)
    x2 = x + o @ w["wo"]
    h2, mean2, rstd2 = e(n, d), e(n), e(n)
    gpu.layernorm(c, x2, w["g2"], w["b2"], h2, mean2, rstd2)
    logits = h2 @ w["table"].t()
    loss, dlog = e(1), e(n, V)
    gpu.cross_entropy_loss(c, logits, dev(targets, torch.int32), loss, dlog)

    grads = {i: torch.zeros_like(t) for i, t in w.items()}
    grads["table"].copy_(dlog.t() @ h2)
    dh2 = dlog @ w["table"]
    dx2 = e(n, d)
    gpu.layernorm_backward(c, dh2, x2, w["g2"], mean2, rstd2, dx2, grads["g2"], grads["b2"])
    grads["wo"].copy_(o.t() @ dx2)
    do = dx2 @ w["wo"].t()
    dq, dk, dv = e(n, d), e(n, d), e(n, d)
    blocks = -(-N // c.config.flash_attn_br)
    gpu.flash_attention_backward(c, *map(buf, (q, k, v, o, L, M, do, dq, e(blocks * n, d),
                                               e(blocks * n, d), dk, dv)), B, N, H, D)
    for i, t in (("wq", dq), ("wk", dk), ("wv", dv)):
        grads[i].copy_(h.t() @ t)
    dh = dq @ w["wq"].t() + dk @ w["wk"].t() + dv @ w["wv"].t()
    dx = e(n, d)
    gpu.layernorm_backward(c, dh, x, w["g1"], mean1, rstd1, dx, grads["g1"], grads["b1"],
                           residual=dx2)
    gpu.embedding_backward(c, dx, ids, grads["table"], accumulate=True)

    r = {i: t.double().cpu().requires_grad_() for i, t in w.items()}
    X = r["table"][ids.cpu().long()] + pos.double().cpu().repeat(B, 1)
    ln = lambda t, a, b: torch.nn.functional.layer_norm(t, (d,), a, b, 1e-5)
    Hh = ln(X, r["g1"], r["b1"])
    Q, K, Vv = ((Hh @ r[i]).view(B, N, H, D).transpose(1, 2) for i in ("wq", "wk", "wv"))
    S = (Q @ K.transpose(-1, -2)) / np.sqrt(D)
    S = S.masked_fill(torch.ones(N, N, dtype=torch.bool).triu(1), -np.inf)
    O = (S.softmax(-1) @ Vv).transpose(1, 2).reshape(n, d)
    H2 = ln(X + O @ r["wo"], r["g2"], r["b2"])
    want = torch.nn.functional.cross_entropy(H2 @ r["table"].t(), torch.from_numpy(targets).long())
    want.backward()
    # nine operators deep, each off by at most the path of its sums, 64 to 101 terms and 30
    # more, times u: relative to a gradient's norm
    tol = 9 * 131 * U
    assert abs(loss.item() - want.item()) < tol * want.item()
    for i in w:
        off = float((grads[i].double().cpu() - r[i].grad).norm() / r[i].grad.norm())
        print(f"{i}: {off:.2e}")
        assert off < tol, i

    old = {i: g64(t) for i, t in w.items()}
    opt = gpu.adamw_create(c, list(w.values()), list(grads.values()))
    gpu.adamw_update(c, opt, **HYPER)
    for i, t in w.items():
        m, v = to.moments(0.0, 0.0, g64(grads[i]), HYPER["beta1"], HYPER["beta2"])
        step = to.stepped(old[i], m, v, 1, **HYPER)
        within(t, step, p_tol(old[i], m.astype(float), v.astype(float), 1, HYPER, step), i)


def test_offsets_past_32_bits(gpu_ctx):
    """More than 2^31 elements: the last rows equal a small call's."""
    from simple_llm_amd.gpu import gpu
    d, rows = 16384, (1 << 17) + 5
    x = torch.empty(rows, d, dtype=BF, device="cuda")
    x.normal_()
    g, b = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(rows).cuda(), torch.empty(rows).cuda()
    gpu.layernorm(gpu_ctx, x, g, b, y, mean, rstd)
    small = torch.empty(8, d, dtype=BF, device="cuda")
    gpu.layernorm(gpu_ctx, x[-8:], g, b, small)
    assert torch.equal(y[-8:], small)
    dg, db = torch.empty(d).cuda(), torch.empty(d).cuda()
    dx = torch.empty_like(x)
    gpu.layernorm_backward(gpu_ctx, y, x, g, mean, rstd, dx, dg, db)
    gpu.layernorm_backward(gpu_ctx, y[-8:], x[-8:], g, mean[-8:].clone(), rstd[-8:].clone(), small, dg,
                           db)
    assert torch.equal(dx[-8:], small)
    t = torch.zeros(rows, dtype=torch.int32, device="cuda")
    loss, one = torch.empty(1).cuda(), torch.empty(1).cuda()
    gpu.cross_entropy_loss(gpu_ctx, x, t, loss, dx, rstd)
    gpu.cross_entropy_loss(gpu_ctx, x[-8:], t[:8].clone(), one, small, mean[:8], grad_scale=8 / rows)
    assert torch.equal(rstd[-8:], mean[:8])
    # the scale is rounded once in one call and twice in the other, then bf16 on both sides
    assert ((dx[-8:].float() - small.float()).abs() <= 2.0 ** -7 * small.float().abs()).all()
    ids = torch.arange(rows, device="cuda").int()
    gpu.embedding(gpu_ctx, ids, x, y)
    assert torch.equal(x[-9:], y[-9:]) and torch.equal(x[:9], y[:9])


def test_gradients_and_weights_past_32_bits(gpu_ctx):
    """A table and a tensor of more than 2^31 elements: rows and weights at both ends."""
    from simple_llm_amd.gpu import gpu
    vocab, d, n = (1 << 20) + 300, 2050, 777
    rng = np.random.default_rng(1)
    ids = np.concatenate([rng.integers(0, 9, n // 2), vocab - 1 - rng.integers(0, 9, n - n // 2)])
    dy = dev(rng.integers(-3, 4, (n, d)))  # whole numbers: exact sums
    grad = torch.full((vocab, d), 7.0, device="cuda")
    gpu.embedding_backward(gpu_ctx, dy, dev(ids, torch.int32), grad)
    want = torch.zeros(18, d, device="cuda")
    want.index_add_(0, dev(np.where(ids < 9, ids, 18 + ids - vocab), torch.int64), dy)
    assert torch.equal(torch.cat([grad[:9], grad[-9:]]), want)
    assert int((grad[9:-9] != 0).sum()) == 0

    p = grad.view(-1)
    p.fill_(0.5)
    size = p.numel()
    g = torch.empty(size, dtype=BF, device="cuda").normal_()
    opt = gpu.adamw_create(gpu_ctx, [p], [g])
    tail = 5000
    p2, g2 = torch.full((tail,), 0.5, device="cuda"), g[-tail:].clone()
    small = gpu.adamw_create(gpu_ctx, [p2], [g2])
    for _ in range(2):
        gpu.adamw_update(gpu_ctx, opt, 1e-2)
        gpu.adamw_update(gpu_ctx, small, 1e-2)
    assert torch.equal(p[-tail:], p2)
    assert torch.equal(opt.v[size - tail:size], small.v[:tail])
    assert not (p == 0.5).any()
