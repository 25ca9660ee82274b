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


# ---- bounds from the kernels' longest sums ---------------------------------------

# Rows on 16, 32 and 64 lanes, 4 and 16 wavefronts; many rows a place.
SUMS = [(70000, 64), (40000, 300), (20000, 1500), (2048, 2048), (3000, 5000), (513, 8192), (3, 16384),
        (300, 16381)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,d", SUMS)
def test_layernorm_sums(gpu_ctx, rows, d, dtype):
    """A row's sum: at most 32 columns in a lane, 6 additions over a wavefront and 4 over
    wavefronts, or 16 + 6 + 16: 42. A column's: the rows of a place, then at most 2 and 8
    over a workgroup's places, 4 + 2 + 16 over the workgroups."""
    from simple_llm_amd.gpu import gpu
    banner(f"layernorm sums {rows} x {d} {dtype}")
    rng, x, gamma, beta = norm_inputs(rows, d, dtype)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows).cuda(), torch.empty(rows).cuda()
    gpu.layernorm(gpu_ctx, x, gamma, beta, y, mean, rstd)
    want, mu, rs = to.layernorm(g64(x), g64(gamma), g64(beta))
    # the deviations' mean: its sum, the deviations' roundings and a quotient, 44 u of a deviation
    within(mean, mu, U * (np.abs(mu) + 44 / rs), "mean")
    # squares of rounded deviations, 3 u each, their sum, a quotient, eps; half of it, and 2 more
    within(rstd, rs, 26 * U * rs, "rstd")
    xh = (g64(x) - mu[:, None]) * rs[:, None]
    tol = U * (np.abs(g64(gamma)) * (30 * np.abs(xh) + 44) + np.abs(g64(beta)) + np.abs(want))
    within(y, want, tol + half_step(dtype) * (np.abs(want) + tol), "y")

    dy = dev(rng.standard_normal((rows, d)), dtype)
    dx, dg, db = torch.empty_like(x), torch.empty(d).cuda(), torch.empty(d).cuda()
    gpu.layernorm_backward(gpu_ctx, dy, x, gamma, mean, rstd, dx, dg, db)
    want, wg, wb = to.layernorm_backward(g64(dy), g64(x), g64(gamma), g64(mean), g64(rstd))
    mu, rs = g64(mean)[:, None], g64(rstd)[:, None]
    xh = np.abs((g64(x) - mu) * rs)
    g = np.abs(g64(dy) * g64(gamma))
    # xh: two roundings; g: one; the means: 42 and 2, their terms 4; then six more
    tol = U * rs * (8 * g + 50 * g.mean(-1, keepdims=True)
                    + 54 * xh * (g * xh).mean(-1, keepdims=True)) + 2 * U * np.abs(want)
    within(dx, want, tol + half_step(dtype) * (np.abs(want) + tol), "dx")
    at_once = 256 * (32 if d <= 128 else 8 if d <= 1024 else 1)  # rows, at the least
    path = -(-rows // at_once) + 10 + 22
    s = np.abs(g64(dy))
    within(dg, wg, U * ((path + 3) * (s * xh).sum(0) + np.abs(wg)), "dgamma")
    within(db, wb, U * (path * s.sum(0) + np.abs(wb)), "dbeta")


@pytest.mark.parametrize("before", [0, 1, 9, 16])
@pytest.mark.parametrize("count", [15, 16, 17, 111, 112, 113, 127, 128, 129, 145, 6000, 30000])
def test_embedding_backward_sums(gpu_ctx, count, before):
    """A row of so many tokens behind `before` others in the sorted order, so that it lies in
    one range of 16, in up to 8 and in more. A range's tokens are added one after the other;
    then up to 8 ranges' parts, or, of more ranges, an eighth of them and 8 sums."""
    from simple_llm_amd.gpu import gpu
    banner(f"embedding_backward of {count} tokens behind {before}")
    rng = np.random.default_rng(count + before)
    n, d = count + before + 40, 65
    ids = np.concatenate([np.zeros(before), np.full(count, 1), rng.integers(2, 9, 40)])
    ids = rng.permutation(ids).astype(np.int32)
    dy = dev(rng.standard_normal((n, d)))
    want = to.embedding_backward(g64(dy), ids, 9, 3.0)
    size = to.embedding_backward(np.abs(g64(dy)), ids, 9, 3.0)
    ranges = count // 16 + 2
    path = 16 + max(8, -(-ranges // 8) + 8) + 2
    for accumulate in (False, True):
        grad = dev(rng.standard_normal((9, d)))
        was = g64(grad) * accumulate
        gpu.embedding_backward(gpu_ctx, dy, dev(ids, torch.int32), grad, 3.0, accumulate)
        within(grad, want + was, U * (path * size + 2 * np.abs(want + was)), f"{accumulate}")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grads", [F32, BF])
def test_adamw_of_many_chunks(gpu_ctx, bits, grads):
    """More chunks of 4096 than workgroups, over tensors of unlike sizes, alignments and
    decay, with copies: moments bit by bit, the codes of two steps too."""
    from simple_llm_amd.gpu import gpu
    banner(f"adamw of many chunks bits={bits} grads={grads}")
    rng = np.random.default_rng(bits)
    shapes = [(700, 1500), (1,), (4097,), (300, 4096), (129,), (511, 1000), (77,), (8192,)]

    def tensors(dtype, scale):
        out = []
        for i, s in enumerate(shapes):
            n = int(np.prod(s))
            flat = torch.zeros(n + i % 2, dtype=dtype, device="cuda")
            flat[i % 2:] = dev(scale * rng.standard_normal(n) * np.exp(2 * rng.standard_normal(n)),
                               dtype)
            out.append(flat[i % 2:].view(s))
        return out

    ps, gs, cs = tensors(F32, 1.0), tensors(grads, 1e-2), tensors(BF, 1.0)
    decay = [i % 3 == 0 for i in range(len(shapes))]
    opt = gpu.adamw_create(gpu_ctx, ps, gs, bits=bits, copies=cs, decay=decay, seed=77)
    assert opt._chunks.shape[0] > 2 * 256
    n = opt.m.numel()
    place = np.concatenate([o + np.arange(p.numel()) for o, p in zip(opt.offsets, ps)])
    dec = np.concatenate([np.full(p.numel(), d) for p, d in zip(ps, decay)])
    flat = lambda ts: np.concatenate([g64(x).ravel() for x in ts])
    m, v, g = (np.zeros(n, np.float32) for _ in range(3))
    g[place] = flat(gs)
    for t in (1, 2):
        old = flat(ps)
        gpu.adamw_update(gpu_ctx, opt, **HYPER)
        m, v = to.moments(m, v, g, HYPER["beta1"], HYPER["beta2"])
        want = np.where(dec, to.stepped(old, m[place], v[place], t, **HYPER),
                        to.stepped(old, m[place], v[place], t, **{**HYPER, "weight_decay": 0}))
        within(flat(ps), want, p_tol(old, m[place].astype(float), v[place].astype(float), t, HYPER,
                                     want), f"step {t}")
        assert all(torch.equal(c, p.bfloat16()) for p, c in zip(ps, cs))
        if bits == 32:
            np.testing.assert_array_equal(opt.m.cpu().numpy(), m)
            np.testing.assert_array_equal(opt.v.cpu().numpy(), v)
            continue
        r, back = to.hashed(77, t, n), []
        for x, name, shift, uns in ((m, "m", 0, False), (v, "v", 16, True)):
            code, byte = to.store(x, (r >> shift) & 0xffff, uns)
            np.testing.assert_array_equal(getattr(opt, name).cpu().numpy(), code)
            np.testing.assert_array_equal(getattr(opt, name + "_scale").cpu().numpy(), byte)
            back.append(to.values(code, byte, uns).astype(np.float32))
        m, v = back
