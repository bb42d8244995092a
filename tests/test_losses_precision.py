"""Softmax cross entropy: digits of the gradients where weights differ by orders
of magnitude, of long sums, and of the few queries that are streamed.

Tolerances as in test_losses.py; what is added to them is derived at each test.
"""
import pytest
import torch
from test_losses import DT, IGN, Ref, U32, UNDERFLOW, half_step, loss_fn, make, relative, run_all, within


def fp16_row_tolerance(r, q, x, t, scale, w):
    """Ref's tolerance of dx with the weighted queries of fp16 rounded in steps of
    2^-25 below 2^-14, the largest of them between 2^14 and 2^15: those steps are
    2^-39 of max_b |u_b| max_t |q_bt|, u_b = w_b (1 - p_t), and not 2^-25 of max |u_b|."""
    u, sub = half_step(torch.float16), 2.0 ** -25
    qd, xd = q.double(), x.double()
    keep, (n, d) = t >= 0, x.shape
    qd = torch.where(keep[:, None], qd, torch.zeros_like(qd))
    s = scale * (qd @ xd.T)
    p = torch.softmax(s, 1)
    rest = -torch.expm1(-r.loss)
    p[torch.arange(len(t)), t.clamp(min=0)] = -rest
    u_b = torch.where(keep, w.double().abs(), torch.zeros(len(t), dtype=torch.float64)) * rest
    smax = s.abs().max().item()
    dp = 2 * scale * (d + 4) * U32 * (qd.abs() @ xd.abs().T).max().item() + (n + 16 + 4 * smax) * U32
    pg = torch.where(rest[:, None] > 0, p.abs() / rest[:, None], torch.zeros_like(p)) * keep[:, None]  # |G| / u_b
    return 1.01 * ((2 * u + dp + len(t) * U32) * scale * (pg.T @ (u_b[:, None] * qd.abs())) + u * r.dx.abs() +
                   sub * 2.0 ** -14 * scale * (u_b[:, None] * qd.abs()).sum(0)[None, :] +
                   sub * 2.0 ** -14 * scale * (u_b * qd.abs().amax(1)).max().item() * pg.sum(0)[:, None]) + sub + UNDERFLOW


def steep(nq, lo, hi, seed):
    """Weights spread evenly over the orders of two between 2^lo and 2^hi, of both signs."""
    g = torch.Generator().manual_seed(seed)
    return torch.exp2(lo + (hi - lo) * torch.rand(nq, generator=g)) * torch.where(torch.rand(nq, generator=g) < 0.5, -1.0, 1.0)


# the largest element of dx, scale * w * max |q| (about 0.2), stays below 65504
@pytest.mark.gpu
@pytest.mark.parametrize("nq,n,d,scale,lo,hi", [(256, 4096, 768, 20.0, -4, 13), (256, 4096, 768, 40.0, -6, 12),
                                                (60, 700, 100, 20.0, -4, 13), (2100, 3000, 64, 10.0, -4, 13),
                                                (3, 500, 64, 10.0, -6, 13), (33, 90, 1030, 6.0, -3, 14)])
def test_fp16_rows_gradient_under_unequal_weights(device, nq, n, d, scale, lo, hi):
    """Every row of dx is as exact as its own digits allow, whatever the weights
    of other queries are."""
    q, x, t, _ = make(nq, n, d, torch.float16, seed=nq + n, ignored=nq // 9)
    w = steep(nq, lo, hi, nq)
    dx = run_all(q, x, t, w, scale)[2]
    r = Ref(q, x, t, scale, w)
    assert r.dx.abs().max().item() < 60000.0
    within(dx, r.dx, fp16_row_tolerance(r, q, x, t, scale, w), "dx")


def pairs(nq, d, seed, found):
    """Query b lies between rows 2 b (its target) and 2 b + 1 alone, closer to the
    target by found[b], and far from all others: their two rows of dx are its own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.linalg.qr(torch.randn(d, 2 * nq, generator=g, dtype=torch.float64))[0].T.contiguous()
    noise = torch.randn(nq, d, generator=g, dtype=torch.float64)
    noise -= noise @ x.T @ x
    q = (0.7 + found[:, None]) * x[::2] + 0.7 * x[1::2] + 0.3 * torch.nn.functional.normalize(noise, dim=1)
    return q.half(), x.half(), 2 * torch.arange(nq)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,d", [(100, 768), (30, 100), (3, 64)])
def test_fp16_rows_of_light_queries(device, nq, d):
    """Rows that only a query of small weight moves, next to queries of up to 2^21
    times its weight."""
    q, x, t = pairs(nq, d, nq, torch.zeros(nq, dtype=torch.float64))
    w = steep(nq, -8, 13, nq)
    w[0], w[-1] = 2.0 ** 13, 2.0 ** -8
    scale = 40.0
    dx = run_all(q, x, t, w, scale)[2]
    r = Ref(q, x, t, scale, w)
    assert r.dx.abs().max().item() < 65000.0
    within(dx, r.dx, fp16_row_tolerance(r, q, x, t, scale, w), "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("nq,d", [(100, 768), (30, 100)])
def test_fp16_rows_gradient_of_trained_queries(device, nq, d):
    """Queries whose 1 - p_t goes from 1/2 down to 1e-7, under one loss scale: every
    row of dx in norm.  Three independent roundings of 0.41 half steps in the mean,
    sqrt(3) of that, and the cut of the logits (below 2^-13 of p) beside it."""
    scale = 40.0
    q, x, t = pairs(nq, d, 5, torch.linspace(0.0, 0.4, nq, dtype=torch.float64))
    w = torch.full((nq,), 4096.0)
    dx = run_all(q, x, t, w, scale)[2].cpu().double()
    r = Ref(q, x, t, scale, w)
    norm = r.dx.norm(dim=1)
    assert norm.min().item() > 2.0 ** -14 * d ** 0.5  # elements of fp16's normal range
    err = (dx - r.dx).norm(dim=1) / norm
    assert err.max().item() < 1.25 * half_step(torch.float16), err.max().item()


@pytest.mark.gpu
def test_fp16_rows_gradient_of_odd_queries(device):
    """Zero queries, tiny ones, ones next to the largest, with weights to match:
    no overflow on the way, and nothing of the others is lost."""
    n, d, scale = 64, 40, 2.0 ** -12
    g = torch.Generator().manual_seed(3)
    x = torch.randn(n, d, generator=g).half()
    q = torch.randn(12, d, generator=g).half()
    q[0] = 0
    q[1] *= 2.0 ** -20
    q[2] = (torch.randn(d, generator=g) * 8000).half()
    t = torch.arange(12)
    for w in (torch.ones(12), torch.tensor([1e30] + [1.0] * 11), torch.tensor([1.0, 1e12, 2.0 ** -10] + [1.0] * 9),
              torch.tensor([1e-30] * 12), torch.zeros(12), torch.tensor([1.0, 1.0, 1e36] + [1.0] * 9)):
        dx = run_all(q, x, t, w, scale)[2]
        r = Ref(q, x, t, scale, w)
        inside = r.dx.abs() < 60000.0
        tol = torch.where(inside, fp16_row_tolerance(r, q, x, t, scale, w), torch.full_like(r.dx, float("inf")))
        got = dx.cpu().double()
        assert not got.isnan().any()
        assert ((got - r.dx).abs() <= tol)[inside].all(), w
    for bad in (float("inf"), float("nan")):
        w = torch.ones(12)
        w[5] = bad
        assert run_all(q, x, t, w, scale)[2].isnan().all()


# ------------------------------------------------------------------ long sums
@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 777, 2 ** 20 + 3])
def test_reduced_loss_is_the_sum_of_the_losses(device, nq):
    """Mean and sum are rounded once from a 64-bit sum of the losses that
    reduction="none" gives (2 u32 for the rounding and the mean's division)."""
    g = torch.Generator(device="cuda").manual_seed(nq)
    q = torch.rand(nq, 16, generator=g, device=device)
    x = torch.rand(9, 16, generator=g, device=device)
    t = torch.randint(0, 9, (nq,), generator=g, device=device)
    t[1::7] = IGN
    each = loss_fn(q, x, t, reduction="none").double()
    count = (t != IGN).sum().item()
    total = each.sum().item()
    assert abs(loss_fn(q, x, t, reduction="sum").item() - total) <= 2 * U32 * total
    assert abs(loss_fn(q, x, t).item() - total / count) <= 2 * U32 * total / count


# An accumulator of the tensor cores is cut towards zero at every instruction (16
# products), by 2^-23 of itself in the mean and less than 2^-22.  A run of up to 8,192
# products is 512 instructions, over which the sum grows: it loses at most
# 512 * 2^-22 / 2 = 2^-14 of itself, and half of that in the mean.  The joins of the
# runs are rounded to either side: 2^7 of them a split here, 2^-18 in the worst case.
LONG = 2.0 ** -14


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("nq", [1, 3])
def test_query_gradient_over_many_rows(device, nq, dtype):
    """2^25 rows of equal logits (zero queries): dq is their mean, G the exact
    2^-11, so that only the sum and the last rounding are off."""
    n, d = 2 ** 25 + 1, 16
    g = torch.Generator(device="cuda").manual_seed(nq)
    x = torch.empty(n, d, dtype=DT[dtype], device=device)
    for part in x.split(2 ** 22):
        part.copy_(torch.rand(part.shape, generator=g, device=device) * 0.5 + torch.linspace(0.5, 1.0, d, device=device))
    x[-1] = 0
    q = torch.zeros(nq, d, dtype=DT[dtype], device=device, requires_grad=True)
    t = torch.full((nq,), n - 1, device=device)
    dq, = torch.autograd.grad(loss_fn(q, x, t, scale=1.0, reduction="sum"), q)
    want = sum(part.double().sum(0) for part in x.split(2 ** 22)) / n
    tol = (half_step(DT[dtype]) + LONG) * want
    assert ((dq.double() - want).abs() <= tol).all(), ((dq.double() - want).abs() / want).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [16, 19])
def test_row_gradient_of_many_queries(device, dim, dtype):
    """2^20 queries against zero rows: p = 1/65, G the exact 256, every row that is
    no target has dx = scale / 65 of the queries' sum.  The weighted queries are
    rounded besides, independently: half a step over sqrt(2^20), 2^-19 at 2^-8."""
    nq, n, scale = 2 ** 20, 65, 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(dim)
    q = (torch.rand(nq, dim, generator=g, device=device) * 0.5 + torch.linspace(0.5, 1.0, dim, device=device)).to(DT[dtype])
    x = torch.zeros(n, dim, dtype=DT[dtype], device=device, requires_grad=True)
    t = torch.zeros(nq, dtype=torch.long, device=device)
    loss = loss_fn(q, x, t, scale=scale, reduction="sum")
    want = scale * q.double().sum(0) / n
    assert abs(loss.item() / nq - torch.log(torch.tensor(65.0)).item()) < 1e-4
    dx, = torch.autograd.grad(loss, x)
    tol = (half_step(DT[dtype]) + LONG + 2.0 ** -16) * want
    assert ((dx[1:].double() - want).abs() <= tol).all(), ((dx[1:].double() - want).abs() / want).max().item()
    # the target's row: (p - 1) of every query
    assert ((dx[0].double() + (n - 1) * want).abs() <= (n - 1) * tol).all()


# ------------------------------------------------------- streamed few queries
@pytest.mark.gpu
@pytest.mark.parametrize("near", [0.0, 0.6, 0.9])
@pytest.mark.parametrize("nq,n,d", [(1, 20000, 768), (4, 20000, 768), (2, 3000, 1024), (3, 5000, 200), (1, 900, 64)])
@pytest.mark.parametrize("dtype", sorted(DT))
def test_errors_in_norm_of_few_queries(device, nq, n, d, dtype, near):
    """As test_errors_in_norm at sizes whose forward pass streams the rows (one
    query, fp32 up to four), also where many rows that are not the target lie close
    to the query and carry the weight: the statistics and G come from logits that
    are rounded alike."""
    q, x, t, w = make(nq, n, d, DT[dtype], seed=n + d)
    if near:
        g = torch.Generator().manual_seed(7)
        x = x.double()
        for b in range(nq):
            k = torch.randperm(n, generator=g)[:20]
            k = k[~torch.isin(k, t)]
            noise = torch.nn.functional.normalize(torch.randn(len(k), d, generator=g, dtype=torch.float64), dim=1)
            x[k] = torch.nn.functional.normalize(near * q[b].double() + (1 - near) * noise, dim=1)
        x = x.to(DT[dtype])
    r = Ref(q, x, t, 20.0, w)
    loss, dq, dx = run_all(q, x, t, w)
    # One loss is no mean of many, and logits come up to 20: the exponent of a part's
    # sum and of its join are rounded by u32 of 20 log2 e, twice each, 80 u32.  Two and
    # more 16-bit queries run on the tensor cores, which cut a logit by up to 2^-22 of
    # itself at each of d / 16 instructions while it grows: 20 d / 16 * 2^-23.
    cut = 20 * d / 16 * 2.0 ** -23 if nq > 1 and dtype != "fp32" else 0.0
    assert ((loss.cpu().double() - r.loss).abs() <= 2.0 ** -20 * r.loss + 80 * U32 + cut).all()
    bound = 2.0 ** -18 if dtype == "fp32" else half_step(DT[dtype])
    assert relative(dq, r.dq) < bound and relative(dx, r.dx) < bound, (relative(dq, r.dq), relative(dx, r.dx))


# --------------------------------------------------- close rows on the tile loops
@pytest.mark.gpu
@pytest.mark.parametrize("near", [0.6, 0.9])
@pytest.mark.parametrize("nq,n,d", [(5, 9000, 768), (128, 4000, 256), (129, 4000, 256), (300, 8000, 512)])
@pytest.mark.parametrize("dtype", sorted(DT))
def test_errors_in_norm_beside_close_rows(device, nq, n, d, dtype, near):
    """Twenty rows beside each query that are not its target carry the weight.  Their
    logits, up to 20, come from the tensor cores, which cut a sum of d products at
    d / 16 instructions (fp32: of the largest planes) by up to 2^-22 of itself while
    it grows: the loss moves by 20 d / 16 * 2^-23 at most; G, over a sum of the same
    terms, by their differences alone."""
    q, x, t, w = make(nq, n, d, DT[dtype], seed=n + d)
    g = torch.Generator().manual_seed(7)
    x = x.double()
    free = torch.randperm(n, generator=g)
    free = free[~torch.isin(free, t)]
    for b in range(nq):
        k = free[20 * b:20 * b + 20]
        noise = torch.nn.functional.normalize(torch.randn(len(k), d, generator=g, dtype=torch.float64), dim=1)
        x[k] = torch.nn.functional.normalize(near * q[b].double() + (1 - near) * noise, dim=1)
    x = x.to(DT[dtype])
    r = Ref(q, x, t, 20.0, w)
    loss, dq, dx = run_all(q, x, t, w)
    cut = 20 * d / 16 * 2.0 ** -23
    assert ((loss.cpu().double() - r.loss).abs() <= 2.0 ** -20 * r.loss + 80 * U32 + cut).all()
    bound = 2.0 ** -18 if dtype == "fp32" else half_step(DT[dtype])
    assert relative(dq, r.dq) < bound and relative(dx, r.dx) < bound, (relative(dq, r.dq), relative(dx, r.dx))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("nq,n,d", [(8192, 3000, 40), (8193, 3000, 40), (9000, 45000, 71), (16500, 700, 256)])
def test_row_gradient_past_one_run(device, nq, n, d, dtype):
    """At and past the queries whose products fit one run, over one piece of the rows
    and two: errors in norm, three independent roundings."""
    g = torch.Generator(device="cuda").manual_seed(nq)
    unit = torch.nn.functional.normalize
    x = unit(torch.randn(n, d, generator=g, device=device), dim=1).to(DT[dtype])
    t = torch.randint(0, n, (nq,), generator=g, device=device)
    q = unit(x[t].float() + unit(torch.randn(nq, d, generator=g, device=device), dim=1), dim=1).to(DT[dtype])
    t[3::50] = IGN
    w = torch.rand(nq, generator=g, device=device) + 0.1
    a, b = q.clone().requires_grad_(), x.clone().requires_grad_()
    dq, dx = torch.autograd.grad(loss_fn(a, b, t, scale=8.0, reduction="none"), (a, b), w)
    xd = x.double()
    want_q, want_x = torch.zeros(nq, d, dtype=torch.float64, device=device), torch.zeros_like(xd)
    for part in torch.arange(nq, device=device).split(1000):
        part = part[t[part] != IGN]
        p = torch.softmax(8.0 * q[part].double() @ xd.T, 1)
        p[torch.arange(len(part), device=device), t[part]] -= 1.0
        p *= 8.0 * w[part].double()[:, None]
        want_q[part] = p @ xd
        want_x += p.T @ q[part].double()
    u = half_step(DT[dtype])
    assert relative(dq, want_q.cpu()) < u and relative(dx, want_x.cpu()) < u
    assert (dq[3::50] == 0).all()
