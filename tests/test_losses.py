"""Softmax cross entropy of queries against every row of a base, and its
gradients, against plain 64-bit arithmetic.

Tolerances, derived before the first run.  With u32 = 2^-24 and u the half step
of the storage type (bf16 2^-8, fp16 2^-11, fp32 2^-24):

* a logit is scale * dot; an fp32 sum of d products in any order is off by at
  most (d + 2) u32 sum|q x| and the scaling adds two roundings:
  ds = scale (d + 4) u32 max sum|q x|.
* the loss is a smooth function of the logits with slope at most 2, and its own
  sum of n terms, exponentials (2 ulp and the rounding of their argument, up to
  |s| u32 each) and logarithm add n u32 + 8 u32 + 4 max|s| u32, relative to
  values of the size of 1 + loss:
  dl = 2 ds + (n + 16 + 4 max|s|) u32 (1 + loss).
* G = g scale (p - [n = t]) is off by |G| (2 ds + (n + 16 + 4 max|s|) u32)
  relative to p, and to p_t - 1 = expm1(-loss); over 1 - p_t it is rounded to
  the storage type once, and for dx the query, times its weight and 1 - p_t, once
  more; a product over k terms adds k u32 of the sum of absolute values:
  dq: (u + dp + n u32) (|G| @ |x|) + u |dq|,
  dx: (2 u + dp + nq u32) (|G|^T @ |q|) + u |dx|.
* what underflows fp32 is off by up to 2^-126 a term: at most 2^12 terms of
  weight up to 2^10 (scale times an element) here, so 2^-104 in all.
* fp16 rounds below its normal range in steps of 2^-24: G is held as
  2^14 (p - [n = t]) / (1 - p_t), the weighted query relative to the largest
  w (1 - p_t).
"""
import ctypes
import os

import pytest
import torch

U32 = 2.0 ** -24
UNDERFLOW = 2.0 ** -104
IGN = -100
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _C():
    import rapidadb._C as mod

    return mod


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(nq, n, d, dtype, seed=0, ignored=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.nn.functional.normalize(torch.randn(n, d, generator=g), dim=1)
    t = torch.randint(0, n, (nq,), generator=g)
    q = torch.nn.functional.normalize(x[t] + 1.2 * torch.nn.functional.normalize(torch.randn(nq, d, generator=g), dim=1),
                                      dim=1)
    if ignored:
        t[torch.randperm(nq, generator=g)[:ignored]] = IGN
    w = torch.rand(nq, generator=g) + 0.1
    return q.to(dtype), x.to(dtype), t, w


class Ref:
    """Loss and gradients in 64 bits, with the tolerances above."""

    def __init__(self, q, x, t, scale, w, ignore=IGN):
        u = half_step(q.dtype)
        qd, xd = q.cpu().double(), x.cpu().double()
        t = t.cpu().long()
        nq, (n, d) = len(t), x.shape
        keep = t != ignore
        qd = torch.where(keep[:, None], qd, torch.zeros_like(qd))
        tc = torch.where(keep, t, torch.zeros_like(t))
        s = scale * (qd @ xd.T)
        lp = torch.log_softmax(s, 1)
        rows = torch.arange(nq)
        self.loss = torch.where(keep, -lp[rows, tc], torch.zeros(nq, dtype=torch.float64))
        w = torch.where(keep, w.double(), torch.zeros(nq, dtype=torch.float64))
        p = lp.exp()
        p[rows, tc] = torch.expm1(-self.loss)
        G = p * (w * scale)[:, None]
        self.dq, self.dx = G @ xd, G.T @ qd
        smax = s.abs().max().item()
        ds = scale * (d + 4) * U32 * (qd.abs() @ xd.abs().T).max().item()
        rel = (n + 16 + 4 * smax) * U32
        dp = 2 * ds + rel
        self.tol_loss = torch.where(keep, 2 * ds + rel * (1 + self.loss) + UNDERFLOW, torch.zeros_like(self.loss))
        # steps of 2^-24 below fp16's normal range
        sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
        rest = -torch.expm1(-self.loss)  # 1 - p_t
        u_b = w * rest
        subG = sub * 2.0 ** -14 * scale
        self.tol_dq = 1.01 * ((u + dp + n * U32) * (G.abs() @ xd.abs()) + u * self.dq.abs() +
                              subG * u_b[:, None] * xd.abs().sum(0)[None, :]) + sub + UNDERFLOW
        pg = torch.where(rest[:, None] > 0, p.abs() / rest[:, None], torch.zeros_like(p)) * scale * keep[:, None]
        self.tol_dx = 1.01 * ((2 * u + dp + nq * U32) * (G.abs().T @ qd.abs()) + u * self.dx.abs() +
                              subG * (u_b[:, None] * qd.abs()).sum(0)[None, :] +
                              sub * u_b.abs().max().item() * pg.sum(0)[:, None]) + sub + UNDERFLOW


def within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first {i}: {got[i]} vs {want[i]} "
                             f"(tolerance {tol[i]})")


def loss_fn(*a, **k):
    from rapidadb.losses import softmax_cross_entropy

    return softmax_cross_entropy(*a, **k)


def run_all(q, x, t, w, scale=20.0, device="cuda", **kw):
    qd, xd = q.to(device).requires_grad_(), x.to(device).requires_grad_()
    loss = loss_fn(qd, xd, t.to(device), scale=scale, reduction="none", **kw)
    dq, dx = torch.autograd.grad(loss, (qd, xd), w.to(device))
    assert loss.dtype == torch.float32 and dq.dtype == q.dtype and dx.dtype == x.dtype
    return loss, dq, dx


def check_all(q, x, t, w, scale=20.0, **kw):
    loss, dq, dx = run_all(q, x, t, w, scale, **kw)
    r = Ref(q, x, t, scale, w, kw.get("ignore_index", IGN))
    within(loss, r.loss, r.tol_loss, "loss")
    within(dq, r.dq, r.tol_dq, "dq")
    within(dx, r.dx, r.tol_dx, "dx")


# ------------------------------------------------------------------ refusals
def test_refusals_without_gpu():
    q = torch.randn(3, 8)
    with pytest.raises(RuntimeError, match="queries must be a CUDA tensor"):
        loss_fn(q, q, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="reduction must be one of"):
        loss_fn(q, q, torch.zeros(3, dtype=torch.long), reduction="max")


def test_abi_refusals_without_gpu():
    """Every bad argument of both entry points is rejected before any device work."""
    lib = ctypes.CDLL(os.path.join(os.path.dirname(__file__), "..", "rapidadb_b200", "librdb_kernels.so"))
    lib.rdb_last_error.restype = ctypes.c_char_p
    i64, vp, i, sz = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    f, b = lib.rdb_softmax_xent, lib.rdb_softmax_xent_backward
    common = [i, vp, i64, i64, vp, i64, i64, i, vp, ctypes.c_float, i64, i]
    f.argtypes = common + [vp, vp, vp, sz, vp]
    b.argtypes = common + [vp, vp, vp, i64, vp, i64, vp, sz, vp]
    for w in (lib.rdb_softmax_xent_workspace, lib.rdb_softmax_xent_backward_workspace):
        w.restype = sz
    lib.rdb_softmax_xent_workspace.argtypes = [i, i64, i64, i, i]
    lib.rdb_softmax_xent_backward_workspace.argtypes = [i, i64, i64, i, i, i]
    assert 0 < lib.rdb_softmax_xent_workspace(2, 1024, 1_000_000, 768, 1) < 1 << 31
    assert 0 < lib.rdb_softmax_xent_backward_workspace(2, 4096, 131072, 768, 1, 1) < 1 << 31
    for dt in (0, 1, 2):  # no queries, one, single rows and columns: plans exist
        for nq, n, d in ((0, 5, 8), (1, 1, 1), (3, 1, 70), (100000, 3, 5000)):
            assert lib.rdb_softmax_xent_workspace(dt, nq, n, d, 0) > 0
            for flags in ((0, 0), (1, 0), (0, 1), (1, 1)):
                assert lib.rdb_softmax_xent_backward_workspace(dt, nq, n, d, *flags) > 0
    for nq, n, d in ((1 << 31, 5, 8), (1 << 40, 5, 8), (5, 1 << 31, 8), (5, 1 << 44, 8), (5, 5, (1 << 31) - 1),
                     (-1, 5, 8), (5, 0, 8), (5, 5, 0)):  # and none where the calls refuse
        assert lib.rdb_softmax_xent_workspace(2, nq, n, d, 0) == 0
        assert lib.rdb_softmax_xent_backward_workspace(2, nq, n, d, 1, 1) == 0
    ok = dict(dt=2, q=1 << 20, nq=2, ldq=16, x=1 << 21, n=4, ldx=16, d=16, t=1 << 22, s=1.0, ign=-100, red=1)
    bad = [(dict(dt=5), b"dtype"), (dict(n=0), b"shape"), (dict(d=0), b"shape"), (dict(ldq=8), b"shape"),
           (dict(s=0.0), b"scale"), (dict(s=-1.0), b"scale"), (dict(s=float("inf")), b"scale"),
           (dict(s=float("nan")), b"scale"), (dict(red=3), b"reduction"), (dict(q=None), b"NULL"),
           (dict(t=None), b"NULL"), (dict(ldx=20), b"multiples of 16"), (dict(x=(1 << 21) + 2), b"aligned"),
           (dict(n=1 << 31), b"2^31"), (dict(nq=1 << 31), b"2^31"),
           (dict(d=(1 << 31) - 1, ldq=1 << 31, ldx=1 << 31), b"2^31 - 256")]
    for kw, msg in bad:
        a = list({**ok, **kw}.values())
        assert f(*a, 1 << 23, 1 << 24, 1 << 25, 1 << 40, None) == 1 and msg in lib.rdb_last_error(), kw
        assert b(*a, 1 << 23, 1 << 24, 1 << 26, 16, 1 << 27, 16, 1 << 25, 1 << 40, None) == 1, kw
        assert msg in lib.rdb_last_error(), kw
    a = list(ok.values())
    assert f(*a, 1 << 23, 1 << 24, 1 << 25, 3, None) == 6 and b"workspace" in lib.rdb_last_error()
    assert b(*a, 1 << 23, 1 << 24, 1 << 26, 16, 1 << 27, 16, 1 << 25, 3, None) == 6
    assert f(*a, None, 1 << 24, 1 << 25, 1 << 40, None) == 1 and b"NULL" in lib.rdb_last_error()
    assert b(*a, None, 1 << 24, 1 << 26, 16, 1 << 27, 16, 1 << 25, 1 << 40, None) == 1
    assert b(*a, 1 << 23, 1 << 24, 1 << 26, 8, 1 << 27, 16, 1 << 25, 1 << 40, None) == 1


@pytest.mark.gpu
def test_refusals(device):
    q, x = torch.randn(3, 8, device=device), torch.randn(5, 8, device=device)
    t = torch.zeros(3, dtype=torch.long, device=device)
    for a, msg in [((q, x[:, :4], t), "dimension mismatch"), ((q, x[:0], t), "database is empty"),
                   ((q, x, t[:2]), "targets must be 1D"), ((q, x, t.float()), "int64 or int32"),
                   ((q, x.half(), t), "same dtype"), ((q.double(), x.double(), t), "float32, float16 or bfloat16"),
                   ((q, x.cpu(), t), "CUDA"), ((q, x, t.cpu()), "same CUDA device"),
                   ((q[0], x, t), "must be 2D"), ((q[:, :0], x[:, :0], t), "at least one column")]:
        with pytest.raises(RuntimeError, match=msg):
            loss_fn(*a)
    for s in (0.0, -1.0, float("inf"), float("nan"), 1e39):
        with pytest.raises(RuntimeError, match="scale must be positive"):
            loss_fn(q, x, t, scale=s)
    many = torch.zeros(1, 8, device=device).expand(1 << 31, 8)
    with pytest.raises(RuntimeError, match="database must have fewer than 2\\^31 rows"):
        loss_fn(q, many, t)
    with pytest.raises(RuntimeError, match="queries must have fewer than 2\\^31 rows"):
        loss_fn(many, x, t[:1].expand(1 << 31))
    loss, stats = _C().softmax_cross_entropy(q, x, t, 1.0, IGN, 0)
    with pytest.raises(RuntimeError, match="stats must be"):
        _C().softmax_cross_entropy_backward(loss, q, x, t, stats[:5], 1.0, IGN, 0)
    with pytest.raises(RuntimeError, match="shape of the loss"):
        _C().softmax_cross_entropy_backward(loss[:2], q, x, t, stats, 1.0, IGN, 0)
    with pytest.raises(RuntimeError, match="reduction"):
        _C().softmax_cross_entropy(q, x, t, 1.0, IGN, 7)


# -------------------------------------------------------------------- values
SIZES = [(1, 1, 1), (1, 300, 64), (2, 5, 7), (3, 64, 8), (31, 255, 63), (32, 256, 64), (33, 257, 65), (64, 1000, 128),
         (77, 503, 100), (127, 129, 200), (128, 512, 256), (129, 130, 257), (255, 640, 96), (256, 256, 384),
         (257, 700, 130), (300, 1025, 768), (5, 2500, 1030), (520, 90, 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("nq,n,d", SIZES)
def test_loss_and_gradients(device, nq, n, d, dtype):
    check_all(*make(nq, n, d, DT[dtype], seed=nq + n + d, ignored=nq // 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("nq,n,d", [(1, 9000, 100), (1, 700, 250), (4, 5001, 130), (3, 333, 511), (1, 2049, 768),
                                    (4, 999, 769), (1, 130, 1024), (2, 40, 1025), (1, 1, 999), (2, 31, 1), (1, 7, 129)])
def test_few_queries(device, nq, n, d, dtype):
    check_all(*make(nq, n, d, DT[dtype], seed=n + d), scale=6.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("nq", [1, 3])
@pytest.mark.parametrize("d", [5, 100, 258, 771])
def test_few_queries_beside_other_values(device, nq, d, dtype):
    """What lies between the rows does not count, and the last row ends with
    the memory; ignored queries and targets that are no row as ever."""
    g = torch.Generator().manual_seed(d)
    n, ld = 77, (d + 7) // 8 * 8 + 8
    buf = torch.full(((n - 1) * ld + d,), float("nan"), dtype=DT[dtype], device=device)
    x = buf.as_strided((n, d), (ld, 1))
    x.copy_(torch.randn(n, d, generator=g))
    qbuf = torch.full(((nq - 1) * ld + d,), float("inf"), dtype=DT[dtype], device=device)
    q = qbuf.as_strided((nq, d), (ld, 1))
    q.copy_(torch.randn(nq, d, generator=g) / d ** 0.5)
    t, w = torch.tensor([76, IGN, 0][:nq]), torch.rand(nq, generator=g)
    got = run_all(q.detach(), x.detach(), t, w, 2.0)
    r = Ref(q, x, t, 2.0, w)
    within(got[0], r.loss, r.tol_loss, "loss")
    within(got[1], r.dq, r.tol_dq, "dq")
    within(got[2], r.dx, r.tol_dx, "dx")
    t[0] = n
    loss = loss_fn(q, x, t.to(device), reduction="none")
    assert loss[0].isnan() and not loss[1:].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reductions(device, dtype, reduction):
    q, x, t, w = make(200, 333, 96, DT[dtype], ignored=31)
    qd, xd = q.to(device).requires_grad_(), x.to(device).requires_grad_()
    loss = loss_fn(qd, xd, t.to(device).int(), scale=9.0, reduction=reduction)
    (3.0 * loss).backward()
    g = 3.0 / (169 if reduction == "mean" else 1)
    r = Ref(q, x, t, 9.0, torch.full((200,), g))
    k = 169 if reduction == "mean" else 1
    # a sum of 200 losses in fp32 on top of their own errors, and the division
    tol = (r.tol_loss.sum() + 202 * U32 * r.loss.sum()) / k
    assert loss.shape == () and abs(loss.item() - r.loss.sum().item() / k) <= tol
    within(qd.grad, r.dq, r.tol_dq * (1 + 4 * U32), "dq")
    within(xd.grad, r.dx, r.tol_dx * (1 + 4 * U32), "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_only_the_gradients_asked_for(device, dtype):
    q, x, t, w = make(60, 400, 72, DT[dtype])
    r = Ref(q, x, t, 20.0, w)
    qd, xd, td, wd = q.to(device), x.to(device), t.to(device), w.to(device)
    q1 = qd.clone().requires_grad_()
    loss = loss_fn(q1, xd, td, scale=20.0, reduction="none")
    within(torch.autograd.grad(loss, q1, wd)[0], r.dq, r.tol_dq, "dq")
    x1 = xd.clone().requires_grad_()
    loss = loss_fn(qd, x1, td, scale=20.0, reduction="none")
    within(torch.autograd.grad(loss, x1, wd)[0], r.dx, r.tol_dx, "dx")
    assert not loss_fn(qd, xd, td).requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        q2 = qd.clone().requires_grad_()
        g, = torch.autograd.grad(loss_fn(q2, xd, td), q2, create_graph=True)
        g.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("nq,n,d", [(6, 40, 24), (130, 300, 64)])
def test_gradients_against_differences(device, nq, n, d):
    """Central differences of the summed loss along random directions.  The
    fp32 inputs move by h = 2^-7; the truncation is h^2 / 6 times the third
    derivative (at most 2 scale^3 |direction of the logits|^3 per query), the
    difference of two losses carries twice their tolerance over 2 h."""
    q, x, t, w = make(nq, n, d, torch.float32, seed=4)
    scale, h = 5.0, 2.0 ** -7
    r = Ref(q, x, t, scale, torch.ones(nq))
    _, dq, dx = run_all(q, x, t, torch.ones(nq), scale)
    gen = torch.Generator().manual_seed(1)
    for which in (0, 1):
        v = torch.nn.functional.normalize(torch.randn((q, x)[which].shape, generator=gen), dim=1)
        up, dn = [q, x], [q, x]
        up[which], dn[which] = up[which] + h * v, dn[which] - h * v
        total = [loss_fn(a.to(device), b.to(device), t.to(device), scale=scale, reduction="none").double().sum().item()
                 for a, b in (up, dn)]
        diff = (total[0] - total[1]) / (2 * h)
        want = ((dq, dx)[which].double().cpu() * v.double()).sum().item()
        tol = nq * (h * h / 6) * 2 * scale ** 3 + 2 * r.tol_loss.sum().item() / h + \
            ((r.tol_dq, r.tol_dx)[which] * v.abs().double()).sum().item() + 2 * nq * scale * U32 / h
        assert abs(diff - want) <= tol, (which, diff, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_matches_torch_cross_entropy(device, dtype):
    q, x, t, w = make(70, 210, 40, DT[dtype], ignored=9)
    loss = loss_fn(q.to(device), x.to(device), t.to(device), scale=3.0)
    ref = torch.nn.functional.cross_entropy(3.0 * q.double() @ x.double().T, t, ignore_index=IGN)
    r = Ref(q, x, t, 3.0, w)
    assert abs(loss.item() - ref.item()) <= r.tol_loss.sum().item() / 61 + 80 * U32 * ref.item()


# --------------------------------------------------------------------- masks
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_an_ignored_query_holds_reaches_nothing(device, dtype, value):
    q, x, t, w = make(140, 300, 80, DT[dtype], ignored=20)
    clean = run_all(q, x, t, w)
    q2, w2 = q.clone(), w.clone()
    q2[t == IGN] = value
    w2[t == IGN] = value
    dirty = run_all(q2, x, t, w2)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert (dirty[0][t.to(device) == IGN] == 0).all() and (dirty[1][t.to(device) == IGN] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_every_query_ignored(device, dtype):
    q, x, _, w = make(9, 20, 16, DT[dtype])
    t = torch.full((9,), IGN)
    loss, dq, dx = run_all(q, x, t, w)
    assert (loss == 0).all() and (dq == 0).all() and (dx == 0).all()
    qd, xd = q.to(device).requires_grad_(), x.to(device).requires_grad_()
    total = loss_fn(qd, xd, t.to(device))
    total.backward()
    assert total.isnan() and (qd.grad == 0).all() and (xd.grad == 0).all()


@pytest.mark.gpu
def test_ignore_index_may_be_a_row(device):
    q, x, t, w = make(50, 12, 32, torch.float32)
    check_all(q, x, t, w, ignore_index=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("target", [-1, 300, 1 << 40, -(1 << 62)])
def test_target_outside_the_base_is_nan(device, dtype, target):
    q, x, t, w = make(140, 300, 80, DT[dtype])
    good = run_all(q, x, t, w)
    t[7] = target
    loss, dq, dx = run_all(q, x, t, w)
    assert loss[7].isnan() and dq[7].isnan().all() and dx.isnan().all()
    rest = torch.arange(140, device=device) != 7
    assert torch.equal(loss[rest], good[0][rest]) and torch.equal(dq[rest], good[1][rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_nan_query_and_row(device, dtype):
    """NaN in a query stays in its loss and dq; NaN in a row is in every logit
    sum."""
    q, x, t, w = make(140, 300, 80, DT[dtype])
    good = run_all(q, x, t, w)
    q2 = q.clone()
    q2[5, 3] = float("nan")
    loss, dq, dx = run_all(q2, x, t, w)
    rest = torch.arange(140, device=device) != 5
    assert loss[5].isnan() and dq[5].isnan().all() and dx.isnan().all()
    assert torch.equal(loss[rest], good[0][rest]) and torch.equal(dq[rest], good[1][rest])
    x2 = x.clone()
    x2[299] = float("nan")
    assert run_all(q, x2, t, w)[0].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_rows_far_below(device, dtype):
    """Logits hundreds below the largest vanish without NaN, whichever tile
    they lie in; a target among them keeps its (large) loss."""
    n, d = 700, 64
    x = torch.zeros(n, d)
    x[:, 0] = -8.0
    x[650, 0] = 8.0
    q = torch.zeros(3, d)
    q[:, 0] = 8.0
    t = torch.tensor([650, 0, 699])
    check_all(q.to(DT[dtype]), x.to(DT[dtype]), t, torch.ones(3), scale=4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_loss_near_zero_keeps_its_digits(device, dtype):
    """Queries that find their row: the loss is the sum of the other terms."""
    d = 64
    x = torch.eye(d)
    q = torch.eye(d)
    t = torch.arange(d)
    scale = 24.0
    loss, dq, _ = run_all(q.to(DT[dtype]), x.to(DT[dtype]), t, torch.ones(d), scale)
    want = torch.log1p(torch.tensor((d - 1), dtype=torch.float64) * torch.exp(torch.tensor(-scale, dtype=torch.float64)))
    # argument 24 log2 e rounds by 2^-20 of a unit; 63 terms; 2 ulp each
    assert ((loss.cpu().double() - want).abs() <= want * (2.0 ** -19 + 80 * U32)).all()
    u = half_step(DT[dtype])
    got = dq.diagonal().cpu().double()
    ref = scale * torch.expm1(-want)
    sub = (2.0 ** -25 * 2.0 ** -14 * scale + 2.0 ** -25) if dtype == "fp16" else 0.0
    assert ((got - ref).abs() <= ref.abs() * (2.0 ** -18 + 2.02 * u) + sub).all()


@pytest.mark.gpu
def test_same_target_many_times_and_duplicate_rows(device):
    q, x, t, w = make(200, 90, 64, torch.bfloat16)
    t[:] = 17
    x[40:60] = x[17]
    check_all(q, x, t, w)


# ----------------------------------------------------------- use of the call
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_strides_and_bases(device, dtype):
    """Columns of wider matrices, odd offsets, transposed and repeated rows
    give what their copies give; what lies beside them is not read."""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(300, 160, generator=g).to(DT[dtype]).to(device)
    qw = torch.randn(40, 160, generator=g).to(DT[dtype]).to(device)
    wide[:, 100:] = float("nan")
    qw[:, 100:] = float("nan")
    t, w = torch.randint(0, 37, (40,), generator=g).to(device), torch.rand(40, generator=g).to(device)
    views = [(qw[:, :100], wide[:, :100]), (qw[:, 3:99], wide[:, 3:99]), (qw[:, 8:96], wide[::2, 8:96]),
             (qw[:, :100:4], wide[:, :100:4]), (qw[:, :88], wide[:, :88].t().contiguous().t()),
             (qw[:1, :64].expand(40, 64), wide[5:6, :64].expand(50, 64))]
    for qv, xv in views:
        got = run_all(qv.detach(), xv.detach(), t, w, 1.0)
        want = run_all(qv.contiguous(), xv.contiguous(), t, w, 1.0)
        for a, b in zip(got, want):
            assert torch.equal(a, b) and not a.isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("d", [64, 37])
def test_saved_tensors_that_come_back_elsewhere(device, d, dtype):
    """Hooks on the saved tensors return them in other memory and other
    strides (offloaded to the host and back, transposed, at odd bases): the
    gradients stay the same."""
    g = torch.Generator().manual_seed(4)
    qw = torch.randn(40, 96, generator=g).to(DT[dtype]).to(device)
    xw = torch.randn(300, 96, generator=g).to(DT[dtype]).to(device)
    q, x = qw[:, :d], xw[::2, 8:8 + d]
    t, w = torch.randint(0, 150, (40,), generator=g).to(device), torch.rand(40, generator=g).to(device)
    want = run_all(q.detach(), x.detach(), t, w)

    def transposed(v):
        return v.t().contiguous().t() if v.dim() == 2 else v.repeat_interleave(2)[::2]

    def odd_base(v):
        out = torch.empty(v.numel() + 1, dtype=v.dtype, device=v.device)[1:].view(v.shape)
        return out.copy_(v)

    hooks = [torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
             torch.autograd.graph.saved_tensors_hooks(lambda v: v, transposed),
             torch.autograd.graph.saved_tensors_hooks(lambda v: v, odd_base)]
    for h in hooks:
        with h:
            got = run_all(q.detach(), x.detach(), t, w)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_saved_tensors_that_come_back_wrong_are_refused(device):
    q, x, t, w = make(6, 40, 32, torch.float32)
    for unpack, message in [(lambda v: v.cpu(), "CUDA"), (lambda v: v.half() if v.is_floating_point() else v, "stats"),
                            (lambda v: v[:-1] if v.dim() == 1 else v, "targets")]:
        qd, xd = q.to(device).requires_grad_(), x.to(device).requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
            loss = loss_fn(qd, xd, t.to(device))
            with pytest.raises(RuntimeError, match=message):
                torch.autograd.grad(loss, (qd, xd))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_no_queries(device, dtype):
    q, x, t, w = make(1, 30, 16, DT[dtype])
    loss, dq, dx = run_all(q[:0], x, t[:0], w[:0])
    assert loss.shape == (0,) and dq.shape == (0, 16) and (dx == 0).all()
    assert loss_fn(q[:0].to(device), x.to(device), t[:0].to(device), reduction="sum").item() == 0
    assert loss_fn(q[:0].to(device), x.to(device), t[:0].to(device)).isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_same_bits_every_time_and_on_any_stream(device, dtype):
    q, x, t, w = make(300, 2000, 128, DT[dtype], ignored=10)
    first = run_all(q, x, t, w)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        other = run_all(q, x, t, w)
    torch.cuda.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_captured_steps(device, dtype):
    """Two captured training steps, replayed with new inputs on two streams at
    once, give what eager calls give; an eager graph of the same leaves lives
    through the capture."""
    C = _C()
    q, x, t, w = (v.to(device) for v in make(150, 700, 96, DT[dtype], ignored=11))

    def step():
        loss, stats = C.softmax_cross_entropy(q, x, t, 20.0, IGN, 1)
        return (loss, *C.softmax_cross_entropy_backward(torch.ones_like(loss), q, x, t, stats, 20.0, IGN, 1))

    leaf = q.clone().requires_grad_()
    eager = loss_fn(leaf, x, t, scale=20.0)
    want = step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        # torch.autograd.grad of fresh leaves: no accumulation node of another stream
        lq = q.detach().requires_grad_()
        lx = x.detach().requires_grad_()
        outs.append((lambda l: (l.detach(), *torch.autograd.grad(l, (lq, lx))))(loss_fn(lq, lx, t, scale=20.0)))
    graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for k in range(2):
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b)
        q2, x2, t2, _ = make(150, 700, 96, DT[dtype], seed=9, ignored=20)
        if k == 0:
            r = Ref(q, x, t, 20.0, torch.full((150,), 1 / 139))
            within(torch.autograd.grad(eager, leaf)[0], r.dq, r.tol_dq * (1 + 4 * U32), "dq of the eager graph")
        q.copy_(q2), x.copy_(x2), t.copy_(t2)
        want = step()


def relative(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("nq,n,d", [(40, 3000, 768), (100, 20000, 256), (300, 4000, 512)])
@pytest.mark.parametrize("dtype", sorted(DT))
def test_errors_in_norm(device, nq, n, d, dtype):
    """Errors of whole results, much below the elementwise worst cases.  A loss
    is the sum of n terms, each off by the cut of its logit (half a step of 2^-24
    per instruction, d / 16 of them, on logits of about one tenth of the scale)
    and a few roundings: 2^-20 covers them four times over.  fp32 gradients are
    sums of such terms: 2^-18.  16-bit gradients round G and the query besides the
    result, independently: sqrt(3) roundings, of 0.41 half steps in the mean."""
    q, x, t, w = make(nq, n, d, DT[dtype], seed=3)
    r = Ref(q, x, t, 20.0, w)
    loss, dq, dx = run_all(q, x, t, w)
    assert relative(loss, r.loss) < 2.0 ** -20
    bound = 2.0 ** -18 if dtype == "fp32" else half_step(DT[dtype])
    assert relative(dq, r.dq) < bound and relative(dx, r.dx) < bound


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [3, 150])
def test_offsets_past_32_bits(device, nq):
    """More than 2^31 elements of rows: losses, and the gradients of queries and
    of rows at the end, in the middle and next to the 2^31st element."""
    n, d = 2_900_000, 768
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(n, d, dtype=torch.bfloat16, device=device)
    for part in x.split(500_000):
        part.copy_(torch.randn(part.shape, generator=g, device=device) / d ** 0.5)
    edge = 2 ** 31 // d
    t = torch.randint(0, n, (nq,), generator=g, device=device)
    t[0], t[1], t[2] = n - 1, edge, edge + 1
    q = (x[t].float() + 0.05 * torch.randn(nq, d, generator=g, device=device)).to(torch.bfloat16)
    qd, xd = q.clone().requires_grad_(), x.requires_grad_()
    loss = loss_fn(qd, xd, t, scale=10.0, reduction="none")
    dq, dx = torch.autograd.grad(loss, (qd, xd), torch.ones_like(loss))
    x = x.detach()
    lse = torch.full((nq,), -float("inf"), dtype=torch.float64, device=device)
    for part in x.split(100_000):
        lse = torch.logaddexp(lse, torch.logsumexp(10.0 * q.double() @ part.double().T, 1))
    want = lse - 10.0 * (q.double() * x[t].double()).sum(1)
    assert ((loss.double() - want).abs() <= 1e-4 * want).all()
    ref = torch.zeros(nq, d, dtype=torch.float64, device=device)
    for i, part in enumerate(x.split(100_000)):
        p = torch.exp(10.0 * q.double() @ part.double().T - lse[:, None])
        own = (t >= i * 100_000) & (t < i * 100_000 + len(part))
        p[own.nonzero()[:, 0], t[own] - i * 100_000] -= 1.0
        ref += 10.0 * p @ part.double()
    assert relative(dq, ref.cpu()) < 2.0 ** -7
    for lo, hi in ((0, 300), (edge - 150, edge + 150), (n - 300, n)):
        p = torch.exp(10.0 * q.double() @ x[lo:hi].double().T - lse[:, None])
        own = (t >= lo) & (t < hi)
        p[own.nonzero()[:, 0], t[own] - lo] -= 1.0
        assert relative(dx[lo:hi], (10.0 * p.T @ q.double()).cpu()) < 2.0 ** -7, (lo, hi)


@pytest.mark.gpu
def test_one_query_past_32_bits(device):
    """One query, whose rows are streamed, over more than 2^31 elements."""
    n, d = 2_900_000, 768
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(n, d, dtype=torch.bfloat16, device=device)
    for part in x.split(500_000):
        part.copy_(torch.randn(part.shape, generator=g, device=device) / d ** 0.5)
    edge = 2 ** 31 // d
    for t in (0, edge, edge + 1, n - 1):
        q = (x[t:t + 1].float() * 1.5).to(torch.bfloat16)
        loss = loss_fn(q, x, torch.tensor([t], device=device), scale=10.0).item()
        s = torch.cat([10.0 * (part.double() @ q[0].double()) for part in x.split(100_000)])
        want = (torch.logsumexp(s, 0) - s[t]).item()
        assert abs(loss - want) <= 1e-4 * want, (t, loss, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_one_query_captured_on_two_streams(device, dtype):
    """Two captured losses of one query, replayed at once on two streams with
    inputs that change between the replays."""
    x = make(5, 3000, 200, DT[dtype])[1].to(device)
    side = [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.zeros(1, 200, dtype=DT[dtype], device=device) for _ in side]
    ts = [torch.zeros(1, dtype=torch.long, device=device) for _ in side]
    loss_fn(qs[0], x, ts[0])
    torch.cuda.synchronize()
    graphs, out = [], []
    for q, t in zip(qs, ts):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out.append(loss_fn(q, x, t, scale=4.0))
    for i in range(8):
        for k in range(2):
            qs[k].copy_(x[17 * i + k:17 * i + k + 1] * 2)
            ts[k].fill_(17 * i + k if i % 3 else 2999 - i)
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for q, t, o in zip(qs, ts, out):
            assert torch.equal(o, loss_fn(q, x, t, scale=4.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
def test_two_threads_at_once(device, dtype):
    from concurrent.futures import ThreadPoolExecutor

    cases = [make(150, 900, 96, DT[dtype], seed=s) for s in (1, 2)]
    want = [run_all(*c) for c in cases]
    torch.cuda.synchronize()

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [run_all(*cases[i]) for _ in range(8)]
        s.synchronize()
        return got

    with ThreadPoolExecutor(2) as ex:
        for i, runs in enumerate(ex.map(work, (0, 1))):
            for got in runs:
                assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("d", [64, 50])
def test_short_calls_in_a_row(device, d, dtype):
    """Calls whose launches overlap (each starts while the one before it ends)
    on inputs that change between them, next to other kernels, give the bits of
    the same calls with a synchronisation after each."""
    q0, x0, t, _ = make(48, 700, d, DT[dtype])
    q0, x0, t = q0.to(device), x0.to(device), t.to(device)

    def run(sync):
        q, x, out = q0.clone(), x0.clone(), []
        for i in range(30):
            a, b = q.detach().requires_grad_(), x.detach().requires_grad_()
            loss = loss_fn(a, b, t, scale=5.0)
            sync()
            dq, dx = torch.autograd.grad(loss, (a, b))
            sync()
            c, s = _C().sq8_encode(x)
            sync()
            qc, qs = _C().sq8_encode(q)
            sync()
            scores = _C().sq8_dot_product(qc, qs, c, s, DT[dtype])
            sync()
            one = _C().sq8_dot_product(qc[i:i + 1], qs[i:i + 1], c, s)
            sync()
            out += [loss.detach(), dq, dx, scores, one]
            q -= dq * 4
            x -= dx * 4  # overwrites what the calls before read
            del a, b, c, s, qc, qs  # the allocator hands their memory on
            sync()
        return out

    want = run(torch.cuda.synchronize)
    got = run(lambda: None)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.isnan().any()


@pytest.mark.gpu
def test_train_quantise_score(device):
    """The operators together: a step of training queries and rows, the rows
    quantised into an int8 base, queries quantised and scored, top-k taken."""
    C = _C()
    q, x, t, _ = make(96, 1500, 64, torch.float32, seed=5)
    qp, xp = q.to(device).requires_grad_(), x.to(device).requires_grad_()
    opt = torch.optim.SGD([qp, xp], lr=0.05)
    r = Ref(q, x, t, 20.0, torch.full((96,), 1 / 96))
    loss = loss_fn(qp, xp, t.to(device), scale=20.0)
    loss.backward()
    within(qp.grad, r.dq, r.tol_dq * (1 + 4 * U32), "dq")
    opt.step()
    within(qp, q.double() - 0.05 * r.dq, 0.05 * r.tol_dq + 2 * U32 * (q.double().abs() + r.dq.abs()), "updated queries")
    codes, scales = C.sq8_encode(xp.detach())
    qc, qs = C.sq8_encode(qp.detach())
    s = C.sq8_dot_product(qc, qs, codes, scales)
    ref = (qc.double() @ codes.double().T) * (qs.double()[:, None] * scales.double()[None, :])  # whole sums: exact
    assert ((s.double() - ref).abs() <= 3.01 * U32 * ref.abs()).all()
    v, i = C.topk(s, 5, True)
    assert torch.equal(v, s.gather(1, i))
    # the quantised scores differ from the float ones by at most half a step per coordinate of either side
    slack = 0.51 * (qs[:, None] * (codes.abs() * scales[:, None]).sum(1)[None, :] +
                    scales[None, :] * qp.detach().abs().sum(1)[:, None])
    assert ((s - qp.detach() @ xp.detach().T).abs() <= slack + 1e-4).all()
