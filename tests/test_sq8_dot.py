"""Int8 scores: quantising a user's rows (_C.sq8_encode) and the product of
codes with a scale per query and per row (_C.sq8_dot_product), against the
oracle's codes and plain 64-bit arithmetic.

The integer sum is exact, so an output is off by the roundings that follow it:
sum -> fp32, qs * xs, and their product (2^-24 each), and one to the output
type (half an eps of it)."""
import numpy as np
import pytest
import torch

import oracle

U32 = 2.0 ** -24


def _C():
    import rapidadb._C as mod

    return mod


def codes_of(rng, n, d, lo=-128):
    return torch.from_numpy(rng.integers(lo, 128, (n, d), dtype=np.int8)), \
        torch.from_numpy(rng.uniform(1e-3, 2e-2, n).astype(np.float32))


def check(out, qc, qs, xc, xs, dtype):
    acc = qc.double() @ xc.double().T
    ref = acc * qs.double()[:, None] * xs.double()[None, :]
    # three fp32 roundings and the output's; fp16 may go below its normal range
    tol = ref.abs() * (3.01 * U32 + torch.finfo(dtype).eps / 2 * (dtype != torch.float32)) + \
        (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert out.dtype == dtype and out.shape == ref.shape
    bad = (out.cpu().double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first {bad.nonzero()[0].tolist()}"


# ------------------------------------------------------------------ refusals
def test_refusals_without_gpu():
    C = _C()
    with pytest.raises(RuntimeError, match="vectors must be a CUDA tensor"):
        C.sq8_encode(torch.randn(3, 4))
    c, s = torch.zeros(3, 16, dtype=torch.int8), torch.ones(3)
    with pytest.raises(RuntimeError, match="query_codes must be a CUDA tensor"):
        C.sq8_dot_product(c, s, c, s)


def test_abi_refusals_without_gpu():
    """Every bad argument is rejected before any device work."""
    import ctypes
    import os

    lib = ctypes.CDLL(os.path.join(os.path.dirname(__file__), "..", "rapidadb_b200", "librdb_kernels.so"))
    lib.rdb_last_error.restype = ctypes.c_char_p
    i64, vp = ctypes.c_int64, ctypes.c_void_p
    f = lib.rdb_sq8_dot
    f.argtypes = [vp, vp, i64, i64, vp, vp, i64, i64, ctypes.c_int, ctypes.c_int, vp, i64, vp]
    ok = dict(qc=1 << 20, qs=1 << 21, nq=2, ldq=16, xc=1 << 22, xs=1 << 23, n=4, ldx=16, d=16, t=0, out=1 << 24, ldo=4)
    for kw, msg in [(dict(t=3), b"dtype"), (dict(d=0), b"shape"), (dict(ldq=8), b"shape"), (dict(ldo=3), b"shape"),
                    (dict(d=131072, ldq=131072, ldx=131072), b"131071"), (dict(qc=None), b"NULL"),
                    (dict(ldx=24), b"multiples of 16"), (dict(xc=(1 << 22) + 4), b"aligned"),
                    (dict(n=1 << 31, ldo=1 << 31), b"2^31")]:
        a = {**ok, **kw}
        rc = f(a["qc"], a["qs"], a["nq"], a["ldq"], a["xc"], a["xs"], a["n"], a["ldx"], a["d"], a["t"], a["out"],
               a["ldo"], None)
        assert rc == 1 and msg in lib.rdb_last_error(), (kw, lib.rdb_last_error())
    assert f(None, None, 0, 16, None, None, 4, 16, 16, 0, None, 4, None) == 0  # nothing to do


def test_row_copy_refusals_without_gpu():
    import ctypes
    import os

    lib = ctypes.CDLL(os.path.join(os.path.dirname(__file__), "..", "rapidadb_b200", "librdb_kernels.so"))
    lib.rdb_last_error.restype = ctypes.c_char_p
    i64, vp = ctypes.c_int64, ctypes.c_void_p
    f = lib.rdb_pad_rows
    f.argtypes = [vp, i64, i64, i64, vp, i64, vp]
    for a, msg in [((1 << 20, -1, 5, 5, 1 << 21, 16), b"shape"), ((1 << 20, 3, 0, 5, 1 << 21, 16), b"shape"),
                   ((1 << 20, 3, 5, 5, 1 << 21, 24), b"multiples of 16"), ((1 << 20, 3, 17, 17, 1 << 21, 16), b"multiples"),
                   ((1 << 20, 3, 5, 5, (1 << 21) + 8, 16), b"multiples"), ((None, 3, 5, 5, 1 << 21, 16), b"NULL"),
                   ((1 << 20, 3, 5, 5, None, 16), b"NULL")]:
        assert f(*a, None) == 1 and msg in lib.rdb_last_error(), (a, lib.rdb_last_error())
    assert f(None, 0, 5, 5, None, 16, None) == 0


@pytest.mark.gpu
def test_refusals(device):
    C = _C()
    c, s = torch.zeros(3, 16, dtype=torch.int8, device=device), torch.ones(3, device=device)
    for args, msg in [((c, s, c[:, :8], s), "dimension mismatch"), ((c, s[:2], c, s), "query_scales must be 1D"),
                      ((c, s, c, s[:2]), "scales must be 1D"), ((c.int(), s, c, s), "codes must be int8"),
                      ((c, s.double(), c, s), "scales must be float32"), ((c[0], s, c, s), "must be 2D"),
                      ((c, s, c.cpu(), s), "CUDA"), ((c, s, c, s.cpu()), "same CUDA device"),
                      ((c, s, c, s, torch.float64), "dtype must be"), ((c[:, :0], s, c[:, :0], s), "at least one")]:
        with pytest.raises(RuntimeError, match=msg):
            C.sq8_dot_product(*args)
    many, ms = c[:1].expand(1 << 31, 16), s[:1].expand(1 << 31)
    for args, msg in [((many, ms, c, s), "query_codes must have"), ((c, s, many, ms), "codes must have")]:
        with pytest.raises(RuntimeError, match=msg + " fewer than 2\\^31 rows"):
            C.sq8_dot_product(*args)
    for d in ((1 << 31) - 256, (1 << 32) + 8):  # the latter is 8 in 32 bits
        with pytest.raises(RuntimeError, match="dim must be <"):
            C.sq8_encode(s[:1].reshape(1, 1).expand(1, d))
    with pytest.raises(RuntimeError, match="must be 2D"):
        C.sq8_encode(s)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        C.sq8_encode(s.double().reshape(1, 3))


# -------------------------------------------------------------------- encode
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(1, 1), (5, 7), (33, 64), (9, 100), (70, 768), (3, 1025), (2, 5000)])
def test_encode_equals_definition(device, n, d, dtype):
    rng = np.random.default_rng(n * 1000 + d)
    x = torch.from_numpy(rng.standard_normal((n, d), dtype=np.float32)).to(dtype)
    x[0] = 0  # a zero row
    if n > 2:
        x[1] = 1e-41 if dtype == torch.float32 else 0.5  # subnormal rows; a constant row
        x[2, 0] = 60000.0
    codes, scales = _C().sq8_encode(x.to(device))
    rc, rs = oracle.sq8_encode(x.float().numpy())
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32
    assert np.array_equal(codes.cpu().numpy(), rc[:, :d]) and np.array_equal(scales.cpu().numpy(), rs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_encode_next_to_halves(device, dtype):
    """Quotients at and next to k + 1/2, subnormal scales, infinities and NaN:
    the codes of the division's definition."""
    k = torch.arange(-127, 127, dtype=torch.float32) + 0.5
    rows = []
    for s in (1.0, 0.37, 2.0 ** -20, 3e-5, 7.0):
        base = torch.cat([k * s, torch.nextafter(k * s, torch.tensor(1e9)), torch.nextafter(k * s, torch.tensor(-1e9)),
                          torch.tensor([127.0 * s] * 6)])
        rows.append(base)
    x = torch.stack(rows).to(dtype)
    extra = x.clone()
    extra[0, 5], extra[1, 700], extra[2, 0] = float("inf"), float("nan"), -float("inf")
    tiny = (x[:2].float() * 2.0 ** -139).to(dtype)  # subnormal rows (zero rows in fp16)
    x = torch.cat([x, extra, tiny])
    assert x.shape[1] % 8 == 0
    for v in (x, x[:, :-3]):
        codes, scales = _C().sq8_encode(v.to(device))
        xf = v.float().numpy()
        amax = np.fmax.reduce(np.abs(xf), axis=1)
        sc = (amax / np.float32(127)).astype(np.float32)
        with np.errstate(all="ignore"):
            c = np.rint(xf / sc[:, None])
        c = np.where(np.isnan(c), -127, np.clip(c, -127, 127))  # a NaN quotient has the lowest code
        c = np.where(sc[:, None] > 0, c, 0).astype(np.int8)
        assert np.array_equal(scales.cpu().numpy(), sc)
        assert np.array_equal(codes.cpu().numpy(), c)


@pytest.mark.gpu
def test_encode_strided_rows(device):
    """Columns of a wider matrix, a transposed matrix, and an odd base offset."""
    x = torch.randn(40, 301, device=device)
    for v in (x[:, 3:103], x.t()[:100, :40], x[:, 1::3], x[::2, :64], x[:0]):
        codes, scales = _C().sq8_encode(v)
        rc, rs = oracle.sq8_encode(np.ascontiguousarray(v.cpu().numpy())) if len(v) else (np.zeros((0, 301)), np.zeros(0))
        assert np.array_equal(codes.cpu().numpy(), rc[:, :v.shape[1]]) and np.array_equal(scales.cpu().numpy(), rs)


# ------------------------------------------------------------------- product
SIZES = [(1, 1, 1), (1, 1000, 768), (2, 37, 16), (3, 255, 100), (8, 129, 64), (9, 256, 128), (16, 300, 200),
         (17, 513, 33), (32, 1000, 768), (33, 256, 129), (64, 31, 1024), (65, 700, 48), (127, 257, 512), (128, 1, 256),
         (129, 520, 96), (255, 300, 130), (256, 256, 256), (257, 511, 640), (300, 2049, 144), (600, 90, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,n,d", SIZES)
def test_dot_product(device, nq, n, d, dtype):
    rng = np.random.default_rng(nq * 7919 + n * 31 + d)
    qc, qs = codes_of(rng, nq, d)
    xc, xs = codes_of(rng, n, d)
    out = _C().sq8_dot_product(qc.to(device), qs.to(device), xc.to(device), xs.to(device), dtype)
    check(out, qc, qs, xc, xs, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq", [1, 2])
@pytest.mark.parametrize("n,d", [(1, 5), (9001, 100), (20000, 128), (6001, 129), (501, 256), (4097, 300), (1000, 512),
                                 (333, 513), (77, 1600), (3, 12289)])
def test_few_queries(device, nq, n, d, dtype):
    """Also with other codes between the rows, where the last one ends with the memory."""
    rng = np.random.default_rng(n + d)
    qc, qs = codes_of(rng, nq, d)
    xc, xs = codes_of(rng, n, d)
    dev = [t.to(device) for t in (qc, qs, xc, xs)]
    out = _C().sq8_dot_product(*dev, dtype)
    check(out, qc, qs, xc, xs, dtype)
    ld = (d + 15) // 16 * 16 + 16
    buf = torch.full(((n - 1) * ld + d,), 77, dtype=torch.int8, device=device)
    rows = buf.as_strided((n, d), (ld, 1))
    rows.copy_(dev[2])
    assert torch.equal(_C().sq8_dot_product(dev[0], dev[1], rows, dev[3], dtype), out)


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [3, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("n,d", [(100_001, 128), (60_000, 1), (40_000, 200)])
def test_many_short_tiles(device, nq, n, d):
    """Many more tiles than accumulators, a K block or two each: sums exact in fp32."""
    g = torch.Generator().manual_seed(nq)
    qc = torch.randint(-128, 128, (nq, d), generator=g, dtype=torch.int8).to(device)
    xc = torch.randint(-128, 128, (n, d), generator=g, dtype=torch.int8).to(device)
    out = _C().sq8_dot_product(qc, torch.ones(nq, device=device), xc, torch.ones(n, device=device))
    # |sums| < 2^24: products of integers in fp32 are exact in any order
    assert torch.equal(out.double(), qc.double() @ xc.double().T)


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 5, 40, 300])
def test_extreme_codes_and_long_rows(device, nq):
    """All codes at -128 / 127 and the largest allowed dimension: the integer
    sum reaches 131071 * 2^14 < 2^31 and stays exact."""
    n, d = 70, 131071
    qc, xc = torch.full((nq, d), -128, dtype=torch.int8), torch.full((n, d), -128, dtype=torch.int8)
    xc[1] = 127
    xc[2, ::2] = 127
    qs, xs = torch.rand(nq) + 0.5, torch.rand(n) + 0.5
    out = _C().sq8_dot_product(qc.to(device), qs.to(device), xc.to(device), xs.to(device))
    check(out, qc, qs, xc, xs, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 6, 50, 290])
def test_special_scales(device, nq):
    """Zero, infinite and NaN scales act on their own query or row only."""
    rng = np.random.default_rng(nq)
    qc, qs = codes_of(rng, nq, 96, lo=1)
    xc, xs = codes_of(rng, 300, 96, lo=1)
    qs[nq // 2], xs[3], xs[7], xs[299] = 0.0, float("inf"), float("nan"), 0.0
    out = _C().sq8_dot_product(qc.to(device), qs.to(device), xc.to(device), xs.to(device)).cpu()
    ref = (qs.double()[:, None] * xs.double()[None, :]) * (qc.double() @ xc.double().T)
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.isinf(), ref.isinf())
    assert (out[:, 299] == 0).all()
    fin = ref.isfinite()
    assert ((out.double() - ref).abs()[fin] <= 3.01 * U32 * ref.abs()[fin]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 4, 20, 270])
def test_strided_operands(device, nq):
    """Index rows (padded stride with other bytes behind the dimension), a
    wider matrix's columns, odd bases and reversed orders."""
    rng = np.random.default_rng(5)
    d = 100
    wide = torch.from_numpy(rng.integers(-127, 128, (600, 176), dtype=np.int8)).to(device)
    qw = torch.from_numpy(rng.integers(-127, 128, (nq, 112), dtype=np.int8)).to(device)
    s = torch.rand(1200, device=device) + 0.1
    views = [wide[:, :d], wide[:, 16:16 + d], wide[:, 5:5 + d], wide[::2, :d], wide.t()[:d, :].t()[:, :d],
             wide[:, :d].expand(600, d), wide[:1, :d].expand(7, d)]
    for x in views:
        for q in (qw[:, :d], qw[:, 7:7 + d]):
            xs = s[:2 * x.shape[0]:2]  # strided scales
            out = _C().sq8_dot_product(q, s[:nq], x, xs)
            check(out, q.cpu(), s[:nq].cpu(), x.cpu(), xs.cpu(), torch.float32)


@pytest.mark.gpu
def test_empty_and_single(device):
    C = _C()
    c, s = torch.ones(3, 20, dtype=torch.int8, device=device), torch.ones(3, device=device)
    assert C.sq8_dot_product(c[:0], s[:0], c, s).shape == (0, 3)
    assert C.sq8_dot_product(c, s, c[:0], s[:0]).shape == (3, 0)
    assert C.sq8_encode(torch.zeros(0, 8, device=device))[0].shape == (0, 8)
    assert C.sq8_dot_product(c[:1, :1], s[:1], c[:1, :1], s[:1]).item() == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 24, 300])
def test_graph_stream_and_two_captures(device, nq):
    """Side streams, a captured and replayed product with new inputs, and two
    captured products replayed together."""
    C = _C()
    rng = np.random.default_rng(3)
    qc, qs = codes_of(rng, nq, 128)
    xc, xs = codes_of(rng, 500, 128)
    qd, qsd, xd, xsd = (t.to(device) for t in (qc, qs, xc, xs))
    want = C.sq8_dot_product(qd, qsd, xd, xsd)
    st, st2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        a = C.sq8_dot_product(qd, qsd, xd, xsd)
    with torch.cuda.stream(st2):
        b = C.sq8_dot_product(qd, qsd, xd, xsd)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(C.sq8_dot_product(qd, qsd, xd, xsd))
        graphs.append(g)
    qc2, _ = codes_of(rng, nq, 128)
    qd.copy_(qc2)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        graphs[0].replay()
    with torch.cuda.stream(st2):
        graphs[1].replay()
    torch.cuda.synchronize()
    for o in outs:
        check(o, qc2, qs, xc, xs, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 5])
def test_codes_past_32_bits(device, nq):
    n, d = 2_900_000, 768
    g = torch.Generator(device="cuda").manual_seed(1)
    xc = torch.empty(n, d, dtype=torch.int8, device=device)
    for part in xc.split(500_000):
        part.copy_(torch.randint(-127, 128, part.shape, generator=g, device=device, dtype=torch.int8))
    qc = torch.randint(-127, 128, (nq, d), generator=g, device=device, dtype=torch.int8)
    qs, xs = torch.rand(nq, generator=g, device=device) + 0.1, torch.rand(n, generator=g, device=device) + 0.1
    out = _C().sq8_dot_product(qc, qs, xc, xs)
    for i in range(0, n, 500_000):
        acc = qc.double() @ xc[i:i + 500_000].double().T
        ref = acc * (qs.double()[:, None] * xs[i:i + 500_000].double()[None, :])
        assert ((out[:, i:i + 500_000].double() - ref).abs() <= 3.01 * U32 * ref.abs()).all(), i


@pytest.mark.gpu
def test_scores_past_32_bits(device):
    """More than 2^31 scores."""
    nq, n, d = 750, 2_900_000, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    xc = torch.randint(-127, 128, (n, d), generator=g, device=device, dtype=torch.int8)
    qc = torch.randint(-127, 128, (nq, d), generator=g, device=device, dtype=torch.int8)
    qs, xs = torch.rand(nq, generator=g, device=device) + 0.1, torch.rand(n, generator=g, device=device) + 0.1
    out = _C().sq8_dot_product(qc, qs, xc, xs, torch.bfloat16)
    for b in (0, 3, 739, 740, 741, 749):
        ref = (qc[b].double() @ xc.double().T) * (qs[b].double() * xs.double())
        assert ((out[b].double() - ref).abs() <= (3.01 * U32 + 2.0 ** -8) * ref.abs()).all(), b


@pytest.mark.gpu
def test_two_threads_at_once(device):
    from concurrent.futures import ThreadPoolExecutor

    rng = np.random.default_rng(8)
    cases = []
    for nq in (2, 300):
        qc, qs = codes_of(rng, nq, 200)
        xc, xs = codes_of(rng, 1500, 200)
        cases.append([t.to(device) for t in (qc, qs, xc, xs)])
    want = [_C().sq8_dot_product(*c) for c in cases]
    torch.cuda.synchronize()

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [_C().sq8_dot_product(*cases[i]) for _ in range(20)]
        s.synchronize()
        return all(torch.equal(g, want[i]) for g in got)

    with ThreadPoolExecutor(2) as ex:
        assert all(ex.map(work, (0, 1)))


@pytest.mark.gpu
def test_scores_of_an_int8_index(device):
    """The codes of a Flat INT8 index scored with quantised queries: close to
    the index's exact scores, by the quantisation of the query alone."""
    from rapidadb import IndexConfig, Metric, RapidaDB
    from rapidadb_b200.config import Precision

    C = _C()
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2000, 100, generator=g).to(device)
    q = torch.randn(9, 100, generator=g).to(device)
    db = RapidaDB(config=IndexConfig(dim=100, metric=Metric.DOT_PRODUCT, precision=Precision.INT8))
    db.add(x)
    idx = db._index
    codes, scales = idx.sq8_codes(), idx.sq8_scales()
    qc, qs = C.sq8_encode(q)
    s = C.sq8_dot_product(qc, qs, codes, scales)
    check(s, qc.cpu(), qs.cpu(), codes.cpu(), scales.cpu(), torch.float32)
    # a query coordinate moves by at most qs / 2
    exact = q.double() @ (codes.double() * scales.double()[:, None]).T
    slack = 0.501 * qs.double()[:, None] * (codes.double().abs() * scales.double()[:, None]).sum(1)[None, :]
    assert ((s.double() - exact).abs() <= slack + 1e-4).all()
    v, i = C.topk(s, 10, True)
    assert torch.equal(v, s.gather(1, i)) and (v[:, :-1] >= v[:, 1:]).all()
