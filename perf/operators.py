"""Cases of the embedding-training and int8-scoring operators.

Each case is one pass through an operator as a user's program calls it:

* ``encode``   rows of embeddings -> int8 codes and one scale per row
* ``dot``      int8 query codes x int8 row codes -> scores, with a scale per
               query (token) and per row (channel)
* ``xent``     softmax cross entropy of queries against every row of a base of
               embeddings (the "vocabulary"), forward only
* ``train``    the same loss with its gradients

``own = False`` runs the plain form (elementary torch operations in 32 bits);
``own = True`` makes the framework's calls.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # quantising the embeddings of a bulk add: 1M bf16 rows of the default dimension
        {"name": "encode_1Mx768_bf16", "op": "encode", "n": 1_000_000, "d": 768, "dtype": "bf16"},
        # quantising one batch of queries before they are scored: latency
        {"name": "encode_32x768_fp32", "op": "encode", "n": 32, "d": 768, "dtype": "fp32"},
        # one query against a base of 100,000 codes: serving, one pass over the codes
        {"name": "dot_1x100000x768_fp32", "op": "dot", "nq": 1, "n": 100_000, "d": 768, "out": "fp32", "pad": 0},
        # a batch of 32 queries against the same base
        {"name": "dot_32x100000x768_fp32", "op": "dot", "nq": 32, "n": 100_000, "d": 768, "out": "fp32", "pad": 0},
        # a large batch against 16,384 centroids in bf16 scores: compute bound
        {"name": "dot_4096x16384x1024_bf16", "op": "dot", "nq": 4096, "n": 16_384, "d": 1024, "out": "bf16", "pad": 0},
        # odd sizes, rows at the padded stride an index stores them with
        {"name": "dot_37x9973x100_fp16", "op": "dot", "nq": 37, "n": 9_973, "d": 100, "out": "fp16", "pad": 12},
        # evaluation loss of a query encoder over a whole base: 1,024 queries, 1M rows
        {"name": "xent_1024x1Mx768_bf16", "op": "xent", "nq": 1024, "n": 1_000_000, "d": 768, "dtype": "bf16",
         "ignored": 0, "reduction": "none"},
        # the loss of a single query (latency, one pass over the rows)
        {"name": "xent_1x100000x768_bf16", "op": "xent", "nq": 1, "n": 100_000, "d": 768, "dtype": "bf16",
         "ignored": 0, "reduction": "none"},
        # training queries and rows together: a large batch over 131,072 rows, both gradients
        {"name": "train_4096x131072x768_bf16", "op": "train", "nq": 4096, "n": 131_072, "d": 768, "dtype": "bf16",
         "ignored": 0, "reduction": "mean", "rows": True},
        # in-batch negatives: the smallest training step
        {"name": "train_256x256x768_bf16", "op": "train", "nq": 256, "n": 256, "d": 768, "dtype": "bf16",
         "ignored": 0, "reduction": "mean", "rows": True},
        # training the query encoder against a fixed fp32 base
        {"name": "train_128x100000x768_fp32", "op": "train", "nq": 128, "n": 100_000, "d": 768, "dtype": "fp32",
         "ignored": 0, "reduction": "mean", "rows": False},
        # odd sizes with unlabelled (ignored) queries, a gradient per query
        {"name": "train_77x5003x100_fp16", "op": "train", "nq": 77, "n": 5_003, "d": 100, "dtype": "fp16",
         "ignored": 9, "reduction": "none", "rows": True},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["encode", "dot", "xent", "train"])
    d = rng.choice([rng.randint(16, 1024), 8 * rng.randint(4, 128), 128 * rng.randint(1, 8)])
    if op == "encode":
        return {"op": op, "n": _log_uniform(rng, 1, 450_000), "d": d, "dtype": rng.choice(sorted(DTYPES))}
    if op == "dot":
        nq = _log_uniform(rng, 1, 4096)
        n = _log_uniform(rng, 64, min(400_000, 60_000_000 // nq))
        return {"op": op, "nq": nq, "n": n, "d": d, "out": rng.choice(sorted(DTYPES)), "pad": rng.choice([0, 0, -d % 16])}
    dtype = rng.choice(sorted(DTYPES))
    if op == "xent":
        nq = _log_uniform(rng, 1, 4096)
        n = _log_uniform(rng, 64, min(600_000, 500_000_000 // nq))
        return {"op": op, "nq": nq, "n": n, "d": d, "dtype": dtype, "ignored": rng.choice([0, nq // 7]),
                "reduction": rng.choice(["none", "mean", "sum"])}
    nq = _log_uniform(rng, 1, 4096)
    n = _log_uniform(rng, 64, min(200_000, 250_000_000 // nq))
    return {"op": op, "nq": nq, "n": n, "d": d, "dtype": dtype, "ignored": rng.choice([0, nq // 7]),
            "reduction": rng.choice(["none", "mean", "sum"]), "rows": rng.choice([True, True, False])}


def _unit_rows(g, n, d):
    x = torch.randn(n, d, generator=g, device="cuda")
    return x / x.square().sum(1, keepdim=True).sqrt()


def _encode_plain(x):
    """code = rint(x / s) in [-127, 127], s = max|x| / 127 of the row (0 for a
    zero row), in fp32 arithmetic: the definition of the stored codes."""
    x = x.float()
    amax = x.abs().amax(1)
    s = amax / torch.full_like(amax, 127.0)  # a true division, not a product with 1/127
    c = (x / s[:, None]).round().clamp(-127, 127)
    return torch.where(s[:, None] > 0, c, torch.zeros_like(c)).to(torch.int8), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "encode":
        # unit embeddings with a few heavy coordinates
        x = _unit_rows(g, case["n"], case["d"])
        x = x * (1.0 + 4.0 * (torch.rand(case["n"], case["d"], generator=g, device="cuda") < 0.01))
        return {"case": case, "x": x.to(DTYPES[case["dtype"]])}
    if case["op"] == "dot":
        xc, xs = _encode_plain(_unit_rows(g, case["n"], case["d"]))
        qc, qs = _encode_plain(_unit_rows(g, case["nq"], case["d"]))
        if case["pad"]:
            buf = torch.zeros(case["n"], case["d"] + case["pad"], dtype=torch.int8, device="cuda")
            buf[:, :case["d"]] = xc
            xc = buf[:, :case["d"]]
        return {"case": case, "xc": xc, "xs": xs, "qc": qc, "qs": qs}
    dt = DTYPES[case["dtype"]]
    x = _unit_rows(g, case["n"], case["d"])
    t = torch.randint(0, case["n"], (case["nq"],), generator=g, device="cuda")
    # a half-trained encoder: queries lean towards their own row
    q = x[t] + 1.2 * _unit_rows(g, case["nq"], case["d"])
    q = q / q.square().sum(1, keepdim=True).sqrt()
    if case["ignored"]:
        t[torch.randperm(case["nq"], generator=g, device="cuda")[:case["ignored"]]] = IGNORE
    state = {"case": case, "q": q.to(dt), "x": x.to(dt), "t": t, "scale": 20.0}
    if case["op"] == "train" and case["reduction"] == "none":
        state["grad"] = torch.rand(case["nq"], generator=g, device="cuda") + 0.1
    return state


def _xent_plain(state):
    """Loss (per query), dlogits (softmax - onehot) and the valid mask, in fp32;
    the sum of exponentials and what is left of it without the target in 64
    bits, since the loss of a query that finds its row is next to 0."""
    q, x, t = state["q"].float(), state["x"].float(), state["t"]
    valid = t != IGNORE
    tc = torch.where(valid, t, torch.zeros_like(t))
    s = (q @ x.t()) * state["scale"]
    m = s.amax(1, keepdim=True)
    away = (m - s.gather(1, tc[:, None])).double()
    e = s.sub_(m).exp_()
    z = e.sum(1, keepdim=True, dtype=torch.float64)
    loss = (z.log() + away).float()[:, 0]
    at = ((e.gather(1, tc[:, None]) - z) / z).float()
    d = e.div_(z.float()).scatter_(1, tc[:, None], at)
    return torch.where(valid, loss, torch.zeros_like(loss)), d, valid


def _reduce(loss, valid, how):
    if how == "none":
        return loss
    return loss.sum() / valid.sum() if how == "mean" else loss.sum()


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "encode":
        return _encode_plain(state["x"])
    if case["op"] == "dot":
        # integer sums this small are exact in fp32
        acc = state["qc"].float() @ state["xc"].float().t()
        return (acc * (state["qs"][:, None] * state["xs"][None, :])).to(DTYPES[case["out"]])
    loss, d, valid = _xent_plain(state)
    total = _reduce(loss, valid, case["reduction"])
    if case["op"] == "xent":
        return total
    g = state["grad"] if case["reduction"] == "none" else torch.ones_like(loss)
    if case["reduction"] == "mean":
        g = g / valid.sum()
    g = torch.where(valid, g, torch.zeros_like(g)) * state["scale"]
    d.mul_(g[:, None])
    dq = (d @ state["x"].float()).to(state["q"].dtype)
    if not case["rows"]:
        return total, dq
    return total, dq, (d.t() @ state["q"].float()).to(state["x"].dtype)


def _run_own(case, state):
    from rapidadb import _C

    if case["op"] == "encode":
        return _C.sq8_encode(state["x"])
    if case["op"] == "dot":
        return _C.sq8_dot_product(state["qc"], state["qs"], state["xc"], state["xs"], DTYPES[case["out"]])
    from rapidadb.losses import softmax_cross_entropy

    q, x = state["q"], state["x"]
    if case["op"] == "xent":
        return softmax_cross_entropy(q, x, state["t"], scale=state["scale"], ignore_index=IGNORE,
                                     reduction=case["reduction"])
    q = q.detach().requires_grad_()
    leaves = [q]
    if case["rows"]:
        x = x.detach().requires_grad_()
        leaves.append(x)
    loss = softmax_cross_entropy(q, x, state["t"], scale=state["scale"], ignore_index=IGNORE,
                                 reduction=case["reduction"])
    return (loss.detach(), *torch.autograd.grad(loss, leaves, state.get("grad")))


def work(case):
    if case["op"] == "encode":
        n, d = case["n"], case["d"]
        return {"bytes": n * d * (SIZE[case["dtype"]] + 1) + 4 * n, "flops": 3 * n * d}
    nq, n, d = case["nq"], case["n"], case["d"]
    if case["op"] == "dot":
        return {"bytes": (nq + n) * (d + 4) + nq * n * SIZE[case["out"]], "flops": 2 * nq * n * d}
    e = SIZE[case["dtype"]]
    if case["op"] == "xent":
        return {"bytes": (nq + n) * d * e + 12 * nq, "flops": 2 * nq * n * d}
    # one product forward, one for each gradient
    grads = 2 if case["rows"] else 1
    out = nq * d * e + (n * d * e if case["rows"] else 0)
    return {"bytes": (nq + n) * d * e + out + 12 * nq, "flops": 2 * nq * n * d * (1 + grads)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "encode":
        # the codes are whole numbers of the fp32 definition; the scale has a value
        return None, st["x"].double().abs().max(dim=1).values / 127.0
    if case["op"] == "dot":
        qd, xd = st["qc"].double() * st["qs"].double()[:, None], st["xc"].double() * st["xs"].double()[:, None]
        return torch.cat([torch.einsum("bd,nd->bn", part, xd) for part in qd.split(512)])
    q, x, t = st["q"].double(), st["x"].double(), st["t"]
    keep = (t != IGNORE).nonzero()[:, 0]
    losses = torch.zeros(case["nq"], dtype=torch.float64, device=q.device)
    train = case["op"] == "train"
    dq, dx = torch.zeros_like(q), torch.zeros_like(x) if train and case["rows"] else None
    if train:
        g = st["grad"].double() if case["reduction"] == "none" else torch.ones_like(losses)
        g = g / len(keep) if case["reduction"] == "mean" else g
    for part in keep.split(256):
        logits = st["scale"] * torch.einsum("bd,nd->bn", q[part], x)
        logp = torch.log_softmax(logits, 1)
        del logits
        rows = torch.arange(len(part), device=q.device)
        losses[part] = -logp[rows, t[part]]
        if train:
            d = logp.exp_()
            d[rows, t[part]] -= 1.0
            d *= g[part][:, None] * st["scale"]
            dq[part] = torch.einsum("bn,nd->bd", d, x)
            if dx is not None:
                dx += torch.einsum("bn,bd->nd", d, q[part])
    total = losses if case["reduction"] == "none" else losses.sum()
    if case["reduction"] == "mean":
        total = total / len(keep)
    if not train:
        return total
    return (total, dq) if dx is None else (total, dq, dx)
