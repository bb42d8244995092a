"""Kernels whose launch overlaps the end of what runs before them (chain.cuh)
are resident while that still writes their inputs.  Loads through the read-only
path (``__ldg``, ``ld.global.nc``, or the ones a compiler makes of a ``const
__restrict__`` parameter) need data that stays as it is for the whole life of
the kernel, and are not held back by the wait."""
import glob
import os
import re

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rapidadb_b200", "csrc")


def code_of(path):
    text = open(path).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def chained_files():
    """chain.cuh, what it includes, and every file that includes it, also through others."""
    names = [os.path.basename(p) for ext in ("*.cu", "*.cuh") for p in glob.glob(os.path.join(CSRC, ext))]
    code = {n: code_of(os.path.join(CSRC, n)) for n in names}
    includes = {n: set(re.findall(r'#include "([^"]+)"', code[n])) & set(names) for n in names}
    files = {"chain.cuh"}
    while True:
        more = {n for n in names if includes[n] & files} - files
        if not more:
            break
        files |= more
    for n in sorted(files):  # headers whose functions the kernels call
        stack = [n]
        while stack:
            for h in includes[stack.pop()] - files:
                files.add(h)
                stack.append(h)
    return {n: code[n] for n in files}


def test_the_files_are_found():
    assert {"chain.cuh", "rows.cu", "sq8.cu", "sq8_dot.cu", "xent.cu", "tile_tc.cuh", "tile_f32.cuh"} <= set(chained_files())


def test_no_read_only_loads_in_chained_kernels():
    for name, code in chained_files().items():
        for pattern in (r"__ldg\s*\(", r"ld\.global(\.\w+)*\.nc", r"\bconst\b[^,;(){}]*\*\s*(const\s+)?__restrict__",
                        r"__constant__\b", r"\btex(1D|2D|3D)?fetch\b|\btex[123]D\b"):
            hit = re.search(pattern, code)
            assert not hit, f"{name}: {hit.group(0)}"


def in_a_row(device, step, inputs, rounds=40):
    """step(i) -> tensors, run back to back on inputs that change between the
    rounds, gives the bits of the same calls with a synchronisation after each
    (step synchronises through its argument)."""
    def run(sync):
        cur = [v.clone() for v in inputs]
        out = []
        for i in range(rounds):
            out += step(cur, i, sync)
            for v in cur:
                v.mul_(-1.0009765625)  # overwrites what the calls before read
        return out

    want = run(torch.cuda.synchronize)
    got = run(lambda: None)
    torch.cuda.synchronize()
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.isnan().any()


DT = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("nq,n,d", [(1, 700, 50), (1, 40000, 50), (1, 3000, 769), (4, 900, 99), (9, 5000, 51),
                                    (100, 3000, 131)])
def test_a_row_copy_right_before_the_loss(device, nq, n, d, dtype):
    """Rows without 16-byte strides are copied by one launch, and the next one
    reads the copy: streamed (one query, fp32 up to four), split on the way
    (fp32), or by TMA."""
    from rapidadb.losses import softmax_cross_entropy

    g = torch.Generator().manual_seed(n + d)
    q = (torch.randn(nq, d, generator=g) / d ** 0.5).to(dtype).to(device)
    x = torch.randn(n, d, generator=g).to(dtype).to(device)
    t = torch.randint(0, n, (nq,), generator=g).to(device)

    def step(cur, i, sync):
        a, b = cur[0].detach().requires_grad_(), cur[1].detach().requires_grad_()
        loss = softmax_cross_entropy(a, b, t, scale=2.0, reduction="none")
        sync()
        dq, dx = torch.autograd.grad(loss, (a, b), torch.ones_like(loss))
        sync()
        alone = softmax_cross_entropy(cur[0], cur[1], t, scale=3.0)
        sync()
        return [loss.detach(), dq, dx, alone]

    in_a_row(device, step, [q, x])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("nq", [1, 2, 3])
@pytest.mark.parametrize("n,d", [(900, 64), (30000, 768), (2000, 50), (700, 333)])
def test_codes_scored_right_after_they_are_made(device, n, d, nq, dtype):
    """Quantise rows and queries, score: every launch reads what the one before
    it wrote (codes and scales; a copy of the codes where d is no multiple of 16)."""
    import rapidadb._C as C

    g = torch.Generator().manual_seed(n + d + nq)
    q = torch.randn(nq, d, generator=g).to(dtype).to(device)
    x = torch.randn(n, d, generator=g).to(dtype).to(device)

    def step(cur, i, sync):
        c, s = C.sq8_encode(cur[1])
        sync()
        qc, qs = C.sq8_encode(cur[0])
        sync()
        one = C.sq8_dot_product(qc, qs, c, s)
        sync()
        c2, s2 = C.sq8_encode(cur[1])  # rows right before the product
        sync()
        two = C.sq8_dot_product(qc, qs, c2, s2)
        sync()
        del c, s, qc, qs, c2, s2  # the allocator hands their memory on
        return [one, two]

    in_a_row(device, step, [q, x])
