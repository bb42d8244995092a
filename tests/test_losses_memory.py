"""Workspace of the softmax cross entropy: the bounds that its header states,
over sizes up to millions of queries, rows and thousands of columns."""
import ctypes
import os

import pytest

MB = 1 << 20
FP32, FP16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(os.path.dirname(__file__), "..", "rapidadb_b200", "librdb_kernels.so"))
    i, i64 = ctypes.c_int, ctypes.c_int64
    lib.rdb_softmax_xent_workspace.restype = lib.rdb_softmax_xent_backward_workspace.restype = ctypes.c_size_t
    lib.rdb_softmax_xent_workspace.argtypes = [i, i64, i64, i, i]
    lib.rdb_softmax_xent_backward_workspace.argtypes = [i, i64, i64, i, i, i]
    return lib


SIZES = [(1, 1, 1), (1, 10 ** 7, 768), (64, 10 ** 6, 768), (128, 10 ** 6, 1024), (129, 10 ** 6, 1024),
         (4096, 131072, 768), (8192, 10 ** 6, 128), (8193, 10 ** 5, 100_000), (20_000, 50_000, 8192),
         (131_072, 10 ** 6, 768), (262_144, 262_144, 1024), (10 ** 6, 10 ** 6, 768), (8 * 10 ** 6, 10 ** 5, 64),
         (2 ** 31 - 1, 5, 8), (300, 2 ** 31 - 1, 16), (3, 7, 10 ** 6)]


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("nq,n,d", SIZES)
def test_forward_bound(lib, dtype, nq, n, d):
    got = lib.rdb_softmax_xent_workspace(dtype, nq, n, d, 1)
    bound = 64 * nq + 32 * MB
    if dtype == FP32:
        d8 = (d + 7) // 8 * 8
        pieces = 1 + n // max(256, 256 * MB // (6 * d8) // 512 * 256) if nq > 128 else 1
        bound += 6 * d8 * nq + (max(256 * MB, 1536 * d8) + pieces * max(10 * MB, 32 * nq) if nq > 128 else 0)
    assert 0 < got <= bound


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("need_dq,need_dx", [(1, 1), (1, 0), (0, 1), (0, 0)])
@pytest.mark.parametrize("nq,n,d", SIZES)
def test_backward_bound(lib, dtype, nq, n, d, need_dq, need_dx):
    got = lib.rdb_softmax_xent_backward_workspace(dtype, nq, n, d, need_dq, need_dx)
    planes = 3 if dtype == FP32 else 1
    d8, d32 = (d + 7) // 8 * 8, (d + 31) // 32 * 32
    per_row = 2 * planes * nq
    bound = max(512 * MB, min(2048 * MB, 4096 * per_row), 256 * per_row) + MB
    if need_dq:
        bound += max(64 * MB, 4 * d32 * nq)
    if need_dx:
        bound += 2 * planes * d8 * nq
    if dtype == FP32:
        bound += 6 * d8 * nq + (max(256 * MB, 1536 * d8) if nq > 128 else 0)
    elif need_dx and nq > 8192:
        bound += max(512 * MB, 1024 * d32)
    assert 0 < got <= bound


def test_common_sizes_stay_small(lib):
    """No more than the sizes that training on one GPU meets need."""
    assert lib.rdb_softmax_xent_backward_workspace(BF16, 4096, 131072, 768, 1, 1) <= 640 * MB
    assert lib.rdb_softmax_xent_backward_workspace(FP32, 128, 10 ** 6, 768, 1, 0) <= 640 * MB
    assert lib.rdb_softmax_xent_workspace(BF16, 1024, 10 ** 6, 768, 1) <= 32 * MB
