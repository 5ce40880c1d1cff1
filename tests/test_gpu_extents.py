"""Extents at which one launch does not hold the threads of a call (fewer than 2^32), or an extent does not fit the C ABI's
32-bit ints: the results of the whole array are those of its parts."""
import numpy as np
import pytest
import torch

from bars import say
from test_gpu_e4m3 import K, dev, host  # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # to the bit, of any type


@pytest.mark.parametrize("n", [33, 36])
def test_reduction_of_more_rows_than_a_launch_has(K, n):
    """33 elements take a wave per row, 36 four rows of a wave."""
    rows = (1 << 26) + 77
    say("reduce_sum", rows, n)
    x = torch.randint(-8, 9, (rows, n), device="cuda", dtype=torch.float32)  # (sums of integers: exact)
    got = K.reduce_sum(x, [1])
    assert got.shape == (rows,)
    step = 1 << 22
    for i in range(0, rows, step):
        assert torch.equal(got[i:i + step], x[i:i + step].sum(1)), i
