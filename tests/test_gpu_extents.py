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


@pytest.mark.parametrize("rows,n", [(1 << 26, 1), ((1 << 26) + 7, 3)])
def test_norm_of_more_rows_than_a_launch_has(K, rows, n):
    say("rms_norm", rows, n)
    x = torch.randn(rows, n, device="cuda")
    w, cut = torch.randn(n, device="cuda"), (1 << 26) - 9
    y, h, rstd = K.rms_norm(x, w, 1e-3, residual=x)
    for part in (slice(0, 50), slice(cut - 1000, cut + 9), slice(rows - 50, rows)):
        for got, want in zip((y, h, rstd), K.rms_norm(x[part], w, 1e-3, residual=x[part])):
            assert same(got[part], want)
    step = 1 << 22
    for i in range(0, rows, step):  # every row, against the definition
        h64 = 2 * x[i:i + step].double()
        want = h64 * (w.double() / (h64.square().mean(1, keepdim=True) + float(np.float32(1e-3))).sqrt())
        assert ((y[i:i + step].double() - want).abs() <= 2.0 ** -24 * (1 + 1e-6) * want.abs() + 2.0 ** -149).all()
    del y, h
    e, _, _ = K.rms_norm_e4m3(x, w, 1e-3)
    part = slice(rows - 50, rows)
    want = K.rms_norm_e4m3(x[part], w, 1e-3)[0]
    assert same(e.q[part], want.q) and same(e.scales[part], want.scales)


@pytest.mark.parametrize("rows,n", [(1, (1 << 26) + 5), (2, (1 << 27) + 5)])
def test_norm_gradient_of_more_columns_than_a_launch_has(K, rows, n):
    say("rms_norm_grad", rows, n)
    h, gy = torch.randn(rows, n, device="cuda"), torch.randn(rows, n, device="cuda")
    w, rstd = torch.randn(n, device="cuda"), torch.full((rows,), 0.75, device="cuda")
    gx, gw = K.rms_norm_grad(h, w, rstd, gy)
    c = [(gy[i].double() * w.double() * h[i].double()).sum() / n * 0.75 ** 3 for i in range(rows)]
    step = 1 << 24
    for i in range(0, n, step):
        s = slice(i, i + step)
        h64, g64, w64 = h[:, s].double(), gy[:, s].double(), w[s].double()
        first, second = 0.75 * w64 * g64, torch.stack([h64[r] * c[r] for r in range(rows)])
        # one rounding of gx (6 u cover the order of c's sum); of gw two roundings a term, `rows` of the sum, one of the result
        assert ((gx[:, s].double() - (first - second)).abs() <= 6 * 2.0 ** -24 * (first.abs() + second.abs()) + 2.0 ** -149).all()
        terms = g64 * h64 * 0.75
        assert ((gw[s].double() - terms.sum(0)).abs() <= (rows + 4) * 2.0 ** -24 * terms.abs().sum(0) + 2.0 ** -149).all()


def test_rounding_of_more_rows_than_a_launch_has(K):
    rows = (1 << 27) + 3
    say("quantize", rows, 1)
    x = torch.randn(rows, 1, device="cuda")
    e = K.quantize_e4m3(x)
    step = 1 << 22
    for i in range(0, rows, step):  # (a row of one element: its block's largest is itself)
        part = K.quantize_e4m3(x[i:i + step])
        assert same(e.q[i:i + step], part.q) and same(e.scales[i:i + step], part.scales), i


def test_rounding_of_a_column_of_more_blocks_than_a_launch_has(K):
    rows = (1 << 31) - 1
    say("quantize, transposed", rows, 1)
    x = torch.empty(rows, 1, device="cuda").normal_()
    t = K.quantize_e4m3(x, transpose=True)
    for i in (0, (1 << 31) - (1 << 20)):  # whole blocks, the last one ragged
        part = K.quantize_e4m3(x[i:i + (1 << 20)].t().contiguous())
        assert same(t.q[:, i:i + (1 << 20)], part.q)
        assert same(t.scales[:, i // 128:i // 128 + part.scales.shape[1]], part.scales)
    # every block: rounded along the rows of the array cut into rows of whole blocks
    whole = rows // 512 * 512
    cut = K.quantize_e4m3(x[:whole].view(-1, 512))
    assert same(t.q[0, :whole].view(-1, 512), cut.q) and same(t.scales[0, :whole // 128].view(-1, 4), cut.scales)


def test_product_of_more_columns_than_a_launch_has(K):
    n, k, m = (1 << 29) + 21, 8, 3
    say("product", m, n, k)
    rng = np.random.default_rng(3)
    a = dev(rng.integers(-3, 4, (m, k)))
    b = torch.empty(n, 128, dtype=torch.uint8, device="cuda").zero_()
    step = 1 << 20
    values = K.quantize_e4m3(dev(rng.integers(-3, 4, (step, k))))
    for i in range(0, n, step):
        b[i:i + step].copy_(values.q.view(torch.uint8)[: n - i])
    scales = torch.full((n, 4), 127, dtype=torch.uint8, device="cuda")
    power = values.scales.view(torch.uint8)[:, 0]
    for i in range(0, n, step):
        scales[i:i + step, 0].copy_(power[: n - i])
    e = K.E4m3(b.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), k)
    want = (a.double() @ values.values().double().t()).float()  # integers: exact
    for got in (K.quantize_matmul_e4m3(a, e), K.matmul_e4m3(K.quantize_e4m3(a), e)):
        for i in range(0, n, step):
            assert torch.equal(got[:, i:i + step], want[:, : n - i]), i


def test_extents_beyond_32_bits_are_refused(K):
    """2^32 + 8 rows would reach the library as 8."""
    from rust_autograd_amd import capi

    rows = (1 << 32) + 8
    x, w = torch.zeros(rows, 1, device="cuda"), torch.ones(1, device="cuda")
    byte, scales = torch.zeros(4, 128, dtype=torch.uint8, device="cuda"), torch.full((4, 4), 127, dtype=torch.uint8, device="cuda")
    e = K.E4m3(byte.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), 1)
    for call in (lambda: K.rms_norm(x, w), lambda: K.rms_norm_e4m3(x, w), lambda: K.rms_norm_grad(x, w, x[:, 0], x), lambda: K.quantize_e4m3(x),
                 lambda: K.quantize_e4m3(x, transpose=True), lambda: K.quantize_e4m3(x.view(1, rows)), lambda: K.quantize_e4m3_both(x),
                 lambda: K.quantize_matmul_e4m3(x, e)):
        before = torch.cuda.memory_allocated()
        with pytest.raises(capi.InvalidDims, match="2147483647"):
            call()
        assert torch.cuda.memory_allocated() == before
