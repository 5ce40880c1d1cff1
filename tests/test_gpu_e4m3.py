"""8-bit operands and their product on the GPU, through the C ABI, against 64-bit forms.

Rounding to 8 bits is exact integer and power-of-two arithmetic plus one rounding, so it is held to the bits.  The product
of two 8-bit values is exact in f32; what is left are the roundings of the sums.  With small integers every partial sum is
an integer below 2^24 and the result is exact whatever the order.  Otherwise, for a result of K terms that is summed in
steps of 64 terms, each step rounding the running sum (at most a whole unit, 2^-23 of it, should the matrix unit cut
instead of rounding) after rounding inside the step (a tree over 64 terms and the running sum: 7 levels, 2^-23 each), and
then over at most 32 slices of the contraction and waves (2^-24 each):
    |got - truth| <= ((K / 64 + 7) * 2^-23 + 32 * 2^-24) * (|A| . |B|).
"""
import numpy as np
import pytest
import torch

import plain64
from bars import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    import __graft_entry__ as entry
    entry.load_package()
    from rust_autograd_amd import kernels
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return kernels


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def scale_bytes(e):
    return e.scales.view(torch.uint8).cpu().numpy()


def assert_same_operand(e, x, what):
    q, b = plain64.quantize(x)
    assert e.q.shape == q.shape and e.scales.shape == b.shape, what
    assert np.array_equal(scale_bytes(e), b), f"{what}: scales"
    got = host(e.q)
    assert np.array_equal(np.isnan(got), np.isnan(q)), f"{what}: NaN"
    assert np.array_equal(np.nan_to_num(got), np.nan_to_num(q)), f"{what}: values"


def tolerance(k, absdot):
    return ((k / 64 + 7) * 2.0 ** -23 + 32 * 2.0 ** -24) * absdot


def sample(rng, rows, n):
    """Rows of very different size, a row and a block of zeros among them."""
    x = rng.standard_normal((rows, n)) * np.exp2(rng.integers(-30, 30, (rows, 1)))
    x[:, : min(n, 128)] *= np.exp2(rng.integers(-20, 1, (rows, 1)))
    if rows > 2:
        x[2] = 0.0
    if n > 256 and rows > 1:
        x[1, 128:256] = 0.0
    return x.astype(np.float32)


SHAPES = [(1, 1), (1, 4096), (3, 127), (2, 128), (5, 129), (4, 512), (7, 513), (33, 1000), (130, 384), (257, 1025), (128, 128), (1000, 3)]


@pytest.mark.parametrize("rows,n", SHAPES)
def test_rounding_has_the_bits_of_the_definition(K, rng, rows, n):
    say("quantize", rows, n)
    x = sample(rng, rows, n)
    assert_same_operand(K.quantize_e4m3(dev(x)), x, "rows")
    assert_same_operand(K.quantize_e4m3(dev(x), transpose=True), x.T, "columns")
    e, t = K.quantize_e4m3_both(dev(x))
    assert_same_operand(e, x, "both: rows")
    assert_same_operand(t, x.T, "both: columns")
    assert np.array_equal(host(e.values()), plain64.rounded(x))


def test_rounding_of_every_f32_exponent_ties_and_what_is_not_finite(K):
    # a tie in every binade of e4m3 (16.5 of 16 steps and the like), the largest value, its neighbours, subnormals
    base = np.concatenate([np.arange(1, 32) / 16.0, [448, 447.99997, 432, 431.99997, 464 / 448 * 448 / 2, 2 ** -9, 2 ** -10, 3 * 2 ** -10, 0.0]])
    x = np.zeros((254, 128), dtype=np.float32)
    for i, e in enumerate(range(-126, 128)):
        with np.errstate(over="ignore"):
            x[i, : len(base)] = (base * 2.0 ** (e - 9)).astype(np.float32)
            x[i, -1] = 448.0 * 2.0 ** (e - 9) if e - 9 < 119 else 2.0 ** e
        x[i, 64:64 + len(base)] = -x[i, : len(base)]
    x[~np.isfinite(x)] = 0.0
    assert_same_operand(K.quantize_e4m3(dev(x)), x, "binades")
    y = np.ones((6, 300), dtype=np.float32)
    y[0, 5] = np.inf
    y[1, 200] = -np.inf
    y[2, 299] = np.nan
    y[3, :128] = np.inf
    y[4] = np.nan
    y[5, 7] = np.finfo(np.float32).max
    assert_same_operand(K.quantize_e4m3(dev(y)), y, "not finite")
    e, t = K.quantize_e4m3_both(dev(y))
    assert_same_operand(e, y, "not finite, rows")
    assert_same_operand(t, y.T, "not finite, columns")
    tiny = np.full((2, 130), np.float32(1e-45))
    tiny[1] = np.float32(2.0 ** -120)
    assert_same_operand(K.quantize_e4m3(dev(tiny)), tiny, "subnormal")


def test_rounding_reads_a_strided_view(K, rng):
    x = sample(rng, 40, 300)
    assert_same_operand(K.quantize_e4m3(dev(x)[:, 17:205]), x[:, 17:205], "view")
    assert_same_operand(K.quantize_e4m3(dev(x).t()), x.T, "transposed view")
    # through the C ABI with a row stride, from a start that is no multiple of 16 bytes
    from rust_autograd_amd import capi
    d = dev(x)
    e, t = K.quantize_e4m3_both(torch.zeros(40, 188, device="cuda"))
    src = d[:, 17:205]
    capi.check(capi.lib().ag_quantize_e4m3_f32(K._stream(), src.data_ptr(), 300, 40, 188, e.q.data_ptr(), e.scales.data_ptr(), t.q.data_ptr(),
                                               t.scales.data_ptr()))
    assert_same_operand(e, x[:, 17:205], "stride, rows")
    assert_same_operand(t, x[:, 17:205].T, "stride, columns")


# extents around the tiles and blocks of the kernels, and the skinny ones
PRODUCTS = [(1, 1, 1), (1, 17, 128), (1, 4096, 512), (2, 100, 300), (5, 33, 129), (16, 16, 128), (16, 1000, 4096), (17, 255, 640), (31, 64, 1000),
            (48, 129, 2048), (63, 500, 513), (64, 128, 128), (65, 127, 384), (128, 128, 1024), (129, 257, 130), (200, 1, 700), (255, 256, 257),
            (256, 256, 256), (257, 513, 1100), (300, 2000, 8192), (512, 512, 640), (1000, 1999, 2500), (1024, 768, 128), (30, 5000, 700),
            (33, 4000, 4100), (20, 4096, 4096), (64, 300, 16400)]
# tiles of 128 four steps and two steps deep and of 256, contractions of one to six steps
PRODUCTS += [(m, n, k) for m, n in ((1030, 3900), (1990, 4000), (2100, 4400)) for k in (100, 256, 300, 512, 640, 768)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_integers_is_exact(K, rng, m, n, k):
    """Integers of magnitude up to 3 (times a power of two per row) are exact in 8 bits and their sums exact in f32."""
    say("product", m, n, k)
    sa, sb = np.exp2(rng.integers(-8, 8, (m, 1))), np.exp2(rng.integers(-8, 8, (n, 1)))
    a, b = rng.integers(-3, 4, (m, k)) * sa, rng.integers(-3, 4, (n, k)) * sb
    got = host(K.matmul_e4m3(K.quantize_e4m3(dev(a)), K.quantize_e4m3(dev(b))))
    want = a @ b.T
    assert np.array_equal(got, want), f"{(got != want).sum()} of {got.size} differ"
    got = host(K.quantize_matmul_e4m3(dev(a), K.quantize_e4m3(dev(b))))
    assert np.array_equal(got, want), f"from f32: {(got != want).sum()} of {got.size} differ"


@pytest.mark.parametrize("m,n,k", [p for p in PRODUCTS if p[2] > 1])
def test_product_within_the_roundings_of_its_sums(K, rng, m, n, k):
    say("product", m, n, k)
    a = rng.standard_normal((m, k)) * np.exp2(rng.integers(-6, 6, (1, k)))
    b = rng.standard_normal((n, k)) * np.exp2(rng.integers(-6, 6, (n, 1)))
    a, b = a.astype(np.float32), b.astype(np.float32)
    ra, rb = plain64.rounded(a), plain64.rounded(b)
    qb = K.quantize_e4m3(dev(b))
    for what, got in (("8-bit", K.matmul_e4m3(K.quantize_e4m3(dev(a)), qb)), ("f32", K.quantize_matmul_e4m3(dev(a), qb))):
        err = np.abs(host(got) - ra @ rb.T)
        size = np.abs(ra) @ np.abs(rb).T
        say(what, "worst error over |A|.|B|: %.2e, allowed %.2e" % ((err / np.maximum(size, 1e-300)).max(), tolerance(k, 1.0)))
        assert (err <= tolerance(k, size)).all(), what


@pytest.mark.parametrize("m,k,n", [(64, 128, 64), (130, 200, 300), (1, 500, 33), (513, 257, 129)])
def test_gradients_are_the_products_of_the_formula(K, rng, m, k, n):
    """y = x . w with integer operands: exact, so the products of the gradients are those of the formula, and a finite
    difference of sum(gy * y) along any direction of integers gives them exactly too."""
    x, w, gy = rng.integers(-3, 4, (m, k)), rng.integers(-3, 4, (k, n)), rng.integers(-2, 3, (m, n))
    (qx, qxt), (qw, qwt), (qg, qgt) = (K.quantize_e4m3_both(dev(a)) for a in (x, w, gy))
    assert np.array_equal(host(K.matmul_e4m3(qx, qwt)), x @ w)
    gx, gw = host(K.matmul_e4m3(qg, qw)), host(K.matmul_e4m3(qxt, qgt))
    assert np.array_equal(gx, gy @ w.T) and np.array_equal(gw, x.T @ gy)
    dx, dw = rng.integers(-1, 2, (m, k)), rng.integers(-1, 2, (k, n))

    def loss(x, w):
        return (host(K.matmul_e4m3(K.quantize_e4m3(dev(x)), K.quantize_e4m3(dev(w), transpose=True))) * gy).sum()

    # exact: the loss is linear in either operand, and integers up to 16 are exact in 8 bits
    assert loss(x + dx, w) - loss(x - dx, w) == 2 * (gx * dx).sum()
    assert loss(x, w + dw) - loss(x, w - dw) == 2 * (gw * dw).sum()


@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (40, 96, 384), (200, 300, 512)])
def test_nan_reaches_its_row_and_column_only(K, rng, m, n, k):
    a, b = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    clean = host(K.matmul_e4m3(K.quantize_e4m3(dev(a)), K.quantize_e4m3(dev(b))))
    a[m // 2, 3], b[n // 3, k - 1] = np.inf, np.nan
    for got in (K.matmul_e4m3(K.quantize_e4m3(dev(a)), K.quantize_e4m3(dev(b))), K.quantize_matmul_e4m3(dev(a), K.quantize_e4m3(dev(b)))):
        got = host(got)
        hit = np.zeros((m, n), dtype=bool)
        hit[m // 2], hit[:, n // 3] = True, True
        assert np.array_equal(np.isnan(got), hit)
        assert np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("m,n,k", [(3, 200, 512), (200, 300, 1000)])
def test_output_rows_keep_what_lies_between_them(K, rng, m, n, k):
    """ldc > N: the columns behind a row of the result are not written; empty contractions give zeros."""
    from rust_autograd_amd import capi
    L = capi.lib()
    a, b = rng.integers(-3, 4, (m, k)), rng.integers(-3, 4, (n, k))
    ea, eb = K.quantize_e4m3(dev(a)), K.quantize_e4m3(dev(b))
    out = torch.full((m, n + 13), 7.0, device="cuda")
    nb = max(L.ag_matmul_e4m3_f32_workspace(m, n, k), 16)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    capi.check(L.ag_matmul_e4m3_f32(K._stream(), m, n, k, ea.q.data_ptr(), ea.scales.data_ptr(), eb.q.data_ptr(), eb.scales.data_ptr(),
                                    out.data_ptr(), n + 13, ws.data_ptr(), nb))
    got = host(out)
    assert np.array_equal(got[:, :n], a @ b.T) and (got[:, n:] == 7.0).all()
    capi.check(L.ag_matmul_e4m3_f32(K._stream(), m, n, 0, None, None, None, None, out.data_ptr(), n + 13, ws.data_ptr(), nb))
    got = host(out)
    assert (got[:, :n] == 0.0).all() and (got[:, n:] == 7.0).all()


@pytest.mark.parametrize("m,n", [(1, 64), (30, 64), (200, 300), (1030, 3900), (2100, 4400)])
def test_products_at_the_ends_of_the_scales(K, m, n):
    """Every value that bf16 holds enters exactly, whatever the byte, and a smaller one rounded to nearest; from 1.9375 * 2^127 on an f32 is rounded to 2^128, which
    counts as an infinity."""
    def product(byte, value, power):
        q, s = torch.zeros(m, 128, device="cuda"), torch.full((m, 4), 127, dtype=torch.uint8, device="cuda")
        q[:, 5], s[:, 0] = value, byte
        b = torch.zeros(n, 128, device="cuda")
        b[:, 5] = 2.0 ** power
        return K.matmul_e4m3(K.E4m3(q.to(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu), 128), K.quantize_e4m3(b))

    for byte, value in ((0, 1.0), (1, 1.0), (1, 1.75 * 2.0 ** -6), (5, 2.0 ** -9), (9, 2.0 ** -9), (10, 2.0 ** -9), (10, 448.0), (247, 2.0 ** -9),
                        (247, -240.0), (248, 1.0), (254, -1.875)):
        power = -60 if byte > 127 else 60
        # multiples of 2^-133 are what bf16 holds below 2^-126: 1.75 * 2^-6 * 2^-126 = 3.5 * 2^-133 lies between two of them
        # and is rounded to the even one, 4 * 2^-133; every other value of the list is a multiple
        held = np.round(value * 2.0 ** (byte - 127 + 133)) * 2.0 ** -133
        assert held == (2.0 ** -131 if value == 1.75 * 2.0 ** -6 else value * 2.0 ** (byte - 127))
        assert (product(byte, value, power) == held * 2.0 ** power).all(), (byte, value)
    assert torch.isinf(product(254, 2.0, -60)).all() and torch.isnan(product(255, 1.0, -60)).all()
    a, b = torch.zeros(m, 128, device="cuda"), torch.zeros(n, 128, device="cuda")
    b[:, 0] = 2.0 ** -20
    for value, want in ((1.9375 * 2.0 ** 127 * (1 - 2.0 ** -23), 1.875 * 2.0 ** 107), (1.9375 * 2.0 ** 127, np.inf), (-3.4028234e38, -np.inf)):
        a[:, 0] = value
        assert (K.quantize_matmul_e4m3(a, K.quantize_e4m3(b)) == want).all(), value


def test_empty_extents(K):
    z = torch.zeros
    assert K.quantize_e4m3(z(0, 40, device="cuda")).q.shape == (0, 128)
    e = K.quantize_e4m3(z(5, 40, device="cuda"))
    assert K.matmul_e4m3(K.quantize_e4m3(z(0, 40, device="cuda")), e).shape == (0, 5)
    assert K.quantize_matmul_e4m3(z(0, 40, device="cuda"), e).shape == (0, 5)
    y = K.matmul_e4m3(K.quantize_e4m3(z(5, 0, device="cuda")), K.quantize_e4m3(z(7, 0, device="cuda")))
    assert y.shape == (5, 7) and not y.any()


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (40, 640, 2048), (128, 256, 4096), (300, 520, 1000)])
def test_same_bits_on_another_stream_and_from_a_graph(K, rng, m, n, k):
    """A captured step (rounding and product) replayed several times on changing inputs, with eager work between the
    replays; and the same call on a side stream."""
    a = dev(rng.standard_normal((m, k)))
    b = K.quantize_e4m3(dev(rng.standard_normal((n, k))))
    eager = K.quantize_matmul_e4m3(a, b).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = K.quantize_matmul_e4m3(a, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = K.quantize_matmul_e4m3(a, b)
        second = K.matmul_e4m3(K.quantize_e4m3(a), b)
    for i in range(4):
        a.copy_(dev(rng.standard_normal((m, k))))
        graph.replay()
        torch.cuda.synchronize()
        want = K.quantize_matmul_e4m3(a, b)
        two = K.matmul_e4m3(K.quantize_e4m3(a), b)
        torch.cuda.synchronize()
        assert torch.equal(captured, want), f"replay {i}"
        assert torch.equal(second, two), f"replay {i}, in two calls"


def test_offsets_beyond_32_bits(K, rng):
    """2.4 * 10^9 elements: the last rows of the array come out as they do alone, in every form that reads or writes them."""
    rows, k, last = 600_000, 4096, 70
    tail = dev(rng.integers(-3, 4, (last, k)))
    x = torch.zeros(rows, k, device="cuda")
    x[-last:] = tail
    small = dev(rng.integers(-3, 4, (40, k)))
    qs, qtail = K.quantize_e4m3(small), K.quantize_e4m3(tail)
    e = K.quantize_e4m3(x)
    assert torch.equal(e.q[-last:].view(torch.uint8), qtail.q.view(torch.uint8)) and torch.equal(e.scales[-last:].view(torch.uint8), qtail.scales.view(torch.uint8))
    want = (tail.double() @ small.double().t()).float()  # integers: exact in every order
    assert torch.equal(K.matmul_e4m3(e, qs)[-last:], want)
    assert torch.equal(K.matmul_e4m3(qs, e)[:, -last:], want.t())
    one = K.quantize_matmul_e4m3(small[:1], e)
    assert torch.equal(one[0, -last:], want[:, 0]) and not one[0, :-last].any()
    del e, one
    torch.cuda.empty_cache()
    e, t = K.quantize_e4m3_both(x)
    assert torch.equal(e.q[-last:].view(torch.uint8), qtail.q.view(torch.uint8))
    assert not t.q[:, rows - last - 1000: rows - last].float().any()
    # 600000 = 4687 * 128 + 64: the last block of a column holds the last 64 rows
    got = host(t.q[:, 4687 * 128: rows]) * np.exp2(t.scales.view(torch.uint8)[:, 4687:4688].cpu().numpy().astype(np.float64) - 127)
    assert np.array_equal(got, host(tail[-64:]).T)
    del e, t
    torch.cuda.empty_cache()
    w = torch.ones(k, device="cuda")
    y, h, rstd = K.rms_norm(x, w, 1e-6, residual=x)
    y1, h1, rstd1 = K.rms_norm(tail, w, 1e-6, residual=tail)
    assert torch.equal(y[-last:], y1) and torch.equal(h[-last:], h1) and torch.equal(rstd[-last:], rstd1)
    gx, _ = K.rms_norm_grad(h, w, rstd, y)
    gx1, _ = K.rms_norm_grad(h1, w, rstd1, y1)
    assert torch.equal(gx[-last:], gx1)
    del y, gx
    outs, clip = K.clip_by_global_norm([x, h], 1.0, outs=[x, h])
    norm = np.sqrt((host(tail) ** 2).sum() * 5)  # h is twice x
    assert abs(host(clip)[0] - norm) <= 2.0 ** -24 * (1 + 1e-6) * norm
    assert torch.equal(x[-last:], tail * clip[1]) and torch.equal(h[-last:], h1 * clip[1])


# ---- every form of the product, by the number of CUs ------------------------------------------------------------------
def form(m, n, k, cus):
    """The form that the extents choose: (tile, steps in flight, whether the contraction is sliced), tile 0 for few rows."""
    steps = -(-k // 128)

    def tiles(t):
        return -(-m // t) * -(-n // t)

    if m <= 16 or (m <= 32 and n <= 16 * cus and steps <= 32):
        return 0, 16 if m <= 16 else 32, False
    if tiles(64) <= 2 * cus:
        return 64, 4, min(cus // tiles(64), steps // 8) > 1
    if tiles(128) <= cus:
        return 128, 4, False
    return (128, 2, False) if -(-tiles(128) // (2 * cus)) * 62 < -(-tiles(256) // cus) * 100 else (256, 2, False)


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def a_tile_of_128_per_cu():
    """Ragged extents of as many tiles of 128 as there are CUs."""
    return 8 * 128 - 4, cus() // 8 * 128 - 6


@pytest.mark.parametrize("k", [1, 100, 128, 256, 300, 512, 640, 768, 1025, 1300])
def test_tiles_of_128_four_steps_deep(K, rng, k):
    """One to eleven steps through a ring of four."""
    m, n = a_tile_of_128_per_cu()
    assert form(m, n, k, cus()) == (128, 4, False)
    test_product_of_integers_is_exact(K, rng, m, n, k)
    if k > 1:
        test_product_within_the_roundings_of_its_sums(K, rng, m, n, k)


def test_the_extents_of_these_tests_reach_every_form():
    reached = {form(m, n, k, cus()) for m, n, k in PRODUCTS} | {form(*a_tile_of_128_per_cu(), 768, cus())}
    assert reached == {(0, 16, False), (0, 32, False), (64, 4, False), (64, 4, True), (128, 4, False), (128, 2, False), (256, 2, False)}


def test_values_of_an_operand_at_the_ends_of_the_scales(K):
    """What values() says is what the product reads: byte 0 is 2^-127, 255 is NaN."""
    q = torch.ones(7, 128, device="cuda")
    scales = torch.tensor([0, 1, 10, 127, 247, 254, 255], dtype=torch.uint8, device="cuda")[:, None].expand(7, 4).contiguous()
    got = host(K.E4m3(q.to(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), 100).values())
    want = np.exp2(np.array([0.0, 1, 10, 127, 247, 254, np.nan]) - 127)
    assert got.shape == (7, 100) and np.array_equal(got, np.repeat(want[:, None], 100, axis=1), equal_nan=True)
