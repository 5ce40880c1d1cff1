"""RMS norm, clipping by the global norm and the clipped Adam update on the GPU, through the C ABI, against 64-bit forms.

u = 2^-24 is half a step of f32.  Tolerances count the roundings that the kernels make:
  h     one addition                                              exact against the f32 sum
  y     64 bits, rounded once                                     u |y|  (and 2^-149, half a step of the smallest values)
  rstd  64 bits, rounded once                                     u |rstd|
  gx    its first term carries the rounding of rstd and two products, its second those of rstd three times over (its
        cube), of c and of the multiply-add, and the sum with gh one more: 6 u (|first| + |second| + |gh|)
  gw    terms gy h rstd carry two roundings, a block adds its rows in f32 in turn (at most `rows`), then 64 bits rounded
        once: (rows + 4) u sum |gy h rstd|
  norm, coefficient   64 bits, rounded once each
"""
import numpy as np
import pytest
import torch

import plain64
from bars import say
from test_gpu_e4m3 import assert_same_operand, dev, host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 2.0 ** -149


@pytest.fixture(scope="module")
def K():
    import __graft_entry__ as entry
    entry.load_package()
    from rust_autograd_amd import kernels
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return kernels


def sample(rng, rows, n):
    return (rng.standard_normal((rows, n)) * np.exp2(rng.integers(-12, 12, (rows, 1)))).astype(np.float32)


WIDTHS = [1, 2, 3, 4, 5, 63, 127, 128, 129, 511, 512, 513, 1000, 1023, 1024, 1025, 2047, 2048, 2050, 4095, 4096, 4097, 5001, 8191, 8192, 8193, 16384,
          16385, 32768, 32769, 40001]


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("rows,with_residual", [(1, True), (5, False), (6, True)])
def test_norm_is_the_formula_rounded_once(K, rng, rows, with_residual, n):
    say("rms_norm", rows, n, with_residual)
    x, w = sample(rng, rows, n), (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    res = sample(rng, rows, n) if with_residual else None
    h32 = x + res if with_residual else x
    eps = np.float32(1e-5)
    y, h, rstd = K.rms_norm(dev(x), dev(w), float(eps), residual=None if res is None else dev(res))
    assert np.array_equal(h.cpu().numpy(), h32)
    want, r = plain64.rms_norm(h32, w, float(eps))
    assert (np.abs(host(y) - want) <= U * (1 + 1e-6) * np.abs(want) + TINY).all()
    assert (np.abs(host(rstd) - r) <= U * (1 + 1e-6) * r).all()
    e, h2, rstd2 = K.rms_norm_e4m3(dev(x), dev(w), float(eps), residual=None if res is None else dev(res))
    assert_same_operand(e, y.cpu().numpy(), "8-bit output")
    assert torch.equal(h2, h) and torch.equal(rstd2, rstd)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 7, 253, 254, 257, 509, 1021, 1022, 1023, 2045, 2047, 4093, 4095, 5003, 8190, 16381, 16383])
@pytest.mark.parametrize("places", [(0, 0, 0, 0), (1, 1, 1, 1), (3, 3, 3, 3), (2, 2, 2, 1), (0, 1, 2, 3)])
def test_rows_and_arrays_that_start_anywhere_in_a_line(K, rng, places, n):
    """Arrays whose first elements lie 0 to 3 elements behind a 16-byte boundary, alike or not: values, and nothing written
    in front of or behind them."""
    from rust_autograd_amd import capi
    L = capi.lib()
    rows = 13

    def array(place, value=None):
        buf = torch.full((rows * n + 16,), 7.0, device="cuda")
        view = buf[4 + place:4 + place + rows * n].view(rows, n)
        if value is not None:
            view.copy_(value)
        return buf, view

    def untouched(buf, place):
        return bool((buf[:4 + place] == 7.0).all()) and bool((buf[4 + place + rows * n:] == 7.0).all())

    w = dev(1 + 0.2 * rng.standard_normal(n))
    x, res, gy = (dev(sample(rng, rows, n)) for _ in range(3))
    (_, vx), (_, vr), (bh, vh), (by, vy) = array(places[0], x), array(places[1], res), array(places[2]), array(places[3])
    rstd = torch.empty(rows, device="cuda")
    capi.check(L.ag_rms_norm_f32(K._stream(), vx.data_ptr(), vr.data_ptr(), w.data_ptr(), 1e-6, vh.data_ptr(), vy.data_ptr(), None, None,
                                 rstd.data_ptr(), rows, n))
    h32 = x.cpu().numpy() + res.cpu().numpy()
    eps = float(np.float32(1e-6))
    want, r = plain64.rms_norm(h32, host(w), eps)
    assert np.array_equal(vh.cpu().numpy(), h32)
    assert (np.abs(host(vy) - want) <= U * (1 + 1e-6) * np.abs(want) + TINY).all()
    assert (np.abs(host(rstd) - r) <= U * (1 + 1e-6) * r).all()
    assert untouched(bh, places[2]) and untouched(by, places[3])
    (_, vg), (bx, vgx) = array(places[2], gy), array(places[3])
    gw_buf = torch.full((n + 8,), 7.0, device="cuda")
    nb = L.ag_rms_norm_grad_f32_workspace(rows, n)
    ws = torch.full((nb // 4 + 8,), 7.0, device="cuda")
    capi.check(L.ag_rms_norm_grad_f32(K._stream(), vh.data_ptr(), w.data_ptr(), rstd.data_ptr(), vg.data_ptr(), vx.data_ptr(), vgx.data_ptr(),
                                      gw_buf[3:].data_ptr(), rows, n, ws.data_ptr(), nb))
    want_x, want_w, size_x, size_w = plain64.rms_norm_grad(h32, host(w), eps, host(gy), host(x))
    assert (np.abs(host(vgx) - want_x) <= 6 * U * size_x + TINY).all()
    assert (np.abs(host(gw_buf[3:3 + n]) - want_w) <= (rows + 4) * U * size_w + TINY).all()
    assert untouched(bx, places[3]) and (gw_buf[:3] == 7.0).all() and (gw_buf[3 + n:] == 7.0).all() and (ws[nb // 4:] == 7.0).all()


def test_norm_of_many_rows_and_leading_axes(K, rng):
    x, w = sample(rng, 3000, 257), sample(rng, 1, 257)[0]
    y, _, _ = K.rms_norm(dev(x).view(30, 100, 257), dev(w), 1e-6)
    want, _ = plain64.rms_norm(x, w, float(np.float32(1e-6)))  # (the operator takes eps in f32)
    assert (np.abs(host(y).reshape(3000, 257) - want) <= U * (1 + 1e-6) * np.abs(want) + TINY).all()


def test_norm_at_the_ends_of_f32(K):
    """Squares beyond f32's range, zeros with eps 0, infinities and NaN."""
    n = 200
    x = np.ones((6, n), dtype=np.float32)
    x[0] *= 3e38
    x[1] *= 1e-40
    x[2] = 0.0
    x[3, 7] = np.inf
    x[4, 9] = np.nan
    w = np.ones(n, dtype=np.float32)
    y, _, rstd = K.rms_norm(dev(x), dev(w), 1e-12)
    y = host(y)
    assert np.allclose(y[0], 1.0, rtol=2 * U, atol=0) and (y[2] == 0).all()
    assert np.allclose(y[1], x[1].astype(np.float64) / np.sqrt((x[1].astype(np.float64) ** 2).mean() + np.float64(np.float32(1e-12))), rtol=2 * U, atol=TINY)
    assert np.isnan(y[3, 7]) and (np.delete(y[3], 7) == 0).all()  # 1 / inf = 0, and inf * 0
    assert np.isnan(y[4]).all() and np.allclose(y[5], 1.0, rtol=1e-6)
    y, _, _ = K.rms_norm(dev(x[2:3]), dev(w), 0.0)
    assert np.isnan(host(y)).all()  # 0 / 0
    e, _, _ = K.rms_norm_e4m3(dev(x), dev(w), 1e-12)
    assert_same_operand(e, K.rms_norm(dev(x), dev(w), 1e-12)[0].cpu().numpy(), "8-bit")


@pytest.mark.parametrize("n", [100, 4096, 20000, 40001])
def test_norm_outputs_may_be_the_inputs(K, rng, n):
    from rust_autograd_amd import capi
    L = capi.lib()
    rows = 9
    x, res, w = dev(sample(rng, rows, n)), dev(sample(rng, rows, n)), dev(sample(rng, 1, n)[0])
    y, h, rstd = K.rms_norm(x, w, 1e-6, residual=res)

    def call(x, res, h, y):
        capi.check(L.ag_rms_norm_f32(K._stream(), x.data_ptr(), res.data_ptr() if res is not None else None, w.data_ptr(), 1e-6,
                                     h.data_ptr() if h is not None else None, y.data_ptr(), None, None, None, rows, n))

    a, b = x.clone(), res.clone()
    call(a, b, b, a)
    assert torch.equal(a, y) and torch.equal(b, h)
    a, b = x.clone(), res.clone()
    call(a, b, a, b)
    assert torch.equal(a, h) and torch.equal(b, y)
    a, b = x.clone(), res.clone()
    call(a, b, None, b)
    assert torch.equal(a, x) and torch.equal(b, y)
    gy, gh = dev(sample(rng, rows, n)), dev(sample(rng, rows, n))
    gx, gw = K.rms_norm_grad(h, w, rstd, gy, gh=gh)
    nb = L.ag_rms_norm_grad_f32_workspace(rows, n)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    for alias in ("gy", "gh"):
        g1, g2, gw2 = gy.clone(), gh.clone(), torch.empty_like(w)
        out = g1 if alias == "gy" else g2
        capi.check(L.ag_rms_norm_grad_f32(K._stream(), h.data_ptr(), w.data_ptr(), rstd.data_ptr(), g1.data_ptr(), g2.data_ptr(), out.data_ptr(),
                                          gw2.data_ptr(), rows, n, ws.data_ptr(), nb))
        assert torch.equal(out, gx) and torch.equal(gw2, gw), alias


@pytest.mark.parametrize("n", [1, 3, 128, 130, 1024, 1025, 2048, 4096, 4099, 8192, 8193, 16384, 16385, 33000])
@pytest.mark.parametrize("rows,with_gh", [(1, False), (7, True), (700, False)])
def test_norm_gradient_is_the_formula(K, rng, rows, with_gh, n):
    say("rms_norm_grad", rows, n, with_gh)
    if rows * n > 10 ** 7:
        rows = 550  # more rows than blocks all the same
    h, w, gy = sample(rng, rows, n), sample(rng, 1, n)[0], sample(rng, rows, n)
    gh = sample(rng, rows, n) if with_gh else None
    eps = float(np.float32(1e-5))
    _, _, rstd = K.rms_norm(dev(h), dev(w), eps)
    gx, gw = K.rms_norm_grad(dev(h), dev(w), rstd, dev(gy), gh=None if gh is None else dev(gh))
    want_x, want_w, size_x, size_w = plain64.rms_norm_grad(h, w, eps, gy, gh)
    ex, ew = np.abs(host(gx) - want_x), np.abs(host(gw) - want_w)
    say("gx error in u of its terms: %.2f; gw: %.2f" % ((ex / size_x).max() / U, (ew / size_w).max() / U))
    assert (ex <= 6 * U * size_x + TINY).all()
    assert (ew <= (rows + 4) * U * size_w + TINY).all()


def test_norm_gradient_against_differences(K, rng):
    """Central differences of sum(gy * y) + sum(gh * h) in f64 around the same point: the step 1e-6 leaves an error of
    about step^2 |f'''| + 2^-53 |f| / step, below 1e-7 of values of order one."""
    rows, n, eps = 3, 40, 1e-5
    h, w, gy, gh = (rng.standard_normal(s).astype(np.float32) for s in ((rows, n), (n,), (rows, n), (rows, n)))
    _, _, rstd = K.rms_norm(dev(h), dev(w), eps)
    gx, gw = (host(t) for t in K.rms_norm_grad(dev(h), dev(w), rstd, dev(gy), gh=dev(gh)))

    def f(h, w):
        return (plain64.rms_norm(h, w, float(np.float32(eps)))[0] * gy).sum() + (gh * h).sum()

    h64, w64, step = h.astype(np.float64), w.astype(np.float64), 1e-6
    for i, j in ((0, 0), (1, 17), (2, 39)):
        d = np.zeros_like(h64)
        d[i, j] = step
        assert abs((f(h64 + d, w64) - f(h64 - d, w64)) / (2 * step) - gx[i, j]) < 1e-6 * (1 + abs(gx[i, j]))
    for j in (0, 20, 39):
        d = np.zeros_like(w64)
        d[j] = step
        assert abs((f(h64, w64 + d) - f(h64, w64 - d)) / (2 * step) - gw[j]) < 1e-6 * (1 + abs(gw[j]))


@pytest.mark.parametrize("n", [3, 200, 1025, 4096, 8192, 16000, 20000, 40001])
@pytest.mark.parametrize("gy_size,w_size", [(1.0, 1.0), (1e-3, 1.0), (1e-19, 1e-24), (1e18, 1e22)])
def test_norm_gradient_over_the_range_of_f32(K, rng, gy_size, w_size, n):
    """Rows whose squares, and products of gradient and weight, lie beyond f32's range while the gradient does not: the
    roundings are counted as for any other rows."""
    sizes = [h for h in (1e-36, 1e-30, 1e-20, 1.0, 1e18, 1e19, 1e20, 1e23, 1e30, 1e37) if 1e-36 <= gy_size * w_size / h <= 1e35]
    rows = len(sizes)
    assert rows >= 3
    h, gy, gh = (rng.standard_normal((rows, n)) for _ in range(3))
    h = (h * np.array(sizes)[:, None]).astype(np.float32)
    gy = (gy * gy_size).astype(np.float32)
    gh = (gh * (gy_size * w_size / np.array(sizes))[:, None]).astype(np.float32)
    w = (rng.standard_normal(n) * w_size).astype(np.float32)
    _, _, rstd = K.rms_norm(dev(h), dev(w), 0.0)
    for other in (None, gh):
        gx, gw = K.rms_norm_grad(dev(h), dev(w), rstd, dev(gy), gh=None if other is None else dev(other))
        want_x, want_w, size_x, size_w = plain64.rms_norm_grad(h, w, 0.0, gy, other)
        ex, ew = np.abs(host(gx) - want_x), np.abs(host(gw) - want_w)
        say("gx error in u of its terms, by row: " + " ".join("%.2g" % v for v in (ex / size_x).max(1) / U))
        assert (ex <= 6 * U * size_x + TINY).all()
        assert (ew <= (rows + 4) * U * size_w + TINY).all()


def test_norm_gradient_without_rows(K):
    z = torch.zeros
    gx, gw = K.rms_norm_grad(z(0, 8, device="cuda"), z(8, device="cuda"), z(0, device="cuda"), z(0, 8, device="cuda"))
    assert gx.shape == (0, 8) and not gw.any()


# ------------------------------------------------------------------------------------------ clipping
SIZES = [[1], [5, 0, 3], [8192], [8193, 8191, 1], [100] * 63, [17] * 64, [33] * 65, [3, 100000, 1, 70001] * 40, [300001, 4194304, 2]]


def arrays(rng, sizes, misaligned=False):
    """Tensors of the sizes inside one buffer, starting anywhere."""
    flat = dev(rng.standard_normal(sum(sizes) + len(sizes) + 8))
    out, at = [], 1 if misaligned else 0
    for i, n in enumerate(sizes):
        out.append(flat[at:at + n])
        at += n + (1 if misaligned else 0)
    return out


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("over", [0.5, 3.0])
def test_clipping(K, rng, sizes, over):
    say("clip", len(sizes), sum(sizes), over)
    xs = arrays(rng, sizes, misaligned=True)
    x64 = [host(x) for x in xs]
    norm = np.sqrt(sum((x * x).sum() for x in x64))
    limit = float(np.float32(norm / over))
    keep = [x.clone() for x in xs]
    outs, clip = K.clip_by_global_norm(xs, limit)
    c = host(clip)
    assert abs(c[0] - norm) <= U * (1 + 1e-6) * norm
    assert c[1] == 1.0 if over < 1 else abs(c[1] - limit / norm) <= U * (1 + 1e-6) * limit / norm
    assert torch.equal(K.global_norm(xs, limit), clip)
    for x, k, o in zip(xs, keep, outs):
        assert torch.equal(x, k) and torch.equal(o, k * clip[1])
    K.clip_by_global_norm(xs, limit, outs=xs)
    for x, o in zip(xs, outs):
        assert torch.equal(x, o)


def test_clipping_of_what_is_not_finite(K):
    big = torch.full((1000,), 3e38, device="cuda")  # its square is beyond f32
    outs, clip = K.clip_by_global_norm([big], 1.0)
    # the coefficient, 1 / (3e38 sqrt(1000)) = 1.05e-40, lies below f32's normal numbers, where half a step is 2^-150
    # whatever the value: 6.7e-6 of it
    coef = 1.0 / (float(np.float32(3e38)) * 1000 ** 0.5)
    assert torch.isinf(clip[0]) and np.allclose(host(outs[0]), 1000 ** -0.5, rtol=4 * U + 2.0 ** -150 / coef, atol=0)
    a, b = torch.ones(5, device="cuda"), torch.ones(9, device="cuda")
    b[3] = float("nan")
    outs, clip = K.clip_by_global_norm([a, b], 1.0)
    assert torch.isnan(clip).all() and torch.isnan(outs[0]).all()
    b[3] = float("inf")
    outs, clip = K.clip_by_global_norm([a, b], 1.0)
    assert clip[1] == 0 and not outs[0].any() and torch.isnan(outs[1][3])
    assert host(K.global_norm([]))[0] == 0 and host(K.global_norm([], 0.0))[1] == 1
    assert host(K.global_norm([torch.zeros(4, device="cuda")], 0.0))[1] == 1  # 0 <= 0: nothing to clip
    assert host(K.global_norm([a], float("inf")))[1] == 1


@pytest.mark.parametrize("sizes", [[7], [100, 1 << 20, 5, (1 << 20) + 77], [50] * 61], ids=lambda s: f"{len(s)}")
@pytest.mark.parametrize("over", [0.5, 4.0])
def test_clipped_adam_has_the_bits_of_clipping_first(K, rng, sizes, over):
    def state():
        r = np.random.default_rng(5)
        p, g, m, v = (arrays(r, sizes) for _ in range(4))
        return p, g, m, [t.square() for t in v], [torch.full((1,), float(i + 1), device="cuda") for i in range(len(sizes))]

    p, g, m, v, t = state()
    limit = float(np.sqrt(sum(sizes)) / over)
    keep = [x.clone() for x in g]
    clip = K.adam_update_clipped(p, g, m, v, t, limit, 1e-2)
    p2, g2, m2, v2, t2 = state()
    g2, clip2 = K.clip_by_global_norm(g2, limit)
    for i in range(0, len(sizes), 24):
        s = slice(i, i + 24)
        K.adam_update_multi(p2[s], g2[s], m2[s], v2[s], t2[s], 1e-2)
    assert torch.equal(clip, clip2)
    for a, b in ((p, p2), (g, keep), (m, m2), (v, v2), (t, t2)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_captured_step_repeats_the_eager_one(K, rng):
    """norm -> 8-bit product -> gradients -> clip -> Adam, captured once and replayed on changing inputs against the eager
    run of the same step."""
    rows, n, k, eps = 200, 300, 512, 1e-6
    x, res, gy = (dev(rng.standard_normal((rows, c))) for c in (k, k, n))
    start = {"w": dev(rng.standard_normal((k, n)) / 20), "g": dev(1 + 0.1 * rng.standard_normal(k))}

    def state():
        return {a: [t.clone(), torch.zeros_like(t), torch.zeros_like(t), torch.ones(1, device="cuda")] for a, t in start.items()}

    def step(s):
        w, g = s["w"][0], s["g"][0]
        y8, h, rstd = K.rms_norm_e4m3(x, g, eps, residual=res)
        qw, qwt = K.quantize_e4m3_both(w)
        y = K.matmul_e4m3(y8, qwt)
        qg, qgt = K.quantize_e4m3_both(gy)
        yn, _, _ = K.rms_norm(h, g, eps)
        gw = K.matmul_e4m3(K.quantize_e4m3(yn, transpose=True), qgt)
        gx, gg = K.rms_norm_grad(h, g, rstd, K.matmul_e4m3(qg, qw))
        clip = K.adam_update_clipped([w, g], [gw, gg], [s["w"][1], s["g"][1]], [s["w"][2], s["g"][2]], [s["w"][3], s["g"][3]], 0.5)
        return y, gx, clip

    a, b = state(), state()
    step(state())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for i in range(4):
        x.copy_(dev(rng.standard_normal((rows, k))))
        graph.replay()
        torch.cuda.synchronize()
        want = step(b)
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), f"replay {i}"
        for name in start:
            assert all(torch.equal(p, q) for p, q in zip(a[name], b[name])), f"replay {i}: {name}"


def test_clipped_adam_refuses_arrays_shared_between_its_launches(K):
    """More parameters than one launch takes, two of them with one step counter, parameter or moment, or a gradient that is
    another's parameter: refused before anything is written, as within one launch."""
    from rust_autograd_amd import capi
    count = capi.lib().ag_adam_update_multi_max() + 6

    def state():
        r = np.random.default_rng(5)
        return [[dev(r.random(40)) for _ in range(count)] for _ in range(4)] + [[torch.ones(1, device="cuda") for _ in range(count)]]

    for table, of in ((0, 0), (2, 2), (3, 3), (4, 4), (1, 0), (1, 2)):
        for first, last in ((1, count - 2), (count - 1, 0)):
            s = state()
            s[table][last] = s[of][first]
            keep = [[t.clone() for t in ts] for ts in s]
            with pytest.raises(capi.InvalidDims, match="separate calls"):
                K.adam_update_clipped(*s, 0.5)
            assert all(torch.equal(p, q) for a, b in zip(s, keep) for p, q in zip(a, b)), (table, of, first, last)
    s = state()
    s[1][count - 1] = s[1][0]  # (a gradient of two parameters is only read)
    K.adam_update_clipped(*s, 0.5)
    assert all(t.item() == 2.0 for t in s[4])


# ---- forms of the norm that the widths above do not reach ---------------------------------------------------------------
@pytest.mark.parametrize("n", [2560, 2561, 5120, 5121, 5125, 5632, 5633, 6143, 6144, 6145, 20480, 20481])
@pytest.mark.parametrize("rows,with_residual", [(1, True), (5, False), (6, True)])
def test_norm_at_the_borders_of_its_forms(K, rng, rows, with_residual, n):
    test_norm_is_the_formula_rounded_once(K, rng, rows, with_residual, n)


@pytest.mark.parametrize("n", [6143, 6144, 6145])
def test_norm_gradient_at_the_borders_of_its_forms(K, rng, n):
    test_norm_gradient_is_the_formula(K, rng, 7, True, n)


@pytest.mark.parametrize("n", [130, 511, 1023, 2046, 2555, 4091, 5115, 6130, 8190, 16380, 20470, 32761, 33001])
def test_arrays_beyond_the_caches_have_the_bits_of_their_parts(K, rng, n):
    """Arrays of 256 MiB and more are read past the caches."""
    rows = (1 << 26) // n + 5
    say("large", rows, n)
    x, res, gy = (torch.randn(rows, n, device="cuda") for _ in range(3))
    w = torch.randn(n, device="cuda")
    y, h, rstd = K.rms_norm(x, w, 1e-6, residual=res)
    e, _, _ = K.rms_norm_e4m3(x, w, 1e-6, residual=res)
    gx, gw = K.rms_norm_grad(h, w, rstd, gy, gh=res)
    sums, sizes = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    step = -(-rows // 4)
    for i in range(0, rows, step):
        s = slice(i, i + step)
        y1, h1, rstd1 = K.rms_norm(x[s], w, 1e-6, residual=res[s])
        e1, _, _ = K.rms_norm_e4m3(x[s], w, 1e-6, residual=res[s])
        gx1, _ = K.rms_norm_grad(h1, w, rstd1, gy[s], gh=res[s])
        for got, want in ((y[s], y1), (h[s], h1), (rstd[s], rstd1), (gx[s], gx1), (e.q[s].view(torch.uint8), e1.q.view(torch.uint8)),
                          (e.scales[s].view(torch.uint8), e1.scales.view(torch.uint8))):
            assert torch.equal(got, want)
        terms = gy[s].double() * h1.double() * rstd1.double()[:, None]
        sums += terms.sum(0)
        sizes += terms.abs().sum(0)
    # (a block adds its rows in f32 in turn: at most all of them)
    assert ((gw.double() - sums).abs() <= (rows + 4) * U * sizes + TINY).all()
    torch.cuda.empty_cache()


def test_nothing_is_clipped_to_an_infinite_norm(K):
    x = torch.full((5000,), 2.0, device="cuda")
    x[77] = float("inf")
    for xs in ([x], [x] * 200):  # one block, several
        outs, clip = K.clip_by_global_norm(xs, float("inf"))
        assert torch.isinf(clip[0]) and clip[1] == 1 and all(torch.equal(o, x) for o in outs)
    assert K.global_norm([x], 3.0e38)[1] == 0
