"""The 8-bit product, the RMS norm and clipping through the graph: how the nodes are built (on the CPU), and their values
and gradients (on the GPU) against 64-bit forms."""
import numpy as np
import pytest

import plain64

U = 2.0 ** -24


@pytest.fixture(scope="module")
def G():
    import torch

    torch.cuda.is_available()  # torch brings up the device before the library does, as in the other GPU tests
    from __graft_entry__ import load_package

    load_package()
    import rust_autograd_amd.graph as graph

    graph.lib()
    return graph


def context(G):
    env = G.VariableEnvironment()
    return env, env.context()


# ---- built without a device --------------------------------------------------------------------------------------------
def test_products_share_the_rounding_of_an_operand(G):
    env, c = context(G)
    x, w, v = c.placeholder("x", [-1, 64]), c.placeholder("w", [64, 32]), c.placeholder("v", [64, 16])
    y = c.matmul_e4m3(x, w)
    before = c.num_nodes
    z = c.matmul_e4m3(x, v)
    # the rounding of v, the extents of x and of v, and the product: x is not rounded again
    assert y.op_name == z.op_name == "MatMulE4m3" and c.num_nodes == before + 4
    assert y.num_inputs == 6


def test_gradients_of_a_product_are_products(G):
    env, c = context(G)
    x, w = c.placeholder("x", [-1, 64]), c.placeholder("w", [64, 32])
    gx, gw = c.grad([c.matmul_e4m3(x, w)], [x, w])
    assert gx.op_name == gw.op_name == "MatMulE4m3"
    # and theirs too
    assert c.grad([gx], [w])[0].op_name == "MatMulE4m3"


def test_misuse_panics(G):
    env, c = context(G)
    x, w = c.placeholder("x", [-1, 64]), c.placeholder("w", [64])
    for eps in (-1.0, float("nan")):
        with pytest.raises(G.Panic, match="eps"):
            c.rms_norm(x, w, eps)
    for limit in (-1.0, float("nan")):
        with pytest.raises(G.Panic, match="max_norm"):
            c.clip_by_global_norm([x], limit)
        with pytest.raises(G.Panic, match="max_norm"):
            c.global_norm([x], limit)
    with pytest.raises(G.Panic, match="no tensors"):
        c.clip_by_global_norm([], 1.0)
    g = c.grad([c.rms_norm(x, w)], [x])[0]
    with pytest.raises(G.Panic, match="second-order"):
        c.grad([g], [x])
    with pytest.raises(G.Panic, match="no gradient"):
        c.grad(c.clip_by_global_norm([x, w], 1.0), [x])
    with pytest.raises(G.Panic, match="no gradient"):
        c.grad([c.global_norm([x])], [x])


# ---- evaluated ---------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("ta", [False, True])
@pytest.mark.parametrize("tb", [False, True])
@pytest.mark.parametrize("m,k,n", [(3, 130, 40), (200, 300, 129)])
def test_product_and_gradients_of_integers_are_exact(G, rng, m, k, n, ta, tb):
    env, c = context(G)
    a, b = rng.integers(-3, 4, (k, m) if ta else (m, k)), rng.integers(-3, 4, (n, k) if tb else (k, n))
    gy = rng.integers(-3, 4, (m, n))
    x, w, g = c.placeholder("a", list(a.shape)), c.placeholder("b", list(b.shape)), c.placeholder("g", [m, n])
    y = c.matmul_e4m3(x, w, ta, tb)
    grads = c.grad_with_default([y], [x, w], [g])
    got = c.eval([y, *grads], {"a": a, "b": b, "g": gy})
    A, B = (a.T if ta else a), (b.T if tb else b)
    ga, gb = gy @ B.T, A.T @ gy
    for p, q in zip(got, (A @ B, ga.T if ta else ga, gb.T if tb else gb)):
        assert np.array_equal(p, q)


@pytest.mark.gpu
def test_second_order_and_a_tensor_against_itself(G, rng):
    """Integers, exact: d/dw of sum(v * d/dx sum(g * x w)) is the product of v and g; the gradient of x x^T has both of x's
    shares, and its two operands are one rounding."""
    env, c = context(G)
    m, k, n = 40, 150, 33
    x, w, g, v = (rng.integers(-2, 3, s) for s in ((m, k), (k, n), (m, n), (m, k)))
    xt, wt = c.placeholder("x", [m, k]), c.placeholder("w", [k, n])
    gt, vt = c.placeholder("g", [m, n]), c.placeholder("v", [m, k])
    gx = c.grad_with_default([c.matmul_e4m3(xt, wt)], [xt], [gt])[0]
    second = c.grad([c.mul(gx, vt)], [wt, gt])
    square = c.matmul_e4m3(xt, xt, False, True)
    st = c.placeholder("s", [m, m])
    s = rng.integers(-2, 3, (m, m))
    gsq = c.grad_with_default([square], [xt], [st])[0]
    dw, dg, sq, gs = c.eval([*second, square, gsq], {"x": x, "w": w, "g": g, "v": v, "s": s})
    assert np.array_equal(dw, v.T @ g) and np.array_equal(dg, v @ w)
    assert np.array_equal(sq, x @ x.T) and np.array_equal(gs, (s + s.T) @ x)


@pytest.mark.gpu
def test_product_of_rounded_operands(G, rng):
    env, c = context(G)
    m, k, n = 70, 400, 200
    a, b = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    y = c.eval([c.matmul_e4m3(c.variable(env.set("a", a)), c.variable(env.set("b", b)))])[0]
    ra, rb = plain64.rounded(a), plain64.rounded(b.T).T
    # sums of 400 exact products: 7 steps of 64 and the roundings inside one, a whole unit each, and at most 32 slices
    assert (np.abs(y - ra @ rb) <= ((k / 64 + 7) * 2 * U + 32 * U) * (np.abs(ra) @ np.abs(rb))).all()


@pytest.mark.gpu
def test_errors_of_extents_come_back_as_results(G, rng):
    env, c = context(G)
    x, w = c.variable(env.set("x", rng.random((4, 8)))), c.variable(env.set("w", rng.random((9, 3))))
    cube, v = c.variable(env.set("cube", rng.random((2, 4, 8)))), c.variable(env.set("v", rng.random(7)))
    for t, text in ((c.matmul_e4m3(x, w), "4 × 8 and 9 × 3"), (c.matmul_e4m3(cube, w), "must be 2D"), (c.rms_norm(x, v), "weight [7]"),
                    (c.rms_norm(x, w), "weight [9, 3]"), (c.rms_norm(x + x, v), "weight [7]")):
        r = c.eval([t])[0]
        assert isinstance(r, G.OpError) and r.kind == "IncompatibleShape" and text in r.message, r


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 300), (2, 3, 128), (64,), (300, 1000)])
def test_norm_and_its_gradient(G, rng, shape):
    env, c = context(G)
    x, w, gy = (rng.standard_normal(s).astype(np.float32) for s in (shape, shape[-1:], shape))
    eps = 2.0 ** -17
    xt, wt = c.placeholder("x", list(shape)), c.variable(env.set("w", w))
    y = c.rms_norm(xt, wt, eps)
    got = c.eval([y, *c.grad_with_default([y], [xt, wt], [c.placeholder("gy", list(shape))])], {"x": x, "gy": gy})
    n = shape[-1]
    want = plain64.rms_norm(x.reshape(-1, n), w, eps)[0].reshape(shape)
    gx, gw, size_x, size_w = plain64.rms_norm_grad(x.reshape(-1, n), w, eps, gy.reshape(-1, n))
    rows = x.size // n
    assert (np.abs(got[0] - want) <= U * (1 + 1e-6) * np.abs(want)).all()
    # the roundings of the gradient's terms: rstd (three times in its cube), two products, the multiply-add
    assert (np.abs(got[1] - gx.reshape(shape)) <= 6 * U * size_x.reshape(shape)).all()
    assert got[2].shape == w.shape and (np.abs(got[2] - gw) <= (rows + 4) * U * size_w).all()


@pytest.mark.gpu
def test_a_residual_is_added_in_the_pass_of_the_norm_with_the_same_bits(G, rng):
    a, b, w = (rng.standard_normal(s).astype(np.float32) for s in ((300, 260), (300, 260), (260,)))
    proj = (rng.standard_normal((260, 70)) / 16).astype(np.float32)

    def run():
        env, c = context(G)
        ta, tb = c.placeholder("a", [300, 260]), c.placeholder("b", [300, 260])
        h = ta + tb
        y = c.rms_norm(h, c.variable(env.set("w", w)))
        z = c.matmul_e4m3(y, c.variable(env.set("proj", proj)))
        s = h + c.matmul_e4m3(y, c.variable(env.set("back", proj[:, :1] * np.ones((1, 260), np.float32))))
        ts = [z, s, y, h, *c.grad([z, s], [ta, tb])]
        return c.eval(ts, {"a": a, "b": b}), c.fused_pairs

    try:
        fused, pairs = run()
        G.set_shortcuts(False)
        plain, none = run()
    finally:
        G.set_shortcuts(True)
    assert pairs == 1 and none == 0
    for p, q in zip(fused, plain):
        assert np.array_equal(p, q)
    assert np.array_equal(fused[3], a + b)


@pytest.mark.gpu
def test_a_weight_that_depends_on_the_sum_is_not_evaluated_with_it(G, rng):
    """The norm's weight comes from the very sum that it norms: the two nodes are evaluated in turn."""
    env, c = context(G)
    a, b = rng.standard_normal((6, 40)).astype(np.float32), rng.standard_normal((6, 40)).astype(np.float32)
    h = c.placeholder("a", [6, 40]) + c.placeholder("b", [6, 40])
    w = c.reduce_mean(h, [0])
    y, wv = c.eval([c.rms_norm(h, w), w], {"a": a, "b": b})
    want = plain64.rms_norm(a + b, wv, float(np.float32(1e-6)))[0]
    assert c.fused_pairs == 0 and (np.abs(y - want) <= U * (1 + 1e-6) * np.abs(want)).all()


@pytest.mark.gpu
def test_sums_that_broadcast_keep_their_own_pass(G, rng):
    env, c = context(G)
    a, b, w = rng.random((6, 40), dtype=np.float32), rng.random((1, 40), dtype=np.float32), rng.random(40, dtype=np.float32)
    y, h = c.eval([c.rms_norm(s := c.placeholder("a", [6, 40]) + c.placeholder("b", [1, 40]), c.variable(env.set("w", w))), s], {"a": a, "b": b})
    assert c.fused_pairs == 0 and np.array_equal(h, a + b)
    want = plain64.rms_norm(a + b, w, float(np.float32(1e-6)))[0]
    assert (np.abs(y - want) <= U * (1 + 1e-6) * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("over", [0.5, 4.0])
def test_clipping_in_the_graph(G, rng, over):
    env, c = context(G)
    xs = [rng.standard_normal(s).astype(np.float32) for s in ((3, 5), (1000, 7), (1,))]
    norm = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in xs))
    limit = float(np.float32(norm / over))
    ts = [c.variable(env.set(f"x{i}", x)) for i, x in enumerate(xs)]
    clip, *outs = c.eval([c.global_norm(ts, limit), *c.clip_by_global_norm(ts, limit)])
    assert abs(clip[0] - norm) <= U * (1 + 1e-6) * norm
    for x, o in zip(xs, outs):
        assert np.array_equal(o, x * clip[1])


@pytest.mark.gpu
def test_a_quantised_network_trains_with_clipped_adam(G, rng):
    """Residual block of norm and 8-bit products in front of a softmax loss, several steps: the clipped optimizer step has
    the bits of clipping the gradients first and updating with them."""
    rows, d, h, classes = 64, 160, 200, 10
    start = {"g": np.ones(d), "up": rng.standard_normal((d, h)) / 12, "down": rng.standard_normal((h, d)) / 14, "out": rng.standard_normal((d, classes))}
    x, t = rng.standard_normal((rows, d)), rng.integers(0, classes, (rows, 1))

    def train(clip_first):
        env = G.VariableEnvironment()
        ids = {k: env.set(k, v) for k, v in start.items()}
        adam = G.Adam(env, list(ids.values()), alpha=1e-2)
        for _ in range(4):
            c = env.context()
            v = {k: c.variable(i) for k, i in ids.items()}
            xt = c.placeholder("x", [-1, d])
            y = c.matmul_e4m3(c.relu(c.matmul_e4m3(c.rms_norm(xt, v["g"]), v["up"])), v["down"])
            logits = c.matmul_e4m3(c.rms_norm(xt + y, v["g"]), v["out"])
            loss = c.reduce_mean(c.sparse_softmax_cross_entropy(logits, c.placeholder("t", [-1, 1])), [0], False)
            params = list(v.values())
            grads = c.grad([loss], params)
            feeds = {"x": x, "t": t}
            if clip_first:
                adam.update(params, c.clip_by_global_norm(grads, 0.25), c, feeds)
            else:
                adam.update(params, grads, c, feeds, max_norm=0.25)
        return [env.array(i) for i in ids.values()]

    a, b = train(False), train(True)
    for p, q, s in zip(a, b, start.values()):
        assert np.isfinite(p).all() and not np.array_equal(p, s.astype(np.float32))
        assert np.array_equal(p, q)


# ---- weights that change within an evaluation (tensors are visited from the last to the first) ---------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("order", ["behind", "in front", "both sides"])
@pytest.mark.parametrize("kind,ta,tb", [("matmul", False, False), ("matmul_e4m3", False, False), ("matmul_e4m3", False, True), ("matmul_e4m3", True, False)])
def test_a_product_reads_the_weight_as_it_is_at_its_turn(G, rng, kind, order, ta, tb):
    """The weight is trained by an update of the same evaluation, whose gradients share the products' operands: a product
    behind the update has the bits of one of the updated weight, a product in front of it those of the old one."""
    k, n = 200, 72
    env = G.VariableEnvironment()
    w = env.set("w", rng.standard_normal((n, k) if tb else (k, n)))
    adam = G.Adam(env, [w], alpha=0.5)
    feeds = {"x": rng.standard_normal((k, 24) if ta else (24, k)), "z": rng.standard_normal((k, 40) if ta else (40, k))}

    def product(c, name):
        x = c.placeholder(name, list(feeds[name].shape))
        return c.matmul(x, c.variable(w)) if kind == "matmul" else c.matmul_e4m3(x, c.variable(w), ta, tb)

    def alone():  # of the weight as it is now
        c = env.context()
        return c.eval([product(c, "z")], feeds)[0]

    old = alone()
    c = env.context()
    y, wt = product(c, "x"), c.variable(w)
    update = adam.get_update_op([wt], c.grad([c.sum_all(c.mul(y, y))], [wt]), c)
    if order == "behind":
        after, before = c.eval([product(c, "z"), update], feeds)[0], None
    elif order == "in front":
        after, before = None, c.eval([update, product(c, "z")], feeds)[1]
    else:
        after, _, before = c.eval([product(c, "z"), update, product(c, "z")], feeds)
    new = alone()
    assert not np.array_equal(old, new)
    assert after is None or np.array_equal(after, new)
    assert before is None or np.array_equal(before, old)


@pytest.mark.gpu
def test_both_operands_and_several_updates(G, rng):
    """x x^T of a variable on both sides, between and behind two updates of it."""
    env = G.VariableEnvironment()
    x = env.set("x", rng.standard_normal((30, 140)))
    adam = G.Adam(env, [x], alpha=0.25)
    c = env.context()
    xt = c.variable(x)

    def square(c):
        return c.matmul_e4m3(c.variable(x), c.variable(x), False, True)

    def update(g):
        return adam.get_update_op([xt], [c.placeholder(g, [30, 140])], c)

    feeds = {"g": rng.standard_normal((30, 140)), "h": rng.standard_normal((30, 140))}
    third, _, second, _, first = c.eval([square(c), update("h"), square(c), update("g"), square(c)], feeds)
    c = env.context()
    assert np.array_equal(third, c.eval([square(c)])[0])
    assert not np.array_equal(first, second) and not np.array_equal(second, third)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["sum first", "norm first", "sum behind"])
def test_a_norm_reads_its_weight_as_it_is_at_its_turn(G, rng, order):
    """A sum and the norm behind it, with an update of the norm's weight between them that does not wait for the norm: with
    and without the pass over both the norm takes the weight of its own turn, and so does a product that reads it."""
    a, b, w = (rng.standard_normal(s) for s in ((50, 260), (50, 260), (260,)))
    proj = rng.standard_normal((260, 40)) / 16

    def run():
        env = G.VariableEnvironment()
        wid, pid = env.set("w", w), env.set("proj", proj)
        adam = G.Adam(env, [wid], alpha=0.5)
        c = env.context()
        h = c.placeholder("a", [50, 260]) + c.placeholder("b", [50, 260])
        y = c.rms_norm(h, c.variable(wid))
        z = c.matmul_e4m3(y, c.variable(pid))
        update = adam.get_update_op([c.variable(wid)], [c.placeholder("g", [260])], c)
        ts = {"sum first": [z, y, update, h], "norm first": [h, update, z, y], "sum behind": [h, z, y, update]}[order]
        got = dict(zip((t.id for t in ts), c.eval(ts, {"a": a, "b": b, "g": np.ones(260)})))
        return [got[t.id] for t in (h, y, z)], env.array(wid)

    try:
        (h, y, z), new = run()
        G.set_shortcuts(False)
        plain, same = run()
    finally:
        G.set_shortcuts(True)
    assert np.array_equal(new, same) and not np.array_equal(new, w.astype(np.float32))
    for p, q in zip((h, y, z), plain):
        assert np.array_equal(p, q)
    weight = w.astype(np.float32) if order == "norm first" else new
    want = plain64.rms_norm(h, weight, float(np.float32(1e-6)))[0]
    assert (np.abs(y - want) <= U * (1 + 1e-6) * np.abs(want)).all()


@pytest.mark.gpu
def test_a_norm_keeps_the_pass_of_the_sum_where_its_weight_is_trained_behind_it(G, rng):
    """The sum is asked for first and the update of the norm's weight waits for the norm, as in a training step."""
    env = G.VariableEnvironment()
    w = env.set("w", 1 + 0.1 * rng.standard_normal(130))
    adam = G.Adam(env, [w], alpha=0.5)
    c = env.context()
    h = c.placeholder("a", [20, 130]) + c.placeholder("b", [20, 130])
    y = c.rms_norm(h, c.variable(w))
    update = adam.get_update_op([c.variable(w)], c.grad([c.sum_all(c.mul(y, y))], [c.variable(w)]), c)
    a, b, old = rng.standard_normal((20, 130)).astype(np.float32), rng.standard_normal((20, 130)).astype(np.float32), env.array(w)
    yv, _, hv = c.eval([y, update, h], {"a": a, "b": b})
    assert c.fused_pairs == 1 and np.array_equal(hv, a + b) and not np.array_equal(env.array(w), old)
    want = plain64.rms_norm(hv, old, float(np.float32(1e-6)))[0]
    assert (np.abs(yv - want) <= U * (1 + 1e-6) * np.abs(want)).all()


@pytest.mark.gpu
def test_a_sum_is_evaluated_where_the_norm_behind_it_is_refused(G):
    """Rows of one element, more of them than the norm takes: its error is its own, the sum in front of it has a value."""
    env, c = context(G)
    shape = [1 << 16, (1 << 15) + 1]  # 2^31 + 2^16 elements, a product of two vectors
    a = c.matmul(c.variable(env.set("a", np.ones((shape[0], 1)))), c.variable(env.set("b", np.full((1, shape[1]), 1.5))))
    x = c.reshape(a, [shape[0] * shape[1], 1])
    h = x + x
    total, y = c.eval([c.reduce_mean(c.reshape(h, shape), [0, 1], False), c.rms_norm(h, c.variable(env.set("w", np.ones(1))))])
    assert isinstance(y, G.OpError) and y.kind == "InvalidDims" and "rms_norm" in y.message
    assert abs(float(np.reshape(total, -1)[0]) - 3.0) < 1e-4
