"""The operators of an 8-bit training and serving step, as cases that can be timed and checked.

Three families, each at the sizes a program meets:

  norm     root-mean-square norm of x (+ a residual), its output in f32 or in e4m3 with a power-of-two scale per block
           of 128 along the row; with its backward pass
  product  matrix product of two e4m3 operands with a scale per row and block of 128 of the contraction; from operands in
           hand, from f32 activations, and as a training step with both gradients
  clip     norm over all gradient tensors together and clipping by it, alone or inside the Adam update

`own` selects what run() does: the operators' plain form (elementary torch operations) or this package's kernels.

Layout of an 8-bit operand of `rows` rows and n elements along the contraction: q [rows, pitch] of float8_e4m3fn with
pitch = n rounded up to 128 and zeros behind n; scales [rows, blocks] of float8_e8m0fnu with one power of two for each
block of 128, the number of blocks rounded up to 4 and ones behind the last.  An element is q * scale.
"""
import math
import random

import torch

own = False

BLOCK = 128
EPS = 2.0 ** -20  # (a number of f32, which is what the operator takes)
ALPHA, ADAM_EPS, B1, B2 = 1e-3, 1e-8, 0.9, 0.999
# gradients of the small convolutional net's parameters (filters, dense layer and biases of its three layers)
SMALL_NET = (32 * 9, 64 * 32 * 9, 3136 * 10, 32 * 28 * 28, 64 * 14 * 14, 10)


def listed():
    return [
        # one token of a decoding step: a single row, where latency is everything
        {"name": "norm8 one token", "kind": "norm8", "rows": 1, "n": 4096},
        # a long prompt, or a training batch's forward: bandwidth
        {"name": "norm8 prompt", "kind": "norm8", "rows": 16384, "n": 8192},
        # f32 output without a residual, rows that are no whole quads or blocks
        {"name": "norm odd rows", "kind": "norm", "rows": 4099, "n": 5001, "residual": False},
        # a training step through the norm: forward, then the gradients of both inputs and the weight
        {"name": "norm training", "kind": "norm_train", "rows": 8192, "n": 4096},
        # one token through a dense layer whose weight was laid out in 8 bits once
        {"name": "product one token", "kind": "product_x", "m": 1, "n": 4096, "k": 4096},
        # a decoding batch through a wide layer
        {"name": "product batch 48", "kind": "product_x", "m": 48, "n": 16384, "k": 4096},
        # ragged in every extent: tiles and blocks that end inside
        {"name": "product odd", "kind": "product", "m": 1000, "n": 1999, "k": 2500},
        # the square product, operands in hand
        {"name": "product square", "kind": "product", "m": 4096, "n": 4096, "k": 4096},
        # a prompt through a large layer
        {"name": "product large", "kind": "product", "m": 16384, "n": 8192, "k": 8192},
        # a training step of a dense layer: the product and both gradients, all three from f32
        {"name": "product training", "kind": "product_train", "m": 8192, "n": 4096, "k": 4096},
        # the small convolutional net's optimizer step: a few small arrays
        {"name": "clip adam small net", "kind": "clip_adam", "net": True, "count": 6, "total": sum(SMALL_NET), "over": 2.0},
        # the gradients of a transformer of some 150 arrays
        {"name": "clip many arrays", "kind": "clip", "net": False, "count": 148, "total": 200000001, "over": 4.0},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["norm8", "norm", "norm_train", "product_x", "product", "product_train", "clip", "clip_adam"])
    if kind in ("norm8", "norm", "norm_train"):
        case = {"kind": kind, "rows": _log(rng, 1, 16384 if kind == "norm8" else 8192), "n": _log(rng, 64, 8192)}
        if kind == "norm":
            case["residual"] = rng.random() < 0.5
        return case
    if kind == "product_x":
        return {"kind": kind, "m": _log(rng, 1, 64), "n": _log(rng, 128, 16384), "k": _log(rng, 128, 8192)}
    if kind == "product":
        return {"kind": kind, "m": _log(rng, 64, 8192), "n": _log(rng, 64, 8192), "k": _log(rng, 64, 8192)}
    if kind == "product_train":
        return {"kind": kind, "m": _log(rng, 64, 8192), "n": _log(rng, 64, 4096), "k": _log(rng, 64, 4096)}
    return {"kind": kind, "net": False, "count": _log(rng, 1, 300), "total": _log(rng, 1000, 1 << 26),
            "over": rng.choice([0.5, 2.0, 10.0])}  # the norm as a multiple of the limit: below it nothing is clipped


def _sizes(case):
    """Element counts of the tensors of a clip case: the small net's, or `count` sizes spread over a factor of a
    thousand that add up to `total`."""
    if case["net"]:
        return list(SMALL_NET)
    count, total = case["count"], case["total"]
    rng = random.Random(count * 1000003 + total)
    weights = [math.exp(rng.uniform(0.0, math.log(1000.0))) for _ in range(count)]
    whole = sum(weights)
    sizes = [max(1, int(total * w / whole)) for w in weights]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def _views(flat, sizes):
    """Tensors that share one buffer, each starting on a multiple of 4 elements, as a trainer keeps its gradients."""
    views, at = [], 0
    for n in sizes:
        views.append(flat[at:at + n])
        at += (n + 3) // 4 * 4
    return views


def _flat_length(sizes):
    return sum((n + 3) // 4 * 4 for n in sizes)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    kind = case["kind"]
    if kind in ("norm8", "norm", "norm_train"):
        rows, n = case["rows"], case["n"]
        x = normal(rows, n)
        x[:, :: 97] *= 20.0  # some channels of a residual stream stand out
        s = {"case": case, "x": x, "weight": 1.0 + 0.1 * normal(n), "residual": None}
        if kind != "norm" or case["residual"]:
            s["residual"] = 0.5 * normal(rows, n)
        if kind == "norm_train":
            s["gy"], s["gh"] = 0.01 * normal(rows, n), 0.01 * normal(rows, n)
        return s
    if kind == "product_x":
        m, n, k = case["m"], case["n"], case["k"]
        x, w = normal(m, k), normal(n, k) / math.sqrt(k)
        q, scales = _quantize(w)
        return {"case": case, "x": x, "q": q, "scales": scales}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a, b = _quantize(normal(m, k)), _quantize(normal(n, k) / math.sqrt(k))
        return {"case": case, "a": a, "b": b}
    if kind == "product_train":
        m, n, k = case["m"], case["n"], case["k"]
        return {"case": case, "x": normal(m, k), "w": normal(k, n) / math.sqrt(k), "gy": 0.01 * normal(m, n)}
    sizes = _sizes(case)
    length = _flat_length(sizes)
    s = {"case": case, "flat": 1e-3 * normal(length)}
    s["grads"] = _views(s["flat"], sizes)
    s["max_norm"] = 1e-3 * math.sqrt(sum(sizes)) / case["over"]
    if kind == "clip":
        s["flat_out"] = torch.zeros(length, device="cuda")
        s["outs"] = _views(s["flat_out"], sizes)
        return s
    s["flat_p"], s["flat_m"], s["flat_v"] = normal(length), 1e-3 * normal(length), (1e-3 * normal(length)).square()
    s["params"], s["ms"], s["vs"] = (_views(s[f], sizes) for f in ("flat_p", "flat_m", "flat_v"))
    s["ts"] = [torch.full((1,), 5.0, device="cuda") for _ in sizes]
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------
def _quantize(x):
    """x [rows, n] -> (q, scales) in the layout above.  The scale of a block is the smallest power of two, at least
    2^-117, that brings the block's largest finite magnitude to at most 448; a block of zeros has scale 1.  Values that
    are not finite become NaN."""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    padded = torch.zeros(rows, blocks * BLOCK, device=x.device)
    padded[:, :n] = x
    padded = padded.view(rows, blocks, BLOCK)
    finite = padded.isfinite()
    amax = torch.where(finite, padded.abs(), torch.zeros_like(padded)).amax(2)
    mantissa, exponent = torch.frexp(amax.double())  # amax = mantissa * 2^exponent, mantissa in [1/2, 1)
    byte = exponent - 9 + (mantissa > 0.875).int() + 127  # 448 = 0.875 * 2^9
    byte = torch.where(amax > 0, byte.clamp(min=10), torch.full_like(byte, 127)).int()
    inverse = ((254 - byte) << 23).view(torch.float32)  # 2^(127 - byte), by its bits
    scaled = padded * inverse[:, :, None]
    q = torch.where(finite, scaled, torch.full_like(scaled, math.nan)).to(torch.float8_e4m3fn)
    scales = torch.full((rows, (blocks + 3) // 4 * 4), 127, dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = byte.to(torch.uint8)
    return q.view(rows, blocks * BLOCK), scales.view(torch.float8_e8m0fnu)


def _values(q, scales):
    """The f32 values that an 8-bit operand stands for, zeros behind n included."""
    rows, pitch = q.shape
    power = (scales.view(torch.uint8)[:, : pitch // BLOCK].int() << 23).view(torch.float32)
    return (q.float().view(rows, pitch // BLOCK, BLOCK) * power[:, :, None]).view(rows, pitch)


def _rounded(x):
    return _values(*_quantize(x))[:, : x.shape[1]]


def _norm_plain(s):
    x = s["x"]
    h = x if s["residual"] is None else x + s["residual"]
    r = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    return h, r, h * r * s["weight"]


def _clip_plain(s):
    total = torch.stack([g.square().sum() for g in s["grads"]]).sum()
    norm = total.sqrt()
    coef = torch.where(norm <= s["max_norm"], torch.ones_like(norm), s["max_norm"] / norm)
    return torch.stack([norm, coef])


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "norm8":
        # in 64 bits up to the f32 value that is rounded to 8: its neighbours there are 6 % apart
        h = s["x"] + s["residual"]
        h64 = h.double()
        r = 1.0 / (h64.square().mean(1, keepdim=True) + EPS).sqrt()
        q, scales = _quantize((h64 * r * s["weight"].double()).float())
        return {"h": h, "q": q, "scales": scales}
    if kind == "norm":
        h, _, y = _norm_plain(s)
        return {"y": y} if s["residual"] is None else {"h": h, "y": y}
    if kind == "norm_train":
        h, r, y = _norm_plain(s)
        gw_rows = s["gy"] * h * r
        g = s["gy"] * s["weight"]
        c = (g * h).mean(1, keepdim=True)
        gx = g * r - h * (c * r * r * r) + s["gh"]
        return {"h": h, "y": y, "gx": gx, "gw": gw_rows.sum(0)}
    if kind == "product_x":
        return {"y": _rounded(s["x"]) @ _values(s["q"], s["scales"])[:, : s["x"].shape[1]].t()}
    if kind == "product":
        return {"y": _values(*s["a"]) @ _values(*s["b"]).t()}
    if kind == "product_train":
        x, w, gy = s["x"], s["w"], s["gy"]
        y = _rounded(x) @ _rounded(w.t()).t()
        gx = _rounded(gy) @ _rounded(w).t()
        gw = _rounded(x.t()) @ _rounded(gy.t()).t()
        return {"y": y, "gx": gx, "gw": gw}
    clip = _clip_plain(s)
    if kind == "clip":
        [torch.mul(g, clip[1], out=o) for g, o in zip(s["grads"], s["outs"])]
        return {"clip": clip, "out": s["flat_out"]}
    [_adam_plain(*a, clip[1]) for a in zip(s["params"], s["grads"], s["ms"], s["vs"], s["ts"])]
    return {"clip": clip, "p": s["flat_p"], "m": s["flat_m"], "v": s["flat_v"], "t": torch.cat(s["ts"])}


def _adam_plain(p, g, m, v, t, coef):
    g = g * coef
    m.copy_(m * B1 + (1 - B1) * g)
    v.copy_(v * B2 + (1 - B2) * g * g)
    m_hat, v_hat = m / (1 - B1 ** t), v / (1 - B2 ** t)
    p.sub_(ALPHA * (m_hat / (v_hat.sqrt() + ADAM_EPS)))
    t.add_(1.0)


# ---- the package's operators ------------------------------------------------------------------------------------------
_package = None


def _kernels():
    global _package
    if _package is None:
        from __graft_entry__ import load_package

        load_package()
        from rust_autograd_amd import kernels

        _package = kernels
    return _package


def _ours(s):
    K = _kernels()
    kind = s["case"]["kind"]
    if kind == "norm8":
        e, h, _ = K.rms_norm_e4m3(s["x"], s["weight"], EPS, residual=s["residual"])
        return {"h": h, "q": e.q, "scales": e.scales}
    if kind == "norm":
        y, h, _ = K.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
        return {"y": y} if s["residual"] is None else {"h": h, "y": y}
    if kind == "norm_train":
        y, h, rstd = K.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
        gx, gw = K.rms_norm_grad(h, s["weight"], rstd, s["gy"], gh=s["gh"])
        return {"h": h, "y": y, "gx": gx, "gw": gw}
    if kind == "product_x":
        return {"y": K.quantize_matmul_e4m3(s["x"], K.E4m3(s["q"], s["scales"], s["case"]["k"]))}
    if kind == "product":
        k = s["case"]["k"]
        return {"y": K.matmul_e4m3(K.E4m3(*s["a"], k), K.E4m3(*s["b"], k))}
    if kind == "product_train":
        x, xt = K.quantize_e4m3_both(s["x"])
        w, wt = K.quantize_e4m3_both(s["w"])
        y = K.matmul_e4m3(x, wt)
        gy, gyt = K.quantize_e4m3_both(s["gy"])
        return {"y": y, "gx": K.matmul_e4m3(gy, w), "gw": K.matmul_e4m3(xt, gyt)}
    if kind == "clip":
        _, clip = K.clip_by_global_norm(s["grads"], s["max_norm"], outs=s["outs"])
        return {"clip": clip, "out": s["flat_out"]}
    clip = K.adam_update_clipped(s["params"], s["grads"], s["ms"], s["vs"], s["ts"], s["max_norm"], ALPHA, ADAM_EPS, B1, B2)
    return {"clip": clip, "p": s["flat_p"], "m": s["flat_m"], "v": s["flat_v"], "t": torch.cat(s["ts"])}


def run(state):
    return _ours(state) if own else _plain(state)


def work(case):
    kind = case["kind"]
    if kind in ("norm8", "norm", "norm_train"):
        cells = case["rows"] * case["n"]
        if kind == "norm8":  # x, residual in; h, q, scales out
            return {"bytes": cells * 13 + cells // BLOCK + 4 * case["n"], "flops": 6 * cells}
        if kind == "norm":
            return {"bytes": cells * (16 if case["residual"] else 8) + 4 * case["n"], "flops": 5 * cells}
        return {"bytes": cells * 32 + 8 * case["n"], "flops": 17 * cells}  # x, residual, gy, gh in; h, y, gx out; gw
    if kind in ("product_x", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        a = m * k * (4 if kind == "product_x" else 1 + 1 / BLOCK)
        return {"bytes": a + n * k * (1 + 1 / BLOCK) + 4 * m * n, "flops": 2.0 * m * n * k}
    if kind == "product_train":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 8.0 * (m * k + k * n + m * n), "flops": 6.0 * m * n * k}
    total = sum(_sizes(case))
    return {"bytes": (8 if kind == "clip" else 28) * total, "flops": (3 if kind == "clip" else 17) * total}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _exact_rounded(x, layout=False):
    """The values of x after rounding to 8 bits, from the bits of each block's largest magnitude: in 64 bits, [rows, n];
    with `layout`: (q, scales) as values, padded as they are stored."""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    v = torch.nn.functional.pad(x.double(), (0, blocks * BLOCK - n)).view(rows, blocks, BLOCK)
    top = v.abs().amax(2).float().view(torch.int32)  # exact: the inputs are f32
    e = (top >> 23) - 127 - 8 + ((top & 0x7FFFFF) > 0x600000).int()
    e = torch.where(top > 0, e.clamp(min=-117), torch.zeros_like(e)).long()
    scale = ((e + 1023) << 52).view(torch.float64)[:, :, None]
    v = v / scale
    _, k = torch.frexp(v)
    step = ((k.long().clamp(min=-5) - 4 + 1023) << 52).view(torch.float64)  # 2^-3 of the leading power, 2^-9 at the least
    v = torch.round(v / step) * step
    if layout:
        scales = torch.nn.functional.pad(scale[:, :, 0], (0, -blocks % 4), value=1.0)
        return v.view(rows, blocks * BLOCK), scales
    return (v * scale).view(rows, blocks * BLOCK)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("norm8", "norm", "norm_train"):
        h32 = s["x"] if s["residual"] is None else s["x"] + s["residual"]
        if kind == "norm8":
            h, w = h32.double(), s["weight"].double()
            y = h * w / torch.sqrt(torch.einsum("ij,ij->i", h, h) / h.shape[1] + EPS)[:, None]
            q, scales = _exact_rounded(y.float(), layout=True)  # what is rounded to 8 bits is the norm's f32 value
            return {"h": s["x"].double() + s["residual"].double(), "q": q, "scales": scales}
        h, w = h32.double(), s["weight"].double()
        d = torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS)
        if kind == "norm":
            return {"y": h * w / d} if s["residual"] is None else {"h": h, "y": h * w / d}
        gy = s["gy"].double()
        gx = gy * w / d - h * ((gy * w * h).sum(1, keepdim=True) / h.shape[1]) / d ** 3 + s["gh"].double()
        return {"h": h, "y": h * w / d, "gx": gx, "gw": (gy * h / d).sum(0)}
    if kind == "product_x":
        return {"y": _exact_rounded(s["x"]) @ (_exact_layout(s["q"], s["scales"])[:, : case["k"]]).t()}
    if kind == "product":
        return {"y": _exact_layout(*s["a"]) @ _exact_layout(*s["b"]).t()}
    if kind == "product_train":
        x, w, gy = s["x"], s["w"], s["gy"]
        return {"y": _exact_rounded(x) @ _exact_rounded(w.t().contiguous()).t(),
                "gx": _exact_rounded(gy) @ _exact_rounded(w).t(),
                "gw": _exact_rounded(x.t().contiguous()) @ _exact_rounded(gy.t().contiguous()).t()}
    total = math.fsum(float((g.double() ** 2).sum()) for g in s["grads"])
    norm = math.sqrt(total)
    coef = 1.0 if norm <= s["max_norm"] else s["max_norm"] / norm
    clip = torch.tensor([norm, coef], dtype=torch.float64)
    out = torch.zeros(s["flat"].numel(), dtype=torch.float64, device="cuda")
    if kind == "clip":
        for g, o in zip(s["grads"], _views(out, _sizes(case))):
            o.copy_(g.double() * coef)
        return {"clip": clip, "out": out}
    # the padding between the arrays keeps what it holds
    g = torch.zeros_like(out)
    inside = torch.zeros_like(out, dtype=torch.bool)
    for a, b, i in zip(s["grads"], _views(g, _sizes(case)), _views(inside, _sizes(case))):
        b.copy_(a.double() * coef)
        i.fill_(True)
    p0, m0, v0 = s["flat_p"].double(), s["flat_m"].double(), s["flat_v"].double()
    m, v = B1 * m0 + (1 - B1) * g, B2 * v0 + (1 - B2) * g * g
    p = p0 - ALPHA * (m / (1 - B1 ** 5.0)) / (torch.sqrt(v / (1 - B2 ** 5.0)) + ADAM_EPS)
    return {"clip": clip, "p": torch.where(inside, p, p0), "m": torch.where(inside, m, m0), "v": torch.where(inside, v, v0),
            "t": torch.full((len(_sizes(case)),), 6.0, dtype=torch.float64)}


def _exact_layout(q, scales):
    rows, pitch = q.shape
    power = scales.view(torch.uint8).long()[:, : pitch // BLOCK] - 127
    power = ((power + 1023) << 52).view(torch.float64)
    return (q.double().view(rows, -1, BLOCK) * power[:, :, None]).view(rows, pitch)
