"""Eager launchers: each function allocates the outputs as torch CUDA tensors (torch is only the
owner of device memory and of the stream) and calls the matching C-ABI entry point of
libag_hip.so.  Names and argument order follow the reference's compute functions
(conv2d_impl, conv2d_filter_grad_impl, conv2d_transpose_impl, max_pool_f32, ...), so that the
parity tests read like the reference's own tests.
"""
import ctypes as C
from typing import NamedTuple

import torch

from . import capi
from .capi import check


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _stream():
    # (the handle itself: making a Stream object of it costs ten times as much as looking it up)
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _f32(t, name):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise capi.TypeUnsupported(f"{name}: expected a CUDA tensor")
    if t.dtype != torch.float32:
        raise capi.TypeUnsupported(f"{name}: only f32 is supported on the GPU path")
    return t.contiguous()   # the reference deep-copies non-contiguous inputs (conv2d.rs:436-452)


def _empty(shape, like, dtype=torch.float32):
    return torch.empty(tuple(int(s) for s in shape), dtype=dtype, device=like.device)


def _ws(nbytes, like):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=like.device)


def conv_out_size(x, k, p, s, d):
    return capi.lib().ag_conv_out_size(x, k, p, s, d)


# ------------------------------------------------------------------------------------------ im2col
def im2col(x, kh, kw, ph, pw, sh, sw, dh, dw):
    x = _f32(x, "im2col")
    B, Cc, H, W = x.shape
    OH, OW = conv_out_size(H, kh, ph, sh, dh), conv_out_size(W, kw, pw, sw, dw)
    cols = _empty((B, Cc * kh * kw, max(OH, 0) * max(OW, 0)), x)
    check(capi.lib().ag_im2col_f32(_stream(), _ptr(x), _ptr(cols), B, Cc, H, W, kh, kw, ph, pw, sh, sw, dh, dw))
    return cols


def col2im(cols, Cc, H, W, kh, kw, ph, pw, sh, sw, dh, dw, OH, OW):
    cols = _f32(cols, "col2im")
    B = cols.shape[0]
    gx = _empty((B, Cc, H, W), cols)
    check(capi.lib().ag_col2im_f32(_stream(), _ptr(cols), _ptr(gx), B, Cc, H, W, kh, kw, ph, pw, sh, sw, dh, dw,
                                   OH, OW))
    return gx


# ------------------------------------------------------------------------------------------ GEMM
def gemm(ta, tb, m, n, k, alpha, a, lda, stride_a, b, ldb, stride_b, beta, c, ldc, stride_c, batch):
    check(capi.lib().ag_gemm_f32(_stream(), int(ta), int(tb), m, n, k, alpha, _ptr(a), lda, stride_a, _ptr(b),
                                 ldb, stride_b, beta, _ptr(c), ldc, stride_c, batch))
    return c


def gemm_batchsum(ta, tb, m, n, k, alpha, a, lda, stride_a, b, ldb, stride_b, beta, c, ldc, batch):
    nbytes = capi.lib().ag_gemm_batchsum_f32_workspace(m, n, k, batch)
    ws = _ws(nbytes, c)
    check(capi.lib().ag_gemm_batchsum_f32(_stream(), int(ta), int(tb), m, n, k, alpha, _ptr(a), lda, stride_a,
                                          _ptr(b), ldb, stride_b, beta, _ptr(c), ldc, batch, _ptr(ws),
                                          ws.numel()))
    return c


def matmul(a, b, transpose_a=False, transpose_b=False):
    """MatMul::compute (dot_ops.rs:564-606)."""
    a, b = _f32(a, "matmul"), _f32(b, "matmul")
    if a.dim() != 2:
        raise capi.IncompatibleShape("lhs input for MatMul must be 2D")
    if b.dim() != 2:
        raise capi.IncompatibleShape("rhs input for MatMul must be 2D")
    m, k = (a.shape[1], a.shape[0]) if transpose_a else a.shape
    k2, n = (b.shape[1], b.shape[0]) if transpose_b else b.shape
    if k != k2:
        raise capi.IncompatibleShape(
            f"ndarray: inputs {m} × {k} and {k2} × {n} are not compatible for matrix multiplication")
    c = _empty((m, n), a)
    L = capi.lib()
    ws = _ws(L.ag_matmul_f32_workspace(m, n, k), a)
    check(L.ag_matmul_f32(_stream(), int(transpose_a), int(transpose_b), m, n, k, _ptr(a), max(a.shape[1], 1), _ptr(b),
                          max(b.shape[1], 1), _ptr(c), max(n, 1), _ptr(ws), ws.numel()))
    return c


def batch_matmul(a, b, transpose_a=False, transpose_b=False):
    """BatchMatMul::compute (dot_ops.rs:631-695)."""
    a, b = _f32(a, "batch_matmul"), _f32(b, "batch_matmul")
    if a.dim() < 2:
        raise capi.IncompatibleShape(f"BatchMatMul: Left-hand-side input's ndim must be >= 2, actual: {a.dim()}")
    if b.dim() < 2:
        raise capi.IncompatibleShape(f"BatchMatMul: Right-hand-side input's ndim must be >= 2, actual: {b.dim()}")
    sa = list(a.shape)
    sb = list(b.shape)
    if transpose_a:
        sa[-2], sa[-1] = sa[-1], sa[-2]
    if transpose_b:
        sb[-2], sb[-1] = sb[-1], sb[-2]
    if len(sa) != len(sb) or sa[:-2] != sb[:-2]:
        raise capi.IncompatibleShape(f"Input shapes mismatch: {sa} vs {sb}")
    m, k, k2, n = sa[-2], sa[-1], sb[-2], sb[-1]
    if k != k2:
        raise capi.IncompatibleShape(f"Input shapes mismatch: {sa} vs {sb}")
    batch = 1
    for s in sa[:-2]:
        batch *= s
    c = _empty(sa[:-2] + [m, n], a)
    return gemm(transpose_a, transpose_b, m, n, k, 1.0, a, max(a.shape[-1], 1), a.shape[-1] * a.shape[-2], b,
                max(b.shape[-1], 1), b.shape[-1] * b.shape[-2], 0.0, c, max(n, 1), m * n, batch)


# ------------------------------------------------------------------------------------------ conv
def conv2d(x, w, pad, stride, dilation=1):
    """Conv2D::compute: returns (y, cols), the op's two outputs (conv2d.rs:531-554)."""
    x, w = _f32(x, "conv2d"), _f32(w, "conv2d")
    if x.dim() != 4:
        raise capi.IncompatibleShape(f"conv2d: lhs input must be 4D (got {list(x.shape)})")
    if w.dim() != 4:
        raise capi.IncompatibleShape(f"conv2d: filter must be 4D (got {list(w.shape)})")
    B, Cc, H, W = x.shape
    K, C2, kh, kw = w.shape
    if Cc != C2:
        raise capi.IncompatibleShape(
            f"conv2d: input channel dim ({Cc}) must match filter's second dim ({C2})")
    OH, OW = conv_out_size(H, kh, pad, stride, dilation), conv_out_size(W, kw, pad, stride, dilation)
    y = _empty((B, K, max(OH, 0), max(OW, 0)), x)
    cols = _empty((B, Cc * kh * kw, max(OH, 0) * max(OW, 0)), x)
    check(capi.lib().ag_conv2d_fwd_f32(_stream(), _ptr(x), _ptr(w), _ptr(y), _ptr(cols), B, Cc, H, W, K, kh, kw,
                                       pad, stride, dilation))
    return y, cols


def conv2d_with_cols(cols, w, OH, OW):
    cols, w = _f32(cols, "conv2d_with_cols"), _f32(w, "conv2d_with_cols")
    B = cols.shape[0]
    K, CK = w.shape[0], w.shape[1] * w.shape[2] * w.shape[3]
    y = _empty((B, K, OH, OW), cols)
    check(capi.lib().ag_conv2d_with_cols_f32(_stream(), _ptr(cols), _ptr(w), _ptr(y), B, CK, OH * OW, K))
    return y


def conv2d_filter_grad(cols, gy, w_shape):
    """Conv2DFilterGrad::compute (conv2d.rs:736-744)."""
    cols, gy = _f32(cols, "conv2d_filter_grad"), _f32(gy, "conv2d_filter_grad")
    B, K, OH, OW = gy.shape
    CK = w_shape[1] * w_shape[2] * w_shape[3]
    gw = _empty(w_shape, gy)
    nbytes = capi.lib().ag_conv2d_filter_grad_f32_workspace(B, CK, OH * OW, K)
    ws = _ws(nbytes, gy)
    check(capi.lib().ag_conv2d_filter_grad_f32(_stream(), _ptr(cols), _ptr(gy), _ptr(gw), B, CK, OH * OW, K,
                                               _ptr(ws), ws.numel()))
    return gw


def conv2d_transpose(gy, w, pad, stride, dilation=1, out_hw=None, return_cols=False):
    """Conv2DTranspose::compute (conv2d_transpose.rs:249-272).  out_hw=None reproduces the
    reference's reconstructed output size (conv2d_transpose.rs:55-56)."""
    gy, w = _f32(gy, "conv2d_transpose"), _f32(w, "conv2d_transpose")
    if gy.dim() != 4:
        raise capi.IncompatibleShape(f"conv2d_transpose: Input must be 4D (got {list(gy.shape)})")
    if w.dim() != 4:
        raise capi.IncompatibleShape(f"conv2d_transpose: Filter must be 4D (got {list(w.shape)})")
    B, ych, yh, yw = gy.shape
    ych2, xch, kh, kw = w.shape
    if ych != ych2:
        raise capi.IncompatibleShape(
            f"conv2d_transpose: Number of input channels ({ych}) must match second filter dim ({ych2})")
    if out_hw is None:
        L = capi.lib()
        out_hw = (L.ag_conv_transpose_out_size(yh, kh, pad, stride, dilation),
                  L.ag_conv_transpose_out_size(yw, kw, pad, stride, dilation))
    xh, xw = out_hw
    gx = _empty((B, xch, xh, xw), gy)
    gcols = _empty((B, xch * kh * kw, yh * yw), gy)
    L = capi.lib()
    if return_cols:
        # the caller wants the columns: the reference's two steps through their own entry points, the GEMM
        # gcols_b = w^T . gy_b (conv2d_transpose.rs:114-116, 167-182) and col2im (conv_ops/mod.rs:178-223), with the
        # operator's argument checks done by a call on an empty batch
        check(L.ag_conv2d_transpose_f32(_stream(), _ptr(gy), _ptr(w), _ptr(gx), _ptr(gcols), 0, ych, yh, yw,
                                        xch, kh, kw, pad, stride, dilation, xh, xw))
        M, P = xch * kh * kw, yh * yw
        if B and M and P:
            check(L.ag_gemm_f32(_stream(), 1, 0, M, P, ych, 1.0, _ptr(w), M, 0, _ptr(gy), P, ych * P, 0.0, _ptr(gcols), P,
                                M * P, B))
        check(L.ag_col2im_f32(_stream(), _ptr(gcols), _ptr(gx), B, xch, xh, xw, kh, kw, pad, pad, stride, stride,
                              dilation, dilation, yh, yw))
        return gx, gcols
    check(L.ag_conv2d_transpose_f32(_stream(), _ptr(gy), _ptr(w), _ptr(gx), _ptr(gcols), B, ych, yh, yw,
                                    xch, kh, kw, pad, stride, dilation, xh, xw))
    return gx


def conv2d_nocols(x, w, pad, stride=1, dilation=1):
    """Column-free forward (stride 1 or 2): (y, xpad) or None when the geometry is not supported.
    `xpad` (the rearranged input) is what conv2d_filter_grad_nocols reads instead of the columns."""
    x, w = _f32(x, "conv2d"), _f32(w, "conv2d")
    B, Cc, H, W = x.shape
    Kf, C2, kh, kw = w.shape
    if Cc != C2:
        raise capi.IncompatibleShape(f"conv2d: Number of input channels ({Cc}) must match second filter dim ({C2})")
    L = capi.lib()
    n = L.ag_conv2d_nocols_scratch_floats(B, Cc, H, W, Kf, kh, kw, pad, stride, dilation)
    if n == 0:
        return None
    xpad = torch.empty(n, dtype=torch.float32, device=x.device)
    OH, OW = conv_out_size(H, kh, pad, stride, dilation), conv_out_size(W, kw, pad, stride, dilation)
    y = _empty((B, Kf, OH, OW), x)
    check(L.ag_conv2d_fwd_nocols_f32(_stream(), _ptr(x), _ptr(w), _ptr(y), _ptr(xpad), B, Cc, H, W, Kf, kh, kw, pad,
                                     stride, dilation))
    return y, xpad


def conv_input_grad_staged(gy, w, pad, x_hw, stride=1, dilation=1):
    """The two stages of the column-free input gradient (stride 1 or 2): (gx, scratch); the scratch
    starts with the zero-bordered gy that conv2d_filter_grad_nocols takes.  None when not supported."""
    gy, w = _f32(gy, "conv2d_transpose"), _f32(w, "conv2d_transpose")
    B, ych, yh, yw = gy.shape
    _, xch, kh, kw = w.shape
    xh, xw = x_hw
    L = capi.lib()
    geom = (B, ych, yh, yw, xch, kh, kw, pad, stride, dilation, xh, xw)
    n = L.ag_conv_input_grad_scratch_floats(*geom)
    if n == 0:
        return None
    scratch = torch.empty(n, dtype=torch.float32, device=gy.device)
    gx = _empty((B, xch, xh, xw), gy)
    check(L.ag_conv_input_grad_prepare_f32(_stream(), _ptr(gy), _ptr(w), _ptr(scratch), *geom))
    check(L.ag_conv_input_grad_gemm_f32(_stream(), _ptr(scratch), _ptr(gx), *geom))
    return gx, scratch


def conv2d_filter_grad_nocols(xpad, gypad, x_shape, w_shape, pad, stride=1, dilation=1):
    """Column-free filter gradient from the rearranged copies of x (conv2d_nocols) and gy
    (conv_input_grad_staged): "same" convolutions for stride 1, any supported geometry for stride 2."""
    B, Cc, H, W = x_shape
    Kf, _, kh, kw = w_shape
    L = capi.lib()
    gw = _empty(w_shape, xpad)
    geom = (B, Cc, H, W, Kf, kh, kw, pad, stride, dilation)
    ws = _ws(L.ag_conv2d_filter_grad_nocols_f32_workspace(*geom), xpad)
    check(L.ag_conv2d_filter_grad_nocols_f32(_stream(), _ptr(xpad), _ptr(gypad), _ptr(gw), *geom, _ptr(ws), ws.numel()))
    return gw


def conv2d_transpose_filter_grad(x, gy, w_shape, pad, stride, dilation=1):
    """Conv2DTransposeFilterGrad::compute (conv2d_transpose.rs:433-451)."""
    x, gy = _f32(x, "conv2d_transpose_filter_grad"), _f32(gy, "conv2d_transpose_filter_grad")
    B, ych, yh, yw = x.shape
    _, xch, H, W = gy.shape
    kh, kw = w_shape[2], w_shape[3]
    gw = _empty(w_shape, x)
    gycols = _empty((B, xch * kh * kw, yh * yw), x)
    nbytes = capi.lib().ag_conv2d_filter_grad_f32_workspace(B, xch * kh * kw, yh * yw, ych)
    ws = _ws(nbytes, x)
    check(capi.lib().ag_conv2d_transpose_filter_grad_f32(_stream(), _ptr(x), _ptr(gy), _ptr(gw), _ptr(gycols), B,
                                                         ych, yh, yw, xch, H, W, kh, kw, pad, stride, dilation,
                                                         _ptr(ws), ws.numel()))
    return gw


# ------------------------------------------------------------------------------------------ pooling
def max_pool2d(x, pool_size, pad, stride):
    """MaxPool2D::compute: returns (y, argmax as f32, tap bytes = exact selection inside each window)."""
    x = _f32(x, "max_pool2d")
    B, Cc, H, W = x.shape
    L = capi.lib()
    OH, OW = L.ag_pool_out_size(H, pool_size, pad, stride), L.ag_pool_out_size(W, pool_size, pad, stride)
    y = _empty((B, Cc, max(OH, 0), max(OW, 0)), x)
    am = torch.empty_like(y)
    il = torch.empty(y.shape, dtype=torch.uint8, device=x.device)
    check(L.ag_maxpool2d_fwd_f32(_stream(), _ptr(x), _ptr(y), _ptr(am), _ptr(il), B, Cc, H, W, pool_size, pad,
                                 stride))
    return y, am, il


def relu_max_pool2d(a, b=None):
    """relu(a) or relu(a + b) followed by max_pool2d(2, pad 0, stride 2) in one launch: (r, y, argmax, taps)."""
    a = _f32(a, "relu_max_pool2d")
    if a.dim() != 4:
        raise capi.IncompatibleShape(f"max_pool2d: input must be 4D (got {list(a.shape)})")
    B, Cc, H, W = a.shape
    r = torch.empty_like(a)
    y = _empty((B, Cc, H // 2, W // 2), a)
    am = torch.empty_like(y)
    taps = torch.empty(y.shape, dtype=torch.uint8, device=a.device)
    bshape = None
    if b is not None:
        b = _f32(b, "relu_max_pool2d")
        if b.dim() != 4:
            raise capi.IncompatibleShape(f"add: operands of rank 4 and {b.dim()}")
        bshape = (C.c_int * 4)(*b.shape)
    check(capi.lib().ag_relu_maxpool2d_2x2_f32(_stream(), _ptr(a), _ptr(b), bshape, _ptr(r), _ptr(y), _ptr(am), _ptr(taps),
                                               B, Cc, H, W))
    return r, y, am, taps


def max_pool2d_grad(gy, argmax, taps, x_shape, pool_size, pad, stride):
    gy = _f32(gy, "max_pool2d_grad")
    B, Cc, H, W = x_shape
    gx = _empty(x_shape, gy)
    check(capi.lib().ag_maxpool2d_bwd_f32(_stream(), _ptr(gy), _ptr(argmax), _ptr(taps), _ptr(gx), B, Cc, H,
                                          W, pool_size, pad, stride))
    return gx


def max_pool2d_grad_relu(gy, argmax, taps, relu_x, pool_size, pad, stride):
    """MaxPool2DGrad and the gradient of the ReLU in front of the pooling in one pass:
    greater(relu_x, 0) * max_pool2d_grad(gy)."""
    gy, relu_x = _f32(gy, "max_pool2d_grad"), _f32(relu_x, "max_pool2d_grad")
    B, Cc, H, W = relu_x.shape
    gx = _empty(tuple(relu_x.shape), gy)
    check(capi.lib().ag_maxpool2d_bwd_relu_f32(_stream(), _ptr(gy), _ptr(argmax), _ptr(taps), _ptr(relu_x), _ptr(gx),
                                               B, Cc, H, W, pool_size, pad, stride))
    return gx


def max_pool2d_grad_grad(ggx, argmax, taps, pool_size, pad, stride):
    ggx = _f32(ggx, "max_pool2d_grad_grad")
    B, Cc, H, W = ggx.shape
    L = capi.lib()
    OH, OW = L.ag_pool_out_size(H, pool_size, pad, stride), L.ag_pool_out_size(W, pool_size, pad, stride)
    ggy = _empty((B, Cc, OH, OW), ggx)
    check(L.ag_maxpool2d_gradgrad_f32(_stream(), _ptr(ggx), _ptr(argmax), _ptr(taps), _ptr(ggy), B, Cc, H, W,
                                      pool_size, pad, stride))
    return ggy


# ------------------------------------------------------------------------------------------ reductions
def sum_all(x):
    x = _f32(x, "sum_all")
    out = _empty((), x)
    ws = _ws(capi.lib().ag_sum_all_f32_workspace(x.numel()), x)
    check(capi.lib().ag_sum_all_f32(_stream(), _ptr(x), x.numel(), _ptr(out), _ptr(ws), ws.numel()))
    return out


def _axes(axes, rank):
    ax = [int(a) % rank if rank else int(a) for a in axes]
    return ax, (C.c_int * max(1, len(ax)))(*ax)


def reduce_sum(x, axes, keep_dims=False, mean=False):
    x = _f32(x, "reduce_sum")
    ax, cax = _axes(axes, x.dim())
    shape = (C.c_int * max(1, x.dim()))(*x.shape)
    red = set(ax)
    out_shape = [1 if i in red else s for i, s in enumerate(x.shape)]
    out = _empty(out_shape, x)
    L = capi.lib()
    ws = _ws(L.ag_reduce_sum_f32_workspace(shape, x.dim(), cax, len(ax)), x)
    check(L.ag_reduce_sum_f32(_stream(), _ptr(x), _ptr(out), shape, x.dim(), cax, len(ax), int(mean), _ptr(ws),
                              ws.numel()))
    if not keep_dims:
        out = out.reshape([s for i, s in enumerate(x.shape) if i not in red])
    return out


def reduce_mean(x, axes, keep_dims=False):
    return reduce_sum(x, axes, keep_dims, mean=True)


def broadcast_grad(gy, x_shape, axes):
    gy = _f32(gy, "reduce_grad")
    rank = len(x_shape)
    ax, cax = _axes(axes, rank)
    shape = (C.c_int * max(1, rank))(*x_shape)
    gx = _empty(x_shape, gy)
    check(capi.lib().ag_broadcast_grad_f32(_stream(), _ptr(gy), _ptr(gx), shape, rank, cax, len(ax)))
    return gx


# ------------------------------------------------------------------------------------------ Adam + glue
def adam_update(param, grad, m, v, t, alpha=1e-3, eps=1e-8, b1=0.9, b2=0.999):
    """AdamOp::compute: in place on param, m, v and the one-element step counter t."""
    for a in (param, grad, m, v, t):
        assert a.is_cuda and a.dtype == torch.float32 and a.is_contiguous()
    check(capi.lib().ag_adam_update_f32(_stream(), _ptr(param), _ptr(grad), _ptr(m), _ptr(v), _ptr(t),
                                        param.numel(), alpha, eps, b1, b2))


def adam_update_multi(params, grads, ms, vs, ts, alpha=1e-3, eps=1e-8, b1=0.9, b2=0.999):
    """One optimizer step over several parameters (one AdamOp::compute each in the reference) as one launch."""
    import ctypes as C
    n = len(params)
    assert len(grads) == len(ms) == len(vs) == len(ts) == n
    for a in (*params, *grads, *ms, *vs, *ts):
        assert a.is_cuda and a.dtype == torch.float32 and a.is_contiguous()
    table = lambda xs: (C.c_void_p * max(n, 1))(*[x.data_ptr() for x in xs])
    sizes = (C.c_size_t * max(n, 1))(*[p.numel() for p in params])
    check(capi.lib().ag_adam_update_multi_f32(_stream(), n, table(params), table(grads), table(ms), table(vs), table(ts),
                                              sizes, alpha, eps, b1, b2))


def relu(x):
    x = _f32(x, "relu")
    y = torch.empty_like(x)
    check(capi.lib().ag_relu_f32(_stream(), _ptr(x), _ptr(y), x.numel()))
    return y


def relu_grad(x, gy):
    x, gy = _f32(x, "relu_grad"), _f32(gy, "relu_grad")
    gx = torch.empty_like(x)
    check(capi.lib().ag_relu_grad_f32(_stream(), _ptr(x), _ptr(gy), _ptr(gx), x.numel()))
    return gx


def add_bias(x, bias):
    x, bias = _f32(x, "add"), _f32(bias, "add")
    y = torch.empty_like(x)
    check(capi.lib().ag_add_bias_f32(_stream(), _ptr(x), _ptr(bias), _ptr(y), x.shape[0], x.shape[1]))
    return y


def add_broadcast(x, b):
    """x + b where b has x's rank and extent 1 on the axes it is broadcast along."""
    x, b = _f32(x, "add"), _f32(b, "add")
    if x.dim() != b.dim():
        raise capi.IncompatibleShape(f"add: operands of rank {x.dim()} and {b.dim()}")
    y = torch.empty_like(x)
    shape = (C.c_int * max(x.dim(), 1))(*x.shape)
    bshape = (C.c_int * max(x.dim(), 1))(*b.shape)
    check(capi.lib().ag_add_broadcast_f32(_stream(), _ptr(x), _ptr(b), _ptr(y), shape, bshape, x.dim()))
    return y


def add_broadcast_relu(x, b):
    """relu(x + b) in one pass, b as for add_broadcast."""
    x, b = _f32(x, "add+relu"), _f32(b, "add+relu")
    if x.dim() != b.dim():
        raise capi.IncompatibleShape(f"add+relu: operands of rank {x.dim()} and {b.dim()}")
    y = torch.empty_like(x)
    shape = (C.c_int * max(x.dim(), 1))(*x.shape)
    bshape = (C.c_int * max(x.dim(), 1))(*b.shape)
    check(capi.lib().ag_add_broadcast_relu_f32(_stream(), _ptr(x), _ptr(b), _ptr(y), shape, bshape, x.dim()))
    return y


def bias_grad(gy):
    gy = _f32(gy, "reduce_sum")
    out = _empty((1, gy.shape[1]), gy)
    check(capi.lib().ag_bias_grad_f32(_stream(), _ptr(gy), _ptr(out), gy.shape[0], gy.shape[1]))
    return out


def add_n(xs):
    xs = [_f32(a, "add_n") for a in xs]
    out = torch.empty_like(xs[0])
    arr = (C.c_void_p * len(xs))(*[a.data_ptr() for a in xs])
    check(capi.lib().ag_add_n_f32(_stream(), arr, len(xs), _ptr(out), out.numel()))
    return out


def mul(a, b):
    a, b = _f32(a, "mul"), _f32(b, "mul")
    out = torch.empty_like(a)
    check(capi.lib().ag_mul_f32(_stream(), _ptr(a), _ptr(b), _ptr(out), a.numel()))
    return out


def scale(a, s):
    a = _f32(a, "scale")
    out = torch.empty_like(a)
    check(capi.lib().ag_scale_f32(_stream(), _ptr(a), float(s), _ptr(out), a.numel()))
    return out


def fill(shape, value, device="cuda"):
    out = torch.empty(tuple(shape), dtype=torch.float32, device=device)
    check(capi.lib().ag_fill_f32(_stream(), _ptr(out), float(value), out.numel()))
    return out


def sparse_softmax_cross_entropy(logits, labels):
    logits, labels = _f32(logits, "SparseSoftmaxCrossEntropy"), _f32(labels, "SparseSoftmaxCrossEntropy")
    if logits.dim() != 2:
        raise capi.IncompatibleShape(
            f"SparseSoftmaxCrossEntropy: given first argument's ndim is not 2: shape={list(logits.shape)}")
    if not (labels.dim() == 1 or (labels.dim() == 2 and labels.shape[1] == 1)):
        raise capi.IncompatibleShape(
            "SparseSoftmaxCrossEntropy: second argument's shape must be (batch_size, 1) or (batch_size,). "
            f"given shape={list(labels.shape)}")
    rows, classes = logits.shape
    loss = _empty((rows, 1), logits)
    lsm = torch.empty_like(logits)
    check(capi.lib().ag_sparse_softmax_xent_f32(_stream(), _ptr(logits), _ptr(labels), _ptr(loss), _ptr(lsm), rows,
                                                classes))
    return loss, lsm


def sparse_softmax_cross_entropy_grad(log_softmax, labels, gy):
    lsm, labels, gy = (_f32(log_softmax, "SparseSoftmaxCrossEntropyGrad"),
                       _f32(labels, "SparseSoftmaxCrossEntropyGrad"), _f32(gy, "SparseSoftmaxCrossEntropyGrad"))
    gx = torch.empty_like(lsm)
    check(capi.lib().ag_sparse_softmax_xent_grad_f32(_stream(), _ptr(lsm), _ptr(labels), _ptr(gy), _ptr(gx),
                                                     lsm.shape[0], lsm.shape[1]))
    return gx


def sparse_softmax_cross_entropy_grad_from_logits(logits, labels, gy):
    """The gradient without the forward's log-softmax; `gy`: a tensor of one value per row, or a float."""
    logits, labels = _f32(logits, "SparseSoftmaxCrossEntropyGrad"), _f32(labels, "SparseSoftmaxCrossEntropyGrad")
    gx = torch.empty_like(logits)
    const = isinstance(gy, (int, float))
    check(capi.lib().ag_sparse_softmax_xent_grad_logits_f32(_stream(), _ptr(logits), _ptr(labels), None if const else _ptr(gy),
                                                            float(gy) if const else 0.0, _ptr(gx), logits.shape[0], logits.shape[1]))
    return gx


# ------------------------------------------------------------------------------------------ 8-bit operands
# The launchers from here on serve calls that take a few microseconds on the device, so what they do on the host counts:
# pointers travel as plain integers, and each tensor is looked at once.
class E4m3(NamedTuple):
    """An 8-bit operand: q [rows, pitch(n)] of float8_e4m3fn, scales [rows, scale_pitch(n)] of float8_e8m0fnu (one power of
    two per block of 128), n elements per row along the contraction; an element is q * scale."""
    q: torch.Tensor
    scales: torch.Tensor
    n: int

    @property
    def rows(self):
        return self.q.shape[0]

    def values(self):
        """The f32 values [rows, n] it stands for."""
        power = self.scales.float()[:, : self.q.shape[1] // 128]
        return (self.q.float().view(self.q.shape[0], -1, 128) * power[:, :, None]).view(self.q.shape)[:, : self.n]


def _here(t, name, dtype=torch.float32):
    """t, contiguous, if it is a tensor of that type on the current device (a launch goes to that device's stream)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise capi.TypeUnsupported(f"{name}: expected a CUDA tensor")
    if t.dtype is not dtype:
        raise capi.TypeUnsupported(f"{name}: expected {dtype} (got {t.dtype})")
    if t.get_device() != torch._C._cuda_getDevice():
        raise capi.TypeUnsupported(f"{name}: a tensor on {t.device} while cuda:{torch.cuda.current_device()} is the current device")
    return t if t.is_contiguous() else t.contiguous()


def _ints(name, m, n, k=0):
    """Refuses extents that the C ABI's ints do not hold (ctypes would pass the low 32 bits)."""
    if m > 0x7FFFFFFF or n > 0x7FFFFFFF or k > 0x7FFFFFFF:
        raise capi.InvalidDims(f"{name}: an extent of {max(m, n, k)} (at most 2147483647)")


def _matrix(x, name):
    x = _here(x, name)
    if x.dim() != 2:
        raise capi.IncompatibleShape(f"{name}: input must be 2D (got {list(x.shape)})")
    return x


def _e4m3_empty(rows, n, device):
    return E4m3(torch.empty((rows, -(-n // 128) * 128), dtype=torch.float8_e4m3fn, device=device),
                torch.empty((rows, -(-n // 512) * 4), dtype=torch.float8_e8m0fnu, device=device), n)


def _e4m3(e, name):
    """Checks an 8-bit operand against the layout that the kernels read: (values, scales, rows, n)."""
    if not isinstance(e, E4m3):
        raise capi.TypeUnsupported(f"{name}: expected an E4m3 of CUDA tensors")
    q, scales = _here(e.q, name, torch.float8_e4m3fn), _here(e.scales, name, torch.float8_e8m0fnu)
    if q.dim() != 2 or q.shape[1] != -(-e.n // 128) * 128 or scales.shape != (q.shape[0], -(-e.n // 512) * 4):
        raise capi.IncompatibleShape(f"{name}: values {list(q.shape)} and scales {list(scales.shape)} are not those of rows of {e.n} elements")
    return q, scales, q.shape[0], e.n


def quantize_e4m3(x, transpose=False):
    """x [rows, cols] rounded to 8 bits along its rows; transpose=True: along its columns, as the transposed array."""
    x = _matrix(x, "quantize_e4m3")
    rows, cols = x.shape
    _ints("quantize_e4m3", rows, cols)
    e = _e4m3_empty(cols, rows, x.device) if transpose else _e4m3_empty(rows, cols, x.device)
    q, s = e.q.data_ptr(), e.scales.data_ptr()
    out = (None, None, q, s) if transpose else (q, s, None, None)
    check(capi.lib().ag_quantize_e4m3_f32(_stream(), x.data_ptr(), cols, rows, cols, *out))
    return e


def quantize_e4m3_both(x):
    """Both of quantize_e4m3's results from one pass over x: (along rows, transposed)."""
    x = _matrix(x, "quantize_e4m3")
    rows, cols = x.shape
    _ints("quantize_e4m3", rows, cols)
    e, t = _e4m3_empty(rows, cols, x.device), _e4m3_empty(cols, rows, x.device)
    check(capi.lib().ag_quantize_e4m3_f32(_stream(), x.data_ptr(), cols, rows, cols, e.q.data_ptr(), e.scales.data_ptr(), t.q.data_ptr(),
                                          t.scales.data_ptr()))
    return e, t


def matmul_e4m3(a, b):
    """a . b^T of two 8-bit operands, in f32.  For y = x . w (x [M,K], w [K,N]): matmul_e4m3(quantize_e4m3(x),
    quantize_e4m3(w, transpose=True)); its gradients are matmul_e4m3(quantize_e4m3(gy), quantize_e4m3(w)) and
    matmul_e4m3(quantize_e4m3(x, transpose=True), quantize_e4m3(gy, transpose=True))."""
    qa, sa, m, k = _e4m3(a, "matmul_e4m3")
    qb, sb, n, kb = _e4m3(b, "matmul_e4m3")
    if k != kb:
        raise capi.IncompatibleShape(f"matmul_e4m3: contractions of {k} and {kb} elements")
    _ints("matmul_e4m3", m, n, k)
    c = torch.empty((m, n), dtype=torch.float32, device=qa.device)
    L = capi.lib()
    nbytes = L.ag_matmul_e4m3_f32_workspace(m, n, k)
    ws = _ws(nbytes, c) if nbytes else None
    check(L.ag_matmul_e4m3_f32(_stream(), m, n, k, qa.data_ptr(), sa.data_ptr(), qb.data_ptr(), sb.data_ptr(), c.data_ptr(), n,
                               ws.data_ptr() if nbytes else None, nbytes))
    return c


def quantize_matmul_e4m3(x, b):
    """quantize_e4m3(x) . b^T in one call: a layer whose weight was laid out in 8 bits once."""
    x = _matrix(x, "quantize_matmul_e4m3")
    q, s, n, kb = _e4m3(b, "quantize_matmul_e4m3")
    m, k = x.shape
    if k != kb:
        raise capi.IncompatibleShape(f"quantize_matmul_e4m3: contractions of {k} and {kb} elements")
    _ints("quantize_matmul_e4m3", m, n, k)
    c = torch.empty((m, n), dtype=torch.float32, device=x.device)
    L = capi.lib()
    nbytes = L.ag_quantize_matmul_e4m3_f32_workspace(m, n, k)
    ws = _ws(nbytes, x) if nbytes else None
    check(L.ag_quantize_matmul_e4m3_f32(_stream(), m, n, k, x.data_ptr(), k, q.data_ptr(), s.data_ptr(), c.data_ptr(), n,
                                        ws.data_ptr() if nbytes else None, nbytes))
    return c


# ------------------------------------------------------------------------------------------ RMS norm
def _rms_norm(x, weight, eps, residual, e4m3):
    x, weight = _here(x, "rms_norm"), _here(weight, "rms_norm")
    if x.dim() < 1 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise capi.IncompatibleShape(f"rms_norm: weight {list(weight.shape)} for rows of {list(x.shape)}")
    n = x.shape[-1]
    rows = x.numel() // n if n else 0
    _ints("rms_norm", rows, n)
    h, res = x, None
    if residual is not None:
        res = _here(residual, "rms_norm")
        if res.shape != x.shape:
            raise capi.IncompatibleShape(f"rms_norm: residual {list(res.shape)} and input {list(x.shape)}")
        h = torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    if e4m3:
        y = _e4m3_empty(rows, n, x.device)
        out = (None, y.q.data_ptr(), y.scales.data_ptr())
    else:
        y = torch.empty_like(x)
        out = (y.data_ptr(), None, None)
    check(capi.lib().ag_rms_norm_f32(_stream(), x.data_ptr(), res.data_ptr() if res is not None else None, weight.data_ptr(), eps,
                                     h.data_ptr() if res is not None else None, *out, rstd.data_ptr(), rows, n))
    return y, h, rstd


def rms_norm(x, weight, eps=1e-6, residual=None):
    """(y, h, rstd): h = x + residual (x itself without one), y = h / sqrt(mean(h^2) + eps) * weight over the last axis."""
    return _rms_norm(x, weight, eps, residual, False)


def rms_norm_e4m3(x, weight, eps=1e-6, residual=None):
    """(e, h, rstd): rms_norm whose y leaves as an 8-bit operand, the bits of quantize_e4m3(y); the rows are those of x
    viewed as a matrix."""
    return _rms_norm(x, weight, eps, residual, True)


def rms_norm_grad(h, weight, rstd, gy, gh=None):
    """(gx, gw) from rms_norm's h and rstd; gh: the gradient that reaches h on other ways, added to gx."""
    h, weight, rstd, gy = (_here(t, "rms_norm_grad") for t in (h, weight, rstd, gy))
    n = h.shape[-1] if h.dim() else 0
    rows = h.numel() // n if n else 0
    if weight.shape != (n,) or rstd.shape != (rows,) or gy.shape != h.shape:
        raise capi.IncompatibleShape(f"rms_norm_grad: h {list(h.shape)}, weight {list(weight.shape)}, rstd {list(rstd.shape)}, "
                                     f"gy {list(gy.shape)}")
    _ints("rms_norm_grad", rows, n)
    if gh is not None:
        gh = _here(gh, "rms_norm_grad")
        if gh.shape != h.shape:
            raise capi.IncompatibleShape(f"rms_norm_grad: gh {list(gh.shape)} and h {list(h.shape)}")
    gx, gw = torch.empty_like(h), torch.empty_like(weight)
    L = capi.lib()
    ws = _ws(L.ag_rms_norm_grad_f32_workspace(rows, n), h)
    check(L.ag_rms_norm_grad_f32(_stream(), h.data_ptr(), weight.data_ptr(), rstd.data_ptr(), gy.data_ptr(), None if gh is None else gh.data_ptr(),
                                 gx.data_ptr(), gw.data_ptr(), rows, n, ws.data_ptr(), ws.numel()))
    return gx, gw


# ------------------------------------------------------------------------------------------ clipping
def _sizes(xs, name):
    """Element counts of dense f32 tensors of the current device."""
    here, f32, ns = torch._C._cuda_getDevice() if len(xs) else 0, torch.float32, []
    for t in xs:
        if t.dtype is not f32 or t.get_device() != here:
            raise capi.TypeUnsupported(f"{name}: only f32 tensors of the current CUDA device are supported")
        if not t.is_contiguous():
            raise capi.IncompatibleShape(f"{name}: tensors must be contiguous")
        ns.append(t.numel())
    return ns


def _pointers(xs):
    return (C.c_void_p * max(len(xs), 1))(*[t.data_ptr() for t in xs])


def _norm_call(xs, ns):
    """Host tables, result and workspace of a norm over the tensors."""
    table = (C.c_size_t * max(len(ns), 1))(*ns)
    clip = torch.empty(2, dtype=torch.float32, device=xs[0].device if len(xs) else "cuda")
    return table, clip, _ws(capi.lib().ag_global_norm_f32_workspace(len(ns), table), clip)


def _global_norm(xs, ns, max_norm):
    table, clip, ws = _norm_call(xs, ns)
    check(capi.lib().ag_global_norm_f32(_stream(), len(ns), _pointers(xs), table, max_norm, clip.data_ptr(), ws.data_ptr(), ws.numel()))
    return clip, table


def global_norm(xs, max_norm=float("inf")):
    """[norm over all elements of the tensors, the coefficient that clips it to max_norm], on the device."""
    return _global_norm(xs, _sizes(xs, "global_norm"), max_norm)[0]


def clip_by_global_norm(xs, max_norm, outs=None):
    """(outs, clip): the tensors times clip[1]; `outs` may be the tensors themselves (default: new ones)."""
    ns = _sizes(xs, "clip_by_global_norm")
    if outs is None:
        outs = [torch.empty_like(x) for x in xs]
    elif _sizes(outs, "clip_by_global_norm") != ns:
        raise capi.IncompatibleShape("clip_by_global_norm: outputs and inputs differ in number or size")
    table, clip, ws = _norm_call(xs, ns)
    check(capi.lib().ag_clip_by_global_norm_f32(_stream(), len(ns), _pointers(xs), _pointers(outs), table, max_norm, clip.data_ptr(), ws.data_ptr(),
                                                ws.numel()))
    return outs, clip


def _adam_shares_nothing(params, grads, ms, vs, ts, ns):
    """What the library refuses within one launch, for all of several: two parameters with an array or a step counter in
    common, and a gradient that is an array another parameter updates."""
    filled = [i for i, n in enumerate(ns) if n]
    shared = len(set(ts)) < len(ns) or any(len({a[i] for i in filled}) < len(filled) for a in (params, ms, vs))
    owner = {a[i]: i for a in (params, ms, vs) for i in filled}
    if shared or any(owner.get(grads[i], i) != i for i in filled):
        raise capi.InvalidDims("adam: parameters share an array; update them in separate calls")


def adam_update_clipped(params, grads, ms, vs, ts, max_norm, alpha=1e-3, eps=1e-8, b1=0.9, b2=0.999):
    """One optimizer step on gradients clipped to max_norm over all of them, in place on params, ms, vs, ts (any number of
    parameters); the gradients themselves are left as they are.  Returns [norm, coefficient] on the device."""
    ns = _sizes(grads, "adam")
    if any(_sizes(xs, "adam") != ns for xs in (params, ms, vs)) or len(ts) != len(ns) or any(t < 1 for t in _sizes(ts, "adam")):
        raise capi.IncompatibleShape("adam: parameter, gradient and moment sizes differ")
    L = capi.lib()
    n, most, word, st = len(ns), L.ag_adam_update_multi_max(), C.sizeof(C.c_void_p), _stream()
    tables = [_pointers(xs) for xs in (params, grads, ms, vs, ts)]
    if n > most:
        _adam_shares_nothing(*tables, ns)
    clip, table = _global_norm(grads, ns, max_norm)
    tables.append(table)
    pc = clip.data_ptr()
    for i in range(0, n, most):
        check(L.ag_adam_update_multi_clipped_f32(st, min(most, n - i), *[C.byref(t, i * word) for t in tables], alpha, eps, b1, b2, pc))
    return clip
