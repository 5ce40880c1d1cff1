"""What the 8-bit product, the RMS norm and clipping refuse: argument checks run on the host before anything is launched, so
they are tested without a GPU, with pointers that are never followed."""
import ctypes as C
import math

import pytest


@pytest.fixture(scope="module")
def capi():
    import __graft_entry__ as entry
    return entry.load_package().capi


@pytest.fixture(scope="module")
def L(capi):
    return capi.lib()


N, P, ODD = None, C.c_void_p(4096), C.c_void_p(4104)  # null, aligned, not aligned to 16 bytes


def table(*at):
    return (C.c_void_p * len(at))(*at)


def sizes(*ns):
    return (C.c_size_t * len(ns))(*ns)


def refused(L, status, code, text):
    assert status == code, (status, L.ag_last_error())
    assert text in L.ag_last_error().decode()


def test_layout_of_an_operand(L):
    assert [L.ag_e4m3_pitch(n) for n in (-1, 0, 1, 128, 129, 4096)] == [0, 0, 128, 128, 256, 4096]
    assert [L.ag_e4m3_scale_pitch(n) for n in (-1, 0, 1, 512, 513, 4096)] == [0, 0, 4, 4, 8, 32]
    assert L.ag_e4m3_pitch(2 ** 31 - 1) == 2 ** 31 and L.ag_e4m3_scale_pitch(2 ** 31 - 1) == 2 ** 24


def test_quantize(L):
    f = L.ag_quantize_e4m3_f32
    refused(L, f(N, P, 4, -1, 4, P, P, N, N), 4, "negative extent")
    refused(L, f(N, P, 3, 2, 4, P, P, N, N), 2, "ldx (3)")
    refused(L, f(N, N, 4, 2, 4, P, P, N, N), 4, "null pointer")
    refused(L, f(N, P, 4, 2, 4, P, N, N, N), 4, "go together")
    refused(L, f(N, P, 4, 2, 4, P, P, N, P), 4, "go together")
    refused(L, f(N, P, 4, 2, 4, N, N, N, N), 4, "no output")
    refused(L, f(N, P, 4, 2, 4, ODD, P, N, N), 4, "16-byte aligned")
    refused(L, f(N, P, 4, 2, 4, N, N, ODD, P), 4, "16-byte aligned")
    assert f(N, N, 4, 0, 4, N, N, N, N) == 0


def test_product(L):
    f = L.ag_matmul_e4m3_f32
    refused(L, f(N, 2, -2, 4, P, P, P, P, P, 4, P, 1 << 30), 4, "negative extent")
    refused(L, f(N, 2, 8, 4, P, P, P, P, P, 7, P, 1 << 30), 2, "ldc (7)")
    refused(L, f(N, 2, 8, (1 << 28) + 1, P, P, P, P, P, 8, P, 1 << 30), 4, "at most 2^28")
    refused(L, f(N, 2, 8, 4, P, C.c_void_p(4098), P, P, P, 8, P, 1 << 30), 4, "4-byte aligned")
    refused(L, f(N, 2, 8, 4, P, P, P, C.c_void_p(4098), P, 8, P, 1 << 30), 4, "4-byte aligned")
    need = L.ag_matmul_e4m3_f32_workspace(64, 1000, 8192)  # a contraction that is cut
    assert need > 0
    refused(L, f(N, 64, 1000, 8192, P, P, P, P, P, 1000, P, need - 1), 4, "workspace")
    refused(L, f(N, 64, 1000, 8192, P, P, P, P, P, 1000, ODD, need), 4, "misaligned workspace")
    for a in ((N, P, P, P, P), (P, N, P, P, P), (P, P, N, P, P), (P, P, P, N, P), (P, P, P, P, N)):
        refused(L, f(N, 2, 8, 4, *a, 8, P, 1 << 30), 4, "null pointer")
    refused(L, f(N, 2, 8, 4, ODD, P, P, P, P, 8, P, 1 << 30), 4, "16-byte aligned")
    refused(L, f(N, 2, 8, 4, P, P, ODD, P, P, 8, P, 1 << 30), 4, "16-byte aligned")
    assert f(N, 0, 8, 4, N, N, N, N, N, 8, N, 0) == 0 and f(N, 8, 0, 4, N, N, N, N, N, 0, N, 0) == 0
    assert L.ag_matmul_e4m3_f32_workspace(0, 4, 4) == 0
    g = L.ag_quantize_matmul_e4m3_f32
    need = L.ag_quantize_matmul_e4m3_f32_workspace(200, 300, 4096)
    assert need >= 200 * 4096
    refused(L, g(N, 200, 300, 4096, P, 4095, P, P, P, 300, P, need), 2, "ldx (4095)")
    refused(L, g(N, 200, 300, 4096, P, 4096, P, P, P, 300, P, need - 1), 4, "workspace")
    refused(L, g(N, 200, 300, 4096, P, 4096, P, P, P, 300, N, need), 4, "workspace")
    refused(L, g(N, 200, 300, 4096, P, 4096, P, P, P, 300, ODD, need), 4, "misaligned workspace")
    refused(L, g(N, 200, 300, 4096, N, 4096, P, P, P, 300, P, need), 4, "null pointer")
    refused(L, g(N, 200, 300, 4096, P, 4096, N, P, P, 300, P, need), 4, "null pointer")


def test_norm(L):
    f = L.ag_rms_norm_f32
    refused(L, f(N, P, N, P, 1e-6, N, P, N, N, N, 2, -8), 4, "negative extent")
    refused(L, f(N, P, N, P, -1.0, N, P, N, N, N, 2, 8), 4, "eps")
    refused(L, f(N, P, N, P, math.nan, N, P, N, N, N, 2, 8), 4, "eps")
    refused(L, f(N, N, N, P, 1e-6, N, P, N, N, N, 2, 8), 4, "null pointer")
    refused(L, f(N, P, N, N, 1e-6, N, P, N, N, N, 2, 8), 4, "null pointer")
    refused(L, f(N, P, N, P, 1e-6, N, P, P, N, N, 2, 8), 4, "go together")
    refused(L, f(N, P, N, P, 1e-6, N, N, N, N, N, 2, 8), 4, "no output")
    refused(L, f(N, P, N, P, 1e-6, P, P, N, N, N, 2, 8), 4, "same array")
    refused(L, f(N, P, N, P, 1e-6, N, P, ODD, P, N, 2, 8), 4, "16-byte aligned")
    assert f(N, N, N, N, 1e-6, N, N, N, N, N, 0, 8) == 0
    g = L.ag_rms_norm_grad_f32
    need = L.ag_rms_norm_grad_f32_workspace(100, 64)
    assert need >= 64 * 4 and L.ag_rms_norm_grad_f32_workspace(0, 64) == 0
    other = C.c_void_p(8192)
    refused(L, g(N, P, P, P, P, N, other, P, -1, 64, P, need), 4, "negative extent")
    for a in ((N, P, P, P), (P, N, P, P), (P, P, N, P), (P, P, P, N)):
        refused(L, g(N, *a, N, other, P, 100, 64, P, need), 4, "null pointer")
    refused(L, g(N, P, P, P, P, N, N, N, 100, 64, P, need), 4, "no output")
    refused(L, g(N, P, P, P, other, N, P, P, 100, 64, P, need), 4, "gx must not be h")
    refused(L, g(N, P, P, P, P, N, other, P, 100, 64, P, need - 1), 4, "workspace")
    refused(L, g(N, P, P, P, P, N, other, P, 100, 64, C.c_void_p(4098), need), 4, "misaligned workspace")


def test_clipping(L):
    f, c = L.ag_global_norm_f32, L.ag_clip_by_global_norm_f32
    xs, ns = table(4096, 8192), sizes(100, 50)
    need = L.ag_global_norm_f32_workspace(2, ns)
    assert need > 0 and L.ag_global_norm_f32_workspace(0, N) == 0
    refused(L, f(N, -1, xs, ns, 1.0, P, P, need), 4, "-1 arrays")
    refused(L, f(N, 2, xs, ns, -1.0, P, P, need), 4, "max_norm")
    refused(L, f(N, 2, xs, ns, math.nan, P, P, need), 4, "max_norm")
    refused(L, f(N, 2, xs, ns, 1.0, N, P, need), 4, "null pointer")
    refused(L, f(N, 2, N, ns, 1.0, P, P, need), 4, "null pointer table")
    refused(L, f(N, 2, table(4096, None), ns, 1.0, P, P, need), 4, "array 1")
    refused(L, f(N, 2, xs, ns, 1.0, P, P, need - 1), 4, "workspace")
    refused(L, f(N, 2, xs, ns, 1.0, P, C.c_void_p(4100), need), 4, "misaligned workspace")
    refused(L, c(N, 2, xs, N, ns, 1.0, P, P, need), 4, "null pointer table")
    refused(L, c(N, 2, xs, table(4096, None), ns, 1.0, C.c_void_p(1 << 20), P, need), 4, "array 1")
    # the same array twice in place, an output over another input, an output over another output, a shifted copy of itself
    F = C.c_void_p(1 << 20)
    refused(L, c(N, 2, table(4096, 4096), table(4096, 4096), ns, 1.0, F, P, need), 4, "overlaps")
    refused(L, c(N, 2, xs, table(16384, 4100), ns, 1.0, F, P, need), 4, "overlaps")
    refused(L, c(N, 2, xs, table(16384, 16396), ns, 1.0, F, P, need), 4, "overlaps")
    refused(L, c(N, 2, xs, table(4100, 16384), ns, 1.0, F, P, need), 4, "overlaps")
    refused(L, c(N, 2, xs, table(4092, 16384), ns, 1.0, F, P, need), 4, "overlaps")
    # the norm and coefficient inside an input, inside an output
    refused(L, c(N, 2, xs, table(16384, 32768), ns, 1.0, C.c_void_p(8200), P, need), 4, "array 1 overlaps the norm")
    refused(L, c(N, 2, xs, table(16384, 32768), ns, 1.0, C.c_void_p(16380), P, need), 4, "array 0 overlaps the norm")


def test_clipped_adam(L):
    f = L.ag_adam_update_multi_clipped_f32
    one, t = sizes(10), table(4096)
    refused(L, f(N, 1, t, table(8192), table(12288), table(16384), table(20480), one, 1e-3, 1e-8, 0.9, 0.999, N), 4, "clipping coefficient")
    refused(L, f(N, 99, t, t, t, t, t, one, 1e-3, 1e-8, 0.9, 0.999, P), 4, "at most")
    refused(L, f(N, 1, t, table(8192), table(12288), table(16384), table(None), one, 1e-3, 1e-8, 0.9, 0.999, P), 4, "step counter")


def test_launchers_refuse_what_is_not_an_f32_tensor_of_the_device(capi):
    """kernels.py looks at its arguments before anything is launched; a CPU tensor is the one that can be made anywhere."""
    import torch
    from rust_autograd_amd import kernels as K

    x, e = torch.zeros(2, 8), None
    for call in (lambda: K.quantize_e4m3(x), lambda: K.quantize_e4m3_both(x), lambda: K.rms_norm(x, x[0]), lambda: K.rms_norm_e4m3(x, x[0]),
                 lambda: K.rms_norm_grad(x, x[0], x[0], x), lambda: K.quantize_matmul_e4m3(x, e), lambda: K.matmul_e4m3(e, e),
                 lambda: K.matmul_e4m3(K.E4m3(x, x, 8), K.E4m3(x, x, 8))):
        with pytest.raises(capi.TypeUnsupported):
            call()
