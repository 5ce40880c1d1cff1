"""HIP counts the threads of a grid in 32 bits per axis: calls whose one launch would need more are refused by name, on the
host, before anything is launched (so without a GPU, with pointers that are never followed)."""
import ctypes as C

import pytest

N, P = None, C.c_void_p(4096)


@pytest.fixture(scope="module")
def L():
    import __graft_entry__ as entry
    return entry.load_package().capi.lib()


def refused(L, status, text):
    assert status == 4 and text in L.ag_last_error().decode(), (status, L.ag_last_error())


@pytest.mark.parametrize("planes", [1 << 24, (1 << 24) + 64, (1 << 28) + 64])
def test_pooling_of_many_small_planes(L, planes):
    # a block of 256 threads per plane: 2^24 planes are 2^32 threads, and 64 more would have run 64 planes
    refused(L, L.ag_maxpool2d_fwd_f32(N, P, P, P, P, planes, 1, 4, 4, 2, 0, 2), "too many tiles")
    refused(L, L.ag_maxpool2d_bwd_f32(N, P, P, P, P, planes, 1, 5, 4, 2, 0, 1), "too many tiles")
    refused(L, L.ag_relu_maxpool2d_2x2_f32(N, P, N, N, P, P, P, P, planes * 4, 1, 16, 16), "too many tiles")


def test_columns_of_many_small_planes(L):
    # [planes, 1, 5, 5], a 3 x 3 filter: padding 1, stride 1, dilation 1
    refused(L, L.ag_im2col_f32(N, P, P, (1 << 24) + 64, 1, 5, 5, 3, 3, 1, 1, 1, 1, 1, 1), "too many tiles")


def test_adam_of_many_elements(L):
    refused(L, L.ag_adam_update_f32(N, P, P, P, P, P, 1 << 36, 1e-3, 1e-8, 0.9, 0.999), "too many elements")
    at = [(C.c_void_p * 1)(4096 * (i + 1)) for i in range(5)]
    refused(L, L.ag_adam_update_multi_f32(N, 1, *at, (C.c_size_t * 1)(1 << 36), 1e-3, 1e-8, 0.9, 0.999), "too many elements")


def test_norm_gradient_of_many_long_rows(L):
    other = C.c_void_p(8192)
    refused(L, L.ag_rms_norm_grad_f32(N, P, P, P, P, N, other, N, 1 << 22, 16385, N, 0), "4194304 rows of 16385")


def test_product_of_many_tiles_and_of_rows_at_the_end_of_an_int(L):
    # K = 0: no operand is read
    most = 2 ** 31 - 1
    f = L.ag_matmul_e4m3_f32
    refused(L, f(N, most - 512, 300, 0, N, N, N, N, P, 300, N, 0), "too many tiles")
    refused(L, f(N, 20, most, 4096, P, P, P, P, P, most, N, 0), "operands of 20 and 2147483647 rows")
    refused(L, f(N, most, 20, 4096, P, P, P, P, P, 20, N, 0), "operands of 2147483647 and 20 rows")
    refused(L, L.ag_quantize_matmul_e4m3_f32(N, 20, most, 4096, P, 4096, P, P, P, most, P, 1 << 40), "operands of 20 and")
