"""A bounded wait of the 8-bit products that runs out reaches the host, and a long kernel ahead does not run one out.

Nothing here faults or hangs: a test build of ``csrc/gemm_int8.cu`` in a library of its own, with a wait limit of 4,096 polls and a
producer that leaves the ring's first stage unsent, lets every role's wait run out; the blocks of a cluster still meet, tensor memory
goes back and the kernel returns."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(**more):
    from nanohybrid_vlm_b200.csrc.build import ensure_variant
    lib = ctypes.CDLL(ensure_variant("gemm_int8.cu", {"NHV_WAIT_LIMIT": 4096, "NHV_OWN_ERROR_TEXT": 1, **more}, folder=""))
    lib.nhv_gemm_int8.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    lib.nhv_gemm_int8.restype = ctypes.c_int
    lib.nhv_gemm_int8_error.restype = ctypes.c_int
    lib.nhv_last_error.restype = ctypes.c_char_p
    return lib


@pytest.fixture(scope="module")
def starved():
    return build(NHV_TEST_DROP_UNIT=0)


def product(lib, ops, x, w, xs, ws, y):
    (T, K), N = x.shape, w.shape[0]
    given = ops._PRODUCT_CALL.pack(y.data_ptr(), x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), 0, 0, N, K, K, ops.F32, T, N, K)
    assert lib.nhv_gemm_int8(given, torch.cuda.current_stream().cuda_stream) == 0, lib.nhv_last_error()


@pytest.mark.parametrize("T,K,N", [(5, 256, 9000), (5, 2048, 512), (300, 512, 512)])        # one part of K, a cluster's parts, pairs
def test_a_wait_that_runs_out(starved, T, K, N):
    from nanohybrid_vlm_b200.kernels import ops
    x, w = ops.new_int8(T, K, "cuda").fill_(2), ops.new_int8(N, K, "cuda").fill_(3)
    xs, ws, y = torch.ones(T, device="cuda"), torch.ones(N, device="cuda"), torch.zeros(T, N, device="cuda")
    product(starved, ops, x, w, xs, ws, y)
    torch.cuda.synchronize()
    assert starved.nhv_gemm_int8_error() in (1, 2, 3, 4)      # the producer's, the issuer's or the epilogue's wait, whichever ran out last
    assert starved.nhv_gemm_int8_error() == 0
    ops.linear_int8(y, x, xs, w, ws)                          # the device is as usable as before
    assert (y == 6 * K).all() and ops.take_wait_errors() == []


@pytest.mark.parametrize("T,K,N", [(5, 256, 9000), (5, 2048, 512), (300, 512, 512)])
def test_a_long_kernel_ahead_does_not_count(T, K, N):
    """One row of 2^28 numbers keeps a single block busy for some milliseconds, which lets the product's blocks start beside it (programmatic
    dependent launch) and lie ready: their 4,096 polls begin when it has ended."""
    from nanohybrid_vlm_b200.kernels import ops
    lib = build()
    x, w = ops.new_int8(T, K, "cuda").fill_(2), ops.new_int8(N, K, "cuda").fill_(3)
    xs, ws, y = torch.ones(T, device="cuda"), torch.ones(N, device="cuda"), torch.zeros(T, N, device="cuda")
    wide = torch.ones(1, 1 << 28, dtype=torch.bfloat16, device="cuda")
    q, s = ops.new_int8(1, 1 << 28, "cuda"), torch.empty(1, device="cuda")
    torch.cuda.synchronize()
    ops.quantize_rows(q, s, wide)
    product(lib, ops, x, w, xs, ws, y)
    torch.cuda.synchronize()
    assert lib.nhv_gemm_int8_error() == 0 and (y == 6 * K).all() and q[0, -1] == 127
