"""A bounded wait of the 8-bit products that runs out reaches the host.  Nothing here faults or hangs: a test build of ``csrc/gemm_int8.cu`` in a
library of its own, with a wait limit of 4,096 polls and a producer that leaves the ring's first stage unsent, lets every role's wait run
out; the blocks of a cluster still meet, tensor memory goes back and the kernel returns."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def starved():
    from nanohybrid_vlm_b200.csrc.build import ensure_variant
    lib = ctypes.CDLL(ensure_variant("gemm_int8.cu", {"NHV_WAIT_LIMIT": 4096, "NHV_TEST_DROP_UNIT": 0, "NHV_OWN_ERROR_TEXT": 1}, folder=""))
    lib.nhv_gemm_int8.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    lib.nhv_gemm_int8.restype = ctypes.c_int
    lib.nhv_gemm_int8_error.restype = ctypes.c_int
    lib.nhv_last_error.restype = ctypes.c_char_p
    return lib


@pytest.mark.parametrize("T,K,N", [(5, 256, 9000), (5, 2048, 512), (300, 512, 512)])        # one part of K, a cluster's parts, pairs
def test_a_wait_that_runs_out(starved, T, K, N):
    from nanohybrid_vlm_b200.kernels import ops
    x, w = ops.new_int8(T, K, "cuda").fill_(2), ops.new_int8(N, K, "cuda").fill_(3)
    xs, ws, y = torch.ones(T, device="cuda"), torch.ones(N, device="cuda"), torch.zeros(T, N, device="cuda")
    given = ops._PRODUCT_CALL.pack(y.data_ptr(), x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), 0, 0, N, K, K, ops.F32, T, N, K)
    assert starved.nhv_gemm_int8(given, torch.cuda.current_stream().cuda_stream) == 0, starved.nhv_last_error()
    torch.cuda.synchronize()
    assert starved.nhv_gemm_int8_error() in (1, 2, 3, 4)      # the producer's, the issuer's or the epilogue's wait, whichever ran out last
    assert starved.nhv_gemm_int8_error() == 0
    ops.linear_int8(y, x, xs, w, ws)                          # the device is as usable as before
    assert (y == 6 * K).all() and ops.take_wait_errors() == []
