"""What the operators over 8-bit integers refuse, before anything runs on a device; the rows that they are given room for."""
import pytest
import torch

from nanohybrid_vlm_b200.kernels import ops
from nanohybrid_vlm_b200.kernels.library import KernelError

BF, I8, F = torch.bfloat16, torch.int8, torch.float32


def product(T=3, K=20, N=5, **other):
    given = dict(out=torch.empty(T, N, dtype=BF), x=torch.zeros(T, K, dtype=I8), x_scales=torch.zeros(T), weight=torch.zeros(N, K, dtype=I8),
                 weight_scales=torch.zeros(N))
    given.update(other)
    ops.linear_int8(**given)


@pytest.mark.parametrize("other, text", [
    (dict(x=torch.zeros(3, 21, dtype=I8)), "weight's rows"),
    (dict(x=torch.zeros(3, 20, dtype=torch.uint8)), "x's rows"),
    (dict(x=torch.zeros(20, 3, dtype=I8).t()), "neighbouring columns"),
    (dict(x=torch.zeros(1, 20, dtype=I8).expand(3, 20)), "do not overlap"),
    (dict(weight=torch.zeros(5, 20)), "weight's rows"),
    (dict(weight=torch.zeros(5, 40, dtype=I8)[:, ::2]), "neighbouring columns"),
    (dict(x_scales=torch.zeros(4)), "x_scales"),
    (dict(x_scales=torch.zeros(3, 1)), "x_scales"),
    (dict(x_scales=torch.zeros(3, dtype=BF)), "x_scales"),
    (dict(weight_scales=torch.zeros(10)[::2]), "weight_scales"),
    (dict(out=torch.empty(3, 6, dtype=BF)), "out is"),
    (dict(out=torch.empty(5, 3, dtype=BF).t()), "out is"),
    (dict(out=torch.empty(1, 5, dtype=BF).expand(3, 5)), "out is"),
    (dict(out=torch.empty(3, 5, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(out=torch.empty(15, dtype=BF)), "matrices"),
    (dict(), "GPU only"),
])
def test_products_refused(other, text):
    with pytest.raises(KernelError, match=text):
        product(**other)


@pytest.mark.parametrize("K", [0, 131072])
def test_sums_that_are_not_exact_are_refused(K):
    with pytest.raises(KernelError, match="131071"):
        product(T=1, N=1, K=K)


def rows(**other):
    return dict(q=torch.empty(4, 10, dtype=I8), scales=torch.empty(4)) | other


@pytest.mark.parametrize("other, text", [
    (dict(q=torch.empty(4, 11, dtype=I8)), "8-bit rows"),
    (dict(q=torch.empty(4, 10, dtype=torch.int16)), "8-bit rows"),
    (dict(q=torch.empty(10, dtype=I8).expand(4, 10)), "do not overlap"),
    (dict(scales=torch.empty(5)), "scales"),
    (dict(scales=torch.empty(4, dtype=torch.float64)), "scales"),
    (dict(), "GPU only"),
])
def test_rows_refused(other, text):
    given = rows(**other)
    for call in (lambda: ops.quantize_rows(x=torch.zeros(4, 10, dtype=BF), **given),
                 lambda: ops.rmsnorm_int8(x=torch.zeros(4, 10, dtype=BF), weight=torch.zeros(10, dtype=BF), eps=1e-6, **given),
                 lambda: ops.silu_mul_int8(gate_up=torch.zeros(4, 20, dtype=BF), **given)):
        with pytest.raises(KernelError, match=text):
            call()


def test_rows_of_other_inputs_refused():
    with pytest.raises(KernelError, match="neighbouring columns"):
        ops.quantize_rows(x=torch.zeros(10, 4).t(), **rows())
    with pytest.raises(KernelError, match="float32 or bfloat16"):
        ops.quantize_rows(x=torch.zeros(4, 10, dtype=torch.float16), **rows())
    with pytest.raises(KernelError, match="no elements"):
        ops.quantize_rows(torch.empty(4, 0, dtype=I8), torch.empty(4), torch.empty(4, 0))
    x, w = torch.zeros(4, 10), torch.zeros(10)
    for other in (dict(x=torch.zeros(10, 4).t(), weight=w), dict(x=x, weight=w.to(BF)), dict(x=x, weight=torch.zeros(20)[::2]),
                  dict(x=x, weight=torch.zeros(9)), dict(x=x, weight=w, residual=torch.zeros(4, 11)),
                  dict(x=x, weight=w, residual=x.to(BF)), dict(x=x, weight=w, residual=x)):
        with pytest.raises(KernelError, match="contiguous|weight|residual"):
            ops.rmsnorm_int8(eps=1e-6, **rows(), **other)
    with pytest.raises(KernelError, match="2 \\* inter"):
        ops.silu_mul_int8(gate_up=torch.zeros(4, 21), **rows())
    with pytest.raises(KernelError, match="contiguous"):
        ops.silu_mul_int8(gate_up=torch.zeros(20, 4).t(), **rows())


def test_values_refused():
    q, s = torch.zeros(4, 10, dtype=I8), torch.zeros(4)
    for out, q_, s_, text in ((torch.empty(4, 11), q, s, "8-bit rows"), (torch.empty(4, 10).t(), q, s, "neighbouring"),
                              (torch.empty(10).expand(4, 10), q, s, "do not overlap"), (torch.empty(4, 10), q, torch.zeros(3), "scales"),
                              (torch.empty(4, 10, dtype=torch.float16), q, s, "float32 or bfloat16"), (torch.empty(4, 10), q, s, "GPU only")):
        with pytest.raises(KernelError, match=text):
            ops.dequantize_rows(out, q_, s_)


@pytest.mark.parametrize("width, pitch", [(1, 16), (16, 16), (17, 32), (4096, 4096)])
def test_room_for_rows(width, pitch):
    t = ops.new_int8(3, width, "cpu")
    assert t.shape == (3, width) and t.dtype == I8 and t.stride() == (pitch, 1)


def test_engine_option(model_dirs):
    from nanohybrid_vlm_b200.config import Config
    from nanohybrid_vlm_b200.config.model_config import ConfigError
    assert Config(model_dirs["A"], quantization="int8").quantization == "int8" and Config(model_dirs["A"]).quantization is None
    with pytest.raises(ConfigError, match="int8"):
        Config(model_dirs["A"], quantization="int4")


def test_call_blocks_have_the_size_of_the_librarys_structs():
    """Eight-byte members come first, and a struct's size is a multiple of eight: the library reads so many bytes."""
    assert (ops._ROWS_CALL.size, ops._BACK_CALL.size, ops._PRODUCT_CALL.size) == (88, 56, 96)
