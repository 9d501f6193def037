"""Calls of the operators over 8-bit integers that stand beside their ordinary ones: operands in one buffer with the outputs.  Tolerances as
in ``test_int8_ops_gpu``."""
import pytest
import torch

from nanohybrid_vlm_b200.kernels.library import KernelError
from test_int8_ops_gpu import BF, F, check_rows, gen, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from nanohybrid_vlm_b200.kernels import ops
    return ops


# ------------------------------------------------------------------------------------------------ one buffer
def test_outputs_that_begin_inside_inputs_are_refused(ops):
    """Refused before anything is launched: the inputs stay as they were."""
    n, w = 6, 64
    x = torch.randn(n, w, device="cuda").to(BF)
    both = torch.randn(n, 2 * w, device="cuda").to(BF)
    scales, weight = torch.empty(n, device="cuda"), torch.ones(w, dtype=BF, device="cuda")
    was, were = x.clone(), both.clone()
    inside = x.view(torch.int8)[:, w // 2:w // 2 + w]                    # neither at x's start nor beyond it
    calls = [
        lambda: ops.quantize_rows(inside, scales, x),
        lambda: ops.rmsnorm_int8(inside, scales, x, weight, 1e-6),
        lambda: ops.rmsnorm_int8(inside, scales, x.clone(), weight, 1e-6, residual=x),
        lambda: ops.silu_mul_int8(both.view(torch.int8)[:, w:2 * w], scales, both),
        lambda: ops.quantize_rows(ops.new_int8(n, w, "cuda"), x.view(F).flatten()[3:3 + n], x),
        lambda: ops.dequantize_rows(x[1:, :w // 2].view(BF), x.view(torch.int8)[:n - 1, w // 2:w], scales[:n - 1]),
        lambda: ops.linear_int8(x.flatten()[8:8 + 2 * n].view(n, 2), x.view(torch.int8), scales, ops.new_int8(2, 2 * w, "cuda"), scales[:2]),
        lambda: ops.linear_int8(x[:2, 8:8 + n], ops.new_int8(2, 2 * w, "cuda"), scales[:2], x.view(torch.int8), scales),
    ]
    sums = torch.randn(n * w + 1, device="cuda").to(BF)
    calls.append(lambda: ops.rmsnorm_int8(ops.new_int8(n - 1, w, "cuda"), scales[:n - 1], sums[:(n - 1) * w].view(n - 1, w), weight, 1e-6,
                                          residual=sums[w:n * w].view(n - 1, w)))
    for i, call in enumerate(calls):
        with pytest.raises(KernelError, match="memory of"):
            call()
            pytest.fail(f"call {i}")
    assert torch.equal(x, was) and torch.equal(both, were)


@pytest.mark.parametrize("T", [9, 300])
def test_columns_of_one_buffer(ops, T):
    """What a call reads and writes may be columns of the same rows: every output beside its inputs, product included."""
    g = gen(T)
    K, N, pitch = 96, 48, 1024
    rows = torch.zeros(T, pitch, dtype=torch.uint8, device="cuda").view(torch.int8)
    x, q = rows[:, :2 * K].view(BF), rows[:, 2 * K:3 * K]                # 0 .. 191, 192 .. 287
    back, y = rows[:, 320:320 + 2 * K].view(BF), rows[:, 512:512 + 4 * N].view(F)
    x.copy_(torch.randn(T, K, generator=g, device="cuda"))
    was, s, w, ws = x.clone(), torch.empty(T, device="cuda"), ints(g, N, K), torch.rand(N, generator=g, device="cuda")
    ops.quantize_rows(q, s, x)
    ops.dequantize_rows(back, q, s)
    ops.linear_int8(y, q, s, w, ws)
    check_rows(q, s, was.double(), 0.0, exact=True)
    assert torch.equal(x, was) and torch.equal(back, (q.float() * s[:, None]).to(BF))
    want = (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()[None]
    assert ((y.double() - want).abs() <= 3.1 * 2.0 ** -24 * want.abs()).all()


# ------------------------------------------------------------------------------------------------ the longest rows
@pytest.mark.parametrize("width", [2 ** 31 - 1, 2 ** 31 - 16])
def test_values_of_the_longest_rows(ops, width):
    """One row of as many columns as 32 bits count: nothing before or behind it is touched."""
    q = torch.empty(1, width, dtype=torch.int8, device="cuda")
    q.random_(-127, 128, generator=gen(width % 97))
    whole = torch.full((width + 512,), 3.0, dtype=BF, device="cuda")
    s = torch.tensor([0.37], device="cuda")
    ops.dequantize_rows(whole[256:256 + width][None], q, s)
    for i in range(0, width, 2 ** 28):
        assert torch.equal(whole[256 + i:256 + min(i + 2 ** 28, width)], (q[0, i:i + 2 ** 28].float() * s).to(BF))
    assert (whole[:256] == 3).all() and (whole[256 + width:] == 3).all()
