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


# ------------------------------------------------------------------------------------------------ gates far from zero
LARGEST = torch.finfo(BF).max


@pytest.mark.parametrize("width", [264, 1031, 32776, 60001])         # pieces in registers, any width, shared memory, read again
@pytest.mark.parametrize("dtype", [BF, F])
def test_gates_far_from_zero(ops, width, dtype):
    """A row for each gate.  In 16 bits the unit is off by (9 + 1.25 |g|) * 2^-24 for negative gates g: the exponent of 2 is g log2 e, rounded, with log2 e
    rounded (together 1.22 |g|), ex2 4, the sum 1, the reciprocal 2, two products 2; for positive ones the 9 alone.  In 32 bits: expf an ulp (2), the sum, the
    division and the product 1 each.  Gates that give 0 have a unit below 2^-119."""
    gates = [-20.0, -40.0, -60.0, -87.0, 30.0, 100.0, LARGEST] + ([-0.75] if dtype == BF else [-88.5])
    none = [-100.0, -LARGEST] + ([-87.5, -88.5] if dtype == BF else [-89.0])
    up = (2 * torch.rand(len(gates + none), width, generator=gen(width), device="cuda") - 1).to(BF).to(dtype)
    gate = torch.tensor(gates + none, device="cuda").to(dtype)
    assert gate.tolist() == pytest.approx(gates + none, rel=1e-6)
    x = torch.cat([gate[:, None].expand(-1, width), up], 1)
    q, s = ops.new_int8(len(gate), width, "cuda").fill_(55), torch.empty(len(gate), device="cuda")
    ops.silu_mul_int8(q, s, x)
    g64 = gate.double()[:, None]
    y = g64 * torch.sigmoid(g64) * up.double()
    for i, g in enumerate(gates):
        check_rows(q[i:i + 1], s[i:i + 1], y[i:i + 1], ((9 + 1.25 * max(0.0, -g)) if dtype == BF else 5) * 2.0 ** -24)
    assert y[len(gates):].abs().max() < 2.0 ** -119 and not s[len(gates):].any() and not q[len(gates):].any()


@pytest.mark.parametrize("spread", [1.5, 12.0, 50.0])
def test_a_row_does_not_depend_on_where_it_lies(ops, spread):
    """The unit and plain rows, without a sum of their own, in either type: pieces of eight, single elements and shared memory give the same."""
    for dtype, n, width in ((BF, 40, 4096), (F, 40, 4096), (BF, 700, 17000), (F, 20, 17000)):
        g = gen(width + n)
        x = (spread * torch.randn(n, 2 * width, generator=g, device="cuda")).to(dtype)
        for call, given in ((ops.silu_mul_int8, x), (ops.quantize_rows, x[:, :width])):
            q, s = ops.new_int8(n, width, "cuda"), torch.empty(n, device="cuda")
            call(q, s, given)
            odd, t = torch.empty(n, width + 1, dtype=torch.int8, device="cuda")[:, :width], torch.empty(n, device="cuda")
            call(odd, t, given)
            few, u = ops.new_int8(3, width, "cuda"), torch.empty(3, device="cuda")
            call(few, u, given[:3])
            assert torch.equal(q, odd) and torch.equal(s, t) and torch.equal(q[:3], few) and torch.equal(s[:3], u)
