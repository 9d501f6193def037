"""The operators over 8-bit integers against their definitions in 64 bits.

Tolerances.  A product's sum is an exact integer: its conversion to 32 bits, the two products with scales round once each (3 * 2^-24) and
the store once more (2^-8 for bfloat16, none for float32).  A row's scale comes from one element y of 32 bits: 2^-24 for the division
by 127 on top of what y is off by.  y of a plain row is exact; of a norm: the sum of squares adds at most about sqrt(width) + 10
roundings that partly cancel, 2e-6 for widths up to 60,000, twice that at most with the root and the products; of the gated unit
with the fast exponential: 2^-21 of its value for the moderate gates here.  Integers of a plain row equal the definition's; others
may be one step off where 127 y / a lies within that error, times 127, of the middle between two integers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F = torch.bfloat16, torch.float32
EIGHT = {BF: 2.0 ** -8, F: 0.0}


@pytest.fixture(scope="module")
def ops():
    from nanohybrid_vlm_b200.kernels import ops
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------ products
def ints(g, rows, cols, pitch=16, shift=0):
    """Random 8-bit integers, rows at multiples of ``pitch`` bytes from an address ``shift`` bytes behind an aligned one; what lies between
    the rows is 77."""
    stride = -(-cols // pitch) * pitch
    flat = torch.full((rows * stride + shift,), 77, dtype=torch.int8, device="cuda")
    t = flat[shift:].view(rows, stride)[:, :cols]
    t.copy_(torch.randint(-127, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int16))
    return t


def check_product(ops, T, K, N, out=BF, pitch=16, shift=0, out_pad=0, seed=0, x=None, w=None, xs=None, ws=None):
    g = gen(seed)
    x = ints(g, T, K, pitch, shift) if x is None else x
    w = ints(g, N, K, pitch, shift) if w is None else w
    xs = torch.rand(T, generator=g, device="cuda") + 0.01 if xs is None else xs
    ws = torch.randn(N, generator=g, device="cuda") if ws is None else ws
    whole = torch.full((T + 1, N + out_pad), 5.0, dtype=out, device="cuda")
    y = whole[:T, :N]
    ops.linear_int8(y, x, xs, w, ws)
    want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()[None]
    err = (y.double() - want).abs() - (EIGHT[out] + 3.1 * 2.0 ** -24) * want.abs()
    assert err.max() <= 0, f"off by {err.max()} at T={T} K={K} N={N}"
    assert (whole[T:] == 5).all() and (whole[:, N:] == 5).all()         # behind the rows and the columns
    assert ops.take_wait_errors() == []
    return y


TOKENS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 129, 255, 257, 300, 600]


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("K,N,out", [(256, 384, BF), (1040, 200, F), (4096, 130, BF), (48, 1000, BF)])
def test_products(ops, T, K, N, out):
    check_product(ops, T, K, N, out, seed=T + K)


@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (1, 17, 1), (3, 15, 2), (5, 31, 9), (70, 127, 65), (130, 129, 257), (33, 1001, 2774), (16, 4095, 24)])
@pytest.mark.parametrize("pitch,shift", [(16, 0), (1, 0), (16, 3), (4, 4), (128, 0)])
def test_products_of_odd_sizes_and_addresses(ops, T, K, N, pitch, shift):
    check_product(ops, T, K, N, F if N % 2 else BF, pitch, shift, out_pad=N % 3, seed=N)


@pytest.mark.parametrize("T,K,N", [(2048, 512, 1024), (1500, 1024, 777), (4097, 144, 640), (1111, 4096, 512)])
@pytest.mark.parametrize("out", [BF, F])
def test_products_of_many_tokens(ops, T, K, N, out):
    check_product(ops, T, K, N, out, seed=T)


@pytest.mark.parametrize("T,K,N,out,pad", [(300, 320, 200, BF, 8), (257, 96, 1000, F, 4), (140, 64, 40, BF, 24), (60, 2048, 200, BF, 3)])
def test_products_into_wider_rows(ops, T, K, N, out, pad):
    """An output that is a slice of columns: what lies beside it stays."""
    check_product(ops, T, K, N, out, out_pad=pad)


@pytest.mark.parametrize("T", [64, 366, 1025])
@pytest.mark.parametrize("N,out,pad", [(55, BF, 1), (129, BF, 7), (300, BF, 4), (53, F, 3), (129, F, 7), (302, F, 2)])
def test_products_whose_rows_end_inside_16_bytes(ops, T, N, out, pad):
    """The rows start at multiples of 16 bytes and end between two: the rest of the last 16 bytes is not the output's."""
    check_product(ops, T, 144, N, out, out_pad=pad, seed=N)


@pytest.mark.parametrize("T", [1, 12, 40, 200, 1300])
def test_sums_at_the_ends_of_32_bits(ops, T):
    """All products at the largest magnitude, -128 among them: K * 2^14 is just below 2^31."""
    K, N = 131071, 24
    x = ops.new_int8(T, K, "cuda").fill_(-128)
    w = ops.new_int8(N, K, "cuda").fill_(-128)
    w[1::2] = 127
    check_product(ops, T, K, N, F, x=x, w=w)


@pytest.mark.parametrize("T", [1, 20, 150, 700])
def test_scales_that_are_no_numbers(ops, T):
    g = gen(3)
    K, N = 320, 96
    x, w = ints(g, T, K), ints(g, N, K)
    xs, ws = torch.rand(T, device="cuda") + 1, torch.rand(N, device="cuda") + 1
    xs[0], ws[3], ws[4] = math.nan, math.inf, 0.0
    y = torch.empty(T, N, device="cuda")
    ops.linear_int8(y, x, xs, w, ws)
    plain = (x.double() @ w.double().t()).float() * xs[:, None] * ws[None]
    torch.testing.assert_close(y, plain, rtol=1e-6, atol=0, equal_nan=True)


def test_no_tokens_and_no_outputs(ops):
    for T, N in ((0, 8), (8, 0), (0, 0)):
        ops.linear_int8(torch.empty(T, N, dtype=BF, device="cuda"), ops.new_int8(T, 64, "cuda"), torch.empty(T, device="cuda"),
                        ops.new_int8(N, 64, "cuda"), torch.empty(N, device="cuda"))


@pytest.mark.parametrize("K,N", [(1024, 4096), (4096, 1040)])
def test_a_row_does_not_depend_on_its_batch(ops, K, N):
    g = gen(9)
    x, w = ints(g, 700, K), ints(g, N, K)
    xs, ws = torch.rand(700, device="cuda"), torch.rand(N, device="cuda")
    whole = torch.empty(700, N, device="cuda")
    ops.linear_int8(whole, x, xs, w, ws)
    for a, b in ((0, 1), (3, 11), (100, 130), (200, 300), (5, 400)):
        part = torch.empty(b - a, N, device="cuda")
        ops.linear_int8(part, x[a:b], xs[a:b], w, ws)
        assert torch.equal(part, whole[a:b])


@pytest.mark.parametrize("T", [1, 8, 48, 200, 1024])
def test_streams_and_graphs(ops, T):
    """Products at once on two streams, and a captured one that is replayed on new inputs beside another one."""
    g = gen(T)
    K, N = 2048, 1536
    x, w = ints(g, T, K), ints(g, N, K)
    xs, ws = torch.rand(T, device="cuda"), torch.rand(N, device="cuda")
    want = ((x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()[None])
    outs = [torch.empty(T, N, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                ops.linear_int8(o, x, xs, w, ws)
    torch.cuda.synchronize()
    for o in outs:
        torch.testing.assert_close(o.double(), want, rtol=3.1 * 2.0 ** -24, atol=0)
    graphs = []
    for o in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.linear_int8(o, x, xs, w, ws)
    x.copy_(ints(g, T, K))
    want = ((x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()[None])
    torch.cuda.synchronize()
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        torch.testing.assert_close(o.double(), want, rtol=3.1 * 2.0 ** -24, atol=0)
    assert ops.take_wait_errors() == []


def far_apart(rows, width, stride, dtype):
    """Rows whose last ones start more than 2^31 elements behind the first; most of the memory is never touched."""
    assert (rows - 1) * stride > 2 ** 31
    return torch.empty((rows - 1) * stride + width, dtype=dtype, device="cuda").as_strided((rows, width), (stride, 1))


@pytest.mark.parametrize("T,odd", [(20, 0), (20, 1), (300, 0), (300, 1)])
def test_product_offsets_beyond_32_bits(ops, T, odd):
    """Rows of both operands and of the output lie far apart; with ``odd`` at places from which the operands are copied first."""
    g = gen(T)
    K, N, xp, wp = 80, 300, 2 ** 31 // (T - 2) // 16 * 16 + 64 + odd, 2 ** 31 // 298 // 16 * 16 + 64 + odd
    x, w = far_apart(T, K, xp, torch.int8), far_apart(N, K, wp, torch.int8)
    x.copy_(ints(g, T, K)), w.copy_(ints(g, N, K))
    xs, ws = torch.rand(T, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    y = far_apart(T, N, xp, BF)
    ops.linear_int8(y, x, xs, w, ws)
    want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()[None]
    assert ((y.double() - want).abs() <= (EIGHT[BF] + 3.1 * 2.0 ** -24) * want.abs()).all()


def test_products_beyond_the_numbers_of_tiles_are_refused(ops):
    """Sizes whose last tile has rows without a number in 32 bits; the call's own block says so, as no memory is that large."""
    from nanohybrid_vlm_b200.kernels.library import KernelError, call
    for T, N in ((2 ** 31 - 511, 1), (1, 2 ** 31 - 511)):
        with pytest.raises(KernelError, match="no number"):
            call("nhv_gemm_int8", ops._PRODUCT_CALL.pack(*[0] * 7, 1, 16, 16, 1, T, N, 16), ops.stream_ptr())


# ------------------------------------------------------------------------------------------------ rows
def definition(y):
    a = y.abs().amax(1)
    safe = torch.where(a == 0, 1.0, a)[:, None]
    return torch.round(127 * y / safe), a / 127


def check_rows(q, scales, y, off, exact=False):
    """q, scales against rows y in 64 bits whose 32-bit forms are off by up to ``off`` relative to the row's largest."""
    want, s = definition(y)
    assert ((scales.double() - s).abs() <= (off + 2.0 ** -23) * s).all()
    if exact:
        assert torch.equal(q.double(), want)
        return
    place = 127 * y / torch.where(s == 0, 1.0, 127 * s)[:, None]
    assert ((q.double() - place).abs() <= 0.5 + 127 * 2.5 * (off + 2.0 ** -23)).all()


def room(ops, n, width, pitch):
    if pitch is None:
        return ops.new_int8(n, width, "cuda")
    return torch.zeros(n, width + pitch, dtype=torch.int8, device="cuda")[:, :width]


WIDTHS = [1, 3, 8, 33, 64, 129, 1000, 1024, 1032, 2048, 4096, 4104, 8192, 12288, 16384, 25600, 32768, 32776]
OFF_NORM = 4e-6


@pytest.mark.parametrize("width", WIDTHS + [51208, 131071])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n,pitch", [(3, None), (300, None), (5, 1)])
def test_plain_rows(ops, width, dtype, n, pitch):
    g = gen(width)
    x = (torch.randn(n, width, generator=g, device="cuda") * torch.exp(3 * torch.randn(n, 1, generator=g, device="cuda"))).to(dtype)
    x[n // 2] = 0
    q, s = room(ops, n, width, pitch), torch.empty(n, device="cuda")
    ops.quantize_rows(q, s, x)
    check_rows(q, s, x.double(), 0.0, exact=dtype == BF)
    assert s[n // 2] == 0
    if pitch:
        assert (q.as_strided((n, width + pitch), (width + pitch, 1))[:, width:] == 0).all()


def test_plain_rows_ties_and_ends_of_the_range(ops):
    """Values in the middle between two integers go to the even one; rows of the smallest and largest numbers keep their shape."""
    n = torch.arange(-254, 255, dtype=torch.float64, device="cuda") / 2            # -127, -126.5, ... 127
    for dtype in (BF, F):
        for e in (0, -20, 60, 100, 119, -100, -125):
            x = (n * 2.0 ** e).to(dtype)[None].contiguous()
            q, s = torch.empty(1, 509, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
            ops.quantize_rows(q, s, x)
            check_rows(q, s, x.double(), 0.0, exact=True)
    x = torch.tensor([[2.0 ** -133, -2.0 ** -133, 0.0, 2.0 ** -133]], dtype=BF, device="cuda")      # bfloat16's smallest
    q, s = torch.empty(1, 4, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    ops.quantize_rows(q, s, x)
    assert q.tolist() == [[127, -127, 0, 127]]
    x = torch.tensor([[3.3e38, -3.3e38, 1.0, 1.65e38]], device="cuda")
    ops.quantize_rows(q, s, x)
    assert q.tolist() == [[127, -127, 0, 64]] and torch.isfinite(s).all()


@pytest.mark.parametrize("odd", [0, 1])
def test_row_offsets_beyond_32_bits(ops, odd):
    g = gen(7)
    n, width, stride = 300, 1024, 2 ** 31 // 298 // 16 * 16 + 64 + odd
    x, q, y = far_apart(n, width, stride, BF), far_apart(n, width, stride, torch.int8), far_apart(n, width, stride, BF)
    x.copy_(torch.randn(n, width, generator=g, device="cuda"))
    s = torch.empty(n, device="cuda")
    ops.quantize_rows(q, s, x)
    check_rows(q, s, x.double(), 0.0, exact=True)
    ops.dequantize_rows(y, q, s)
    assert torch.equal(y, (q.float() * s[:, None]).to(BF))
    near = torch.randn(n, width, generator=g, device="cuda").to(BF)
    ops.rmsnorm_int8(q, s, near, torch.ones(width, dtype=BF, device="cuda"), 1e-5)
    y64 = near.double()
    check_rows(q, s, y64 / torch.sqrt(y64.pow(2).mean(1, keepdim=True) + 1e-5), OFF_NORM)


@pytest.mark.parametrize("width", [5, 264, 4096, 40000])
@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_that_hold_no_numbers(ops, width, dtype):
    x = torch.randn(6, width, device="cuda").to(dtype)
    x[1, width - 1], x[2, 0], x[3, width // 2], x[4] = math.inf, -math.inf, math.nan, 0
    want = [False, True, True, True, False, False]
    up = torch.ones(6, width, device="cuda").to(dtype)
    w = torch.ones(width, device="cuda").to(dtype)
    for call in (lambda q, s: ops.quantize_rows(q, s, x), lambda q, s: ops.rmsnorm_int8(q, s, x, w, 1e-6),
                 lambda q, s: ops.silu_mul_int8(q, s, torch.cat([up, x], 1))):
        q, s = ops.new_int8(6, width, "cuda").fill_(55), torch.empty(6, device="cuda")
        call(q, s)
        assert s.isnan().tolist() == want and not q[torch.tensor(want)].any()
        assert s[4] == 0 and not q[4].any()


@pytest.mark.parametrize("width", WIDTHS + [51200])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n,residual,offset", [(3, True, 0.0), (290, True, 1.0), (4, False, 0.0)])
def test_norm(ops, width, dtype, n, residual, offset):
    g = gen(width + n)
    x = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    r = (3 * torch.randn(n, width, generator=g, device="cuda")).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(width, generator=g, device="cuda")).to(dtype)
    s64 = x.double() + (r.double() if residual else 0)
    y = s64 / torch.sqrt(s64.pow(2).mean(1, keepdim=True) + 1e-5) * (w.double() + offset)
    q, s = ops.new_int8(n, width, "cuda"), torch.empty(n, device="cuda")
    kept = r.clone() if residual else None
    if residual:
        ops.rmsnorm_int8(q, s, x, w, 1e-5, residual=kept, write_residual=False, weight_offset=offset)
        assert torch.equal(kept, r)
        check_rows(q, s, y, OFF_NORM)
    ops.rmsnorm_int8(q, s, x, w, 1e-5, residual=r, weight_offset=offset)
    check_rows(q, s, y, OFF_NORM)
    if residual:
        assert torch.equal(r, (x.float() + kept.float()).to(dtype))


def test_norm_refuses_rows_beyond_its_buffer(ops):
    from nanohybrid_vlm_b200.kernels.library import KernelError
    with pytest.raises(KernelError, match="51200"):
        ops.rmsnorm_int8(ops.new_int8(1, 51201, "cuda"), torch.empty(1, device="cuda"), torch.zeros(1, 51201, device="cuda"),
                         torch.zeros(51201, device="cuda"), 1e-6)


@pytest.mark.parametrize("n", [1, 40, 500])
def test_norm_in_32_bits_does_not_depend_on_the_batch(ops, n):
    g = gen(n)
    x, w = torch.randn(n, 2048, generator=g, device="cuda"), torch.randn(2048, generator=g, device="cuda")
    q, s = ops.new_int8(n, 2048, "cuda"), torch.empty(n, device="cuda")
    ops.rmsnorm_int8(q, s, x, w, 1e-6)
    q1, s1 = ops.new_int8(1, 2048, "cuda"), torch.empty(1, device="cuda")
    ops.rmsnorm_int8(q1, s1, x[n // 2:n // 2 + 1], w, 1e-6)
    assert torch.equal(q1[0], q[n // 2]) and torch.equal(s1[0], s[n // 2])


@pytest.mark.parametrize("width", WIDTHS + [60001])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n", [3, 280])
def test_unit(ops, width, dtype, n):
    g = gen(width + n)
    x = (1.5 * torch.randn(n, 2 * width, generator=g, device="cuda")).to(dtype)
    x[1] = 0
    q, s = ops.new_int8(n, width, "cuda"), torch.empty(n, device="cuda")
    ops.silu_mul_int8(q, s, x)
    gate, up = x.double().split(width, 1)
    check_rows(q, s, gate * torch.sigmoid(gate) * up, 2.0 ** -20)


def test_rows_of_strided_inputs(ops):
    """A slice of columns of a wider matrix, as it lies: its rows start anywhere."""
    for dtype in (BF, F):
        wide = torch.randn(9, 1003, device="cuda").to(dtype)
        x = wide[:, 3:1000]
        q, s = ops.new_int8(9, 997, "cuda"), torch.empty(9, device="cuda")
        ops.quantize_rows(q, s, x)
        check_rows(q, s, x.double(), 0.0, exact=dtype == BF)


@pytest.mark.parametrize("n,width,pitch,pad", [(1, 1, 16, 0), (3, 16, 16, 0), (5, 33, 16, 3), (300, 4096, 16, 0), (7, 48, 1, 1), (2, 100000, 16, 0)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_values(ops, n, width, pitch, pad, dtype):
    """Integer times scale, rounded once: to 32 bits and, for bfloat16, from there once more (the product's 8 and 24 bits do not fit 32)."""
    g = gen(width)
    q, s = ints(g, n, width, pitch), torch.randn(n, generator=g, device="cuda")
    s[n // 2] = math.nan if n > 2 else 0.0
    whole = torch.full((n, width + pad), 3.0, dtype=dtype, device="cuda")
    ops.dequantize_rows(whole[:, :width], q, s)
    assert torch.equal(whole[:, :width].nan_to_num(nan=77), (q.float() * s[:, None]).to(dtype).nan_to_num(nan=77)) and (whole[:, width:] == 3).all()


def test_outputs_over_inputs_are_refused(ops):
    from nanohybrid_vlm_b200.kernels.library import KernelError
    x, s = torch.randn(4, 64, device="cuda"), torch.empty(4, device="cuda")
    over = x.view(torch.int8)[:, :64]
    for call in (lambda: ops.quantize_rows(over, s, x), lambda: ops.rmsnorm_int8(over, s, x, x[0].clone(), 1e-6),
                 lambda: ops.silu_mul_int8(over[:, :32], s, x), lambda: ops.dequantize_rows(x, over, s)):
        with pytest.raises(KernelError, match="memory of"):
            call()
    with pytest.raises(KernelError, match="memory of"):
        ops.rmsnorm_int8(over, s, x.clone(), x[0].clone(), 1e-6, residual=x)
    x = ops.new_int8(4, 64, "cuda").fill_(1)
    with pytest.raises(KernelError, match="memory of"):
        ops.linear_int8(x.view(torch.float32)[:, :4], x, s, x[:4].clone(), s)


def test_no_rows(ops):
    e = lambda *shape: torch.empty(*shape, dtype=BF, device="cuda")      # noqa: E731
    q, s = ops.new_int8(0, 64, "cuda"), torch.empty(0, device="cuda")
    ops.quantize_rows(q, s, e(0, 64))
    ops.silu_mul_int8(q, s, e(0, 128))
    ops.rmsnorm_int8(q, s, e(0, 64), e(64), 1e-6, residual=e(0, 64))
    ops.dequantize_rows(e(0, 64), q, s)
    ops.dequantize_rows(e(3, 0), ops.new_int8(3, 0, "cuda"), torch.empty(3, device="cuda"))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("T", [1, 37, 400])
@pytest.mark.parametrize("dtype", [BF, F])
def test_a_feed_forward_in_8_bits(ops, T, dtype):
    """Norm with the residual, gate and up, unit, down: each operator reads what the one before it wrote.  Against 64 bits from the
    integers that the kernels made; and, as a whole, near the product of the unrounded numbers."""
    g = gen(T)
    W, I = 512, 1376
    x = torch.randn(T, W, generator=g, device="cuda").to(dtype)
    r = torch.randn(T, W, generator=g, device="cuda").to(dtype)
    nw = (1 + 0.1 * torch.randn(W, generator=g, device="cuda")).to(dtype)
    w1, w2 = (torch.randn(2 * I, W, generator=g, device="cuda") * 0.05).to(dtype), (torch.randn(W, I, generator=g, device="cuda") * 0.05).to(dtype)
    eight = []
    for w in (w1, w2):
        q, s = ops.new_int8(*w.shape, "cuda"), torch.empty(w.shape[0], device="cuda")
        ops.quantize_rows(q, s, w)
        eight.append((q, s))
    s64 = x.double() + r.double()
    h64 = s64 / torch.sqrt(s64.pow(2).mean(1, keepdim=True) + 1e-6) * nw.double()
    h, hs = ops.new_int8(T, W, "cuda"), torch.empty(T, device="cuda")
    ops.rmsnorm_int8(h, hs, x, nw, 1e-6, residual=r)
    gu = torch.empty(T, 2 * I, dtype=dtype, device="cuda")
    ops.linear_int8(gu, h, hs, *eight[0])
    a, sa = ops.new_int8(T, I, "cuda"), torch.empty(T, device="cuda")
    ops.silu_mul_int8(a, sa, gu)
    y = torch.empty(T, W, dtype=dtype, device="cuda")
    ops.linear_int8(y, a, sa, *eight[1])

    def product(q, s, w, ws):       # the sum of the integers first: it is exact in 64 bits, zero where it is zero
        return (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()[None]

    off = EIGHT[dtype] + 3.1 * 2.0 ** -24
    want = product(h, hs, *eight[0])
    assert ((gu.double() - want).abs() <= off * want.abs()).all()
    gate, up = gu.double().split(I, 1)
    check_rows(a, sa, gate * torch.sigmoid(gate) * up, 2.0 ** -20)
    want = product(a, sa, *eight[1])
    assert ((y.double() - want).abs() <= off * want.abs()).all()
    # Each rounding to 8 bits is off by up to half a step, 1/254 of the row's largest (here 3 to 4.5 times its rms), evenly spread: 4.5 / 254 / sqrt(3)
    # = 1.0 % of the rms at most; four of them (rows and weights of two products; the unit's first factor passes its
    # error on about once more) stay under 4 %.
    gate, up = (h64 @ w1.double().t()).split(I, 1)
    plain = (gate * torch.sigmoid(gate) * up) @ w2.double().t()
    assert (y.double() - plain).norm() <= 0.04 * plain.norm()
