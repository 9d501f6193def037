"""What the operators over 8-bit integers write shares no byte with what they read; columns of one buffer side by side do not count.

The library looks at that before anything else: without a device a call that passes ends with the device's absence, and one that does not with
the refusal.  Places and sizes here are numbers, no memory lies there, so nothing of this runs where a device would take them."""
import random

import pytest
import torch

from nanohybrid_vlm_b200.kernels import ops
from nanohybrid_vlm_b200.kernels.library import KernelError, call

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="places without memory")
APART = 1 << 30     # far behind everything else


def refused(name, given):
    with pytest.raises(KernelError) as e:
        call(name, given, 0)
    return "memory of its own" in str(e.value) or "memory of their own" in str(e.value)


def held(at, rows, pitch, width):
    return {at + r * pitch + c for r in range(rows) for c in range(width)}


def product(out=APART, x=2 * APART, xs=3 * APART, w=4 * APART, ws=5 * APART, pitches=(16, 32, 32), dtype=ops.BF16, T=3, N=5, K=20):
    return ops._PRODUCT_CALL.pack(out, x, xs, w, ws, 6 * APART, 7 * APART, *pitches, dtype, T, N, K)


def rows(q=APART, scales=2 * APART, x=3 * APART, residual=0, weight=0, pitches=(16, 16), kind=0, dtype=ops.BF16, n=4, width=16, write=0):
    return ops._ROWS_CALL.pack(q, scales, x, residual, weight, *pitches, kind, dtype, n, width, write, 1e-6, 0.0)


def values(out=APART, q=2 * APART, scales=3 * APART, pitches=(16, 16), dtype=ops.BF16, n=4, width=16):
    return ops._BACK_CALL.pack(out, q, scales, *pitches, dtype, n, width)


def test_apart_is_not_refused():
    assert not refused("nhv_gemm_int8", product())
    for kind in (0, 1, 2):
        assert not refused("nhv_rows_int8", rows(kind=kind, weight=4 * APART, residual=5 * APART if kind == 1 else 0, write=kind == 1))
    assert not refused("nhv_rows_from_int8", values())


@pytest.mark.parametrize("other", ["x", "xs", "w", "ws"])
def test_products(other):
    """The output, 3 rows of 10 bytes 32 apart, ends at byte 74; operands are rows of 20 bytes 32 apart, scales 12 and 20 bytes."""
    size = {"x": 2 * 32 + 20, "xs": 12, "w": 4 * 32 + 20, "ws": 20}[other]
    for at in (0, 1, 9, 73, 1 - size):
        assert refused("nhv_gemm_int8", product(**{other: APART + at})), at
    for at in (74, -size):
        assert not refused("nhv_gemm_int8", product(**{other: APART + at})), at


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_rows(kind):
    """q: 4 rows of 16 bytes; a row of x has 32, of the unit's 64."""
    more = dict(kind=kind, weight=6 * APART) if kind == 1 else dict(kind=kind)
    pitch = 32 if kind == 2 else 16
    for at in (0, 5, 63, 1 - 4 * 2 * pitch):
        assert refused("nhv_rows_int8", rows(x=APART + at, pitches=(16, pitch), **more)), at
    assert not refused("nhv_rows_int8", rows(x=APART + 64, pitches=(16, pitch), **more))
    assert refused("nhv_rows_int8", rows(scales=APART + 60, **more))                        # the outputs among themselves
    assert refused("nhv_rows_int8", rows(scales=3 * APART + 100, **more))                   # scales in x
    if kind == 1:
        for place in (dict(q=5 * APART + 127), dict(q=6 * APART + 30), dict(scales=5 * APART - 15), dict(scales=6 * APART + 31)):
            for write in (0, 1):
                assert refused("nhv_rows_int8", rows(**(more | dict(residual=5 * APART, write=write) | place)))
        for at in (3 * APART + 2, 3 * APART - 126, 6 * APART - 2):                          # the sum over other rows of x, or the weight
            assert refused("nhv_rows_int8", rows(residual=at, write=1, **more))
            assert not refused("nhv_rows_int8", rows(residual=at, write=0, **more))         # only read


def test_values():
    for at in (0, 1, 127, -63):
        assert refused("nhv_rows_from_int8", values(q=APART + at))
    for at in (0, 126, -15):
        assert refused("nhv_rows_from_int8", values(scales=APART + at))
    assert not refused("nhv_rows_from_int8", values(q=APART + 128)) and not refused("nhv_rows_from_int8", values(q=APART - 64))


def test_columns_side_by_side():
    """One buffer of rows of 64 bytes: the integers at its columns 0 to 15, their values at 16 to 47, what else may be behind."""
    assert not refused("nhv_rows_from_int8", values(out=APART + 16, q=APART, pitches=(32, 64)))
    assert refused("nhv_rows_from_int8", values(out=APART + 15, q=APART, pitches=(32, 64)))
    assert refused("nhv_rows_from_int8", values(out=APART + 33, q=APART, pitches=(32, 64)))        # a row's last byte is the next row's first
    assert not refused("nhv_rows_from_int8", values(out=APART + 32, q=APART, pitches=(32, 64)))
    assert not refused("nhv_rows_int8", rows(q=APART + 32, x=APART, pitches=(64, 32)))


def test_any_places():
    """Against the bytes themselves, counted one by one: equal and unequal pitches, one row, rows of an operand that lie on each other."""
    rng = random.Random(5)
    met = 0
    for _ in range(4000):
        n, width = rng.randint(1, 6), rng.randint(1, 9)
        out_pitch, q_pitch = rng.randint(width, 14), rng.choice((0, rng.randint(1, 30), 2 * rng.randint(width, 14)))
        if rng.random() < 0.4:
            q_pitch = 2 * out_pitch
        out, q = APART + rng.randint(0, 80), APART + rng.randint(0, 80)
        want = bool(held(out, n, 2 * out_pitch, 2 * width) & held(q, n, q_pitch, width))
        assert refused("nhv_rows_from_int8", values(out, q, pitches=(out_pitch, q_pitch), n=n, width=width)) == want, (out, q, n, width, out_pitch, q_pitch)
        N, K = rng.randint(1, 6), rng.randint(1, 9)
        w_pitch = rng.randint(1, 20)
        out_pitch = rng.randint(N, 9)
        want = bool(held(out, n, 2 * out_pitch, 2 * N) & held(q, N, w_pitch, K))
        assert refused("nhv_gemm_int8", product(out, w=q, pitches=(out_pitch, 32, w_pitch), T=n, N=N, K=K)) == want
        met += want
    assert 500 < met < 3500
