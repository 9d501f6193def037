"""Products of 8-bit integers under each plan that real layers meet, on random operands.  Every case names the plan that it is here for, so that
another plan for the same sizes does not go untested unseen.  Tolerances as in ``test_int8_ops_gpu``."""
import pytest
import torch

from test_int8_ops_gpu import BF, F, check_product

pytestmark = pytest.mark.gpu
SMS = 148


@pytest.fixture(scope="module")
def ops():
    from nanohybrid_vlm_b200.kernels import ops
    assert torch.cuda.get_device_properties(0).multi_processor_count == SMS
    return ops


# a pair's tiles one after another: both accumulators again and again, the ring carried from tile to tile
TURNS = [
    (60001, 63, 64, 4), (60000, 64, 64, 4),
    (547, 9433, 128, 3), (547, 9432, 128, 3), (2064, 6200, 128, 6),
    (288, 18949, 192, 3), (288, 18952, 192, 3), (547, 25112, 192, 6),
    (288, 21328, 256, 3), (288, 28465, 256, 4), (2048, 24576, 256, 11), (4500, 5120, 256, 5), (5000, 4100, 192, 6),
]


@pytest.mark.parametrize("K", [144, 600, 1040])
@pytest.mark.parametrize("out", [BF, F])
@pytest.mark.parametrize("T,N,width,turns", TURNS)
def test_tiles_in_turns(ops, T, N, width, turns, out, K):
    """Sums of 2, 5 and 9 turns of a ring of 6, 8 or 9 stages, so that tiles begin at several of its stages; none of them whole, and most tiles at the
    edges are not.  Outputs leave by TMA where N allows it, else element by element."""
    plan = ops.int8_plan(T, N, K, SMS)
    assert (plan.pairs, plan.outputs, plan.turns) == (1, width, turns)
    check_product(ops, T, K, N, out, seed=N + K)


# (tokens, K, N): rows of a tile, parts of K, stages
FEW = [
    (8, 400, 24576, 84, 1, None), (33, 400, 24576, 84, 1, None), (64, 400, 24576, 84, 1, None), (100, 400, 24576, 84, 1, None), (128, 400, 24576, 84, 1, None),
    (8, 400, 51203, 87, 1, None), (64, 400, 51203, 87, 1, None), (128, 400, 51203, 87, 1, None),       # two waves of blocks
    (8, 4112, 10240, 128, 3, None), (64, 2064, 10240, 70, 1, 8), (100, 2064, 10240, 70, 1, 8), (128, 2064, 10240, 70, 1, None),
    (8, 4112, 6144, 128, 4, None), (64, 4112, 6144, 128, 4, None), (100, 4112, 6144, 128, 2, None), (128, 4112, 6144, 128, 2, None),
    (33, 4112, 5120, 128, 4, None), (100, 4112, 5120, 128, 3, None), (128, 12304, 5120, 128, 3, None),
    (5, 256, 9000, 61, 1, None),
]


@pytest.mark.parametrize("T,K,N,rows,parts,stages", FEW)
def test_few_tokens(ops, T, K, N, rows, parts, stages):
    """Tiles of heights that are no whole groups of eight rows, K in two and three parts for many tokens, blocks in waves, the large ring of a block alone."""
    plan = ops.int8_plan(T, N, K, SMS)
    assert plan.pairs == 0 and (plan.outputs, plan.parts) == (rows, parts) and stages in (None, plan.stages)
    check_product(ops, T, K, N, F if T % 2 else BF, seed=T + N)


def test_what_is_reached(ops):
    plans = [ops.int8_plan(T, N, K, SMS) for T, K, N, *_ in FEW]
    assert sum(p.outputs % 8 != 0 for p in plans) >= 6                                        # boxes of odd heights
    assert any(p.tiles * p.parts > 2 * SMS for p in plans)                                    # more blocks than run at once
    assert any(p.parts == 2 for p in plans) and any(p.parts == 3 and p.tokens > 64 for p in plans)
    assert any(p.parts == 1 and p.shared_bytes > 113 * 1024 for p in plans)                   # a block that has its SM to itself
