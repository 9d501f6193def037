"""How products of 8-bit integers are cut, without a device: over random sizes every plan stays within what its kernel allows."""
import math
import random

import pytest

from nanohybrid_vlm_b200.kernels import ops
from nanohybrid_vlm_b200.kernels.library import KernelError

LONGEST_T = 2 ** 31 - 512


def sizes(rng, tokens):
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))      # noqa: E731
    return min(log(*tokens), tokens[1]), min(log(1, 2 ** 31 - 512), 2 ** 31 - 512) if rng.random() < 0.1 else log(1, 100000), log(1, 131071)


@pytest.mark.parametrize("sms", [148, 132, 2, 7])
def test_up_to_128_tokens(sms):
    rng, seen = random.Random(sms), set()
    for _ in range(6000):
        T, N, K = sizes(rng, (1, 128))
        p = ops.int8_plan(T, N, K, sms)
        assert p.pairs == 0 and T <= p.tokens <= 128 and p.tokens % 16 == 0 and p.turns == 1
        assert 1 <= p.outputs <= 128 and p.tiles == -(-N // p.outputs) and 1 <= p.parts <= min(8, -(-K // 128))      # no part of K is empty
        assert 1 <= p.stages <= 8 and p.shared_bytes <= 225 * 1024
        ring = (p.stages - 1) * (-(-p.outputs * 128 // 1024) * 1024 + p.tokens * 128) + 128 * 128 + p.tokens * 128
        share = -(-(-(-p.tokens // p.parts)) // 4) * 4
        assert share * p.parts >= p.tokens                      # each token has a block that finishes it
        assert p.shared_bytes >= 1024 + ring + (p.parts * share * 512 if p.parts > 1 else 0) + (2 * p.stages + 1) * 8 + 4
        seen.add((p.parts, p.outputs in (32, 64, 128)))
    if sms == 148:
        assert {parts for parts, _ in seen} == set(range(1, 9)) and (1, False) in seen


@pytest.mark.parametrize("sms", [148, 132, 2, 7])
def test_more_tokens(sms):
    rng, seen = random.Random(sms), {}
    for _ in range(6000):
        T, N, K = sizes(rng, (129, LONGEST_T if rng.random() < 0.1 else 20000))
        p = ops.int8_plan(T, N, K, sms)
        assert p.pairs == 1 and p.tokens == 256 and p.outputs in (64, 128, 192, 256) and p.parts == 1
        assert p.tiles == -(-T // 256) * -(-N // p.outputs) and p.turns == -(-p.tiles // (sms // 2))
        stage = 128 * 128 + p.outputs // 2 * 128
        assert p.stages * stage + 8 * p.outputs // 2 * 4 + 8 * 2560 + (2 * p.stages + 4) * 8 + 4 + 1024 <= p.shared_bytes <= 227 * 1024
        least = min((-(-T // 256) * -(-N // w) + sms // 2 - 1) // (sms // 2) * (w + 64) for w in (64, 128, 192, 256))
        assert p.turns * (p.outputs + 64) == least
        seen.setdefault(p.outputs, set()).add(min(p.turns, 3))
    if sms == 148:
        # in several turns tiles of 64 outputs are taken for up to 64 of them alone: else tiles of 128 need half as many
        assert seen == {w: {1, 2, 3} for w in (64, 128, 192, 256)}


@pytest.mark.parametrize("T,N,K,sms", [(0, 1, 1, 148), (1, 0, 1, 148), (1, 1, 0, 148), (1, 1, 131072, 148), (2 ** 31 - 511, 1, 1, 148), (1, 2 ** 31 - 511, 1, 148),
                                       (1, 1, 1, 1)])
def test_no_plan(T, N, K, sms):
    with pytest.raises(KernelError, match="no plan"):
        ops.int8_plan(T, N, K, sms)
