"""The host's part of attention with scored keys: the plan and the scratch it asks for, without a GPU."""
import math
import subprocess
import sys

import pytest
import torch

from conftest import ROOT


@pytest.mark.parametrize("dtype,d", [("bfloat16", 64), ("float32", 64), ("bfloat16", 33), ("float32", 256)])
@pytest.mark.parametrize("keys", [1, 40, 100000])
def test_a_step_without_new_tokens_has_a_plan(dtype, d, keys):
    """In a process of its own: a division by zero would end it."""
    code = (f"import torch; from nanohybrid_vlm_b200.kernels import ops; "
            f"print('bytes', ops.attention_scored_scratch_bytes(torch.{dtype}, 2, 0, 0, 0, {keys}, 4, 2, {d}, 16))")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    assert 0 < int(r.stdout.split("bytes")[1]) < 2 ** 31


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_call_takes_more_scratch_than_the_bound(dtype):
    """What an engine sets aside for steps of up to so many requests, tokens and keys is enough for every one of them."""
    import random
    from nanohybrid_vlm_b200.kernels import ops
    rng = random.Random(5)
    log = lambda a, b: int(round(2 ** rng.uniform(math.log2(a), math.log2(b))))     # noqa: E731
    for most_seqs, most_tokens, most_keys, nq, nkv, d in [(512, 16384, 4096, 32, 8, 128), (256, 2048, 32768, 32, 8, 128), (1, 8192, 131072, 64, 8, 128),
                                                          (64, 4096, 40960, 16, 16, 64), (16, 1024, 2000, 6, 2, 32), (300, 700, 9000, 40, 1, 256),
                                                          (32, 2048, 8192, 5, 1, 80), (8, 64, 1 << 20, 8, 1, 128), (100, 5000, 5000, 129, 1, 64)]:
        bound = ops.attention_scored_most_scratch_bytes(dtype, most_seqs, most_tokens, most_keys, nq, nkv, d)
        sizes = [(most_seqs, 1, most_tokens, most_keys), (1, most_tokens, most_tokens, most_keys)]
        sizes += [(log(1, most_seqs), log(1, most_tokens), log(1, most_tokens), log(1, most_keys)) for _ in range(1500)]
        for seqs, longest, tokens, keys in sizes:
            longest = min(longest, keys, tokens)
            tokens = min(max(tokens, longest), longest * seqs)
            for shortest in {0, 1, longest, max(0, tokens - longest * (seqs - 1))}:
                if shortest * seqs <= tokens:
                    took = ops.attention_scored_scratch_bytes(dtype, seqs, tokens, shortest, longest, keys, nq, nkv, d, 64)
                    assert took <= bound, (seqs, tokens, shortest, longest, keys, nq, nkv, d, took / bound)
        assert bound < 3 << 30                              # and no more than a few GiB


def test_sizes_that_three_samples_of_a_step_missed():
    from nanohybrid_vlm_b200.kernels import ops
    for most, size in [((512, 16384, 4096), (366, 15821, 1, 78, 622)), ((256, 2048, 32768), (256, 2048, 1, 8, 32768))]:
        assert ops.attention_scored_scratch_bytes(torch.bfloat16, *size, 32, 8, 128, 256) <= ops.attention_scored_most_scratch_bytes(torch.bfloat16, *most, 32, 8, 128)
