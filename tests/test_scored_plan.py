"""The host's part of attention with scored keys: the plan and the scratch it asks for, without a GPU."""
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
