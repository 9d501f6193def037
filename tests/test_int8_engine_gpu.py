"""The engine with its layers' matrices in 8-bit integers (``quantization="int8"``) against the plain model with the same roundings:
every matrix of a layer row by row, and what it multiplies token by token, to a = max |x|, round(127 x / a), a / 127.

Tolerance in float32.  Both sides round the same numbers, but for what their sums are off before that, some 1e-6; where a number lies that
near the middle between two integers they come out a step apart.  Of the 640 (A) to 1,632 (B) numbers that a token's products read, one
does so with a chance of 2 * 127 * 1e-6 each: 0.2 to 0.4 a token.  All roundings together, 0.29 steps rms each, are 7 to 12 steps and
move the logits by 0.5 to 2 % of their norm (plain model against plain model): one step moves them by 0.25 % at most.  Two of them, and
what earlier tokens pass on through the attention: 0.6 %."""
import numpy as np
import pytest
import torch

import plain_qwen3 as plain
from conftest import TINY, TINY_C
from test_generate_gpu import make_llm, prompts_for

pytestmark = pytest.mark.gpu
TOL = 0.006


def eight(x):
    top = x.double().abs().amax(-1, keepdim=True)
    return torch.round(127 * x.double() / torch.where(top == 0, 1.0, top)) * (top / 127)


class Plain8(plain.PlainQwen3):
    """The plain model, its layers' products in 8 bits (the head's are not)."""

    def logits(self, token_ids, rows=None):
        whole, head = plain.linear, self.w["lm_head.weight"]
        plain.linear = lambda x, w: whole(x, w) if w is head else (eight(x) @ eight(w).t()).to(x.dtype)
        try:
            return super().logits(token_ids, rows)
        finally:
            plain.linear = whole


@pytest.fixture(scope="module")
def plain8(model_dirs):
    return {name: Plain8(d) for name, d in model_dirs.items()}


class Driver:
    """Requests with given tokens through ``ModelRunner.step``, which returns the logits of every token."""

    def __init__(self, model_dir, dtype="float32", **kw):
        from nanohybrid_vlm_b200.config import Config
        from nanohybrid_vlm_b200.engine.runner import ModelRunner
        opts = dict(dtype=dtype, kvcache_block_size=8, num_kvcache_blocks=80, max_num_seqs=8, max_num_batched_tokens=256, max_model_len=128,
                    enable_prefix_cache=False, poison_cache=True, quantization="int8")
        self.runner = ModelRunner(Config(model_dir, **(opts | kw)))
        self.held = {}

    def step(self, parts):
        from nanohybrid_vlm_b200.engine.batch import StepItem
        items = []
        for rid, tokens in parts:
            at = self.held.get(rid, 0)
            self.runner.cache.allocate(rid, at + len(tokens))
            items.append(StepItem(rid, tokens, at, list(range(len(tokens)))))
            self.held[rid] = at + len(tokens)
        logits = self.runner.step(items).clone()
        self.runner.check_kernels()
        return list(logits.split([len(t) for _, t in parts]))


@pytest.mark.parametrize("name", list(TINY))
def test_logits_follow_the_plain_model_in_8_bits(name, model_dirs, plain8, plain_models):
    d = Driver(model_dirs[name])
    prompts = prompts_for(name, (1, 9, 40, 71), seed=4)
    got = d.step(list(enumerate(prompts)))
    for tokens, lg in zip(prompts, got):
        want = plain8[name].logits(tokens)
        off = (lg.cpu() - want).norm(dim=1) / want.norm(dim=1)
        assert off.max() <= TOL, f"{len(tokens)} tokens: {off.max():.4f}"
    weights = sum(t.numel() * t.element_size() for t in (d.runner.model.embedding.w_weight, d.runner.model.final_norm.w_weight))
    assert weights < d.runner.model.weight_bytes() < 0.45 * sum(w.numel() * 4 for n, w in plain_models[name].w.items() if "layers" in n) + 2 * weights


@pytest.mark.parametrize("name", list(TINY))
def test_float32_logits_do_not_depend_on_the_cutting(name, model_dirs):
    """Whole prompts together, each alone, in portions, and token by token: the sums are integers, so the bits are the same."""
    prompts = prompts_for(name, (3, 26, 90), seed=5)
    together = Driver(model_dirs[name]).step(list(enumerate(prompts)))
    d = Driver(model_dirs[name])
    for i, (tokens, want) in enumerate(zip(prompts, together)):
        rows, at = [], 0
        for n in (1, 12, 9, 1, 1, 33, 2):
            if at < len(tokens):
                rows += d.step([(i, tokens[at:at + n])])
                at += n
        while at < len(tokens):
            rows += d.step([(i, tokens[at:at + 1])])
            at += 1
        assert torch.equal(torch.cat(rows), want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_with_and_without_graphs(dtype, model_dirs, plain8):
    """Greedy tokens are the plain model's best, or as good as it within what the roundings to 8 bits (and to bfloat16) leave open; the same
    through captured decode steps, launched ahead, as one by one."""
    from nanohybrid_vlm_b200 import SamplingParams
    prompts = prompts_for("B", (5, 17, 33), seed=6)
    sp = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    outs = []
    for eager in (True, False):
        llm = make_llm(model_dirs["B"], "B", dtype=dtype, enforce_eager=eager, quantization="int8")
        outs.append([o["token_ids"] for o in llm.generate(prompts, sp, use_tqdm=False)])
        assert llm.model_runner.model.streamed_weights() and all(w.shape[0] == TINY["B"][0]["vocab_size"] for w, _ in llm.model_runner.model.streamed_weights())
        del llm
    if dtype == "float32":
        assert outs[0] == outs[1]
    for out in outs:
        for prompt, tokens in zip(prompts, out):
            seq = list(prompt)
            for t in tokens:
                lg = plain8["B"].logits(seq)[-1]
                # in bfloat16 the 8-bit steps fall differently all over (2^-9 against half a step of 1 / 254): twice the roundings' own 2 %
                assert lg[t] >= lg.max() - (TOL if dtype == "float32" else 0.04) * lg.norm(), f"token {t} at {len(seq)}"
                seq.append(t)


def test_a_batch_of_each_kernels_size(tmp_path):
    """A model with widths that divide by little, in steps of 3, 30 and 200 tokens: each family of products, one after another."""
    from nanohybrid_vlm_b200.weights import write_random_model
    write_random_model(str(tmp_path), TINY_C, 3)
    want = Plain8(str(tmp_path))
    rng = np.random.default_rng(7)
    for total in (3, 30, 200):
        d = Driver(str(tmp_path), kvcache_block_size=64, num_kvcache_blocks=16, max_model_len=256)
        tokens = rng.integers(0, TINY_C["vocab_size"], total).tolist()
        lg, ref = d.step([("a", tokens)])[0].cpu(), want.logits(tokens)
        assert ((lg - ref).norm(dim=1) / ref.norm(dim=1)).max() <= TOL


def test_with_a_bounded_cache(model_dirs):
    from nanohybrid_vlm_b200 import SamplingParams
    llm = make_llm(model_dirs["A"], "A", quantization="int8", cache_budget=32, max_num_batched_tokens=128)
    out = llm.generate(prompts_for("A", (60, 7), seed=8), SamplingParams(temperature=0.0, max_tokens=30, ignore_eos=True), use_tqdm=False)
    assert [len(o["token_ids"]) for o in out] == [30, 30]


def test_a_model_without_such_a_form_is_refused(tmp_path):
    from test_muvonex_config import CFG

    from nanohybrid_vlm_b200.config import Config
    from nanohybrid_vlm_b200.engine.runner import ModelRunner
    import json
    (tmp_path / "config.json").write_text(json.dumps(CFG))
    with pytest.raises(ValueError, match="8-bit"):
        ModelRunner(Config(str(tmp_path), dtype="float32", quantization="int8", max_model_len=64, num_kvcache_blocks=4), random_weights_seed=1)


def test_command_line(model_dirs, plain8):
    import json
    from test_cli import CLI, run
    r = run(CLI + ["generate", "--model", model_dirs["A"], "--dtype", "float32", "--quantization", "int8", "--temperature", "0", "--max-tokens", "4",
                   "--ignore-eos", "--num-kvcache-blocks", "8", "--max-num-seqs", "2", "--max-model-len", "64", "--quiet", "--prompt-ids", "5,9,2"])
    assert r.returncode == 0, r.stderr[-2000:]
    tokens = next(json.loads(x)["token_ids"] for x in r.stdout.splitlines() if x.startswith("{"))
    lg = plain8["A"].logits([5, 9, 2])[-1]
    assert len(tokens) == 4 and lg[tokens[0]] >= lg.max() - TOL * lg.norm()


def test_replay(model_dirs, tmp_path):
    """``bin/trace_run --quantization int8`` gives the runner's logits, bit for bit in float32."""
    import json
    import subprocess
    import sys
    from trace_tools import TRACE_RUN
    tokens = prompts_for("A", (37,), seed=9)[0]
    line = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": tokens, "want": list(range(len(tokens)))}], "end": ["a"]})
    r = subprocess.run([sys.executable, TRACE_RUN, "--model", model_dirs["A"], "--dtype", "float32", "--out", str(tmp_path), "--max-tokens", "64",
                        "--quantization", "int8", "--poison"], input=line + "\n", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    got = np.fromfile(tmp_path / "0.f32", dtype="<f4").reshape(len(tokens), -1)
    assert np.array_equal(got, Driver(model_dirs["A"]).step([("a", tokens)])[0].cpu().numpy())
