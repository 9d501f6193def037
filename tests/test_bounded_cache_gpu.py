"""Generation with a cache that drops keys, against a plain model that does the same one token at a time: per layer and KV head a
list of keys with the weight each has gathered, cut down to the budget after the prompt and whenever a page has come together."""
import math

import pytest
import torch

import plain_qwen3 as plain
from conftest import TINY
from test_generate_gpu import make_llm, prompts_for

pytestmark = pytest.mark.gpu


class PlainBounded:
    """A request's life in the plain model's parts.  Keys are kept as (birth, key, value, score) per layer and KV head, in no order."""

    def __init__(self, model, budget, page, first, recent):
        self.m, self.budget, self.page, self.first, self.recent = model, budget, page, first, recent
        cfg = model.cfg
        self.heads = [[[] for _ in range(cfg["num_key_value_heads"])] for _ in range(cfg["num_hidden_layers"])]
        self.seen = 0

    def attend(self, i, q, k, v):
        """q [T, nq, d], k, v [T, nkv, d] of the new tokens, which see all kept keys and the new ones up to their own."""
        T, nq, d = q.shape
        out = torch.zeros(T, nq, d)
        for g, kept in enumerate(self.heads[i]):
            old = len(kept)
            kept += [[self.seen + t, k[t, g], v[t, g], 0.0] for t in range(T)]
            ks, vs = torch.stack([x[1] for x in kept]).double(), torch.stack([x[2] for x in kept]).double()
            for h in range(g * nq // k.shape[1], (g + 1) * nq // k.shape[1]):
                s = q[:, h].double() @ ks.T * d ** -0.5
                for t in range(T):
                    s[t, old + t + 1:] = -math.inf
                p = torch.softmax(s, dim=1)
                out[:, h] = (p @ vs).float()
                for j, w in enumerate(p.sum(0).tolist()):
                    kept[j][3] += w
        return out

    def step(self, tokens):
        m, cfg, w = self.m, self.m.cfg, self.m.w
        nq, nkv, d, eps = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], cfg["rms_norm_eps"]
        at = torch.arange(self.seen, self.seen + len(tokens))
        h, residual = w["model.embed_tokens.weight"][torch.tensor(tokens)], None
        for i in range(cfg["num_hidden_layers"]):
            p = f"model.layers.{i}."
            if residual is None:
                residual, x = h, plain.rms_norm(h, w[p + "input_layernorm.weight"], eps)
            else:
                x, residual = plain.add_rms_norm(h, residual, w[p + "input_layernorm.weight"], eps)
            q, k, v = (plain.linear(x, w[f"{p}self_attn.{n}_proj.weight"]).view(len(tokens), c, d) for n, c in (("q", nq), ("k", nkv), ("v", nkv)))
            q = plain.apply_rope(plain.rms_norm(q, w[p + "self_attn.q_norm.weight"], eps), m.cos[at], m.sin[at])
            k = plain.apply_rope(plain.rms_norm(k, w[p + "self_attn.k_norm.weight"], eps), m.cos[at], m.sin[at])
            o = self.attend(i, q, k, v).reshape(len(tokens), nq * d)
            x, residual = plain.add_rms_norm(plain.linear(o, w[p + "self_attn.o_proj.weight"]), residual, w[p + "post_attention_layernorm.weight"], eps)
            h = plain.swiglu_mlp(x, w, p + "mlp.")
        h, _ = plain.add_rms_norm(h, residual, w["model.norm.weight"], eps)
        self.seen += len(tokens)
        return plain.linear(h[-1:], w["lm_head.weight"])[0].float()

    def cut(self):
        """Drops keys if a page more than the budget has come together; says how close the choice was."""
        closest = math.inf
        for layer in self.heads:
            for kept in layer:
                if len(kept) < self.budget + self.page:
                    return closest
                held = [x for x in kept if x[0] < self.first or x[0] >= self.seen - self.recent]
                rest = sorted((x for x in kept if not (x[0] < self.first or x[0] >= self.seen - self.recent)), key=lambda x: -x[3])
                n = self.budget - len(held)
                closest = min(closest, (rest[n - 1][3] - rest[n][3]) / rest[n][3])
                kept[:] = held + rest[:n]
        return closest

    def births(self):
        return [[sorted(x[0] for x in kept) for kept in layer] for layer in self.heads]


def held_by_engine(llm, seq_id, n):
    """Per layer and KV head: the sorted births and the scores of the slots that a request holds."""
    runner = llm.model_runner
    table = runner.cache.block_table(seq_id)
    births, scores = [], []
    for b, s in zip(runner.storage.births, runner.storage.scores):
        births.append([sorted(torch.cat([b[p, g] for p in table])[:n].tolist()) for g in range(b.shape[1])])
        scores.append(torch.stack([torch.cat([s[p, g] for p in table])[:n] for g in range(s.shape[1])]))
    return births, scores


@pytest.mark.parametrize("name,lengths,new,budget,first,recent", [("A", (5, 61, 100), 60, 32, 2, 8), ("B", (1, 70), 50, 24, 0, 5)])
def test_generation_with_dropped_keys_matches_plain(name, lengths, new, budget, first, recent, model_dirs, plain_models):
    from nanohybrid_vlm_b200 import SamplingParams
    page = 16 if name == "A" else 8
    prompts = prompts_for(name, lengths, seed=7)
    llm = make_llm(model_dirs[name], name, cache_budget=budget, cache_first=first, cache_recent=recent, max_num_batched_tokens=256,
                   num_kvcache_blocks=60 // page * 3 + 20)
    ids = [llm.add_request(p, SamplingParams(temperature=0.0, max_tokens=new, ignore_eos=True)) for p in prompts]
    plains = {i: PlainBounded(plain_models[name], budget, page, first, recent) for i in ids}
    fed = {i: list(p) for i, p in zip(ids, prompts)}
    outputs, drops, compared = {}, 0, 0
    live = {i: s for i, s in zip(ids, llm.scheduler.waiting)}
    while not llm.is_finished():
        finished, _ = llm.step()
        outputs.update(finished)
        for i in [i for i in llm.last_sampled_ids if i in plains]:
            # the plain model goes through the same tokens: its choice is the engine's, or so close that either may be
            lg = plains[i].step(fed[i])
            token = outputs[i][-1] if i in outputs else live[i].token_ids[-1]
            assert lg[token] >= lg.max() - 2e-4, (i, len(live[i]), float(lg.max() - lg[token]))
            fed[i] = [token]
            near = plains[i].cut()
            drops += near < math.inf
            if near < 1e-4:                                 # so close that rounding decides: either choice is right, and the two part here
                del plains[i]
            if i in outputs or i not in plains:
                continue
            kept = len(plains[i].heads[0][0])
            births, scores = held_by_engine(llm, i, kept)
            assert live[i].num_kept_tokens == kept <= max(len(prompts[ids.index(i)]), budget + page)
            assert births == plains[i].births()
            for a, b in zip(scores, plains[i].heads):
                want = torch.tensor([[x[3] for x in kv] for kv in b], dtype=torch.float64)
                assert torch.allclose(a.cpu().double().sort(1).values, want.sort(1).values, rtol=1e-3, atol=1e-6)
            compared += 1
    assert drops >= len(ids) and compared > new
    assert all(len(outputs[i]) == new for i in ids)
    llm.model_runner.cache.check()
    assert llm.model_runner.cache.num_live() == 0


@pytest.mark.parametrize("name,lengths,new", [("A", (5, 17, 33), 8), ("B", (1, 9, 40, 71), 12)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_budget_that_is_never_reached_changes_nothing(name, lengths, new, dtype, model_dirs, plain_models):
    from nanohybrid_vlm_b200 import SamplingParams
    from test_generate_gpu import assert_greedy_follows
    prompts = prompts_for(name, lengths)
    llm = make_llm(model_dirs[name], name, dtype=dtype, cache_budget=200)
    out = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=new, ignore_eos=True), use_tqdm=False)
    if dtype == "float32":
        assert [o["token_ids"] for o in out] == [plain_models[name].greedy(p, new) for p in prompts]
    else:
        for p, o in zip(prompts, out):
            assert_greedy_follows(plain_models[name], p, o["token_ids"], slack=0.03)


def test_preempted_requests_start_over_and_finish(model_dirs):
    """A pool that cannot hold all requests at once: those that give way are computed again from their first token."""
    from nanohybrid_vlm_b200 import SamplingParams
    llm = make_llm(model_dirs["A"], "A", cache_budget=32, cache_first=2, cache_recent=8, num_kvcache_blocks=8, max_num_batched_tokens=256)
    prompts = prompts_for("A", (40, 50, 30, 20), seed=3)
    out = llm.generate(prompts, SamplingParams(temperature=0.7, max_tokens=70, ignore_eos=True, seed=5), use_tqdm=False)
    assert all(len(o["token_ids"]) == 70 for o in out)
    assert llm.scheduler.num_preemptions > 0
    llm.model_runner.cache.check()
    assert llm.model_runner.cache.num_live() == 0


def test_models_that_cannot_drop_keys_say_so(tmp_path):
    from nanohybrid_vlm_b200 import LLM
    from test_kilisun_gpu import KIL_A, write_model          # a design with windows
    write_model(str(tmp_path), KIL_A, 0)
    with pytest.raises(ValueError, match="cache_budget"):
        LLM(str(tmp_path), dtype="float32", cache_budget=32, num_kvcache_blocks=16, max_num_seqs=2, max_model_len=64)


@pytest.mark.parametrize("name,lengths,new,budget,first,recent,pages", [("A", (40, 50, 30), 70, 40, 2, 8, 9), ("B", (20, 33, 9, 41), 60, 20, 1, 5, 10)])
def test_preempted_requests_keep_what_they_kept(name, lengths, new, budget, first, recent, pages, model_dirs, plain_models):
    """Requests that give way and are computed again hold the same keys behind it as the plain model, which nobody interrupts."""
    from nanohybrid_vlm_b200 import SamplingParams
    page = 16 if name == "A" else 8
    prompts = prompts_for(name, lengths, seed=11)
    llm = make_llm(model_dirs[name], name, cache_budget=budget, cache_first=first, cache_recent=recent, max_num_batched_tokens=64, num_kvcache_blocks=pages)
    ids = [llm.add_request(p, SamplingParams(temperature=0.0, max_tokens=new, ignore_eos=True)) for p in prompts]
    plains = {i: PlainBounded(plain_models[name], budget, page, first, recent) for i in ids}
    fed, outputs = {i: list(p) for i, p in zip(ids, prompts)}, {}
    live = {i: s for i, s in zip(ids, llm.scheduler.waiting)}
    after_preemption = 0
    while not llm.is_finished():
        outputs.update(llm.step()[0])
        for i in [i for i in llm.last_sampled_ids if i in plains]:
            lg = plains[i].step(fed[i])
            token = outputs[i][-1] if i in outputs else live[i].token_ids[-1]
            assert lg[token] >= lg.max() - 2e-4, (i, len(live[i]), float(lg.max() - lg[token]))
            fed[i] = [token]
            if plains[i].cut() < 1e-4:                      # so close that rounding decides: the two may part here
                del plains[i]
            if i in outputs or i not in plains:
                continue
            kept = len(plains[i].heads[0][0])
            births, scores = held_by_engine(llm, i, kept)
            assert live[i].num_kept_tokens == kept and births == plains[i].births()
            for a, b in zip(scores, plains[i].heads):
                want = torch.tensor([[x[3] for x in kv] for kv in b], dtype=torch.float64)
                assert torch.allclose(a.cpu().double().sort(1).values, want.sort(1).values, rtol=1e-3, atol=1e-6)
            after_preemption += live[i].num_preemptions > 0 and live[i].num_dropped_tokens > page
    assert llm.scheduler.num_preemptions > 0 and after_preemption > 20
    assert all(len(outputs[i]) == new for i in ids)
    llm.model_runner.cache.check()
