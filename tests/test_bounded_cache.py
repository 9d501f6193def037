"""The host's part of a cache that drops keys: options, pages that go back when a request shrinks, and the scheduler's books."""
import json

import pytest

from conftest import TINY_A
from nanohybrid_vlm_b200.cache import CacheManager, GroupSpec
from nanohybrid_vlm_b200.config import Config
from nanohybrid_vlm_b200.config.model_config import ConfigError
from nanohybrid_vlm_b200.engine import Scheduler, Sequence, SequenceStatus
from nanohybrid_vlm_b200.sampling.params import SamplingParams


@pytest.fixture
def folder(tmp_path):
    (tmp_path / "config.json").write_text(json.dumps(TINY_A))
    return str(tmp_path)


def test_options(folder):
    cfg = Config(folder, cache_budget=64)
    assert (cfg.cache_first, cfg.cache_recent) == (4, 16) and cfg.enforce_eager and cfg.enable_prefix_cache is False
    assert Config(folder).enforce_eager is False and Config(folder).enable_prefix_cache is None
    for wrong in (dict(cache_budget=-1), dict(cache_budget=8, cache_first=4, cache_recent=4), dict(cache_budget=64, cache_first=-1),
                  dict(cache_budget=64, enable_prefix_cache=True)):
        with pytest.raises(ConfigError):
            Config(folder, **wrong)


def test_a_request_that_shrinks_gives_its_last_pages_back():
    cm = CacheManager([GroupSpec(None)], 4, 10)
    cm.allocate("a", 27)
    table = list(cm.block_table("a"))
    assert cm.shrink("a", 9) == 4 and cm.block_table("a") == table[:3] and cm.num_tokens("a") == 9
    cm.check()
    assert cm.shrink("a", 12) == 0 and cm.num_tokens("a") == 9          # never grows
    cm.allocate("a", 13)
    assert len(cm.block_table("a")) == 4
    assert cm.shrink("a", 0) == 4 and cm.pools[0].num_free == 10
    cm.check()
    cm.free("a")
    cm.check()
    for other in (CacheManager([GroupSpec(8)], 4, 10), CacheManager([GroupSpec(None)], 4, 10, num_state_slots=2),
                  CacheManager([GroupSpec(None)], 4, 10, enable_prefix_cache=True)):
        other.allocate("a", 9)
        with pytest.raises(ValueError):
            other.shrink("a", 4)


def run_one(scheduler, seen):
    """A step without a model: every request that reaches its end chooses token 1."""
    plan = scheduler.schedule()
    for s in plan.seqs:
        start, n = s.num_cached_tokens, s.num_scheduled_tokens
        assert len(scheduler.cache.block_table(s.seq_id)) * scheduler.cache.page_size >= s.num_kept_tokens + n
        seen.setdefault(s.seq_id, []).extend(range(start, start + n))
    done = [s.num_cached_tokens + s.num_scheduled_tokens == len(s) for s in plan.seqs]
    scheduler.postprocess(plan.seqs, [1 if d else None for d in done])
    over = scheduler.over_budget(plan.seqs)
    for s in over:
        scheduler.dropped(s)
    scheduler.cache.check()
    return plan, over


@pytest.mark.parametrize("pages", [64, 13])
def test_the_scheduler_counts_slots_and_positions_apart(pages):
    """Requests hold at most a page above the budget once their prompt is done, every position is computed (again after a
    preemption), and a pool that could never hold the whole requests is enough."""
    budget, page = 16, 4
    cm = CacheManager([GroupSpec(None)], page, pages)
    sch = Scheduler(cm, max_num_seqs=8, max_num_batched_tokens=32, max_model_len=200, cache_budget=budget)
    seqs = [Sequence([5] * n, SamplingParams(max_tokens=60, ignore_eos=True)) for n in (40, 3, 21)]
    for s in seqs:
        sch.add(s)
    seen, drops = {}, 0
    for _ in range(2000):
        if sch.is_finished():
            break
        _, over = run_one(sch, seen)
        drops += len(over)
        for s in seqs:
            if s.status == SequenceStatus.RUNNING:
                assert s.num_kept_tokens < budget + page
    assert sch.is_finished() and drops >= 3 * 8
    for s in seqs:
        assert s.num_completion_tokens == 60
        positions = seen[s.seq_id]
        assert set(positions) == set(range(len(s) - 1))
        if s.num_preemptions == 0:
            assert positions == list(range(len(s) - 1))
    assert cm.pools[0].num_free == pages


def test_requests_that_never_fit_are_refused():
    cm = CacheManager([GroupSpec(None)], 4, 6)
    sch = Scheduler(cm, max_num_seqs=8, max_num_batched_tokens=32, max_model_len=200, cache_budget=16)
    sch.add(Sequence([5] * 20, SamplingParams(max_tokens=100)))          # 24 slots at most
    with pytest.raises(ValueError, match="never fit"):
        sch.add(Sequence([5] * 25, SamplingParams(max_tokens=2)))         # the prompt is held whole
    with pytest.raises(ValueError, match="never fit"):
        Scheduler(cm, max_num_seqs=8, max_num_batched_tokens=32, max_model_len=200).add(Sequence([5] * 20, SamplingParams(max_tokens=100)))


def run_bounded(budget, page, pages, batched, requests, policy="decode_first", max_num_seqs=8, max_portion=None, most_steps=20000):
    """Requests (arrival step, prompt, new tokens) through a scheduler without a model.  Returns them and, per request and life between
    preemptions, the places (numbers of cached tokens) at which its keys were cut down."""
    cm = CacheManager([GroupSpec(None)], page, pages)
    sch = Scheduler(cm, max_num_seqs=max_num_seqs, max_num_batched_tokens=batched, max_model_len=100000, cache_budget=budget, policy=policy,
                    max_portion=max_portion)
    todo = sorted(requests)
    seqs, seen, cuts, lives, step = [], {}, {}, {}, 0
    while todo or not sch.is_finished():
        while todo and (todo[0][0] <= step or sch.is_finished()):
            _, prompt, new = todo.pop(0)
            seqs.append(Sequence([5] * prompt, SamplingParams(max_tokens=new, ignore_eos=True)))
            sch.add(seqs[-1])
        step += 1
        assert step < most_steps, "no end in sight"
        _, over = run_one(sch, seen)
        for s in over:
            key = (s.seq_id, s.num_preemptions)
            cuts.setdefault(key, []).append(s.num_cached_tokens)
            assert s.num_kept_tokens == budget
        for s in seqs:
            if not s.is_finished and s.seq_id in cm:
                assert s.num_kept_tokens < max(s.num_prompt_tokens, budget + page) and cm.num_tokens(s.seq_id) <= max(s.num_prompt_tokens, budget + page)
    assert cm.pools[0].num_free == pages and cm.num_live() == 0
    for s in seqs:
        assert set(seen[s.seq_id]) == set(range(len(s) - 1))
        first = max(s.num_prompt_tokens, budget + page)
        lives = [v for (i, _), v in cuts.items() if i == s.seq_id]
        for places in lives:                                # the same places in every life, as far as it went
            assert places == list(range(first, len(s), page))[:len(places)]
        if len(s) - 1 > first:
            assert max(map(len, lives)) == len(range(first, len(s) - 1, page))
    return seqs


def test_a_request_that_outgrew_the_pool_comes_back():
    """Preempted with more tokens than the pool has slots: computed again under the bound, not from its whole length."""
    for requests, budget, pages, batched in [([(0, 10, 300), (200, 30, 20)], 18, 13, 8), ([(0, 1, 99), (0, 34, 105)], 24, 13, 32)]:
        seqs = run_bounded(budget, 4, pages, batched, requests)
        assert any(s.num_preemptions for s in seqs) and all(s.num_completion_tokens == new for s, (_, _, new) in zip(seqs, requests))


@pytest.mark.parametrize("policy", ["decode_first", "prefill_first"])
def test_bounded_requests_of_every_kind_finish(policy):
    import random
    preempted = outgrown = 0
    for seed in range(400):
        rng = random.Random(seed)
        page = rng.choice((1, 3, 4, 8))
        budget = rng.randint(6, 40)
        full = -(-(budget + page) // page)
        pages = full + rng.randint(0, 2 * full)
        requests = [(rng.choice((0, 0, rng.randint(0, 120))), rng.randint(1, min(60, pages * page)), rng.randint(1, 160)) for _ in range(rng.randint(1, 6))]
        seqs = run_bounded(budget, page, pages, rng.choice((1, 8, 32, 256)), requests, policy, rng.choice((1, 2, 8)), rng.choice((None, None, 5)))
        preempted += sum(s.num_preemptions > 0 for s in seqs)
        outgrown += sum(s.num_preemptions > 0 and len(s) > pages * page for s in seqs)
    assert preempted > 100 and outgrown > 10


def test_new_requests_do_not_wait_for_one_that_is_computed_again():
    """Its portions end where its keys are cut; what they leave of a step goes to the requests behind it."""
    cm = CacheManager([GroupSpec(None)], 4, 40)
    sch = Scheduler(cm, max_num_seqs=8, max_num_batched_tokens=64, max_model_len=1000, cache_budget=16)
    long = Sequence([5] * 10, SamplingParams(max_tokens=100, ignore_eos=True))
    sch.add(long)
    seen = {}
    for _ in range(60):
        run_one(sch, seen)
    sch._preempt(long, sch.schedule())
    fresh = Sequence([5] * 30, SamplingParams(max_tokens=5, ignore_eos=True))
    sch.add(fresh)
    plan, _ = run_one(sch, seen)
    assert plan.seqs == [long, fresh] and plan.num_prefill_tokens == 20 + 30
    while not sch.is_finished():
        run_one(sch, seen)
    assert long.num_completion_tokens == 100 and fresh.num_completion_tokens == 5
