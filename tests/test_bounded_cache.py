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
