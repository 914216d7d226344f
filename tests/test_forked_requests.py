"""Requests that share their first positions' pages: the allocator's holders, forks in the cache manager, and families in the
scheduler, on the host."""
import random
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from tlie_amd.cache.manager import CacheManager, RunNeed
from tlie_amd.cache.pages import PageAllocator
from tlie_amd.engine.scheduler import Request, SamplingParams, Scheduler
from tlie_amd.errors import EngineError
from tlie_amd.parts.base import CacheNeed, StateNeed


def manager(pages=40, requests=8, page_size=4, window=None, state=False):
    need = RunNeed(cache_of=0, cache=CacheNeed((2, 1), 3, window), state=StateNeed((2,)) if state else None)
    return CacheManager([need], page_size, pages, requests, torch.float32, "cpu")


def grow(cache, request, count):
    cache.reserve(request, count)
    cache.commit(request, count)


def test_a_page_comes_back_with_its_last_holder():
    pages = PageAllocator(3)
    held = pages.alloc(2)
    pages.share(held)
    pages.release(held)
    assert pages.num_free == 1 and all(pages.in_use(page) for page in held)
    pages.release(held)
    assert pages.num_free == 3 and not any(pages.in_use(page) for page in held)
    for wrong in ([held[0]], [99], [-1]):
        with pytest.raises(EngineError):
            pages.share(wrong)


@pytest.mark.parametrize("length", [1, 3, 4, 5, 8, 10])
def test_a_fork_holds_the_same_pages_and_a_copy_of_the_last(length):
    cache = manager()
    cache.admit("a")
    grow(cache, "a", 10)
    pool = cache.bindings[0].cache
    pool.copy_(torch.randn_like(pool))
    cache.fork("a", "b", length)
    mine, its = cache.page_list("b", 0), cache.page_list("a", 0)
    whole = length // 4
    assert mine[:whole] == its[:whole] and len(mine) == (length + 3) // 4 and cache.length("b") == length
    if length % 4:
        assert mine[-1] not in its and torch.equal(pool[mine[-1]], pool[its[whole]])
    cache.check()
    held = [cache.held(name) for name in "ab"]
    assert all((info.family != 0) == (whole > 0) for info in held)
    assert not whole or held[0].family == held[1].family and min(info.shared for info in held) == whole * 4
    grow(cache, "b", 7)
    grow(cache, "a", 2)
    cache.check()
    cache.release("a")
    cache.check()
    cache.release("b")
    assert cache.free_pages() == [40]
    cache.check()


def test_forks_of_forks_claim_no_more_than_they_share():
    cache = manager()
    cache.admit("a")
    grow(cache, "a", 12)
    cache.fork("a", "b", 8)
    grow(cache, "b", 12)
    cache.fork("b", "c", 20)                     # more than b has in common with a
    cache.fork("b", "d", 4)
    lists = {name: cache.page_list(name, 0) for name in "abcd"}
    held = {name: cache.held(name) for name in "abcd"}
    for one in "abcd":
        for other in "abcd":
            blocks = min(held[one].shared, held[other].shared) // 4
            assert held[one].family == held[other].family and lists[one][:blocks] == lists[other][:blocks]
    cache.check()


def test_forks_that_are_refused_take_nothing():
    cache = manager(pages=3, requests=2)
    cache.admit("a")
    grow(cache, "a", 10)
    for source, length in (("a", 11), ("a", 0), ("x", 2)):
        with pytest.raises(EngineError):
            cache.fork(source, "b", length)
    with pytest.raises(EngineError):
        cache.fork("a", "b", 5)                  # no page for the copy
    assert not cache.is_live("b") and cache.free_slots == 1
    cache.fork("a", "b", 8)
    with pytest.raises(EngineError):
        cache.fork("a", "c", 4)                  # no slot
    cache.check()
    for kind in (dict(window=8), dict(state=True)):
        other = manager(**kind)
        other.admit("a")
        grow(other, "a", 10)
        assert not other.can_fork
        with pytest.raises(EngineError):
            other.fork("a", "b", 4)


def family_of(count, prompt, **params):
    family = []
    for index in range(count):
        family.append(Request(id=("answer", index), prompt=list(prompt), params=SamplingParams(**params), family=family))
    return family


def run(scheduler, cache, steps=400):
    """Plans and commits; tokens are their place in the request.  Returns the planned tokens of every step."""
    seen = []
    for _ in range(steps):
        if not scheduler.has_work():
            break
        plan = scheduler.schedule()
        assert plan
        assert cache.reserve_all([(item.request.id, item.count) for item in plan])
        for item in plan:
            cache.commit(item.request.id, item.count)
        cache.check()
        seen.append([(item.request.id, item.first, item.count) for item in plan])
        scheduler.update(plan, [item.first + item.count for item in plan if item.samples])
    assert not scheduler.has_work()
    return seen


def test_answers_compute_the_prompt_once():
    cache = manager(pages=60)
    scheduler = Scheduler(cache)
    family = family_of(4, range(21), max_tokens=5)
    for request in family:
        scheduler.add(request)
    seen = run(scheduler, cache)
    brought = {request.id: sum(count for step in seen for name, _, count in step if name == request.id) for request in family}
    assert brought[family[0].id] == 21 + 4 and all(brought[request.id] == 1 + 4 for request in family[1:])
    assert all(len(request.generated) == 5 for request in family)
    assert cache.free_pages() == [60]


def test_a_family_stands_side_by_side():
    cache = manager(pages=100, requests=8)
    scheduler = Scheduler(cache)
    one, two = family_of(3, range(9), max_tokens=6), family_of(3, range(13), max_tokens=6)
    for request in two:
        request.id = ("other", request.id[1])
    for first in range(3):
        scheduler.add(one[first])
        scheduler.add(two[first])
    for step in run(scheduler, cache):
        kinds = [name[0] for name, _, _ in step]
        assert kinds == sorted(kinds, key=kinds.index)


def test_short_prompts_and_caches_that_cannot_fork_run_as_ever():
    for cache, length in ((manager(pages=60), 4), (manager(pages=60, window=8), 21), (manager(pages=60, state=True), 21)):
        scheduler = Scheduler(cache)
        family = family_of(3, range(length), max_tokens=3)
        for request in family:
            scheduler.add(request)
        seen = run(scheduler, cache)
        assert all(sum(count for step in seen for name, _, count in step if name == request.id) == length + 2 for request in family)


@pytest.mark.parametrize("seed", range(12))
def test_pools_too_small_for_all_lose_nothing(seed):
    """Preempted, readmitted, aborted members: every request gets its tokens, every page comes back."""
    rng = random.Random(seed)
    cache = manager(pages=rng.randint(12, 30), requests=rng.randint(2, 6))
    scheduler = Scheduler(cache, max_tokens_per_step=rng.randint(3, 30), chunk_size=rng.randint(2, 12), admit_partial=rng.random() < 0.5)
    families = [family_of(rng.randint(1, 5), range(rng.randint(1, 25)), max_tokens=rng.randint(1, 14)) for _ in range(3)]
    for index, family in enumerate(families):
        for request in family:
            request.id = (index, request.id[1])
            scheduler.add(request)
    victim = families[0][0].id
    scheduler.abort(victim)
    run(scheduler, cache, steps=3000)
    for family in families:
        for request in family:
            assert len(request.generated) == request.params.max_tokens or request.id == victim
    assert cache.free_pages() == [cache.num_pages] and cache.free_slots == cache.max_requests


@pytest.mark.parametrize("bad", [dict(top_k=-1), dict(top_k=1 << 31), dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=float("nan"))])
def test_sampling_options_that_are_refused(bad):
    with pytest.raises(EngineError):
        SamplingParams(**bad).validate()


def test_the_numbers_of_many_rows_are_the_numbers_of_each():
    from tlie_amd.sampling.sampler import uniform01, uniforms01
    rng = random.Random(0)
    seeds, counters = [rng.randrange(-2 ** 63, 2 ** 64) for _ in range(100)], [rng.randrange(1 << 20) for _ in range(100)]
    assert uniforms01(seeds, counters).tolist() == [uniform01(seed, counter) for seed, counter in zip(seeds, counters)]


def test_a_family_of_two_prompts_is_refused():
    cache = manager()
    scheduler = Scheduler(cache, max_tokens_per_step=64)
    family = family_of(2, range(1, 12), max_tokens=2)
    family[1].prompt[3] = 40
    scheduler.add(family[0])
    with pytest.raises(EngineError):
        scheduler.add(family[1])


def test_a_plan_made_within_a_step_is_waited_for_by_the_next(monkeypatch):
    """The host's buffer of a recorded plan is written again only behind the event that stands after its last transfer."""
    from tlie_amd.engine import step
    log = []
    monkeypatch.setattr(step, "ops_RecordedPrefixPlan", lambda *sizes: SimpleNamespace(plan="plan", fill=lambda *work: log.append("fill")))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    graph = step.SharedDecodeGraph.__new__(step.SharedDecodeGraph)
    graph.bucket, graph.longest, graph._plans, graph.shared, graph._rows_filled = 4, 256, {}, [(0, 2, 64)], 2
    graph.host = {"seq_start": np.arange(5), "seq_len": np.array([70, 71, 1, 1])}
    graph.device_flat, graph.copied = torch.zeros(1), SimpleNamespace(record=lambda: log.append("record"))
    assert graph.prefix_plan(8, 2, 64, torch.bfloat16) == "plan"
    assert log == ["fill", "record"]
    assert graph.prefix_plan(8, 2, 64, torch.bfloat16) == "plan" and log == ["fill", "record"]


@pytest.mark.parametrize("length", [16, 17, 21])
def test_a_member_that_does_not_fit_yet_is_not_forked(monkeypatch, length):
    """Blocked over many steps, for want of pages: no fork is made (each copies a page of every layer) until one that then runs.
    Prompts whose shared positions end inside a page and at its end."""
    cache = manager(pages=11, requests=8)
    forks, real = [], cache.fork
    monkeypatch.setattr(cache, "fork", lambda *call: (forks.append(call[1]), real(*call))[1])
    scheduler = Scheduler(cache)
    family = family_of(2, range(length), max_tokens=9)
    other = Request(id="other", prompt=list(range(13)), params=SamplingParams(max_tokens=8))
    for request in (family[0], other, family[1]):
        scheduler.add(request)
    blocked = 0
    for _ in range(60):
        if not scheduler.has_work():
            break
        before = len(forks)
        plan = scheduler.schedule()
        assert cache.reserve_all([(item.request.id, item.count) for item in plan])
        for item in plan:
            cache.commit(item.request.id, item.count)
        cache.check()
        planned = [item.request.id for item in plan]
        assert all(name in planned for name in forks[before:])
        blocked += family[1].state == "waiting" and family[0].computed >= length
        scheduler.update(plan, [item.first + item.count for item in plan if item.samples])
    assert not scheduler.has_work() and blocked > 2
    assert forks.count(family[1].id) <= 1 + family[1].preemptions
    assert [len(request.generated) for request in (*family, other)] == [9, 9, 8]


@pytest.mark.parametrize("length,count", [(1, 1), (3, 1), (4, 1), (5, 3), (8, 9), (10, 1)])
def test_the_pages_that_a_fork_takes(length, count):
    cache = manager()
    cache.admit("a")
    grow(cache, "a", 10)
    free, wanted = cache.free_pages(), cache.pages_to_fork(length, count)
    cache.fork("a", "b", length)
    cache.reserve("b", count)
    assert cache.free_pages() == [have - need for have, need in zip(free, wanted)]


def test_requests_behind_a_member_that_waits_for_its_familys_keys_go_on():
    """A long prompt is computed in portions; its second answer waits for that, other prompts do not.  Its turn is the first when
    the keys are there."""
    cache = manager(pages=200, requests=8)
    scheduler = Scheduler(cache, max_tokens_per_step=16, chunk_size=8)
    family = family_of(3, range(80), max_tokens=4)
    others = [Request(id=("other", index), prompt=list(range(6 + index)), params=SamplingParams(max_tokens=4)) for index in range(3)]
    for request in (*family, *others):
        scheduler.add(request)
    seen = run(scheduler, cache)
    begins = lambda name: next(index for index, step in enumerate(seen) if any(one == name for one, _, _ in step))
    assert begins(("other", 0)) == 0 and begins(("other", 2)) < begins(family[1].id)
    assert begins(family[1].id) == begins(family[2].id) == 1 + max(index for index, step in enumerate(seen) if (family[0].id, 72, 8) in step)


def test_a_member_that_waits_for_pages_lets_nobody_ahead():
    """First come, first served, once the keys are there: a request behind it that would fit does not take the pages it waits for."""
    cache = manager(pages=9, requests=8)
    scheduler = Scheduler(cache)
    family = family_of(2, range(17), max_tokens=16)
    small = Request(id="small", prompt=[1, 2], params=SamplingParams(max_tokens=3))
    family[1].generated = [3] * 8                         # (preempted before: it brings these too, on three pages)
    scheduler.add(family[0])
    scheduler.add(family[1])
    seen = []
    while scheduler.has_work():
        plan = scheduler.schedule()
        assert cache.reserve_all([(item.request.id, item.count) for item in plan])
        for item in plan:
            cache.commit(item.request.id, item.count)
        seen.append([item.request.id for item in plan])
        scheduler.update(plan, [item.first + item.count for item in plan if item.samples])
        if len(seen) == 1:                                # (the prompt's keys are there now; its second answer does not fit beside the first)
            scheduler.add(small)
    begins = lambda name: next(index for index, step in enumerate(seen) if name in step)
    assert begins("small") >= begins(family[1].id) > 2


def runner_of(cache, kv_heads=8, dim=128):
    from tlie_amd.engine.step import ModelRunner
    mixer = SimpleNamespace(nkv=kv_heads, d=dim, takes_shared_prefix=True)
    model = SimpleNamespace(device="cpu", spec=SimpleNamespace(vocab_size=100), blocks=[SimpleNamespace(mixer=mixer)])
    return ModelRunner(model, cache, use_graphs=False)


def test_steps_without_families_are_not_looked_through(monkeypatch):
    """A step of an engine without forks asks no request for its pages; the last fork's end brings that back."""
    from tlie_amd.engine.step import StepEntry
    cache = manager(pages=200, requests=8, page_size=16)
    runner = runner_of(cache)
    asked, real = [], cache.held
    monkeypatch.setattr(cache, "held", lambda request: (asked.append(request), real(request))[1])
    for name in "abcd":
        cache.admit(name)
        grow(cache, name, 40)
    entries = [StepEntry(name, [1], [0]) for name in "abcd"]
    assert runner.shared_groups(entries) == [] and not asked and not cache.has_families
    cache.fork("a", "e", 33)
    assert cache.has_families
    runner.shared_groups(entries)
    assert asked == list("abcd")
    cache.release("a")
    assert cache.has_families
    cache.release("e")
    asked.clear()
    assert runner.shared_groups(entries[1:]) == [] and not asked and not cache.has_families
    cache.fork("b", "e", 15)                     # (less than a page: nothing is held together)
    assert not cache.has_families


def test_groups_are_runs_of_one_family(monkeypatch):
    from tlie_amd.engine import step
    monkeypatch.setattr(step, "ops_shared_prefix_pays", lambda *sizes: True)
    rng = random.Random(1)
    for _ in range(60):
        cache = manager(pages=400, requests=40, page_size=16)
        names, live = iter(range(1000)), []
        for _ in range(4):
            root = next(names)
            cache.admit(root)
            grow(cache, root, rng.randint(1, 90))
            live.append(root)
            for _ in range(rng.randint(0, 4)):
                fork = next(names)
                source = rng.choice(live)
                cache.fork(source, fork, rng.randint(1, cache.length(source)))
                live.append(fork)
        for name in rng.sample(live, rng.randint(0, 3)):
            cache.release(name)
            live.remove(name)
        assert cache.has_families == any(cache.held(name).family for name in live)
        rng.shuffle(live)
        live.sort(key=lambda name: cache.held(name).family if rng.random() < 0.8 else 0)
        covered = [None] * len(live)
        for group, (first, count, prefix) in enumerate(runner_of(cache).shared_groups([step.StepEntry(name, [1], [0]) for name in live])):
            held = [cache.held(name) for name in live[first:first + count]]
            assert count > 1 and prefix == min(info.shared for info in held) > 0 and len({info.family for info in held}) == 1 and held[0].family
            covered[first:first + count] = [group] * count
        for index in range(1, len(live)):
            one, other = cache.held(live[index - 1]), cache.held(live[index])
            assert (covered[index] is not None and covered[index] == covered[index - 1]) == (one.family == other.family != 0)


def test_what_the_rows_of_a_step_ask():
    """The same as row by row, and without looking at each when nobody asks."""
    from tlie_amd.sampling.sampler import what_rows_ask
    rng = random.Random(4)
    kinds = [dict(), dict(temperature=0.7), dict(temperature=0.7, top_k=5), dict(top_k=5), dict(temperature=1.0, min_p=0.1), dict(min_p=0.1), dict(logprobs=True),
             dict(temperature=0.5, top_k=3, min_p=0.2, logprobs=True)]
    for _ in range(300):
        params = [SamplingParams(**rng.choice(kinds[:rng.randint(1, len(kinds))])) for _ in range(rng.randint(1, 6))]
        filtered = [one.temperature > 0 and (one.top_k > 0 or one.min_p > 0) for one in params]
        assert what_rows_ask(params) == (any(one.logprobs for one in params), filtered if any(filtered) else None)
    bare = [SimpleNamespace(temperature=0.5, top_p=1.0, seed=1)]
    assert what_rows_ask(bare) == (False, None)
    assert what_rows_ask(bare + [SamplingParams(temperature=0.5, top_k=2, logprobs=True)]) == (True, [False, True])

    class Asked(SamplingParams):
        @property
        def filtered(self):
            raise AssertionError("looked at row by row")
    assert what_rows_ask([Asked(temperature=0.9) for _ in range(3)]) == (False, None)
