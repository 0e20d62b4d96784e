"""Prefixes and samples in the scheduler, with a stand-in for the step function: what is computed once, what waits for what, what is given back when."""
import pytest

from test_scheduler import ArgmaxSampler, FakeRunner, Request, Scheduler
from wllm_b200.engine.request import RequestStatus
from wllm_b200.sampling import SamplingParams
from wllm_b200.sampling.params import sample_seed


def make(pages=24, **kw):
    runner = FakeRunner(pages)
    return runner, Scheduler(runner, ArgmaxSampler(), **kw)


def request(rid, prompt, prefix=None, max_tokens=4, **kw):
    return Request(rid, list(prompt), SamplingParams(max_tokens=max_tokens, ignore_eos=True, **kw), prefix=prefix)


def alone(prompt, max_tokens=4):
    _, s = make()
    r = request("x", prompt, max_tokens=max_tokens)
    s.add_request(r)
    s.run_to_completion()
    return r.output_token_ids


@pytest.mark.parametrize("length", [1, 3, 4, 5, 8, 11])
@pytest.mark.parametrize("budget", [None, 3])
@pytest.mark.parametrize("async_scheduling", [False, True])
def test_a_prefix_is_computed_once_and_changes_no_token(length, budget, async_scheduling):
    begin = [(5 * i) % 50 for i in range(length)]
    runner, s = make(chunked_prefill_tokens=budget, async_scheduling=async_scheduling)
    prefix = s.add_prefix(begin)
    assert not prefix.ready and s.has_unfinished()
    tails = [[7], [7, 9, 30], [1, 2, 3, 4, 5, 6]]
    reqs = [request(i, begin + t, prefix) for i, t in enumerate(tails)]
    for r in reqs:
        s.add_request(r)
    assert prefix.users == 3
    with pytest.raises(ValueError, match="unfinished"):
        s.drop_prefix(prefix)
    s.run_to_completion()
    assert prefix.ready and prefix.users == 0 and s.stats["prefill_tokens"] == length + sum(map(len, tails))
    assert [r.output_token_ids for r in reqs] == [alone(begin + t) for t in tails]
    assert runner.cache.free_pages() == [24 - -(-length // 4)]       # the prefix stays
    late = request("late", begin + [9, 9], prefix)
    s.add_request(late)
    s.run_to_completion()
    assert late.output_token_ids == alone(begin + [9, 9])
    s.drop_prefix(prefix)
    runner.cache.check()
    assert runner.cache.free_pages() == [24] and prefix.holder.status == RequestStatus.FINISHED
    for wrong in (lambda: s.drop_prefix(prefix), lambda: s.add_request(request("y", begin + [1], prefix))):
        with pytest.raises(ValueError, match="dropped"):
            wrong()


def test_prompts_that_do_not_begin_with_their_prefix_are_refused():
    _, s = make()
    prefix = s.add_prefix([1, 2, 3])
    for prompt in ([1, 2, 3], [1, 2], [1, 2, 4, 5], [9]):
        with pytest.raises(ValueError, match="begins with"):
            s.add_request(request("x", prompt, prefix))
    assert prefix.users == 0
    for bad in ([], [60], [1] * 64):
        with pytest.raises(ValueError):
            s.add_prefix(bad)
    assert len(s.prefixes) == 1 and len(s.waiting) == 1
    s.drop_prefix(prefix)
    assert not s.has_unfinished()


def test_prefixes_of_prefixes_and_those_made_for_a_few():
    runner, s = make()
    system = s.add_prefix([3, 1, 4, 1, 5])
    document = s.add_prefix([3, 1, 4, 1, 5, 9, 2, 6, 5], prefix=system, auto=True)
    reqs = [request(i, document.token_ids + [i], document) for i in range(3)] + [request(9, system.token_ids + [8], system)]
    for r in reqs:
        s.add_request(r)
    assert system.users == 2 and document.users == 3
    s.run_to_completion()
    assert [r.output_token_ids for r in reqs] == [alone(r.prompt_token_ids) for r in reqs]
    assert document.dropped and not system.dropped and system.users == 0 and s.prefixes == [system]
    s.drop_prefix(system)
    assert runner.cache.free_pages() == [24]


def test_cancelled_users_give_a_prefix_back():
    runner, s = make()
    prefix = s.add_prefix([3, 1, 4, 1, 5], auto=True)
    reqs = [request(i, prefix.token_ids + [i], prefix) for i in range(2)]
    for r in reqs:
        s.add_request(r)
    s.step()
    s.step()
    assert s.cancel(0) and not prefix.dropped and s.cancel(1) and prefix.dropped
    assert not s.cancel(("prefix", 0)) and runner.cache.free_pages() == [24] and not s.has_unfinished()
    # before it was computed
    prefix = s.add_prefix([3, 1, 4], auto=True)
    s.add_request(request("a", [3, 1, 4, 1], prefix))
    assert s.cancel("a") and prefix.dropped and not s.has_unfinished()


@pytest.mark.parametrize("admission", ["worst_case", "optimistic"])
def test_scarce_pages(admission):
    """Requests are admitted by what they need beside the prefix's full pages; preempted ones are forked again."""
    begin = list(range(18))                                           # 4 full pages of 4 and two tokens
    runner, s = make(pages=12, admission=admission)
    prefix = s.add_prefix(begin)
    reqs = [request(i, begin + [i], prefix, max_tokens=9) for i in range(5)]
    for r in reqs:
        s.add_request(r)                                              # 7 pages each at the end, 3 of their own; 5 are the prefix's
    most = 0
    while s.has_unfinished():
        s.step()
        runner.cache.check()
        most = max(most, len(s.live))
    assert most >= 2 and [r.output_token_ids for r in reqs] == [alone(r.prompt_token_ids, 9) for r in reqs]
    assert (s.stats["preemptions"] > 0) == (admission == "optimistic")
    with pytest.raises(ValueError, match="prefixes"):
        s.add_request(request("big", list(range(20)) + [1], max_tokens=20))     # 11 pages: more than the prefix leaves
    assert s.largest_need() == 5
    s.drop_prefix(prefix)
    assert runner.cache.free_pages() == [12] and s.largest_need() == 0


def test_slots_are_left_for_no_more_than_there_are():
    runner = FakeRunner(24, max_requests=3)
    s = Scheduler(runner, ArgmaxSampler())
    prefix = s.add_prefix([1, 2, 3, 4, 5])
    reqs = [request(i, prefix.token_ids + [i], prefix) for i in range(4)]
    for r in reqs:
        s.add_request(r)
    while s.has_unfinished():
        s.step()
        assert len(s.live) <= 2
    assert all(len(r.output_token_ids) == 4 for r in reqs)


def test_prefixes_leave_what_was_taken_on_its_pages_and_a_slot():
    """A request that was taken on can finish whatever prefixes come after it."""
    runner, s = make(pages=8)
    big = request("big", range(20), max_tokens=9)                     # 8 pages at the end
    s.add_request(big)
    for auto in (False, True):
        with pytest.raises(ValueError, match="pages"):
            s.add_prefix([1, 2, 3], auto=auto)
    s.step()
    with pytest.raises(ValueError, match="pages"):
        s.add_prefix([1])
    assert not s.prefixes
    s.run_to_completion()
    assert big.output_token_ids == alone(list(range(20)), 9)
    prefix = s.add_prefix(range(10))                                  # 3 pages, two of them full
    s.add_request(request("a", list(range(10)) + [1], prefix, max_tokens=16))      # 7 pages, 5 beside the prefix's
    with pytest.raises(ValueError, match="pages"):
        s.add_prefix([5])
    nested = s.prefix_refusal(12, prefix)
    assert nested and "pages" in nested
    s.run_to_completion()
    assert s.prefix_refusal(12, prefix) is None and s.prefix_refusal(4, None, 16) is None and "pages" in s.prefix_refusal(4, None, 25)
    runner = FakeRunner(24, max_requests=3)
    s = Scheduler(runner, ArgmaxSampler())
    kept = [s.add_prefix([i, 2, 3]) for i in range(2)]
    with pytest.raises(ValueError, match="none would be left"):
        s.add_prefix([9])
    r = request("r", kept[0].token_ids + [4], kept[0])
    s.add_request(r)
    s.run_to_completion()
    assert r.output_token_ids == alone(r.prompt_token_ids)


def test_samples_draw_from_seeds_of_their_own():
    seeds = [sample_seed(7, k) for k in range(100)]
    assert seeds[0] == 7 and len(set(seeds)) == 100 and all(0 <= x < 1 << 63 for x in seeds[1:])
    with pytest.raises(ValueError):
        SamplingParams(n=0)


def test_ids_that_callers_choose_meet_no_prefix():
    """Samples are named (id of the prompt, sample): also those of a prompt called "prefix" are nobody else."""
    runner, s = make()
    prefix = s.add_prefix([1, 2, 3, 4, 5], auto=True)
    reqs = [request(("prefix", k), prefix.token_ids + [7], prefix) for k in range(2)]
    for r in reqs:
        s.add_request(r)
    s.run_to_completion()
    assert [r.output_token_ids for r in reqs] == [alone(r.prompt_token_ids) for r in reqs]
    assert prefix.dropped and runner.cache.free_pages() == [24]


@pytest.mark.parametrize("name", ["fork", "open"])
def test_a_request_whose_cache_cannot_be_made_stays_in_the_queue(monkeypatch, name):
    runner, s = make()
    prefix = s.add_prefix([1, 2, 3, 4, 5], auto=True)
    r = request("r", prefix.token_ids + [7], prefix)
    s.add_request(r)
    s.step()
    if name == "open":
        s.add_request(request("first", [9], max_tokens=1))
    wrong, right = s.waiting[-1 if name == "open" else 0], getattr(runner.cache, name)
    s.waiting = [wrong] + [x for x in s.waiting if x is not wrong]

    def fail(*args, **kw):
        raise MemoryError("no copy")
    monkeypatch.setattr(runner.cache, name, fail)
    with pytest.raises(MemoryError):
        s.step()
    assert s.waiting[0] is wrong and wrong not in s.live and wrong.cache is None and prefix.users == 1
    monkeypatch.setattr(runner.cache, name, right)
    s.run_to_completion()
    assert r.output_token_ids == alone(r.prompt_token_ids) and prefix.dropped and runner.cache.free_pages() == [24]


def test_one_id_twice_is_run_one_behind_the_other():
    runner, s = make()
    pair = [request("same", [4, 9], max_tokens=3), request("same", [8], max_tokens=2)]
    for r in pair:
        s.add_request(r)
    s.run_to_completion()
    assert [r.output_token_ids for r in pair] == [alone([4, 9], 3), alone([8], 2)] and runner.cache.free_pages() == [24]


@pytest.mark.parametrize("admission", ["worst_case", "optimistic"])
@pytest.mark.parametrize("async_scheduling", [False, True])
def test_what_was_made_for_a_few_refuses_nothing_behind_them(admission, async_scheduling):
    """A request that would not fit beside the prompt of the samples in front of it fits when they are over, as it does when it is added first."""
    runner, s = make(pages=12, admission=admission, async_scheduling=async_scheduling)
    for turn in range(2):
        begin = [(7 * i + turn) % 50 for i in range(22)]              # 6 pages
        prefix = s.add_prefix(begin, auto=True)
        few = [request(("few", k), begin + [k], prefix, max_tokens=5) for k in range(3)]
        big = request("big", [(3 * i) % 50 for i in range(30)], max_tokens=14)      # 11 pages
        small = request("small", [5], max_tokens=3)
        for r in few + [big, small]:
            s.add_request(r)
        with pytest.raises(ValueError, match="pages"):                # what it would need beside what is kept now
            s.add_prefix([1] * 8)
        while s.has_unfinished():
            s.step()
            runner.cache.check()
        assert [r.output_token_ids for r in few + [big, small]] == [alone(r.prompt_token_ids, r.sampling.max_tokens) for r in few + [big, small]]
        assert prefix.dropped and runner.cache.free_pages() == [12]
    kept = s.add_prefix([1] * 8)                                      # one that is kept counts, and so does a request's own
    with pytest.raises(ValueError, match="for prefixes"):
        s.add_request(request("big", range(30), max_tokens=14))
    nested = s.add_prefix([1] * 30, prefix=kept, auto=True)
    with pytest.raises(ValueError, match="for prefixes"):
        s.add_request(request("own", [1] * 31, nested, max_tokens=14))          # 12 pages, 7 of them the prefix's, which has one more
    own = request("own", [1] * 31, nested, max_tokens=10)
    s.add_request(own)
    s.run_to_completion()
    assert own.output_token_ids == alone([1] * 31, 10) and nested.dropped


def samples_of(s, i, prompt, n, max_tokens):
    """n samples of a prompt, as the engine adds them: forks of all but its last token."""
    prefix = s.add_prefix(prompt[:-1], auto=True)
    reqs = [request((i, k), prompt, prefix, max_tokens=max_tokens) for k in range(n)]
    for r in reqs:
        s.add_request(r)
    return reqs


@pytest.mark.parametrize("budget", [None, 320])
def test_prompts_with_samples_are_taken_on_together(budget):
    """Sixteen prompts of four samples: their tokens in the first step, the samples from the second on; a request behind them runs in the first."""
    runner = FakeRunner(600, max_requests=100)
    s = Scheduler(runner, ArgmaxSampler(), chunked_prefill_tokens=budget)
    reqs = [r for i in range(16) for r in samples_of(s, i, [(i + 3 * j) % 50 for j in range(20)], 4, 8)]
    late = request("late", [9, 8, 7], max_tokens=8)
    s.add_request(late)
    s.step()
    assert s.stats["prefill_tokens"] == 16 * 19 + 3 and len(late.output_token_ids) == 1
    s.run_to_completion()
    assert s.stats["steps"] == 9
    assert all(r.output_token_ids == alone(r.prompt_token_ids, 8) for r in reqs + [late])
    # whoever can run is taken in the order of the queue
    first = [[rid for rid, _, _ in b] for b in runner.batches[1:2]][0]
    assert first == ["late"] + [(i, k) for i in range(16) for k in range(4)]


def test_who_waits_for_its_prefix_is_passed_only_by_those_that_fit_beside_it():
    runner, s = make(pages=16, chunked_prefill_tokens=8)
    few = samples_of(s, "few", [(7 * i) % 50 for i in range(30)], 2, 4)       # 29 tokens: 8 pages, for four steps
    big = request("big", [(3 * i) % 50 for i in range(30)], max_tokens=6)     # 9 pages: not beside those
    small = request("small", [5], max_tokens=3)
    for r in (big, small):
        s.add_request(r)
    s.step()
    assert [rid for rid, _, _ in runner.batches[0]] == [s.prefixes[0].holder.request_id] and not big.passed
    s.run_to_completion()
    assert all(r.output_token_ids == alone(r.prompt_token_ids, r.sampling.max_tokens) for r in few + [big, small])
    runner, s = make(pages=24, chunked_prefill_tokens=8)
    few = samples_of(s, "few", [(7 * i) % 50 for i in range(24)], 2, 4)
    small = request("small", [5], max_tokens=9)
    s.add_request(small)
    for _ in range(3):
        s.step()
    assert small.passed and len(small.output_token_ids) > 0 and not few[0].output_token_ids
    s.run_to_completion()
    assert all(r.output_token_ids == alone(r.prompt_token_ids, r.sampling.max_tokens) for r in few + [small])


@pytest.mark.parametrize("seed", range(12))
def test_any_mixture_comes_to_an_end(seed):
    """Prefixes that are kept, dropped or made for a few, requests with and without, cancelled ones, scarce pages and slots: everything that was taken on finishes with its own tokens."""
    import random
    rng = random.Random(seed)
    pages, slots = rng.randint(6, 30), rng.choice([3, 5, 8, 20])
    runner = FakeRunner(pages, max_requests=slots)
    s = Scheduler(runner, ArgmaxSampler(), chunked_prefill_tokens=rng.choice([None, 5, 16]), admission=rng.choice(["worst_case", "optimistic"]), async_scheduling=rng.random() < 0.5)
    reqs, kept, refused = [], [], 0
    for turn in range(60):
        for _ in range(rng.choice([0, 0, 1, 3])):
            begin = rng.choice(kept) if kept and rng.random() < 0.4 else None
            prompt = (begin.token_ids if begin else []) + [rng.randrange(50) for _ in range(rng.randint(1, 24))]
            most, what = rng.randint(1, 12), rng.random()
            try:
                if what < 0.3 and len(prompt) - (len(begin.token_ids) if begin else 0) > 1 and not s.prefix_refusal(len(prompt) - 1, begin, len(prompt) + most):
                    auto, made = s.add_prefix(prompt[:-1], prefix=begin, auto=True), []
                    for k in range(rng.randint(1, 4)):
                        made.append(request((turn, len(reqs) + k), prompt, auto, max_tokens=most))
                        s.add_request(made[-1])
                    reqs += made
                elif what < 0.45:
                    kept.append(s.add_prefix(prompt, prefix=begin))
                else:
                    r = request((turn, len(reqs)), prompt, begin, max_tokens=most)
                    s.add_request(r)
                    reqs.append(r)
            except ValueError:
                refused += 1
        for p in [p for p in kept if p.users == 0 and rng.random() < 0.1]:
            s.drop_prefix(p)
            kept.remove(p)
        if reqs and rng.random() < 0.1:
            s.cancel(rng.choice(reqs).request_id)
        if s.has_unfinished():
            s.step()
            runner.cache.check()
    s.run_to_completion(max_steps=4000)
    assert not s.has_unfinished() and all(r.finished for r in reqs)
    for r in reqs:
        if r.finish_reason != "cancelled":
            assert r.output_token_ids == alone(r.prompt_token_ids, r.sampling.max_tokens), r.request_id
    while any(not p.dropped for p in kept):
        for p in [p for p in kept if not p.dropped and p.users == 0]:
            s.drop_prefix(p)
    assert runner.cache.free_pages() == [pages] and runner.cache.slots.num_free == slots and not s.prefixes


@pytest.mark.parametrize("states,most", [((), 4), (("state",), 3)])
def test_prefixes_cost_requests_of_models_without_state_no_place(states, most):
    """Four samples of a prompt run at once where four requests do, beside the prompt; one request at a time may have a prefix."""
    import torch

    from wllm_b200.cache import CacheGroupSpec, CacheManager, StateSpec

    def scheduler(requests):
        runner = FakeRunner(40)
        runner.cache = CacheManager([CacheGroupSpec("all", 1, 1, 8)], 4, 40, requests, [StateSpec(n, (3,), torch.float32) for n in states], prefix_slots=requests)
        assert runner.cache.slots.num_free == requests
        return Scheduler(runner, ArgmaxSampler(), max_num_seqs=requests)
    s, live = scheduler(4), 0
    reqs = samples_of(s, 0, list(range(10)), 4, 6)
    while s.has_unfinished():
        s.step()
        live = max(live, len(s.live))
    assert live == most and all(r.output_token_ids == alone(r.prompt_token_ids, 6) for r in reqs) and s.cache.slots.num_free == 4
    assert (scheduler(1).prefix_refusal(5) is None) == (not states)


def test_adding_many_prompts_with_samples_is_no_work_of_its_own():
    """What the requests in the queue need beside each other's prompts is added up once a prompt, not prompt by prompt for every request: 64 and 128 prompts, in lines that the interpreter runs."""
    import sys

    def steps(prompts):
        s, count = Scheduler(FakeRunner(20000, max_requests=2000), ArgmaxSampler()), 0

        def trace(frame, event, arg):
            nonlocal count
            count += event == "line"
            return trace
        for i in range(prompts):
            if i == prompts - 1:
                sys.settrace(trace)
            try:
                assert not s.prefix_refusal(9, None, 14)
                samples_of(s, i, [(i + j) % 50 for j in range(10)], 4, 4)
            finally:
                sys.settrace(None)
        return count
    few, many = steps(64), steps(128)
    assert many < 3 * few                                             # (proportional to the queue; by every pair of a request and a prompt it would be four times)
