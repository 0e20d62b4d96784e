"""Prefixes and samples through the engine: what is computed and read once for several requests gives what each alone would get, to the last bit in 32 bits."""
import pytest
import torch

from wllm_b200 import LLM, SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def always(monkeypatch):
    """Shared pages are attended to once however few they are."""
    from wllm_b200.kernels import ops
    monkeypatch.setattr(ops, "PREFIX_SAVED", {2: 1, 4: 1})
    monkeypatch.setattr(ops, "PREFIX_PORTION", (1, 0.0))
    plan = ops.prefix_plan
    monkeypatch.setattr(ops, "prefix_plan", lambda *a, **k: plan(*a, **{**k, "min_keys": 1}))


def folders(tmp_path):
    import fusanex_configs
    import gudarax_configs
    import pesanex_configs
    import taritar_configs
    import vifirax_configs
    import zafilix_configs
    from helpers import make_folder
    return {"A": lambda: make_folder(tmp_path, "A"), "B": lambda: make_folder(tmp_path, "B"),
            "pesanex": lambda: pesanex_configs.write_folder(str(tmp_path / "p"), "mix"), "taritar": lambda: taritar_configs.write_folder(str(tmp_path / "t"), "wide"),
            "zafilix": lambda: zafilix_configs.write_folder(str(tmp_path / "z"), "heads64"), "gudarax": lambda: gudarax_configs.write_folder(str(tmp_path / "g"), "heads64"),
            "fusanex": lambda: fusanex_configs.write_folder(str(tmp_path / "f"), "heads64"), "vifirax": lambda: vifirax_configs.write_folder(str(tmp_path / "v"), "heads64")}


def tokens(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


# every architecture: pages of one and two sizes, windows, blocks, latent rows, recurrent state of every kind
@pytest.mark.parametrize("name", ["A", "B", "pesanex", "taritar", "zafilix", "gudarax", "fusanex", "vifirax"])
def test_samples_are_what_each_alone_would_draw(tmp_path, always, name):
    folder = folders(tmp_path)[name]()
    kw = dict(dtype="float32", block_size=16, num_blocks=96, chunked_prefill_tokens=40)
    llm = LLM(folder, poison_pages=True, **kw)
    vocab = llm.model.plan.vocab_size
    prompts = [tokens(75, vocab, 1), tokens(1, vocab, 2), tokens(17, vocab, 3)]
    sp = SamplingParams(temperature=0.9, seed=11, max_tokens=9, ignore_eos=True)
    outs = llm.generate(prompts, SamplingParams(temperature=0.9, seed=11, max_tokens=9, ignore_eos=True, n=4))
    assert [(o.request_id, o.sample) for o in outs] == [((i, k), k) for i in range(3) for k in range(4)]
    assert (llm.runner.prefix_steps > 0) == bool(llm.runner.prefix_layouts) and llm.runner.cache.free_pages() == [96] * len(llm.runner.cache.groups)
    from dataclasses import replace
    from wllm_b200.sampling.params import sample_seed
    plain = LLM(folder, **kw)
    for i, p in enumerate(prompts):
        for k in range(4):
            want = plain.generate([p], replace(sp, seed=sample_seed(11, k)))[0]
            got = outs[4 * i + k]
            # The logits are the same bits; the sampler adds up a row's exponentials in 32 pieces where a step samples more than eight rows and in 64 else, each a chain of at most
            # 32 additions and then a chain of the pieces: (32 + 64) x 2^-24 of the sum on either side, as much in its logarithm, and half a step of a number below 16.
            assert got.token_ids == want.token_ids, (name, i, k)
            assert all(abs(a - b) <= 2 * 96 * 2.0 ** -24 + 2.0 ** -20 for a, b in zip(got.logprobs, want.logprobs)), (name, i, k)
    assert plain.runner.prefix_steps == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs,asynchronous", [(False, False), (True, False), (True, True)])
def test_prompts_behind_a_prefix(tmp_path, always, dtype, graphs, asynchronous):
    folder = folders(tmp_path)["A"]()
    kw = dict(dtype=dtype, block_size=16, num_blocks=80, chunked_prefill_tokens=64, cuda_graphs=graphs, async_scheduling=asynchronous)
    llm, plain = LLM(folder, poison_pages=True, **kw), LLM(folder, **kw)
    vocab = llm.model.plan.vocab_size
    begin, tails = tokens(150, vocab, 5), [tokens(n, vocab, 10 + n) for n in (1, 2, 3, 14, 40)]
    sp = SamplingParams(max_tokens=12, ignore_eos=True)
    prefix = llm.add_prefix(begin)
    outs = llm.generate(tails, sp, prefix=prefix)
    assert llm.runner.prefix_steps > 5
    computed = llm.stats["prefill_tokens"]
    assert computed == 150 + sum(map(len, tails))
    wants = plain.generate([begin + t for t in tails], sp)
    for got, want in zip(outs, wants):
        assert got.prompt_token_ids == want.prompt_token_ids
        if dtype == "float32":
            assert got.token_ids == want.token_ids and got.logprobs == want.logprobs
        else:                                                    # up to the first place where a near-tie went the other way
            same = next((i for i, (a, b) in enumerate(zip(got.token_ids, want.token_ids)) if a != b), len(want.token_ids))
            assert all(abs(a - b) < 2e-2 for a, b in zip(got.logprobs[:same + 1], want.logprobs[:same + 1]))
    llm.resize_cache(30)                                         # the prefix moves with the cache
    again = llm.generate(tails[:2], sp, prefix=prefix)
    if dtype == "float32":
        assert [o.token_ids for o in again] == [o.token_ids for o in outs[:2]]
    with pytest.raises(ValueError):
        llm.resize_cache(9)
    llm.drop_prefix(prefix)
    assert llm.runner.cache.free_pages() == [30] * len(llm.runner.cache.groups)


def test_scarce_pages_and_preemption_with_forks(tmp_path, always):
    folder = folders(tmp_path)["A"]()
    llm = LLM(folder, dtype="float32", block_size=16, num_blocks=14, admission="optimistic", poison_pages=True, cuda_graphs=True)
    begin = tokens(70, llm.model.plan.vocab_size, 3)
    prefix = llm.add_prefix(begin)
    sp = SamplingParams(max_tokens=40, ignore_eos=True)
    tails = [tokens(5, llm.model.plan.vocab_size, 20 + i) for i in range(5)]
    outs = llm.generate(tails, sp, prefix=prefix)
    assert sum(o.preemptions for o in outs) > 0
    plain = LLM(folder, dtype="float32", block_size=16, num_blocks=80)
    assert [o.token_ids for o in outs] == [o.token_ids for o in plain.generate([begin + t for t in tails], sp)]


def test_captured_steps_of_changing_batches(tmp_path, always):
    """Batches with and without shared pages in turn, of sizes that one capture serves, beside requests that share nothing."""
    folder = folders(tmp_path)["B"]()
    llm, plain = (LLM(folder, dtype="float32", block_size=16, num_blocks=120, cuda_graphs=g) for g in (True, False))
    vocab = llm.model.plan.vocab_size
    sp = SamplingParams(max_tokens=10, ignore_eos=True)
    for turn in range(3):
        alone = [tokens(20 + turn, vocab, turn), tokens(7, vocab, 50 + turn)]
        begin = tokens(48 + 16 * turn, vocab, 90 + turn)
        prefix = llm.add_prefix(begin)
        reqs = [llm.add_request(a, sp) for a in alone] + [llm.add_request([turn + i], sp, prefix=prefix) for i in range(3 + turn)]
        llm.scheduler.run_to_completion()
        llm.drop_prefix(prefix)
        want = plain.generate([r.prompt_token_ids for r in reqs], sp)
        assert [r.output_token_ids for r in reqs] == [o.token_ids for o in want]
    assert llm.runner._graphs and llm.runner._prefix_graphs
    assert all(rec["meta"] is llm.runner._meta for g in (llm.runner._graphs, llm.runner._prefix_graphs) for rec in g.values())


def test_samples_without_room_for_their_prompt_beside_them(tmp_path):
    """Three pages hold a request to its end, but not the prompt that its samples would share beside one of them; nor are there slots for all prompts of a batch."""
    folder = folders(tmp_path)["A"]()
    kw = dict(dtype="float32", block_size=16, max_num_seqs=3)
    sp = SamplingParams(max_tokens=8, ignore_eos=True, temperature=0.8, seed=5, n=3)
    for blocks, lengths in ((3, (40,)), (40, (20, 33, 17, 40))):
        llm, roomy = LLM(folder, num_blocks=blocks, **kw), LLM(folder, dtype="float32", block_size=16, num_blocks=80)
        prompts = [tokens(n, llm.model.plan.vocab_size, n) for n in lengths]
        assert [o.token_ids for o in llm.generate(prompts, sp)] == [o.token_ids for o in roomy.generate(prompts, sp)]
        assert llm.runner.cache.free_pages() == [blocks] * len(llm.runner.cache.groups) and not llm.scheduler.prefixes


@pytest.mark.parametrize("name,asynchronous", [("A", False), ("A", True), ("gudarax", False), ("zafilix", False)])
def test_another_size_of_the_cache_and_new_requests_between_steps(tmp_path, always, name, asynchronous):
    """The cache grows and shrinks while requests decode and a prefix is half computed; requests come, are cancelled and begin with prefixes between steps."""
    folder = folders(tmp_path)[name]()
    kw = dict(dtype="float32", block_size=16, chunked_prefill_tokens=24)
    llm, plain = LLM(folder, num_blocks=40, cuda_graphs=True, async_scheduling=asynchronous, poison_pages=True, **kw), LLM(folder, num_blocks=96, **kw)
    vocab = llm.model.plan.vocab_size
    sp = SamplingParams(max_tokens=14, ignore_eos=True)
    first = [llm.add_request(tokens(20 + 9 * i, vocab, i), sp) for i in range(2)]
    for _ in range(5):
        llm.step()
    prefix = llm.add_prefix(tokens(50, vocab, 7))
    behind = [llm.add_request(tokens(1 + 6 * i, vocab, 20 + i), sp, prefix=prefix) for i in range(3)]
    gone = llm.add_request(tokens(9, vocab, 40), sp, prefix=prefix)
    llm.step()
    llm.resize_cache(64)
    for _ in range(6):
        llm.step()
    assert llm.scheduler.cancel(gone.request_id)
    llm.resize_cache(36)
    llm.step()
    late = llm.add_request(tokens(4, vocab, 30), SamplingParams(max_tokens=14, ignore_eos=True, n=2, seed=3, temperature=0.7), prefix=prefix)
    llm.step()
    llm.resize_cache(50)
    llm.scheduler.run_to_completion()
    llm.runner.cache.check()
    for r in first + behind:
        assert r.output_token_ids == plain.generate([r.prompt_token_ids], sp)[0].token_ids
    want = plain.generate([late[0].prompt_token_ids], SamplingParams(max_tokens=14, ignore_eos=True, n=2, seed=3, temperature=0.7))
    assert [r.output_token_ids for r in late] == [o.token_ids for o in want]
    llm.drop_prefix(prefix)
    assert llm.runner.cache.free_pages() == [50] * len(llm.runner.cache.groups) and not llm.scheduler.prefixes


def test_the_command(tmp_path, capsys):
    import json

    from wllm_b200.cli import main
    folder = folders(tmp_path)["A"]()
    assert main(["--model", folder, "--dtype", "float32", "--prefix-ids", "2,7,9,4,4", "--prompt-ids", "5", "--prompt-ids", "6,8", "--n", "2", "--max-tokens", "3", "--ignore-eos",
                 "--log-level", "ERROR"]) == 0
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert [(x["request"], x["sample"], x["prompt_tokens"]) for x in lines] == [([0, 0], 0, 6), ([0, 1], 1, 6), ([1, 0], 0, 7), ([1, 1], 1, 7)]
    llm = LLM(folder, dtype="float32")
    want = llm.generate([[2, 7, 9, 4, 4, 5], [2, 7, 9, 4, 4, 6, 8]], SamplingParams(max_tokens=3, ignore_eos=True))
    assert [x["token_ids"] for x in lines] == [want[0].token_ids] * 2 + [want[1].token_ids] * 2
