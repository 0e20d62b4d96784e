"""Prefixes in the engine beside what else is in it: when their kernels are built, what the requests' places are, whom a step's plan takes."""
import pytest
import torch

from test_gpu_prefixes import always, folders, tokens  # noqa: F401
from wllm_b200 import LLM, SamplingParams

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_no_step_waits_for_a_compiler(tmp_path, always, monkeypatch, dtype):  # noqa: F811
    """The kernels of a model's head sizes are there when it is loaded."""
    from wllm_b200.kernels import ops
    bound, bind = [], ops._bind
    ops._host_calls()
    monkeypatch.setattr(ops, "_bind", lambda what: (bound.append(what), bind(what))[1])
    llm = LLM(folders(tmp_path)["A"](), dtype=dtype, block_size=16, num_blocks=80)
    (_, _, _, hd, vd), = llm.runner.prefix_layouts
    assert ((hd, vd) in bound) == (dtype == "bfloat16")
    bound.clear()
    prefix = llm.add_prefix(tokens(70, llm.model.plan.vocab_size, 1))
    llm.generate([[1], [2], [3]], SamplingParams(max_tokens=4, ignore_eos=True), prefix=prefix)
    assert llm.runner.prefix_steps > 0 and (hd, vd) not in bound


def test_places_of_requests_beside_prefixes(tmp_path):
    """One request at a time, and four samples at once where four requests run at once: tokens as without a prefix."""
    folder = folders(tmp_path)["A"]()
    kw = dict(dtype="float32", block_size=16, num_blocks=80)
    plain = LLM(folder, **kw)
    vocab = plain.model.plan.vocab_size
    begin, tails = tokens(40, vocab, 3), [tokens(3, vocab, 4), tokens(9, vocab, 5)]
    sp = SamplingParams(max_tokens=6, ignore_eos=True)
    llm = LLM(folder, max_num_seqs=1, **kw)
    outs = llm.generate(tails, sp, prefix=llm.add_prefix(begin))
    assert [o.token_ids for o in outs] == [o.token_ids for o in plain.generate([begin + t for t in tails], sp)]
    llm, live = LLM(folder, max_num_seqs=4, **kw), 0
    reqs = llm.add_request(begin, SamplingParams(max_tokens=6, ignore_eos=True, temperature=0.9, seed=2, n=4))
    while llm.has_unfinished():
        llm.step()
        live = max(live, len(llm.scheduler.live))
    assert live == 4 and len({tuple(r.output_token_ids) for r in reqs}) > 1
