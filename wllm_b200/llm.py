"""The Python entry point: token ids in, generated token ids out.

    llm = LLM("/path/to/model", dtype="bfloat16", num_blocks=4096, chunked_prefill_tokens=2048)
    outs = llm.generate([[2, 651, 6037]], SamplingParams(temperature=0.8, seed=1, max_tokens=32))

The reference has no single class for offline use; it is assembled by hand from
load_native, KVCacheManager, Scheduler, add_request and run_to_completion
(tests/test_gemma_architecture.py:119-124).  `LLM` wraps that assembly, with the
reference's option names: num_blocks, block_size, dtype, chunked_prefill_tokens,
cuda_graphs (src/wllm/cli.py:30-35).  `add_request` / `step` expose the loop itself.

What several requests begin with is computed once, and attended to once a step for all of them:

    system = llm.add_prefix([2, 651, 6037, ...])
    outs = llm.generate([[108, 17], [99]], SamplingParams(max_tokens=32), prefix=system)   # prompts behind the prefix
    outs = llm.generate([[2, 651, 6037]], SamplingParams(temperature=0.8, n=4))            # four samples of one prompt
    llm.drop_prefix(system)
"""
from __future__ import annotations

from dataclasses import dataclass, replace

from .config import EngineConfig
from .engine.build import build_model, build_runner
from .engine.request import Prefix, Request
from .engine.scheduler import Scheduler
from .sampling import SamplingParams
from .sampling.params import sample_seed
from .sampling.sampler import Sampler


@dataclass
class RequestOutput:
    request_id: object
    prompt_token_ids: list
    token_ids: list
    logprobs: list
    finish_reason: str | None
    preemptions: int = 0
    sample: int = 0               # which of its prompt's n samples it is


class LLM:
    def __init__(self, model: str | None = None, *, config=None, random_seed: int | None = None,
                 dtype="bfloat16", block_size: int = 16, num_blocks: int = 256,
                 chunked_prefill_tokens: int | None = None, max_num_seqs: int = 256, max_model_len: int | None = None,
                 cuda_graphs: bool = False, device: str = "cuda:0", admission: str = "worst_case", seed: int = 0,
                 async_scheduling: bool = False, poison_pages: bool = False, prefill_row_quantum: int | None = None):
        """`model`: a folder with config.json and model.safetensors.  Without it, `config` (a typed
        configuration) and `random_seed` make a model with random weights on the device."""
        self.engine_config = EngineConfig(dtype=dtype, block_size=block_size, num_blocks=num_blocks,
                                          chunked_prefill_tokens=chunked_prefill_tokens, max_num_seqs=max_num_seqs,
                                          max_model_len=max_model_len, cuda_graphs=cuda_graphs, device=device,
                                          poison_pages=poison_pages, prefill_row_quantum=prefill_row_quantum)
        ec = self.engine_config
        self.model = build_model(model, ec.dtype, ec.device, config=config, random_seed=random_seed)
        self.runner = build_runner(self.model, ec, poison_pages=ec.poison_pages)
        if cuda_graphs:
            self.runner.enable_graphs()
        self.sampler = Sampler(ec.device)
        self.scheduler = Scheduler(self.runner, self.sampler, chunked_prefill_tokens=chunked_prefill_tokens,
                                   max_num_seqs=max_num_seqs, max_model_len=max_model_len, admission=admission, seed=seed,
                                   async_scheduling=async_scheduling, row_quantum=ec.prefill_row_quantum)
        self.eos_token_id = self.model.plan.eos_token_id
        self._next_id = 0

    def add_prefix(self, token_ids) -> Prefix:
        """Tokens for requests to begin with (a system prompt, a document): computed once, by the steps to come, and kept until they are dropped.  It takes pages, and in a model with state of every
        request the place of one of `max_num_seqs`, of which one is left; what could not be kept beside the requests at hand is refused."""
        return self.scheduler.add_prefix(token_ids)

    def drop_prefix(self, prefix: Prefix) -> None:
        """Give a prefix's pages back; every request that begins with it has finished."""
        self.scheduler.drop_prefix(prefix)

    def resize_cache(self, num_blocks: int) -> None:
        """Another number of cache blocks: what is live moves to the front of the new pools.  Refused where a request that was taken on could not finish (ValueError), or what is
        live now holds more (OutOfPages); everything is as it was then."""
        need = self.scheduler.largest_need()
        if need > num_blocks:
            raise ValueError(f"{num_blocks} blocks: the requests and prefixes at hand need {need}")
        self.runner.resize_cache(num_blocks)
        self.engine_config.num_blocks = num_blocks

    def add_request(self, prompt_token_ids, sampling_params: SamplingParams | None = None, request_id=None, prefix: Prefix | None = None):
        """`prefix`: what the prompt begins with; `prompt_token_ids` are the tokens behind it.  The request, or with n > 1 the list of its n samples' requests, whose
        ids are (request_id, sample)."""
        if request_id is None:
            request_id = self._next_id
            self._next_id += 1
        sp = sampling_params or SamplingParams()
        prompt = (list(prefix.token_ids) if prefix is not None else []) + list(prompt_token_ids)
        if sp.n == 1:
            return self._add(request_id, prompt, sp, prefix)
        begin = prefix
        if len(prompt) > 1 + (len(prefix.token_ids) if prefix is not None else 0) and not self.scheduler.prefix_refusal(len(prompt) - 1, prefix, len(prompt) + sp.max_tokens):
            # the samples are forks of the prompt without its last token, which each of them runs for its own first draw; a prompt that cannot be kept beside them is computed by each
            begin = self.scheduler.add_prefix(prompt[:-1], prefix=prefix, auto=True)
        one = [replace(sp, n=1, seed=None if sp.seed is None else sample_seed(sp.seed, k)) for k in range(sp.n)]
        made = []
        try:
            for k in range(sp.n):
                made.append(self._add((request_id, k), prompt, one[k], begin))
        except BaseException:
            for r in made:
                self.scheduler.cancel(r.request_id)
            if begin is not prefix and not made:
                self.scheduler.drop_prefix(begin)
            raise
        return made

    def _add(self, request_id, prompt: list, sampling: SamplingParams, prefix) -> Request:
        req = Request(request_id, prompt, sampling, eos_token_id=self.eos_token_id, prefix=prefix)
        self.scheduler.add_request(req)
        return req

    def step(self) -> list:
        """One scheduler step; returns the requests that got a token (with `async_scheduling`: the tokens of
        the step before, read while this one runs)."""
        return self.scheduler.step()

    def has_unfinished(self) -> bool:
        return self.scheduler.has_unfinished()

    def generate(self, prompts, sampling_params=None, prefix: Prefix | None = None) -> list:
        """Generate for a batch of prompts (lists of token ids); results in the order of the prompts, a prompt's n samples one behind the other.  `prefix`: what all of them
        begin with; the prompts are the tokens behind it."""
        prompts = [list(p) for p in prompts]
        if sampling_params is None or isinstance(sampling_params, SamplingParams):
            sampling_params = [sampling_params or SamplingParams()] * len(prompts)
        if len(sampling_params) != len(prompts):
            raise ValueError("one SamplingParams for all prompts, or one per prompt")
        reqs = []
        for p, sp in zip(prompts, sampling_params):
            made = self.add_request(p, sp, prefix=prefix)
            reqs += enumerate(made) if isinstance(made, list) else [(0, made)]
        self.scheduler.run_to_completion()
        return [RequestOutput(r.request_id, r.prompt_token_ids, list(r.output_token_ids), list(r.logprobs),
                              r.finish_reason, r.preemptions, sample) for sample, r in reqs]

    @property
    def stats(self) -> dict:
        s = dict(self.scheduler.stats)
        s["pages_high_water"] = list(self.runner.cache.pages_high_water)
        return s
