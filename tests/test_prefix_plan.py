"""The plan of attention over shared prefixes, on the host: every (token, key) that is to be seen stands in exactly one item, results are listed in the order of their keys."""
import random

import numpy as np
import pytest
import torch

from prefix_refs import Batch
from wllm_b200.kernels import ops

HEADER = 16


def parts(plan):
    h = plan.host.numpy()
    items = h[h[2]:h[2] + 8 * h[0]].reshape(-1, 8)
    tokens = h[h[3]:].copy()
    starts = h[h[4]:h[4] + h[1] + 1]
    listed = h[h[5]:h[5] + starts[-1]]
    positions = h[h[6]:h[6] + h[1]]
    return items, tokens, starts, listed, positions


def check(plan, tables, q_lens, ctx_lens, ps, rep, tile_rows, align):
    items, tokens, starts, listed, positions = parts(plan)
    n = sum(q_lens)
    owner = [r for r, q in enumerate(q_lens) for _ in range(q)]
    pos = [c - q + t for q, c in zip(q_lens, ctx_lens) for t in range(q)]
    assert positions.tolist() == pos
    seen = [np.zeros(p + 1, dtype=np.int32) for p in pos]
    rows = {}
    for first, count, lo, hi, request, own, row, _ in items.tolist():
        assert 0 < count * rep <= tile_rows and lo < hi and lo % align == 0 and (own or hi % align == 0)
        for i in range(count):
            token, at = tokens[2 * (first + i)], tokens[2 * (first + i) + 1]
            assert at == pos[token] and (own or hi <= at - 0) and (not own or owner[token] == request)
            top = min(hi, at + 1)
            if top > lo:
                seen[token][lo:top] += 1
            pages = range(lo // ps, -(-hi // ps))
            assert all(tables[request][p] == tables[owner[token]][p] for p in pages)     # the item's keys are the token's own
            keys = 64 if tile_rows == 32 else 128
            costs = ops._prefix_costs(torch.float32 if tile_rows == 32 else torch.bfloat16, 8, 8)
            for side in range(costs[6] if count * rep <= costs[4] and hi - lo > keys else 1):
                key = row + (side * count + i) * rep
                assert key not in rows and key + rep <= plan.rows
                rows[key] = (token, lo)
    assert all((s == 1).all() for s in seen)
    assert len(rows) == len(listed) and starts[0] == 0
    for t in range(n):
        mine = [rows[int(k)] for k in listed[starts[t]:starts[t + 1]]]
        assert mine and all(m[0] == t for m in mine) and [m[1] for m in mine] == sorted(m[1] for m in mine)
    taken = sorted(rows)
    assert all(b - a >= rep for a, b in zip(taken, taken[1:]))
    costs = ops._prefix_costs(torch.float32 if tile_rows == 32 else torch.bfloat16, 8, 8)
    keys = 64 if tile_rows == 32 else 128
    dear = [-(-int(i[3] - i[2]) // keys) * costs[2 if i[1] * rep <= costs[4] else 0] for i in items]
    assert dear == sorted(dear, reverse=True)
    for first, count, *_, begins in items.tolist():
        mine = [int(tokens[2 * (first + i)]) for i in range(count)]
        assert begins == (mine[0] if mine == list(range(mine[0], mine[0] + count)) else -1)


TREES = [
    (0, [(5, 1)]),                                                        # one request, nothing shared
    (0, [(0, 1), (0, 1)]),                                                # first tokens
    (512, [(3, 1), (0, 1), (40, 1)]),                                     # a prefix, one right behind it
    (256, [(512, [(1, 1), (17, 3), (0, 9)]), (1024, [(5, 1)] * 30), (70, 1)]),      # two levels, a branch that ends early
    (1024, [(0, 40), (33, 1)] * 9),                                       # portions beside decoded tokens
    (64, [(200, 1)] * 3),                                                 # too short to share
    (0, [(512, [(0, 1)] * 5), (512, [(7, 2)] * 5), (99, 1)]),             # several prompts
    (128, [(128, [(128, [(128, [(3, 1), (2, 1)]), (2, 1)]), (1, 1)]), (0, 1)]),     # a chain of forks
    (16384, [(100, 1)] * 20),
]


@pytest.mark.parametrize("tree", TREES)
@pytest.mark.parametrize("nq,nkv,dtype", [(8, 1, torch.bfloat16), (7, 1, torch.bfloat16), (4, 4, torch.bfloat16), (6, 2, torch.float32), (32, 1, torch.float32), (128, 1, torch.bfloat16)])
@pytest.mark.parametrize("ps", [16, 64])
def test_every_key_stands_in_one_item(tree, nq, nkv, dtype, ps):
    if tree[0] > 4000 and nq > 8:
        tree = (1024, tree[1])
    b = Batch(tree, nq, nkv, 8, 8, ps)
    plan = ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, ps, nq, nkv, 8, 8, dtype)
    assert plan.n_tokens == b.n
    bf16 = dtype == torch.bfloat16
    check(plan, b.table.tolist(), b.q_lens, b.ctx_lens, ps, nq // nkv, ops.prefix_rows(dtype), 1 if bf16 else 64)


def test_shared_keys_are_counted_once_for_all():
    b = Batch((1024, [(256, [(3, 1), (4, 1)]), (9, 1)]), 4, 1, 8, 8, 64)
    plan = ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, 64, 4, 1, 8)
    assert plan.saved_keys == 2 * 1024 + 256
    assert ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, 64, 4, 1, 8, min_keys=300).saved_keys == 2 * 1024
    assert ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, 64, 4, 1, 8, min_keys=2000).saved_keys == 0
    # a page that new tokens are written to is nobody else's, whatever the table says: only the keys in front of every new token are shared
    table = np.array([[3, 4, 5], [3, 4, 5]], dtype=np.int32)
    plan = ops.prefix_plan(table, [1, 70], [140, 190], 64, 4, 1, 8, min_keys=1)
    assert plan.saved_keys == 64


def test_requests_that_bring_nothing_and_empty_batches():
    table = np.array([[3, 4], [-1, -1], [3, 9]], dtype=np.int32)
    plan = ops.prefix_plan(table, [1, 0, 2], [70, 0, 71], 64, 4, 2, 8, min_keys=64)
    check(plan, table.tolist(), [1, 0, 2], [70, 0, 71], 64, 2, 128, 1)
    empty = ops.prefix_plan(np.zeros((2, 3), dtype=np.int32), [0, 0], [0, 5], 64, 4, 2, 8)
    assert empty.n_tokens == empty.items == empty.rows == 0
    none = ops.prefix_plan(np.zeros((0, 3), dtype=np.int32), [], [], 64, 4, 2, 8)
    assert none.items == 0


def test_refusals():
    table = np.array([[3, 4], [3, 9]], dtype=np.int32)
    good = dict(tables=table, q_lens=[1, 2], ctx_lens=[70, 71], page_size=64, nq=4, nkv=2, hd=8)
    ops.prefix_plan(**good)
    for wrong in (dict(q_lens=[1]), dict(q_lens=[-1, 2]), dict(q_lens=[71, 2]), dict(ctx_lens=[129, 71]), dict(tables=np.array([[3, -1], [3, 9]], dtype=np.int32)),
                  dict(tables=table.astype(np.int64)), dict(tables=table[0]), dict(nq=5), dict(nq=512), dict(hd=12), dict(hd=264), dict(vd=0), dict(page_size=8), dict(page_size=48),
                  dict(caps=(0, 8, 8, 8)), dict(caps=(8, 8, 8, -1)), dict(caps=(8, 8, 8)), dict(dtype=torch.float16), dict(dtype=torch.float32, nq=128), dict(ctx_lens=[0, 71]), dict(q_lens=[1.0, 2.0])):
        with pytest.raises(ops.KernelError):
            ops.prefix_plan(**{**good, **wrong})


def test_when_sharing_pays():
    pays = lambda saved, dtype=torch.bfloat16, nkv=1, **kw: ops.prefix_pays(saved, nkv, 256, 256, dtype, **kw)  # noqa: E731
    assert pays(24 << 10) and not pays((24 << 10) - 1) and pays(128, torch.float32) and not pays(127, torch.float32)
    assert pays(3 * 512, holders=4, tokens=1.5) and not pays(3 * 512 - 1, holders=4, tokens=1.5)
    assert not pays(3 * 512, nkv=16, holders=4, tokens=100) and pays(3 * 1120, nkv=16, holders=4, tokens=100)
    assert not pays(0, holders=1, tokens=2) and not pays(0)


def test_a_long_chain_of_branchings():
    """Every request leaves the others one page after the last: the plan follows some hundred of them and is right for all."""
    n = 400
    table = np.array([[j if j < r else 1000 + r * n + j for j in range(n)] for r in range(n)], dtype=np.int32)
    ctx = [16 * (r + 1) + 1 if r + 1 < n else 16 * n for r in range(n)]
    plan = ops.prefix_plan(table, [1] * n, ctx, 16, 1, 1, 8, min_keys=1)
    assert plan.saved_keys > 0
    check(plan, table.tolist(), [1] * n, ctx, 16, 1, 128, 1)


def test_a_plan_laid_out_for_more_than_the_batch_has():
    b = Batch((512, [(3, 1), (0, 1), (40, 1)]), 4, 1, 8, 8, 64)
    for dtype in (torch.bfloat16, torch.float32):
        plan = ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, 64, 4, 1, 8, 8, dtype, caps=(64, 64, 128, 9))
        items, tokens, starts, listed, _ = parts(plan)
        h = plan.host.numpy()
        assert plan.n_tokens == 9 and h[h[4]:h[4] + 10].tolist() == starts.tolist() + [starts[-1]] * 6 and h[h[6]:h[6] + 9].tolist() == [c - 1 for c in b.ctx_lens] + [-1] * 6
        for caps in ((1, 64, 128, 9), (64, 1, 128, 9), (64, 64, 1, 9), (64, 64, 128, 2)):
            assert ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, 64, 4, 1, 8, 8, dtype, caps=caps) is None


@pytest.mark.parametrize("seed", range(8))
def test_random_trees(seed):
    rng = random.Random(seed)
    ps = rng.choice([16, 32, 128])

    def node(depth):
        if depth == 0 or rng.random() < 0.4:
            return (rng.randint(0, 300), rng.choice([1, 1, 1, rng.randint(2, 90)]))
        return (ps * rng.randint(0, 900 // ps), [node(depth - 1) for _ in range(rng.randint(1, 6))])
    b = Batch((0, [node(3) for _ in range(4)]), 1, 1, 8, 8, ps, seed)
    nkv, rep = rng.choice([1, 3]), rng.choice([1, 2, 5, 16])
    for dtype in (torch.bfloat16, torch.float32):
        plan = ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, ps, nkv * rep, nkv, 8, 8, dtype, min_keys=rng.choice([1, 64, 128]))
        bf16 = dtype == torch.bfloat16
        check(plan, b.table.tolist(), b.q_lens, b.ctx_lens, ps, rep, ops.prefix_rows(dtype), 1 if bf16 else 64)


@pytest.mark.parametrize("nq,nkv,hd,vd,shared", [(8, 1, 256, 256, True), (6, 2, 48, 48, True), (16, 4, 128, 64, False), (4, 2, 72, 72, False), (6, 2, 72, 40, False), (4, 2, 20, 20, False)])
def test_bfloat16_layers_with_32_bit_weights_are_not_planned(nq, nkv, hd, vd, shared):
    """Layers whose other kernels weigh values in 32 bits (values of a size of their own, head sizes that are no multiple of 16) keep them whoever shares pages beside a request."""
    from wllm_b200.parts import MIXERS, spec
    make = lambda dtype, **kw: MIXERS.build(spec("attention", num_heads=nq, num_kv_heads=nkv, head_dim=hd, value_dim=vd, position=spec("rope", theta=1e4, head_dim=hd), q_proj="q",  # noqa: E731
                                                 k_proj="k", v_proj="v", o_proj="o", **kw), hidden_size=64, model_dtype=dtype)
    held = [nq, nkv, -(-hd // 8) * 8, -(-vd // 8) * 8]
    assert make(torch.bfloat16).prefix_layout(16) == (tuple(held) if shared else None)
    assert make(torch.float32).prefix_layout(16) == tuple(held)
    assert make(torch.float32, window=8).prefix_layout(16) is None and make(torch.bfloat16).prefix_layout(24) is None


def step(sharers, others, fresh=0):
    """(tables, new tokens, contexts, who shares): (count, new tokens, shared keys), (count, context), a whole prompt of its own; pages of 64."""
    (count, new, shared), (more, ctx) = sharers, others
    reqs = [(new, shared + 20 + new + 7 * i, shared) for i in range(count)] + [(1, ctx + 13 * (i % 29), 0) for i in range(more)] + ([(fresh, fresh, 0)] if fresh else [])
    free = iter(range(shared // 64, 10 ** 6))
    table = np.full((len(reqs), -(-max(c for _, c, _ in reqs) // 64)), -1, dtype=np.int32)
    for r, (_, c, s) in enumerate(reqs):
        mine = list(range(s // 64)) + [next(free) for _ in range(-(-c // 64) - s // 64)]
        table[r, :len(mine)] = mine
    return table, [n for n, _, _ in reqs], [c for _, c, _ in reqs], [s > 0 for _, _, s in reqs]


F32, B16 = torch.float32, torch.bfloat16
# steps that were timed both ways, with the faster one: (heads, kv heads, size, type), sharers, others, a fresh prompt
TIMED = [((8, 1, 256, B16), (2, 16, 576), (0, 0), 2048, False), ((8, 1, 256, B16), (2, 1, 576), (62, 3000), 2048, False), ((16, 16, 256, B16), (2, 1, 576), (62, 3000), 2048, False),
         ((16, 16, 256, B16), (16, 1, 1024), (62, 3000), 0, False), ((16, 16, 256, B16), (16, 1, 8192), (62, 3000), 0, True), ((8, 1, 256, B16), (16, 16, 1024), (16, 1000), 2048, True),
         ((8, 1, 256, B16), (2, 1, 576), (0, 0), 256, True), ((16, 4, 128, B16), (2, 1, 576), (62, 3000), 2048, True), ((16, 16, 256, F32), (2, 1, 256), (62, 3000), 0, False),
         ((16, 16, 256, F32), (16, 1, 1024), (62, 500), 0, False), ((16, 16, 256, F32), (16, 1, 1024), (0, 0), 0, True), ((16, 16, 256, F32), (4, 1, 8192), (62, 500), 0, True),
         ((8, 1, 256, F32), (2, 1, 256), (62, 3000), 0, True), ((32, 8, 64, F32), (2, 1, 256), (16, 3000), 0, False), ((16, 16, 256, F32), (16, 1, 1024), (62, 500), 512, True)]


@pytest.mark.parametrize("layout,sharers,others,fresh,faster", TIMED)
def test_a_step_goes_by_its_plan_where_all_of_it_is_the_faster(layout, sharers, others, fresh, faster):
    """Also by way of the runner, whose decision stands for everything that is in the step."""
    from types import SimpleNamespace

    from wllm_b200.engine.runner import ModelRunner
    nq, nkv, size, dtype = layout
    table, q_lens, ctx_lens, holds = step(sharers, others, fresh)
    plan = ops.prefix_plan(table, q_lens, ctx_lens, 64, nq, nkv, size, size, dtype)
    assert ops.prefix_beside(plan, q_lens, ctx_lens, holds) == faster
    runner = object.__new__(ModelRunner)
    runner.prefix_layouts, runner.cache, runner.model = [(0, nq, nkv, size, size)], SimpleNamespace(page_size=64), SimpleNamespace(dtype=dtype)
    host = np.concatenate([np.array(q_lens, dtype=np.int32), np.array(ctx_lens, dtype=np.int32), table.reshape(-1)])
    R, P = table.shape
    offsets = {"req_q_len": (0, R), "req_ctx_len": (R, R), "table0": (2 * R, R * P)}
    entries = [SimpleNamespace(cache=SimpleNamespace(forked=c - n if h else 0)) for n, c, h in zip(q_lens, ctx_lens, holds)]
    pays = ops.prefix_pays(plan.saved_keys, nkv, size, size, dtype, sum(holds), sum(q_lens) / R)
    assert bool(runner._prefix_plans(entries, host, offsets, (sum(q_lens), R, P), False)[1]) == (faster and pays)


def test_steps_of_sharers_alone_and_small_ones_go_by_their_plan():
    for nq, nkv, size, dtype in ((8, 1, 256, B16), (16, 16, 256, B16), (4, 2, 32, F32), (2, 2, 64, F32), (8, 1, 256, F32)):
        for sharers in ((4, 1, 64), (3, 20, 128)):
            table, q_lens, ctx_lens, holds = step(sharers, (0, 0))
            assert ops.prefix_beside(ops.prefix_plan(table, q_lens, ctx_lens, 64, nq, nkv, size, size, dtype, min_keys=1), q_lens, ctx_lens, holds)


def test_pages_past_the_pools_are_refused():
    table = np.array([[3, 1, 9, -7], [3, 1, 2, 99]], dtype=np.int32)       # (99 holds no key)
    plan = ops.prefix_plan(table, [1, 1], [48, 40], 16, 2, 1, 64, min_keys=1)
    assert plan.top_page == 9 and ops.prefix_plan(table, [1, 1], [16, 33], 16, 2, 1, 64).top_page == 3 and ops.prefix_plan(table, [0, 0], [0, 0], 16, 2, 1, 64).top_page == -1
    q, pages = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(9, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="page 9 of a pool of 9"):
        ops.prefix_attention(q, q, pages, pages, torch.from_numpy(table), plan, plan.host, 2, 1, 64, 16, 0.1, torch.zeros(plan.scratch_floats))


def test_no_plan_is_made_where_the_best_one_would_not_do(monkeypatch):
    """What a plan can save at most is known without it."""
    for layout, sharers, others, fresh, faster in TIMED:
        nq, nkv, size, dtype = layout
        table, q_lens, ctx_lens, holds = step(sharers, others, fresh)
        plan = ops.prefix_plan(table, q_lens, ctx_lens, 64, nq, nkv, size, size, dtype, min_keys=1)
        forked = [c - n if h else 0 for n, c, h in zip(q_lens, ctx_lens, holds)]
        bound = ops.PrefixBound(plan.key, ctx_lens, forked)
        assert bound.saved_keys >= plan.saved_keys and bound.key_tiles <= plan.key_tiles
        assert ops.prefix_beside(bound, q_lens, ctx_lens, holds) or not faster
    from types import SimpleNamespace

    from wllm_b200.engine.runner import ModelRunner
    runner = object.__new__(ModelRunner)
    runner.prefix_layouts, runner.cache, runner.model = [(0, 16, 16, 256, 256)], SimpleNamespace(page_size=64), SimpleNamespace(dtype=F32)
    table, q_lens, ctx_lens, holds = step((2, 1, 256), (62, 3000))
    host = np.concatenate([np.array(q_lens, dtype=np.int32), np.array(ctx_lens, dtype=np.int32), table.reshape(-1)])
    R, P = table.shape
    monkeypatch.setattr(ops, "prefix_plan", lambda *a, **k: pytest.fail("a plan was made"))
    entries = [SimpleNamespace(cache=SimpleNamespace(forked=256 if h else 0)) for h in holds]
    assert not runner._prefix_plans(entries, host, {"req_q_len": (0, R), "req_ctx_len": (R, R), "table0": (2 * R, R * P)}, (R, R, P), False)[1]
