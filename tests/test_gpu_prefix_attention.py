"""Attention over shared prefixes against its definition in 64 bits, and in 32 bits against the engine's other kernels bit for bit."""
import pytest
import torch

from prefix_refs import Batch

DEV = "cuda:0"
pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

SHAPES = [                      # (query heads, kv heads, key size, value size)
    (8, 1, 256, 256), (16, 4, 128, 128), (6, 2, 72, 40), (7, 1, 64, 64), (4, 4, 96, 96), (128, 1, 8, 256), (5, 1, 192, 64), (16, 8, 200, 136), (2, 1, 256, 8),
          (3, 1, 192, 256), (6, 3, 136, 200)]
TREES = [
    (0, [(5, 1)]),
    (0, [(0, 1), (0, 1)]),
    (512, [(3, 1), (0, 1), (40, 1)]),
    (256, [(512, [(1, 1), (17, 3), (0, 9)]), (1024, [(5, 1)] * 30), (70, 1)]),
    (1024, [(0, 40), (33, 1)] * 6),
    (0, [(512, [(0, 1)] * 5), (512, [(7, 2)] * 5), (99, 130)]),
    (128, [(128, [(128, [(128, [(3, 1), (2, 1)]), (2, 1)]), (1, 1)]), (0, 1)]),
]
RULES = {"plain": {}, "all": {"sinks": True, "cap": 5.0, "slopes": True}, "cap": {"cap": 3.0}, "slopes": {"slopes": True}, "sinks": {"sinks": True}}


def rule_args(b, rule, device=None):
    r = RULES[rule]
    move = (lambda t: t.to(device)) if device else (lambda t: t)
    return {"cap": r.get("cap", 0.0), **({"sinks": move(b.sinks)} if "sinks" in r else {}), **({"slopes": move(b.slopes)} if "slopes" in r else {})}


def attend(b, dtype, rule="plain", plan=None, **kw):
    from wllm_b200.kernels import ops
    q, k, v, table = b.on(DEV)
    if plan is None:
        plan = ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, b.ps, b.nq, b.nkv, b.hd, b.vd, dtype, **kw)
    wide = torch.full((b.n, b.nq * b.vd + 8), float("nan"), dtype=dtype, device=DEV)
    out = wide[:, :b.nq * b.vd]
    scratch = torch.full((plan.scratch_floats,), float("nan"), device=DEV)
    ops.prefix_attention(q, out, k, v, table, plan, plan.to(DEV), b.nq, b.nkv, b.hd, b.ps, b.hd ** -0.5, scratch, vd=b.vd, **rule_args(b, rule, DEV))
    torch.cuda.synchronize()
    assert ops.tc_gemm_status(DEV) == 0 and bool(wide[:, b.nq * b.vd:].isnan().all())
    return out.cpu(), plan


def magnitude(b, rule):
    """sum of weight x |value|: what a relative error of the weights is relative to"""
    signed, b.v = b.v, b.v.abs()
    a = b.exact(b.hd ** -0.5, **rule_args(b, rule))
    b.v = signed
    return a


# Each weight is rounded to bfloat16 (2^-8 of it at most), the output again; sixteen-fold smaller is what 32-bit scores, exponentials and sums come to (scores of magnitude 20 summed over
# 256 products: some 1e-5; the capped scores' quotient and exponential 1e-6 of the cap).
@pytest.mark.parametrize("nq,nkv,hd,vd", SHAPES)
@pytest.mark.parametrize("tree", range(len(TREES)))
@pytest.mark.parametrize("ps", [16, 64, 128])
def test_bfloat16(nq, nkv, hd, vd, tree, ps):
    if nq == 128 and tree in (3, 4):
        pytest.skip("the same rows by the hundred")
    rule = list(RULES)[(tree + ps // 16) % len(RULES)]
    b = Batch(TREES[tree], nq, nkv, hd, vd, ps, seed=tree, dtype=BF16)
    got, plan = attend(b, BF16, rule)
    want = b.exact(hd ** -0.5, **rule_args(b, rule))
    err, bound = (got.double() - want).abs(), 2.0 ** -8 * (1 + 2.0 ** -4) * magnitude(b, rule) + 2.0 ** -8 * want.abs()
    assert bool(got.isfinite().all()) and bool((err <= bound).all()), (float((err / bound).max()), rule)


@pytest.mark.parametrize("nq,nkv,hd,vd", [s for s in SHAPES if s[0] // s[1] <= 32])
@pytest.mark.parametrize("tree", range(len(TREES)))
def test_float32_gives_the_tiled_kernels_bits(nq, nkv, hd, vd, tree):
    from wllm_b200.kernels import ops
    ps = (16, 32, 64, 128)[tree % 4]
    rule = list(RULES)[(tree + hd // 8) % len(RULES)]
    b = Batch(TREES[tree], nq, nkv, hd, vd, ps, seed=tree)
    got, plan = attend(b, F32, rule)
    q, k, v, table = b.on(DEV)
    want = torch.empty(b.n, nq * vd, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    starts = [sum(b.q_lens[:r]) for r in range(b.R)]
    ops.paged_attention_simt_tiled(q, want, k, v, i32(starts), i32(b.q_lens), i32(b.ctx_lens), table, max(b.q_lens), nq, nkv, hd, ps, 0, hd ** -0.5, vd=vd, **rule_args(b, rule, DEV))
    assert bool(got.isfinite().all()) and torch.equal(got, want.cpu())


def test_float32_against_64_bits():
    # scores: 72 products of up to 40 in sum, each step off by 2^-24 of the partial sum: 72 x 40 x 2^-24 = 1.7e-4 at most, in the exponent of every weight; the sums over
    # 600 keys 600 x 2^-24 = 4e-5 at most
    b = Batch((512, [(20, 1), (3, 5), (60, 1)]), 6, 2, 72, 40, 16)
    for rule in RULES:
        got, _ = attend(b, F32, rule)
        want = b.exact(72 ** -0.5, **rule_args(b, rule))
        assert bool(((got.double() - want).abs() <= 4e-4 * magnitude(b, rule)).all())


def test_rows_with_masked_infinities_and_zero_queries():
    """Keys of the largest size in places that no row of a request sees (another request's own, slots behind the end) change nothing; queries of zero weigh all keys alike."""
    b = Batch((256, [(10, 1), (30, 2)]), 4, 2, 64, 64, 16, dtype=BF16)
    plain, _ = attend(b, BF16)
    b.k[b.k.isnan()] = float("inf")
    b.v[b.v.isnan()] = float("-inf")
    again, _ = attend(b, BF16)
    assert torch.equal(plain, again)
    b.q.zero_()
    got, _ = attend(b, BF16)
    want = b.exact(64 ** -0.5)
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * (1.0625 * magnitude(b, "plain") + want.abs())).all())


def test_a_key_that_is_no_number_stays_with_those_that_see_it():
    b = Batch((256, [(128, [(10, 1), (30, 2)]), (5, 1)]), 2, 1, 64, 64, 64, dtype=BF16)
    b.k[int(b.table[0, 5]), 0, 3] = float("nan")              # in the stretch that the first two requests share
    got, plan = attend(b, BF16)
    assert plan.saved_keys > 0 and bool(got[:3].isnan().all()) and bool(got[3:].isfinite().all())


def test_the_cut_into_items_changes_roundings_alone():
    b = Batch((2048, [(100, 1)] * 12), 8, 1, 128, 128, 64, dtype=BF16)
    want, bound = b.exact(128 ** -0.5), 2.0 ** -8 * (1.0625 * magnitude(b, "plain"))
    for min_keys in (1, 1 << 20):
        got, plan = attend(b, BF16, min_keys=min_keys)
        assert (plan.saved_keys > 0) == (min_keys == 1)
        assert bool(((got.double() - want).abs() <= bound + 2.0 ** -8 * want.abs()).all())
    one, _ = attend(b, BF16)
    two, _ = attend(b, BF16)
    assert torch.equal(one, two)                              # the same plan, the same bits


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_in_a_graph_on_a_stream_and_twice_at_once(dtype):
    from wllm_b200.kernels import ops
    a, b = (Batch((512, [(20 + s, 1), (3, 4), (60, 1)] * 3), 8, 2, 64, 64, 16, seed=s, dtype=dtype) for s in (1, 2))
    want = [attend(x, dtype)[0] for x in (a, b)]
    streams, outs, kept = [torch.cuda.Stream() for _ in range(2)], [], []
    for x, stream in zip((a, b), streams):
        plan = ops.prefix_plan(x.table, x.q_lens, x.ctx_lens, 16, 8, 2, 64, 64, dtype)
        with torch.cuda.stream(stream):
            args = x.on(DEV)
            out, arrays, scratch = torch.zeros(x.n, 512, dtype=dtype, device=DEV), plan.to(DEV), torch.empty(plan.scratch_floats, device=DEV)
            for _ in range(5):
                ops.prefix_attention(args[0], out, *args[1:], plan, arrays, 8, 2, 64, 16, 64 ** -0.5, scratch)
            outs.append(out)
            kept.append((args, arrays, scratch, plan))
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), w) for o, w in zip(outs, want))
    (q, k, v, table), arrays, scratch, plan = kept[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prefix_attention(q, outs[0], k, v, table, plan, arrays, 8, 2, 64, 16, 64 ** -0.5, scratch)
    outs[0].zero_()
    scratch.fill_(float("nan"))
    graph.replay()
    assert torch.equal(outs[0].cpu(), want[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_captured_call_for_plans_of_several_batches(dtype):
    """A call laid out for twelve tokens replayed for batches of twelve, five and one: the rows behind the last token stay as they were."""
    from wllm_b200.kernels import ops
    caps, width = (64, 96, 400, 12), 24
    batches = [Batch(tree, 8, 2, 64, 64, 16, seed=i, dtype=dtype) for i, tree in enumerate([(256, [(5, 1)] * 12), (0, [(128, [(9, 1)] * 3), (70, 1), (0, 1)]), (0, [(33, 1)])])]
    made = []
    for b in batches:
        table = torch.full((b.R, width), -1, dtype=torch.int32)
        table[:, :b.table.shape[1]] = torch.as_tensor(b.table)
        made.append((ops.prefix_plan(torch.cat([table, torch.full((12 - b.R, width), -1, dtype=torch.int32)]), b.q_lens + [0] * (12 - b.R), b.ctx_lens + [0] * (12 - b.R), 16, 8, 2, 64, 64,
                                     dtype, caps=caps), table))
    pages = max(b.k.shape[0] for b in batches)
    q, out, k, v = (torch.zeros(*s, dtype=dtype, device=DEV) for s in ((12, 512), (12, 512), (pages, 2, 16, 64), (pages, 2, 16, 64)))
    table = torch.zeros(12, width, dtype=torch.int32, device=DEV)
    plan = made[0][0]
    arrays, scratch = torch.zeros(plan.used, dtype=torch.int32, device=DEV), torch.full((plan.scratch_floats,), float("nan"), device=DEV)

    def put(i):
        b, (p, t) = batches[i], made[i]
        assert p.used == plan.used and p.launch == plan.launch and p.places == plan.places
        arrays.copy_(p.host)
        table[:b.R] = t.to(DEV)
        q[:b.n], k[:b.k.shape[0]], v[:b.v.shape[0]] = (x.to(DEV) for x in (b.q, b.k, b.v))
        out.fill_(7.0)
        scratch.fill_(float("nan"))
    put(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prefix_attention(q, out, k, v, table, plan, arrays, 8, 2, 64, 16, 64 ** -0.5, scratch)
    for i in (0, 1, 2, 0):
        put(i)
        graph.replay()
        torch.cuda.synchronize()
        b = batches[i]
        assert bool((out[b.n:] == 7.0).all())
        # bfloat16: a weight's and the output's rounding, as above; 32 bits: as in test_float32_against_64_bits, sums of 64 products and of 300 keys
        bound = 2.0 ** -8 * (1.0625 * magnitude(b, "plain") + b.exact(64 ** -0.5).abs()) if dtype == BF16 else 4e-4 * magnitude(b, "plain")
        assert bool(((out[:b.n].cpu().double() - b.exact(64 ** -0.5)).abs() <= bound).all()), i


def test_pools_past_32_bits():
    """Keys that lie more than 2^32 bytes into the pools, at places above 2^31 elements."""
    b = Batch((256, [(70, 1), (5, 2)]), 8, 1, 256, 256, 64, dtype=BF16)
    pages = 140000
    k, v = (torch.zeros(pages, 1, 64, 256, dtype=BF16, device=DEV) for _ in range(2))
    far = pages - 1 - torch.arange(b.k.shape[0])
    k[far.to(DEV)], v[far.to(DEV)] = b.k.to(DEV), b.v.to(DEV)
    table = torch.where(b.table >= 0, pages - 1 - b.table, b.table)
    from wllm_b200.kernels import ops
    plan = ops.prefix_plan(table, b.q_lens, b.ctx_lens, 64, 8, 1, 256)
    out = torch.empty(b.n, 2048, dtype=BF16, device=DEV)
    ops.prefix_attention(b.on(DEV)[0], out, k, v, table.to(DEV), plan, plan.to(DEV), 8, 1, 256, 64, 1 / 16, torch.empty(plan.scratch_floats, device=DEV))
    assert torch.equal(out.cpu(), attend(b, BF16)[0])
    del k, v


def test_refusals():
    from wllm_b200.kernels import ops
    b = Batch((128, [(20, 1), (3, 4)]), 4, 2, 64, 64, 16, dtype=BF16)
    q, k, v, table = b.on(DEV)
    plan = ops.prefix_plan(b.table, b.q_lens, b.ctx_lens, 16, 4, 2, 64)
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    good = dict(q=q, out=z(b.n, 256), k_pages=k, v_pages=v, block_table=table, plan=plan, arrays=plan.to(DEV), nq=4, nkv=2, hd=64, page_size=16, scale=0.1, scratch=z(plan.scratch_floats, dt=F32))
    ops.prefix_attention(**good)
    for wrong in (dict(q=q[:-1]), dict(q=q.float()), dict(out=z(b.n, 264)), dict(out=z(b.n, 256, dt=F32)), dict(k_pages=k.transpose(1, 2)), dict(v_pages=v[1:]), dict(k_pages=k.float()),
                  dict(block_table=table[:, :-1]), dict(block_table=table.long()), dict(arrays=good["arrays"][:-4]), dict(scratch=good["scratch"][1:]), dict(nq=8), dict(nkv=1), dict(hd=32),
                  dict(page_size=32), dict(vd=32), dict(scale=0.0), dict(scale=float("nan")), dict(cap=-1.0), dict(sinks=z(4)), dict(slopes=z(3, dt=F32)), dict(q=q.cpu()),
                  dict(q=torch.zeros(b.n, 260, dtype=BF16, device=DEV)[:, 4:])):
        with pytest.raises(ops.KernelError):
            ops.prefix_attention(**{**good, **wrong})
    torch.cuda.synchronize()
    assert ops.tc_gemm_status(DEV) == 0
