"""Pages of the cache copied on the device: every byte that a move names and no other, at odd sizes, types, alignments and counts."""
import pytest
import torch

from wllm_b200.cache import CacheGroupSpec, CacheManager, StateSpec

DEV = "cuda:0"
pytestmark = pytest.mark.gpu


def plain(src, dst, src_pages, dst_pages, slots):
    out, old = dst.clone(), src.clone()
    for i, (s, d) in enumerate(zip(src_pages, dst_pages)):
        n = src.shape[-2] if slots is None else slots[i]
        out[..., d, :, :n, :] = old[..., s, :, :n, :]
    return out


def bits(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("outer,heads,slots,row,dtype", [((3, 2), 2, 16, 64, torch.bfloat16), ((5,), 1, 64, 256, torch.bfloat16), ((), 3, 32, 72, torch.float32), ((2,), 2, 16, 5, torch.bfloat16),
                                                         ((4,), 1, 1, 771, torch.float32), ((2, 2), 1, 16, 2, torch.bfloat16), ((2,), 3, 7, 9, torch.uint8), ((1,), 4, 128, 40, torch.float32)])
@pytest.mark.parametrize("count", [1, 2, 17, 600])
@pytest.mark.parametrize("other", [False, True])
def test_moves(outer, heads, slots, row, dtype, count, other):
    g = torch.Generator().manual_seed(count + heads)
    pages = 2 * count + 3
    make = lambda n: (torch.randint(0, 255, (*outer, n, heads, slots, row * torch.empty((), dtype=dtype).element_size()), generator=g).to(torch.uint8)).to(DEV).view(dtype)  # noqa: E731
    src = make(pages)
    dst = make(count + 5) if other else src
    order = torch.randperm(pages, generator=g).tolist()
    from_, to = order[:count], torch.randperm(count + 5, generator=g).tolist()[:count] if other else order[count:2 * count]
    used = torch.randint(0, slots + 1, (count,), generator=g).tolist() if count != 2 else None
    want = plain(src, dst, from_, to, used)
    kept = src.clone()
    from wllm_b200.kernels import ops
    before = ops.launches
    ops.copy_pages([(src, dst, from_, to, used)])
    assert torch.equal(bits(dst), bits(want)) and ops.launches - before == (2 if count > 512 + sum(u == 0 for u in used or []) else 1 if used is None or any(used) else 0)
    if other:
        assert torch.equal(bits(src), bits(kept))


def test_several_pools_an_unaligned_one_and_far_offsets():
    from wllm_b200.kernels import ops
    g = torch.Generator(device=DEV).manual_seed(3)
    a = torch.randn(2, 9, 1, 16, 24, generator=g, device=DEV)
    flat = torch.randn(4 * 6 * 5 + 1, generator=g, device=DEV)
    b = flat[1:].view(6, 1, 4, 5)                         # starts 4 bytes past a 16-byte boundary
    # a pool above 2^31 elements and 2^32 bytes: the offset of its last pages does not fit 32 bits
    far = torch.zeros(3, 600, 8, 64, 2560, dtype=torch.bfloat16, device=DEV)
    far[2, 597] = torch.randn(8, 64, 2560, generator=g, device=DEV).to(torch.bfloat16)
    moves = [(a, a, [0, 3], [1, 8], [16, 3]), (b, b, [5], [0], None), (far, far, [597, 0], [599, 2], None)]
    want = [plain(a, a, *moves[0][2:]), plain(b, b, *moves[1][2:])]
    ops.copy_pages(moves)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(far[2, 599], far[2, 597]) and not bool(far[:, 598].any())
    del far


def test_refusals_leave_everything_as_it_was():
    from wllm_b200.kernels import ops
    a, b = torch.ones(2, 6, 1, 4, 8, device=DEV), torch.zeros(2, 6, 1, 4, 8, device=DEV)
    kept = [a.clone(), b.clone()]
    layer = torch.zeros(3, 4, 1, 4, 8, device=DEV)
    for wrong in ([(a, b, [6], [0], None)], [(a, b, [-1], [0], None)], [(a, b, [0], [6], None)], [(a, b, [0], [-1], None)], [(a, b, [0], [1], [5])], [(a, b, [0], [1], [-1])],
                  [(a, b, [0, 1], [2, 2], None)], [(a, a, [0, 1], [1, 2], None)], [(a, a, [0], [0], None)], [(a, b, [0], [1], None), (b, a, [0], [1], None)],
                  [(a, b, [0], [1], None), (a, b, [1], [2], None)], [(layer[:2], layer[1:], [0], [1], None)], [(a, b.cpu(), [0], [1], None)],
                  [(a, b, torch.tensor([0], device=DEV), [1], None)]):
        with pytest.raises(ops.KernelError):
            ops.copy_pages(wrong)
    assert torch.equal(a, kept[0]) and torch.equal(b, kept[1])
    ops.copy_pages([(a, a, [0], [1], None), (b, b, [0], [1], None)])


def test_on_a_stream_of_its_own_and_in_a_graph():
    from wllm_b200.kernels import ops
    a = torch.randn(2, 8, 1, 16, 64, device=DEV)
    ops.copy_pages([(a, a, [0], [7], None)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages([(a, a, [1, 2], [3, 4], [16, 5])])
    fresh = torch.randn_like(a)
    a.copy_(fresh)
    graph.replay()
    assert torch.equal(a, plain(fresh, fresh, [1, 2], [3, 4], [16, 5]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.copy_(fresh)
        ops.copy_pages([(a, a, [5], [6], None)])
    side.synchronize()
    assert torch.equal(a, plain(fresh, fresh, [5], [6], None))


def _written(m, rc, n, seed):
    """Commits n tokens whose keys and values are numbers of their own."""
    g = torch.Generator().manual_seed(seed)
    start = rc.num_tokens
    m.reserve([(rc, n)])
    for gi, group in enumerate(m.groups):
        for i, slot in enumerate(m.token_slots(rc, gi, start, n)):
            for t in group.tensors():
                t.view(*t.shape[:-4], -1, *t.shape[-3:])[..., slot // m.page_size, :, slot % m.page_size, :] = torch.randn(1, generator=g).item() + i
    m.commit(rc, n)


def _tokens(m, rc):
    out = []
    for gi, group in enumerate(m.groups):
        first = max(0, group.spec.first_needed(rc.num_tokens))
        for t in group.tensors():
            for slot in m.token_slots(rc, gi, first, rc.num_tokens - first):
                out.append(t[..., slot // m.page_size, :, slot % m.page_size, :].reshape(-1))
    return torch.cat(out)


def test_a_fork_has_its_parents_tokens_and_state_and_goes_its_own_way():
    groups = [CacheGroupSpec("all", 3, 2, 8), CacheGroupSpec("v", 1, 1, 16, None, 24), CacheGroupSpec("w", 2, 1, 8, 20), CacheGroupSpec("in", 2, 1, 24, None, 16, values_in_keys=True)]
    m = CacheManager(groups, 16, 12, 4, [StateSpec(f"s{i}", (7 + i,)) for i in range(20)], torch.float32, DEV, poison=True)
    a = m.open("a")
    _written(m, a, 45, 1)
    for i, t in enumerate(m.slots.tensors.values()):
        t[a.slot] = float(i + 1)
    b = m.fork(a, "b")
    m.check()
    assert torch.equal(_tokens(m, a), _tokens(m, b)) and all(torch.equal(t[a.slot], t[b.slot]) for t in m.slots.tensors.values())
    # slots that hold no token stay as they are: no numbers
    assert bool(m.groups[0].pages[:, :, b.tables[0][2], :, 13:].isnan().all()) and not bool(m.groups[0].pages[:, :, b.tables[0][2], :, :13].isnan().any())
    parent = _tokens(m, a)
    _written(m, b, 9, 2)
    assert torch.equal(_tokens(m, a), parent)
    mine = _tokens(m, b)
    m.close(a)                                            # shared pages stay, its own become no numbers
    assert torch.equal(_tokens(m, b), mine) and bool(mine.isfinite().all())
    m.resize(6)
    m.check()
    assert torch.equal(_tokens(m, b), mine)
    m.resize(30)
    _written(m, b, 40, 3)
    m.check()
    m.close(b)
    assert m.free_pages() == [30] * 4 and bool(m.groups[0].pages.isnan().all())
