"""Thin items of plans of shared prefixes (up to 16 rows): one tile and many, in turns that let one item's warps run ahead into the next."""
import pytest
import torch

from prefix_refs import Batch
from test_gpu_prefix_attention import BF16, attend, magnitude

pytestmark = pytest.mark.gpu

# (query heads, kv heads, key size, value size): tiles worked off by both groups of warps apart (keys of up to 192 columns; values of one stage a tile and of two), by all warps together
APART = [(8, 1, 128, 256), (4, 1, 64, 256), (8, 1, 128, 128), (16, 4, 128, 128), (4, 2, 64, 64), (2, 1, 192, 192), (6, 2, 72, 200)]
TOGETHER = [(8, 1, 256, 256), (3, 1, 192, 256)]


def lengths(count, seed):
    """Keys of requests of their own: half of them within a tile of 128."""
    g = torch.Generator().manual_seed(seed)
    return [int(torch.randint(0, 128 if i % 2 else 700, (1,), generator=g)) for i in range(count)]


def check(b, runs, **kw):
    want = b.exact(b.hd ** -0.5)
    # a weight's rounding to bfloat16 and the output's; 32-bit scores, exponentials and sums sixteen-fold smaller
    bound = 2.0 ** -8 * (1 + 2.0 ** -4) * magnitude(b, "plain") + 2.0 ** -8 * want.abs()
    first, plan = attend(b, BF16, **kw)
    assert bool(((first.double() - want).abs() <= bound).all())
    for _ in range(runs):
        assert torch.equal(attend(b, BF16, plan=plan)[0], first)
    return plan


@pytest.mark.parametrize("nq,nkv,hd,vd", APART + TOGETHER)
def test_items_of_one_tile_behind_longer_ones(nq, nkv, hd, vd):
    """Several items a multiprocessor, those of several tiles first: the second group of warps, which has nothing to do in an item of one tile, is through with it while the item before is being stored."""
    b = Batch((256, [(n, 1) for n in lengths(600 // nkv, hd + vd)]), nq, nkv, hd, vd, 16, seed=hd, dtype=BF16)
    plan = check(b, 6)
    assert plan.items * nkv > 3 * 148 and plan.saved_keys > 0


@pytest.mark.parametrize("nq,nkv,hd,vd", [(8, 1, 128, 256), (16, 2, 128, 128), (4, 1, 64, 64), (8, 1, 256, 256)])
def test_long_runs_of_thin_items_with_wide_ones_between(nq, nkv, hd, vd):
    """Thin items go on without the thread that issues the tensor core's products, wide ones wait for it: runs of the one kind between the others, eight items and more a multiprocessor."""
    g = torch.Generator().manual_seed(hd)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    groups = [(128 * (1 + i % 4), [(draw(700 if i % 3 else 60), 1) for _ in range(32 if i % 5 else 3)]) for i in range(48)]
    b = Batch((0, groups), nq, nkv, hd, vd, 64, seed=vd, dtype=BF16)
    plan = check(b, 6, min_keys=1)
    assert plan.items * nkv > 8 * 148 and plan.saved_keys > 0


@pytest.mark.parametrize("nq,nkv,hd,vd", [(8, 1, 128, 256), (16, 4, 128, 128), (4, 1, 64, 64), (8, 1, 256, 256)])
@pytest.mark.parametrize("ps", [16, 128])
def test_values_cleared_behind_the_last_key_leave_the_next_tile_alone(nq, nkv, hd, vd, ps):
    """Tiles that hold a few keys, their other rows cleared in a stage of the ring that the next item's full tiles are brought to."""
    own = [(1 + i % 120) if i % 2 else 127 + 128 * (i % 3) for i in range(400 // nkv)]
    check(Batch((0, [(n, 1) for n in own]), nq, nkv, hd, vd, ps, seed=ps, dtype=BF16), 6)
