"""Forked requests and resized caches on the host: holders are counted, nobody writes to a page that another holder reads, nothing is lost or half done."""
import random

import pytest
import torch

from wllm_b200.cache import CacheGroupSpec, CacheManager, OutOfPages, PagePool, StateSpec
from wllm_b200.kernels import ops


def manager(pages=16, page_size=4, window=None, max_requests=6, states=(), groups=None, **kw):
    return CacheManager(groups or [CacheGroupSpec("all", 2, 1, 8, window, **kw)], page_size, pages, max_requests, states, torch.float32, None)


def grow(m, rc, n):
    m.reserve([(rc, n)])
    m.commit(rc, n)


def test_a_page_is_free_when_its_last_holder_has_given_it_back():
    p = PagePool(2)
    a = p.take()
    p.share(a)
    assert p.holders(a) == 2 and not p.give(a) and p.is_held(a) and p.num_free == 1
    assert p.give(a) and not p.is_held(a)
    with pytest.raises(RuntimeError, match="freed twice"):
        p.give(a)
    with pytest.raises(RuntimeError, match="not held"):
        p.share(a)
    with pytest.raises(RuntimeError, match="not held"):
        p.share(7)


@pytest.mark.parametrize("tokens", [0, 1, 3, 4, 5, 8, 11])
def test_full_pages_are_shared_and_the_last_one_is_not(tokens):
    m = manager()
    a = m.open("a")
    if tokens:
        grow(m, a, tokens)
    b = m.fork(a, "b")
    m.check()
    full = tokens // 4
    assert b.tables[0][:full] == a.tables[0][:full] and len(b.tables[0]) == len(a.tables[0])
    assert b.tables[0][full:] != a.tables[0][full:] or tokens % 4 == 0
    for rc in (a, b):
        grow(m, rc, 6)                                  # both go on writing, each to pages of its own
        m.check()
    assert not set(a.tables[0][full:]) & set(b.tables[0][full:])
    m.close(a)
    m.check()
    m.close(b)
    assert m.free_pages() == [16]
    m.check()


def test_forks_of_forks_and_forks_at_an_earlier_token():
    m = manager(pages=32)
    a = m.open("a")
    grow(m, a, 18)
    b = m.fork(a, "b", num_tokens=9)
    grow(m, b, 7)
    c = m.fork(b, "c")
    d = m.fork(a, "d", num_tokens=0)
    grow(m, d, 3)
    m.check()
    assert b.num_tokens == 16 and b.tables[0][:2] == a.tables[0][:2] and c.tables[0] == b.tables[0] and d.num_tokens == 3
    for rc in (a, b, d):
        m.close(rc)
        m.check()
    assert m.free_pages() == [28]


def test_a_fork_that_does_not_fit_changes_nothing():
    m = manager(pages=3)
    a = m.open("a")
    grow(m, a, 9)
    with pytest.raises(OutOfPages):
        m.fork(a, "b")
    assert m.free_pages() == [0] and m.slots.num_free == 5 and list(m.live) == ["a"] and m.groups[0].pool.holders(a.tables[0][0]) == 1
    b = m.fork(a, "b", num_tokens=8)                    # whole pages need none
    m.check()
    m.close(b)
    few = manager(max_requests=1)
    a = few.open("a")
    grow(few, a, 8)
    with pytest.raises(OutOfPages, match="slots"):
        few.fork(a, "b")
    assert few.groups[0].pool.holders(a.tables[0][0]) == 1
    few.check()


def test_a_fork_whose_copy_fails_changes_nothing(monkeypatch):
    m = CacheManager([CacheGroupSpec("all", 2, 1, 8)], 4, 8, 3, [StateSpec("s", (5,))], torch.float32, "cpu")
    a = m.open("a")
    grow(m, a, 6)
    with pytest.raises(ops.KernelError):                # no device: the copy is refused
        m.fork(a, "b")
    assert m.free_pages() == [6] and m.slots.num_free == 2 and m.groups[0].pool.holders(a.tables[0][0]) == 1
    m.check()


def test_refusals():
    m = manager()
    a = m.open("a")
    grow(m, a, 6)
    for n in (-1, 7):
        with pytest.raises(ValueError):
            m.fork(a, "b", num_tokens=n)
    with pytest.raises(KeyError):
        m.fork(a, "a")
    m.reserve([(a, 2)])
    with pytest.raises(RuntimeError, match="in a step"):
        m.fork(a, "b")
    with pytest.raises(RuntimeError, match="in a step"):
        m.resize(20)
    m.commit(a, 2)
    m.close(a)
    with pytest.raises(RuntimeError, match="closed"):
        m.fork(a, "b")
    m = manager(states=[StateSpec("s", (3,))])
    a = m.open("a")
    grow(m, a, 6)
    with pytest.raises(ValueError, match="state"):
        m.fork(a, "b", num_tokens=4)
    m.fork(a, "b")


def test_windows_give_pages_back_holder_by_holder():
    m = manager(pages=24, window=6)
    a = m.open("a")
    grow(m, a, 10)
    b = m.fork(a, "b")
    m.check()
    with pytest.raises(ValueError, match="window"):
        m.fork(a, "c", num_tokens=4)                    # the token behind 4 reads what the window has passed
    grow(m, a, 12)
    m.check()
    assert a.tables[0][1] == -1 and b.tables[0][1] >= 0 and m.groups[0].pool.holders(b.tables[0][1]) == 1
    grow(m, b, 12)
    m.check()
    m.close(a)
    m.close(b)
    assert m.free_pages() == [24]


def test_kept_first_keys_are_shared():
    m = manager(pages=24, window=6, keep_first=3)
    a = m.open("a")
    grow(m, a, 30)
    b = m.fork(a, "b")
    assert b.tables[0][0] == a.tables[0][0] >= 0 and -1 in b.tables[0]
    grow(m, b, 5)
    m.check()


def test_resizing_moves_live_pages_to_the_front():
    m = manager(pages=12, groups=[CacheGroupSpec("all", 2, 1, 8), CacheGroupSpec("w", 1, 1, 8, 6)])
    a, b = m.open("a"), m.open("b")
    grow(m, a, 9)
    grow(m, b, 13)
    c = m.fork(b, "c")
    m.close(a)
    before = {rc.request_id: [list(t) for t in rc.tables] for rc in (b, c)}
    held = [g.pool.num_pages - g.pool.num_free for g in m.groups]
    with pytest.raises(OutOfPages) as e:
        m.resize(held[0] - 1)
    assert e.value.needed == held[0] and {rc.request_id: rc.tables for rc in (b, c)} == before
    versions = [rc.version for rc in (b, c)]
    m.resize(held[0])
    m.check()
    assert m.free_pages() == [0, held[0] - held[1]] and all(rc.version > v for rc, v in zip((b, c), versions))
    for gi, g in enumerate(m.groups):
        assert {p for rc in (b, c) for p in rc.tables[gi] if p >= 0} == set(range(held[gi]))
        for rc in (b, c):                               # the same pages are shared, the same ones gone
            for x, y in zip(before[rc.request_id][gi], rc.tables[gi]):
                assert (x < 0) == (y < 0)
        assert [x == y for x, y in zip(b.tables[gi], c.tables[gi])] == [x == y for x, y in zip(before["b"][gi], before["c"][gi])]
    m.resize(40)
    grow(m, b, 20)
    m.check()
    for rc in (b, c):
        m.close(rc)
    assert m.free_pages() == [40, 40]


@pytest.mark.parametrize("seed", range(6))
def test_random_orders_lose_nothing(seed):
    rng = random.Random(seed)
    m = CacheManager([CacheGroupSpec("all", 1, 1, 8), CacheGroupSpec("w", 1, 1, 8, 7, keep_first=2)], 4, 40, 8, (), torch.float32, None)
    live, serial = [], 0
    for _ in range(400):
        what = rng.random()
        serial += 1
        try:
            if what < 0.2 or not live:
                live.append(m.open(serial))
            elif what < 0.4:
                live.append(m.fork(rng.choice(live), serial))
            elif what < 0.75:
                grow(m, rng.choice(live), rng.randint(1, 9))
            elif what < 0.8:
                m.resize(rng.randint(30, 50))
            else:
                m.close(live.pop(rng.randrange(len(live))))
        except OutOfPages:
            if live:
                m.close(live.pop(rng.randrange(len(live))))
        m.check()
    for rc in live:
        m.close(rc)
    assert all(g.pool.num_free == g.pool.num_pages for g in m.groups)


def test_what_copies_are_refused_on_the_host():
    z = lambda *s: torch.zeros(s)  # noqa: E731
    a = z(2, 5, 1, 4, 8)
    for wrong in ([(a, z(2, 5, 1, 4, 6), [0], [1], None)], [(a, a.double(), [0], [1], None)], [(a[:, :, :, ::2], a[:, :, :, ::2], [0], [1], None)],
                  [(a, a, [0, 1], [1], None)], [(a, a, [0], [1], [1, 2])], [(a, a, [0.5], [1], None)], [(a, a, [0], [1 << 40], None)], [(a[0, 0], a[0, 0], [0], [1], None)],
                  [(a, a, [[0]], [[1]], None)], [(z(2, 0, 1, 4, 8), a, [0], [1], None)], [(a, a, [], [], None)] * (ops.MAX_COPY_POOLS + 1),
                  [(a, a, [0], [1], None)]):            # (the last is in order, but not on a device)
        with pytest.raises(ops.KernelError):
            ops.copy_pages(wrong)
    ops.copy_pages([])
    ops.copy_pages([(a, a, [], [], None)])              # nothing to do needs no device
