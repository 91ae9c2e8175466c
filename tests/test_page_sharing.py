"""Holder counts and compaction of the page allocator, native and Python alike (CPU)."""
import random

import pytest

from mesh_b200 import _runtime
from mesh_b200.engine.pages import _PyPageAllocator

KINDS = [_runtime.PageAllocator, _PyPageAllocator]


@pytest.mark.parametrize("kind", KINDS)
def test_shared_pages_are_freed_by_their_last_holder(kind):
    a = kind(8, 1)
    pages = a.alloc(3)
    a.share(pages[:2])
    a.share(pages[:1])
    assert [a.refs(p) for p in pages] == [3, 2, 1] and a.refs(7) == 0
    a.free(pages)
    assert a.num_used == 2 and a.num_free == 5 and a.alloc(1) == [3]
    a.free(pages[:2])
    assert a.num_used == 2 and a.refs(1) == 1  # page 1 has a holder left, page 3 is the new one
    with pytest.raises(ValueError):
        a.free([2])
    a.free([1])
    with pytest.raises(ValueError):
        a.free([1])
    with pytest.raises(ValueError):
        a.share([1])
    assert a.refs(3) == 1
    with pytest.raises(ValueError):
        a.share([3, 5])
    assert a.refs(3) == 1  # a refused call counts nothing


@pytest.mark.parametrize("kind", KINDS)
def test_remap_keeps_holders_and_frees_the_rest(kind):
    a = kind(10, 1)
    pages = a.alloc(9)
    a.free([p for p in pages if p not in (2, 7, 9)])
    a.share([7])
    remap = [0, -1, 2, -1, -1, -1, -1, 1, -1, 3]
    a.remap(remap)
    assert [a.refs(p) for p in range(10)] == [0, 2, 1, 1, 0, 0, 0, 0, 0, 0]
    assert a.num_used == 3 and a.alloc(2) == [4, 5]
    for bad in ([0] * 9, [0, 1, 2, 3, -1, 5, 6, 7, 8, 9], [0, 1, 2, 3, 4, 4, 6, 7, 8, 9], [0, 1, 2, 3, 0, 5, 6, 7, 8, 9],
                [0, 1, 2, 3, 10, 5, 6, 7, 8, 9]):
        with pytest.raises(ValueError):
            a.remap(bad)
    assert a.num_used == 5 and a.refs(1) == 2


def test_native_and_python_agree():
    r = random.Random(5)
    native, plain = (k(40, 2) for k in KINDS)
    held = []
    for _ in range(2000):
        op = r.random()
        if op < 0.4:
            n = r.randint(0, 6)
            got = native.alloc(n)
            assert plain.alloc(n) == got
            if got:
                held.append(got)
        elif op < 0.6 and held:
            pages = r.choice(held)
            native.share(pages)
            plain.share(pages)
            held.append(list(pages))
        elif op < 0.95 and held:
            pages = held.pop(r.randrange(len(held)))
            native.free(pages)
            plain.free(pages)
        else:
            live = sorted({p for h in held for p in h})
            n = 2 + len(live)
            holes = [p for p in range(2, n) if p not in live]
            remap = [p if p < 2 or p in live else -1 for p in range(40)]
            for p, q in zip([p for p in live if p >= n], holes):
                remap[p] = q
            native.remap(remap)
            plain.remap(remap)
            held = [[remap[p] for p in h] for h in held]
        assert native.num_free == plain.num_free and native.num_used == plain.num_used
        assert all(native.refs(p) == plain.refs(p) for p in range(40))
