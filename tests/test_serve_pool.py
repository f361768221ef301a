"""The paged decoder's page pool (host side)."""
import pytest

from lnsb200.serve import PagePool


def test_pages_are_handed_out_once():
    p = PagePool(8, 4)
    a, b = p.open(), p.open()
    p.grow([(a, 5), (b, 4)])
    p.grow([(a, 3), (b, 1)])
    assert p.length == {a: 8, b: 5}
    assert [len(p.pages[s]) for s in (a, b)] == [2, 2]
    held = p.pages[a] + p.pages[b] + p.free
    assert sorted(held) == list(range(8))


def test_no_room_changes_nothing():
    p = PagePool(3, 4)
    a, b = p.open(), p.open()
    p.grow([(a, 8)])
    before = (dict(p.length), {s: list(v) for s, v in p.pages.items()}, list(p.free))
    with pytest.raises(MemoryError):
        p.grow([(a, 1), (b, 5)])
    with pytest.raises(KeyError):
        p.grow([(b, 1), (99, 1)])
    with pytest.raises(ValueError):
        p.grow([(b, 1), (b, 1)])
    assert (p.length, p.pages, p.free) == before


def test_closed_pages_return():
    p = PagePool(2, 4)
    a = p.open()
    p.grow([(a, 8)])
    p.close(a)
    b = p.open()
    assert b != a
    p.grow([(b, 8)])
    assert sorted(p.pages[b]) == [0, 1]
