import pytest
from hypothesis import given, settings, strategies as st


def test_basic_allocation():
    from llama_cpp.kv_pages import OutOfPages, PageAllocator
    a = PageAllocator(8, 16)
    assert a.ensure(0, 1) and a.table(0) == [0]
    assert not a.ensure(0, 16)
    assert a.ensure(0, 17) and len(a.table(0)) == 2
    a.ensure(1, 16 * 6)
    assert a.free_pages == 0
    with pytest.raises(OutOfPages):
        a.ensure(2, 1)
    a.release(0)
    assert a.free_pages == 2 and a.table(0) == []
    a.truncate(1, 20)
    assert len(a.table(1)) == 2 and a.free_pages == 6


@settings(max_examples=200, deadline=None)
@given(st.lists(st.tuples(st.sampled_from(["ensure", "release", "truncate"]), st.integers(0, 5), st.integers(0, 300)), max_size=60))
def test_no_page_is_leaked_or_shared(ops):
    from llama_cpp.kv_pages import OutOfPages, PageAllocator
    a = PageAllocator(12, 32)
    for op, seq, n in ops:
        try:
            if op == "ensure":
                a.ensure(seq, n)
            elif op == "release":
                a.release(seq)
            else:
                a.truncate(seq, n)
        except OutOfPages:
            pass
        owned = [p for s in range(6) for p in a.table(s)]
        assert len(owned) == len(set(owned))
        assert len(owned) + a.free_pages == 12
        assert all(0 <= p < 12 for p in owned)
        for s in range(6):
            pass


@settings(max_examples=300, deadline=None)
@given(st.lists(st.tuples(st.sampled_from(["ensure", "release", "truncate", "share", "own"]), st.integers(0, 5), st.integers(0, 5), st.integers(0, 300)), max_size=60))
def test_shared_pages_are_counted_and_never_written(ops):
    """A page is free exactly when no table holds it; pages that two tables hold are their leading ones, at the same places; after own_from nobody else holds
    what is written from there on."""
    from llama_cpp.kv_pages import OutOfPages, PageAllocator
    a = PageAllocator(12, 32)
    for op, seq, other, n in ops:
        before = a.table(seq)
        try:
            if op == "ensure":
                a.ensure(seq, n)
                assert a.table(seq)[:len(before)] == before
            elif op == "release":
                a.release(seq)
            elif op == "truncate":
                a.truncate(seq, n)
            elif op == "share" and seq != other:
                if before:
                    with pytest.raises(ValueError):
                        a.share(seq, other, n)
                else:
                    kept = a.share(seq, other, n)
                    assert kept % 32 == 0 and kept <= n and a.table(seq) == a.table(other)[:kept // 32]
            elif op == "own":
                kept = a.own_from(seq, n)
                assert kept == n or (kept < n and kept % 32 == 0 and len(a.table(seq)) == kept // 32)
                mine = a.table(seq)[n // 32:]
                assert not any(p in a.table(s) for p in mine for s in range(6) if s != seq)
                assert before[:len(a.table(seq))] == a.table(seq)
        except OutOfPages:
            pass
        tables = [a.table(s) for s in range(6)]
        held = {p for t in tables for p in t}
        assert all(len(t) == len(set(t)) for t in tables) and len(held) + a.free_pages == 12
        assert held.isdisjoint(a._free) and len(set(a._free)) == len(a._free)
        for p in held:
            assert len({t.index(p) for t in tables if p in t}) == 1


def test_negative_tokens_are_refused():
    """a negative count would be counted from the other table's end"""
    from llama_cpp.kv_pages import PageAllocator
    a = PageAllocator(20, 16)
    assert a.ensure(0, 100)
    for call in (lambda: a.share(1, 0, -1), lambda: a.share(1, 0, -17), lambda: a.own_from(0, -1)):
        with pytest.raises(ValueError):
            call()
    assert a.table(1) == [] and len(a.table(0)) == 7 and a.free_pages == 13
    assert a.share(1, 0, 0) == 0 and a.share(1, 0, 33) == 32
    assert a.own_from(0, 20) == 16 and a.free_pages == 18      # (its second page is the other's too)


def test_sharing_that_is_refused_leaves_the_slot_its_pages():
    from llama_cpp.engine import EngineBase
    from llama_cpp.kv_pages import PageAllocator
    eng = EngineBase.__new__(EngineBase)
    eng.pages, eng.max_seqs, eng._h, eng.lib, told = PageAllocator(20, 16), 3, None, None, []
    eng._set_table = told.append
    eng.pages.ensure(0, 100)
    eng.pages.ensure(1, 50)
    for slot, other, n in ((1, 0, -1), (1, 3, 32), (3, 0, 32), (-1, 0, 32), (1, -1, 32), (1, 1, 32)):
        with pytest.raises(ValueError):
            eng.share_pages(slot, other, n)
    assert len(eng.pages.table(1)) == 4 and eng.pages.free_pages == 9 and not told
    assert eng.share_pages(1, 0, 40) == 32 and told == [1] and eng.pages.free_pages == 13
