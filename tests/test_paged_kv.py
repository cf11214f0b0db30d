"""Host bookkeeping of the paged KV cache (no GPU needed)."""

from __future__ import annotations

import pytest

from memory.paged_kv import PageAllocator, PagedKVCache, PagedKVSpec


def _spec(**kw):
    base = dict(layers=2, kv_heads=2, head_dim=64, dtype="float32", page_size=8, num_pages=10, rows=3, max_pages=4)
    return PagedKVSpec(**{**base, **kw})


@pytest.mark.parametrize("kw,message", [(dict(dtype="float16"), "dtype"), (dict(page_size=12), "page_size"),
                                        (dict(head_dim=96), "head_dim"), (dict(rows=0), "rows"),
                                        (dict(num_pages=0), "num_pages"), (dict(layers=-1), "layers")])
def test_spec_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        PagedKVCache(_spec(**kw), device="cpu")


def test_spec_sizes():
    s = _spec(dtype="bfloat16")
    assert s.slots == 32 and s.nbytes == 2 * 2 * 10 * 2 * 8 * 64 * 2


def test_allocator_takes_each_page_once_and_refuses_strangers():
    a = PageAllocator(5)
    first = a.take(3)
    assert first == [0, 1, 2] and a.free == 2
    with pytest.raises(MemoryError):
        a.take(3)
    assert a.free == 2
    a.give([1])
    with pytest.raises(ValueError):
        a.give([1])
    assert a.take(1) == [1] and sorted(a.take(2)) == [3, 4]


def test_rows_grow_by_pages_and_give_them_back():
    c = PagedKVCache(_spec(), device="cpu")
    assert c.reserve([1, 8, 9]) and [len(h) for h in c.held] == [1, 1, 2]
    assert not c.reserve([8, 8, 16])  # nothing more is needed
    assert c.reserve([9, 0, 16]) and [len(h) for h in c.held] == [2, 1, 2]
    c.upload()
    for row, held in enumerate(c.held):
        assert c.table[row, :len(held)].tolist() == held
    assert len({p for h in c.held for p in h}) == 5
    with pytest.raises(ValueError, match="33 slots"):
        c.reserve([33])
    with pytest.raises(MemoryError):
        c.reserve([32, 32, 32])
    assert [len(h) for h in c.held] == [2, 1, 2] and c.allocator.free == 5  # all or nothing
    c.trim([3, 8, 0])
    assert [len(h) for h in c.held] == [1, 1, 0] and c.allocator.free == 8
    c.release(1)
    assert c.allocator.free == 9


def test_shared_prompt_pages_leave_every_row_its_own_tail():
    c = PagedKVCache(_spec(num_pages=12), device="cpu", track=True)
    assert c.weights.shape == (2, 3, 2, 32) and c.slot_positions.shape == (2, 3, 2, 32)
    c.reserve([32, 32, 32])
    c.share_prompt(19)  # two full pages and three slots
    c.upload()
    t = c.table.tolist()
    assert t[0][:2] == t[1][:2] == t[2][:2]
    tails = [p for row in t for p in row[2:]]
    assert len(set(tails)) == 6 and not set(tails) & set(t[0][:2])
    assert c.allocator.free == 4
    for row in range(3):
        c.release(row)
    assert c.allocator.free == 12


def test_reserving_after_sharing_keeps_the_shared_pages_and_the_tails():
    c = PagedKVCache(_spec(num_pages=12), device="cpu")
    c.reserve([20, 20, 20])
    c.share_prompt(19)
    c.upload()
    before, free = c.table.clone(), c.allocator.free
    assert not c.reserve([24, 24, 20])  # what the rows have already
    c.upload()
    assert c.table.tolist() == before.tolist() and c.allocator.free == free
    assert c.reserve([20, 25, 32])  # a page more for the last two rows, behind the ones that they have
    c.upload()
    t = c.table.tolist()
    assert [r[:3] for r in t] == before[:, :3].tolist() and c.allocator.free == free - 2
    assert t[1][3] != t[2][3] and not {t[1][3], t[2][3]} & {p for r in t for p in r[:3]}


def test_a_shared_page_is_free_when_its_last_holder_goes():
    c = PagedKVCache(_spec(num_pages=12), device="cpu")
    c.reserve([20, 20, 20])
    c.share_prompt(19)
    shared = c.held[0][:2]
    c.release(0)
    assert c.allocator.free == 12 - 2 - 2  # row 0's tail went, the two shared pages and two tails did not
    c.reserve([24, 0, 0])
    c.upload()
    assert not set(c.table[0, :3].tolist()) & set(c.held[1] + c.held[2])
    assert c.table[1, :2].tolist() == c.table[2, :2].tolist() == shared
    c.trim([24, 16, 0])
    assert c.held[1] == shared and c.held[2] == []
    c.trim([24, 0, 0])
    c.release(0)
    assert c.allocator.free == 12


def test_rows_that_take_the_prompt_of_row_0_need_pages_for_their_tails_only():
    c = PagedKVCache(_spec(num_pages=5), device="cpu")
    c.reserve([19])
    c.share_prompt(19)
    assert c.reserve([19, 19, 19]) and c.allocator.free == 0
    c.upload()
    t = c.table.tolist()
    assert t[0][:2] == t[1][:2] == t[2][:2] and len({r[2] for r in t}) == 3
    c.share_prompt(19)  # again: nothing changes
    c.upload()
    assert c.table.tolist() == t and c.allocator.free == 0
    with pytest.raises(ValueError, match="row 0 has 3 pages"):
        c.share_prompt(32)


def test_a_row_is_not_cut_inside_a_page_that_others_hold():
    """The row's next token would go into that page, which is part of the other rows' prompt."""
    c = PagedKVCache(_spec(num_pages=12), device="cpu")
    c.reserve([20, 20, 20])
    c.share_prompt(19)
    for slots in ([19, 9, 19], [12, 19, 19]):
        with pytest.raises(ValueError, match="other rows hold"):
            c.trim(slots)
        assert [len(h) for h in c.held] == [3, 3, 3]
    c.trim([19, 16, 17])


def test_giving_a_page_twice_changes_nothing():
    a = PageAllocator(4)
    a.take(3)
    with pytest.raises(ValueError, match="page 1"):
        a.give([0, 1, 1])
    assert a.free == 1
    a.give([0, 1])
    assert a.free == 3
