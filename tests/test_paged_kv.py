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
