"""PagedKVCache's dealing of pages (CPU)."""
import pytest
import torch

from torchplusplus_amd.llmops.paged import PagedKVCache


def cache(pages=6, page=16):
    return PagedKVCache(pages, page, 2, 2, 64, torch.float16, torch.device("cpu"))


def test_pages_are_dealt_once_and_come_back():
    c = cache()
    assert c.k_pages.shape == (2, 6, 2, 16, 64) and c.free_pages == 6
    a, b = c.allocate(17), c.allocate(16)
    assert len(c.pages_of(a)) == 2 and len(c.pages_of(b)) == 1 and c.free_pages == 3
    c.grow(b, 33)
    c.grow(b, 5)  # never fewer
    assert len(c.pages_of(b)) == 3
    held = c.pages_of(a) + c.pages_of(b)
    assert len(set(held)) == 5 and all(0 <= x < 6 for x in held)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.grow(a, 16 * 4)
    assert len(c.pages_of(a)) == 2 and c.free_pages == 1
    with pytest.raises(RuntimeError, match="out of pages"):
        c.allocate(100)
    with pytest.raises(ValueError):
        c.allocate(-1)
    c.free(a)
    assert c.free_pages == 3
    with pytest.raises(KeyError):
        c.free(a)
    d = c.allocate()
    assert c.pages_of(d) == [] and d not in (a, b)


def test_tables_and_slots():
    c = cache(8)
    a, b, e = c.allocate(40), c.allocate(10), c.allocate()
    t = c.block_tables([a, b, e])
    assert t.dtype == torch.int32 and t.shape == (3, 3)
    assert t[0].tolist() == c.pages_of(a) and t[1].tolist() == c.pages_of(b) + [-1, -1] and t[2].tolist() == [-1] * 3
    assert c.block_tables([b], 5).shape == (1, 5) and c.block_tables([]).shape == (0, 0)
    with pytest.raises(ValueError):
        c.block_tables([a], 2)
    pos, slots = c.slots([a, b], [14, 0], [4, 3])
    pa, pb = c.pages_of(a), c.pages_of(b)
    assert pos.dtype == torch.int32 and slots.dtype == torch.int64
    assert pos.tolist() == [14, 15, 16, 17, 0, 1, 2]
    assert slots.tolist() == [pa[0] * 16 + 14, pa[0] * 16 + 15, pa[1] * 16, pa[1] * 16 + 1] + [pb[0] * 16 + i for i in range(3)]
    for args in (([b], [0], [17]), ([b], [-1], [2]), ([b], [0], [-1])):
        with pytest.raises(ValueError):
            c.slots(*args)
    assert c.slots([], [], [])[1].shape == (0,)
    nxt = c.next_slots(t, torch.tensor([39, 16, 0], dtype=torch.int32))
    assert nxt.tolist() == [pa[2] * 16 + 7, -1, -1]
    assert c.next_slots(t, torch.tensor([48, 3, -1], dtype=torch.int32)).tolist() == [-1, pb[0] * 16 + 3, -1]


def test_steps():
    c = cache(8)
    a, b = c.allocate(), c.allocate(3)
    s = c.prefill_step([a, b], [0, 0], [20, 3])
    assert s.cu_seqlens.dtype == torch.int32 and s.cu_seqlens.tolist() == [0, 20, 23] and s.key_slots is None
    assert s.positions.tolist() == [*range(20), 0, 1, 2] and len(set(s.slots.tolist())) == 23
    assert len(c.pages_of(a)) == 2 and s.block_tables is None
    t = c.prefill_step([b, a], [3, 20], [1, 13])
    assert t.cu_seqlens.tolist() == [0, 1, 14] and t.cu_seqlens_k.tolist() == [0, 4, 37]
    assert t.key_slots[:3].tolist() == s.slots[20:].tolist() and t.key_slots[4:24].tolist() == s.slots[:20].tolist()
    assert t.slots.tolist() == [t.key_slots[3].item()] + t.key_slots[24:].tolist()
    before = c.pages_of(a), c.pages_of(b), c.free_pages
    with pytest.raises(RuntimeError, match="out of pages"):
        c.prefill_step([a, b], [33, 4], [40, 60])
    assert before == (c.pages_of(a), c.pages_of(b), c.free_pages)
    with pytest.raises(ValueError, match="twice"):
        c.prefill_step([a, a], [33, 34], [1, 1])
    d = c.decode_step(c.block_tables([a, b]), torch.tensor([33, 4], dtype=torch.int32))
    assert d.seqlens.tolist() == [34, 5] and d.seqlens.dtype == torch.int32 and d.cu_seqlens is None
    assert d.slots.tolist() == [c.pages_of(a)[2] * 16 + 1, c.pages_of(b)[0] * 16 + 4]


def test_read_gathers_rows():
    c = cache()
    a = c.allocate(20)
    c.k_pages.copy_(torch.arange(c.k_pages.numel()).view_as(c.k_pages) % 2039)
    _, slots = c.slots([a], [0], [20])
    k, v = c.read(1, slots)
    assert k.shape == (20, 2, 64) and torch.equal(k[17], c.k_pages[1, c.pages_of(a)[1], :, 1]) and (v == 0).all()


@pytest.mark.parametrize("page", [8, 24, 2048])
def test_page_sizes(page):
    with pytest.raises(ValueError, match="page_size"):
        cache(4, page)
