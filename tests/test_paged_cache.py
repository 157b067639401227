"""Who has which pages of a cache, without a GPU."""
import pytest
import torch

from cats_amd.paged import PagedCache


def _cache(pages=10, page=16):
    return PagedCache(2, pages, 1, 32, page, device="cpu")


def test_pages_come_and_go():
    c = _cache()
    a, b = c.open(), c.open()
    c.reserve([a, b], [17, 0])
    assert len(c.pages_of(a)) == 2 and c.pages_of(b) == [] and c.free == 8
    c.reserve([a], 16)
    assert len(c.pages_of(a)) == 2
    c.reserve([a, b], 33)
    assert c.free == 4 and not set(c.pages_of(a)) & set(c.pages_of(b))
    t = c.table([b, a, b])
    assert t.dtype == torch.int32 and t.tolist() == [c.pages_of(b), c.pages_of(a), c.pages_of(b)]
    c.trim(a, 16)
    assert c.free == 6 and c.table([a, b]).tolist() == [c.pages_of(a) + [-1, -1], c.pages_of(b)]
    c.close(b)
    assert c.free == 9
    c.trim(a, 0)
    assert c.free == 10 and c.table([a]).tolist() == [[-1]]


def test_too_many_take_none():
    c = _cache(3)
    a, b = c.open(), c.open()
    with pytest.raises(RuntimeError, match="4 pages are needed and 3 are free"):
        c.reserve([a, b], [32, 17])
    assert c.free == 3 and c.pages_of(a) == c.pages_of(b) == []
    c.reserve([a], 40)
    with pytest.raises(RuntimeError, match="are free"):
        c.fork(a, 1, 40)
    assert len(c.fork(a, 5, 32)) == 5 and c.free == 0


def test_forks_share_whole_pages():
    c = _cache()
    a = c.open()
    c.reserve([a], 40)
    pages = c.pages_of(a)
    for i, x in enumerate((c.k, c.v)):
        x.copy_(torch.arange(x.numel()).reshape(x.shape) % 1000 + i)
    x, y = c.fork(a, 2, 40)
    assert c.pages_of(x)[:2] == c.pages_of(y)[:2] == pages[:2] and len({pages[2], c.pages_of(x)[2], c.pages_of(y)[2]}) == 3
    for t in (c.k, c.v):
        assert torch.equal(t[:, c.pages_of(x)[2], :, :8], t[:, pages[2], :, :8]) and not torch.equal(t[:, c.pages_of(x)[2], :, 8:], t[:, pages[2], :, 8:])
    assert c.free == 5
    c.close(a)
    assert c.free == 6 and pages[2] in c._free and pages[0] not in c._free
    c.close(x)
    assert c.free == 7
    c.close(y)
    assert c.free == 10 and sorted(c._free) == list(range(10))


def test_an_end_within_a_shared_page_is_the_sequence_s_own():
    c = _cache()
    a = c.open()
    c.reserve([a], 32)
    c.k.copy_(torch.arange(c.k.numel()).reshape(c.k.shape) % 1000)
    (b,) = c.fork(a, 1, 32)
    c.trim(b, 32)
    assert c.pages_of(b) == c.pages_of(a)
    c.trim(b, 20)
    old, new = c.pages_of(a)[1], c.pages_of(b)[1]
    assert old != new and torch.equal(c.k[:, old, :, :4], c.k[:, new, :, :4]) and c.free == 7
    c.trim(a, 3)
    assert c.pages_of(a)[0] != c.pages_of(b)[0] and c.free == 7  # its second page is free, and it has a copy of the first


@pytest.mark.parametrize("more", [0, 1])
def test_an_end_that_finds_no_page_takes_nothing(more):
    """Where the page in which the end lies is shared and none is there for the copy, the sequence stays as it was; a page that it gives back itself is one."""
    c = _cache(2 + more)
    a = c.open()
    c.reserve([a], 32)
    (b,) = c.fork(a, 1, 32)
    if more:
        c.reserve([a], 48)  # somebody's
    c.k.copy_(torch.arange(c.k.numel()).reshape(c.k.shape) % 1000)
    before = c.pages_of(a), c.pages_of(b), list(c._users), list(c._free), c.k.clone()
    assert c.free == 0
    for length in (4, 20):
        with pytest.raises(RuntimeError, match="1 page is needed and 0 are free"):
            c.trim(b, length)
        assert before[:4] == (c.pages_of(a), c.pages_of(b), c._users, c._free) and torch.equal(c.k, before[4])
    c.trim(b, 16)  # whole pages need none
    assert c.pages_of(b) == c.pages_of(a)[:1]
    if more:
        c.trim(a, 20)
        assert c.free == 1 and c.pages_of(a) == before[0][:2]  # nobody else has that one now
        c.trim(a, 4)
        assert c.pages_of(a)[0] != c.pages_of(b)[0] and c.free == 1 and torch.equal(c.k[:, c.pages_of(a)[0], :, :4], c.k[:, c.pages_of(b)[0], :, :4])


def test_an_end_may_lie_in_a_page_that_comes_free():
    c = _cache(3)
    a = c.open()
    c.reserve([a], 16)
    (b,) = c.fork(a, 1, 16)
    c.reserve([b], 48)
    c.k.copy_(torch.arange(c.k.numel()).reshape(c.k.shape) % 1000)
    assert c.free == 0
    c.trim(b, 5)
    assert c.free == 1 and c.pages_of(b) != c.pages_of(a) and torch.equal(c.k[:, c.pages_of(b)[0], :, :5], c.k[:, c.pages_of(a)[0], :, :5])


def test_a_table_in_place():
    c = _cache()
    a = c.open()
    c.reserve([a], 20)
    t = torch.full((1, 4), 7, dtype=torch.int32)
    assert c.table([a], out=t) is t and t.tolist() == [c.pages_of(a) + [-1, -1]]
    c.reserve([a], 80)
    with pytest.raises(ValueError, match="up to 5 pages"):
        c.table([a], out=t)


@pytest.mark.parametrize("change,what", [(dict(dtype=torch.float32), "float16 and bfloat16"), (dict(head_dim=48), "heads of"), (dict(page=48), "power of two"), (dict(page=8), "power of two"),
                                         (dict(layers=0), "at least"), (dict(pages=0), "at least"), (dict(kv_heads=0), "at least")])
def test_caches_that_are_none(change, what):
    with pytest.raises(ValueError, match=what):
        PagedCache(**{**dict(layers=1, pages=2, kv_heads=1, head_dim=32, page=16, device="cpu"), **change})


def test_calls_that_are_none():
    c = _cache()
    a = c.open()
    c.reserve([a], 16)
    for call in (lambda: c.fork(a, 1, 17), lambda: c.fork(a, 1, -1), lambda: c.trim(a, 17), lambda: c.trim(a, -1), lambda: c.reserve([a, a], 20), lambda: c.reserve([a], [1, 2])):
        with pytest.raises(ValueError):
            call()
    assert c.free == 9
    c.close(a)
    with pytest.raises(KeyError):
        c.close(a)
