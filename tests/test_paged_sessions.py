"""Page lists of PagedKVCache on the CPU, with plain stand-ins for the device functions: what every session
reads back is what was appended to it, whatever was forked, trimmed, closed and compacted around it."""
import random

import pytest
import torch

from lagunalab_amd import paged
from lagunalab_amd.paged import PAGE, OutOfPages, PagedKVCache

H, D = 2, 128


@pytest.fixture
def plain(monkeypatch):
    """Appends, reads and copies without a GPU: a row's first code holds its tag."""
    def append(k, v, keys, values, table, starts, counts):
        seen, at = set(), 0
        for b, (s, c) in enumerate(zip(starts.tolist(), counts)):
            for i in range(c):
                slot = (int(table[b, (s + i) // PAGE]), (s + i) % PAGE)
                assert slot not in seen, "two rows of a call in one slot"
                seen.add(slot)
                keys[0][slot[0], :, slot[1], 0] = k[at, :, 0].to(torch.uint8)
                values[0][slot[0], :, slot[1], 0] = v[at, :, 0].to(torch.uint8)
                at += 1

    def copy(keys, values, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for t in (*keys, *values):
            t[list(dst)] = t[list(src)]

    monkeypatch.setattr(paged, "paged_append", append)
    monkeypatch.setattr(paged, "copy_pages", copy)
    monkeypatch.setattr(paged._lib, "require_device", lambda *t: t[0].device)


def rows(tags):
    return torch.tensor(tags, dtype=torch.bfloat16)[:, None, None].expand(-1, H, D)


def held(cache, session):
    """The tags of a session's rows."""
    pages, n = cache._sessions[session]
    assert len(pages) == -(-n // PAGE)
    got = []
    for buf in (cache.keys, cache.values):
        got.append([int(buf[0][pages[i // PAGE], 1, i % PAGE, 0]) for i in range(n)])
    assert got[0] == got[1]
    return got[0]


def check(cache, want):
    uses = [0] * len(cache._uses)
    for s, tags in want.items():
        assert held(cache, s) == tags and cache.length(s) == len(tags)
        for p in cache.pages(s):
            uses[p] += 1
    assert uses == cache._uses
    assert sorted(cache._free) == [p for p, n in enumerate(uses) if n == 0]


@pytest.mark.parametrize("seed", range(6))
def test_sessions_hold_their_rows(plain, seed):
    rng = random.Random(seed)
    cache = PagedKVCache(24, H, device="cpu")
    want = {}
    for step in range(150):
        op = rng.choice(["open", "append", "append", "append", "fork", "fork", "trim", "close", "compact",
                         "resize"])
        some = rng.sample(sorted(want), rng.randint(0, min(4, len(want))))
        if op == "open":
            want[cache.open()] = []
        elif op == "append" and some:
            counts = [rng.choice([0, 1, 1, 5, rng.randint(1, 100)]) for _ in some]
            tags = [rng.randint(0, 255) for _ in range(sum(counts))]
            before = (sorted(cache._free), [list(cache.pages(s)) for s in want])
            try:
                cache.append(some, rows(tags), rows(tags), counts)
            except OutOfPages:
                assert before == (sorted(cache._free), [list(cache.pages(s)) for s in want])
                continue
            for s, c in zip(some, counts):
                want[s] = want[s] + tags[:c]
                tags = tags[c:]
        elif op == "fork" and some:
            want[cache.fork(some[0])] = want[some[0]]
        elif op == "trim" and some:
            n = rng.randint(0, 80)
            assert cache.trim(some[0], n) == min(n, len(want[some[0]]))
            want[some[0]] = want[some[0]][:max(0, len(want[some[0]]) - n)]
        elif op == "close" and some:
            cache.close(some[0])
            del want[some[0]]
        elif op == "compact":
            n = cache.compact()
            assert all(p < n for s in want for p in cache.pages(s)) and cache.free_pages == len(cache._uses) - n
        elif op == "resize":
            used = len(cache._uses) - cache.free_pages
            cache.resize(max(1, used, rng.randint(16, 30)))
        check(cache, want)


def test_a_shared_page_is_copied_for_all_writers_but_the_last(plain):
    cache = PagedKVCache(8, H, device="cpu")
    a = cache.open()
    cache.append([a], rows([1] * 70), rows([1] * 70))
    b, c = cache.fork(a), cache.fork(a)
    assert cache.free_pages == 6 and cache.pages(b) == cache.pages(a)
    cache.append([a, b, c], rows([2, 3, 4]), rows([2, 3, 4]))
    assert cache.free_pages == 4  # the full page is still one, the partly filled one became three
    assert len({cache.pages(s)[0] for s in (a, b, c)}) == 1 and len({cache.pages(s)[1] for s in (a, b, c)}) == 3
    check(cache, {a: [1] * 70 + [2], b: [1] * 70 + [3], c: [1] * 70 + [4]})
    # one that is not written to keeps its page as it is
    d = cache.fork(b)
    cache.append([b], rows([9]), rows([9]))
    check(cache, {a: [1] * 70 + [2], b: [1] * 70 + [3, 9], c: [1] * 70 + [4], d: [1] * 70 + [3]})


def test_nothing_changes_when_the_pages_run_out(plain):
    cache = PagedKVCache(3, H, device="cpu")
    a = cache.open()
    cache.append([a], rows([1] * 100), rows([1] * 100))
    b = cache.fork(a)
    with pytest.raises(OutOfPages):  # a copy for one of them and a page for each
        cache.append([a, b], rows([2] * 80), rows([2] * 80))
    check(cache, {a: [1] * 100, b: [1] * 100})
    cache.append([a, b], rows([2, 3]), rows([2, 3]))
    check(cache, {a: [1] * 100 + [2], b: [1] * 100 + [3]})


def test_common_positions():
    cache = PagedKVCache(8, H, device="cpu")
    assert cache._common([[[0, 1], 100]]) == 0
    assert cache._common([[[0, 1], 100], [[0, 1], 128]]) == 64
    assert cache._common([[[0, 1, 2], 192], [[0, 1, 3], 150]]) == 128
    assert cache._common([[[0, 1, 2], 192], [[4, 1, 2], 192]]) == 0
    assert cache._common([[[0], 10], [[0], 10]]) == 0


def test_refusals(plain):
    cache = PagedKVCache(4, H, device="cpu")
    a, b = cache.open(), cache.open()
    with pytest.raises(ValueError, match="no session"):
        cache.fork(7)
    with pytest.raises(ValueError, match="twice"):
        cache.append([a, a], rows([1, 2]), rows([1, 2]))
    with pytest.raises(ValueError, match="same number"):
        cache.append([a, b], rows([1] * 3), rows([1] * 3))
    with pytest.raises(ValueError, match="rows of"):
        cache.append([a, b], rows([1] * 3), rows([1] * 3), [1, 1])
    with pytest.raises(ValueError, match="bfloat16"):
        cache.append([a], rows([1]).float(), rows([1]).float())
    with pytest.raises(ValueError, match="trim"):
        cache.trim(a, -1)
    cache.append([a], rows([1] * 65), rows([1] * 65))
    with pytest.raises(ValueError, match="in use"):
        cache.resize(1)
    cache.close(b)
    with pytest.raises(ValueError, match="no session"):
        cache.length(b)
    with pytest.raises(ValueError):
        PagedKVCache(0, H, device="cpu")
    batch = cache.batch([a, cache.open()])
    with pytest.raises(ValueError, match="offset"):
        batch.offset
    with pytest.raises(ValueError, match="sessions"):
        batch.update_and_fetch(torch.zeros(1, H, 1, D, dtype=torch.bfloat16),
                               torch.zeros(1, H, 1, D, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="shorter"):
        batch.attend(torch.zeros(2, 4, 3, D, dtype=torch.bfloat16), 0.1)


def test_batches_follow_the_page_lists(plain):
    cache = PagedKVCache(12, H, device="cpu")
    a, b = cache.open(), cache.open()
    one, two = cache.batch([a, b]), cache.batch([b])
    step = lambda tag, n, L: torch.full((n, H, L, D), tag, dtype=torch.bfloat16)  # noqa: E731
    one.update_and_fetch(step(1, 2, 60), step(1, 2, 60))
    two.update_and_fetch(step(2, 1, 10), step(2, 1, 10))
    assert two.offset == 70 and two.trim(3) == 3
    cache.append([a], rows([3] * 7), rows([3] * 7))
    one.update_and_fetch(step(4, 2, 1), step(4, 2, 1))
    check(cache, {a: [1] * 60 + [3] * 7 + [4], b: [1] * 60 + [2] * 7 + [4]})
    one._refresh(one._states())
    assert one._lens.tolist() == [68, 68] and one.offset == 68 and not one.empty()
    assert one._table[:, :2].tolist() == [cache.pages(a), cache.pages(b)]
    assert one.make_mask(5) == "causal" and one.make_mask(1) is None and one.is_trimmable()
    assert one.nbytes == 4 * cache.nbytes // 12
