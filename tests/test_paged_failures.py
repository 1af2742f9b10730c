"""PagedKVCache when a call fails on the way, on the CPU: nothing of it stays, and what is forked and written
afterwards is each session's own."""
import pytest
import torch

from lagunalab_amd import paged
from lagunalab_amd.paged import PagedKVCache
from test_paged_sessions import D, H, check, plain, rows  # noqa: F401


class Lost(Exception):
    pass


def fail_once(monkeypatch, owner, name):
    """owner.name raises at its next call and works again afterwards."""
    real = getattr(owner, name)

    def broken(*args, **kwargs):
        monkeypatch.setattr(owner, name, real)
        raise Lost(name)
    monkeypatch.setattr(owner, name, broken)


def step(tag, B, L):
    return torch.full((B, H, L, D), tag, dtype=torch.bfloat16)


# what raises: the rows' launch, the upload of the tables, the copy of a page that is shared; the row goes to a
# new page or to a part-filled one
@pytest.mark.parametrize("what,had", [("paged_append", 64), ("paged_append", 100), ("_tables", 64),
                                      ("_tables", 100), ("copy_pages", 100)])
@pytest.mark.parametrize("through", ["append", "batch"])
def test_an_append_that_fails_leaves_no_pages_behind(plain, monkeypatch, what, had, through):  # noqa: F811
    cache = PagedKVCache(12, H, device="cpu")
    a = cache.open()
    cache.append([a], rows([1] * had), rows([1] * had))
    if what == "copy_pages":
        keep = cache.fork(a)
    batch = cache.batch([a])
    free = cache.free_pages
    fail_once(monkeypatch, PagedKVCache if what == "_tables" else paged, what)
    with pytest.raises(Lost):
        if through == "append":
            cache.append([a], rows([9] * 140), rows([9] * 140))
        else:
            batch.update_and_fetch(step(9, 1, 140), step(9, 1, 140))
    want = {a: [1] * had}
    if what == "copy_pages":
        want[keep] = [1] * had
        assert cache.free_pages == free
    check(cache, want)
    # forks of it write to pages of their own, also through the batch made before
    b = cache.fork(a)
    cache.append([b], rows([3]), rows([3]))
    batch.update_and_fetch(step(2, 1, 1), step(2, 1, 1))
    want[a], want[b] = want[a] + [2], want[a] + [3]
    check(cache, want)
    batch._refresh(batch._states())
    assert batch._lens.tolist() == [had + 1]
    assert batch._table[0, :len(cache.pages(a))].tolist() == cache.pages(a)


def test_lengths_that_cannot_be_made_leave_a_batch_as_it_was(plain, monkeypatch):  # noqa: F811
    """The step's new lengths are a device tensor: if there is none, the step did not happen."""
    cache = PagedKVCache(6, H, device="cpu")
    a, b = cache.open(), cache.open()
    batch = cache.batch([a, b])
    batch.update_and_fetch(step(1, 2, 63), step(1, 2, 63))

    class Full:
        def __add__(self, n):
            raise Lost("out of memory")

        def tolist(self):
            return [63, 63]
    batch._lens = Full()
    with pytest.raises(Lost):
        batch.update_and_fetch(step(9, 2, 1), step(9, 2, 1))
    check(cache, {a: [1] * 63, b: [1] * 63})
    batch.update_and_fetch(step(2, 2, 2), step(2, 2, 2))
    check(cache, {a: [1] * 63 + [2] * 2, b: [1] * 63 + [2] * 2})
    assert batch._lens.tolist() == [65, 65]


class Stored:
    """A contiguous cache of n rows, as adopt reads one."""

    def __init__(self, n, words=torch.bfloat16):
        def buf():
            return (torch.ones(1, H, n, D, dtype=torch.uint8), torch.ones(1, H, n, 2, dtype=words),
                    torch.zeros(1, H, n, 2, dtype=words))
        self.state = buf(), buf()


class Unreadable(torch.Tensor):
    def __getitem__(self, i):
        raise Lost("copy")


@pytest.mark.parametrize("n", [200, 128, 10])
def test_a_cache_that_cannot_be_copied_takes_no_pages(plain, n):  # noqa: F811
    cache = PagedKVCache(6, H, device="cpu")
    src = Stored(n)
    src.state[1][2].__class__ = Unreadable  # the last of the copies
    with pytest.raises(Lost):
        cache.adopt(src)
    assert cache.free_pages == 6 and not cache._sessions
    s = cache.adopt(Stored(n))
    check(cache, {s: [1] * n})


@pytest.mark.parametrize("words", [torch.float16, torch.float32])
@pytest.mark.parametrize("part", [0, 1])
def test_a_cache_of_other_scales_is_not_adopted(plain, words, part):  # noqa: F811
    """Its scales or biases would be rounded to bf16: other values than the cache holds."""
    cache = PagedKVCache(6, H, device="cpu")
    src = Stored(70)
    src.state = tuple(Stored(70, words).state[i] if i == part else src.state[i] for i in range(2))
    with pytest.raises(ValueError, match="bfloat16"):
        cache.adopt(src)
    assert cache.free_pages == 6 and not cache._sessions


def test_a_resize_that_fails_keeps_the_pool(plain, monkeypatch):  # noqa: F811
    cache = PagedKVCache(6, H, device="cpu")
    s = cache.open()
    cache.append([s], rows([7] * 100), rows([7] * 100))

    class NoStores(torch.Tensor):
        def __setitem__(self, i, x):
            raise Lost("copy")
    real = paged.page_pool

    def broken(*args):
        made = real(*args)
        made[1][0].__class__ = NoStores
        return made
    monkeypatch.setattr(paged, "page_pool", broken)
    with pytest.raises(Lost):
        cache.resize(9)
    check(cache, {s: [7] * 100})
    assert cache.keys[0].shape[0] == 6 and cache.free_pages == 4
    monkeypatch.setattr(paged, "page_pool", real)
    cache.resize(9)
    check(cache, {s: [7] * 100})
    assert cache.keys[0].shape[0] == 9 and cache.free_pages == 7


def test_masks_of_a_window_that_ends_before_the_rows_are_refused(plain):  # noqa: F811
    """attend() is causal over all rows: a sliding-window layer gets that only while its window covers them."""
    cache = PagedKVCache(6, H, device="cpu")
    batch = cache.batch([cache.open(), cache.open()])
    batch.update_and_fetch(step(1, 2, 60), step(1, 2, 60))
    with pytest.raises(ValueError, match="window"):
        batch.make_mask(1, window_size=60)
    with pytest.raises(ValueError, match="window"):
        batch.make_mask(8, window_size=67)
    with pytest.raises(ValueError, match="window"):
        batch.make_mask(1, window_size=0)
    for n, window in ((1, 61), (8, 68), (8, 500)):  # the whole of what the rows see
        q, k = torch.arange(60, 60 + n)[:, None], torch.arange(60 + n)[None]
        assert torch.equal(batch.make_mask(n, window_size=window), k <= q)
    assert batch.make_mask(8) == "causal" and batch.make_mask(1) is None
    assert torch.equal(batch.make_mask(8, return_array=True), batch.make_mask(8, window_size=68))


def test_a_model_with_a_sliding_window_layer_is_refused(plain):  # noqa: F811
    from tiny_model import TinyArgs, TinyLM
    model = TinyLM(TinyArgs(layer_types=["sliding_attention"]))
    cache = PagedKVCache(6, H, device="cpu")
    s = cache.open()
    with pytest.raises(ValueError, match="window"), torch.no_grad():
        model(torch.tensor([[1, 2, 3, 4, 5, 6, 7, 8, 9]]), cache=[cache.batch([s])])
    assert cache.length(s) == 0 and cache.free_pages == 6


def test_nothing_of_the_session_layer_runs_in_a_captured_graph(plain, monkeypatch):  # noqa: F811
    """Its lists and lengths move on the host, once: a replay would write the same rows again."""
    cache = PagedKVCache(8, H, device="cpu")
    a, b = cache.open(), cache.open()
    cache.append([a, b], rows([1] * 80), rows([1] * 80))
    cache.close(cache.fork(a))
    batch = cache.batch([a, b])
    q = torch.zeros(2, 4, 1, D, dtype=torch.bfloat16)
    monkeypatch.setattr(paged._lib, "capturing", lambda dev: True)
    for call in (lambda: cache.append([a], rows([2]), rows([2])), lambda: cache.rows([a]),
                 lambda: cache.attention([a, b], q, 0.1), lambda: cache.compact(), lambda: cache.resize(9),
                 lambda: cache.adopt(Stored(70)), lambda: batch.update_and_fetch(step(2, 2, 1), step(2, 2, 1)),
                 lambda: batch.attend(q, 0.1)):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    check(cache, {a: [1] * 40, b: [1] * 40})
    monkeypatch.undo()
    assert paged._lib.capturing(torch.device("cpu")) is False
