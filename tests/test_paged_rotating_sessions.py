"""Sessions whose rows are rotated on their way in, and batches with windows, on the CPU with plain stand-ins for the
device functions: what a session holds after appends, forks and appends that fail, and which masks a batch takes."""
import pytest
import torch

from lagunalab_amd import paged
from lagunalab_amd.paged import OutOfPages, PagedKVCache
from test_paged_failures import Lost, fail_once
from test_paged_sessions import D, H, check, plain, rows  # noqa: F401


@pytest.fixture
def rotating(plain, monkeypatch):  # noqa: F811
    """The rotated append stores rows as the plain stand-in does; queries come back as they are."""
    def append(q, k, v, keys, values, table, starts, rotary, counts=None, q_norm=None, k_norm=None, eps=1e-6, fetch=False):
        assert rotary == "rotary" and (q_norm, k_norm, eps) == ("qw", "kw", 1e-5)
        paged.paged_append(k, v, keys, values, table, starts, counts)
        return (q, k, v) if fetch else q
    monkeypatch.setattr(paged, "paged_append_rotated", append)


HOW = dict(rotary="rotary", q_norm="qw", k_norm="kw", eps=1e-5)


def step(tags, L, heads=H):
    return torch.tensor(tags, dtype=torch.bfloat16)[:, None, None, None].expand(-1, L, heads, D)


def test_rows_go_to_their_sessions(rotating):
    cache = PagedKVCache(12, H, device="cpu")
    a, b = cache.open(), cache.open()
    x = rows([1] * 70 + [2] * 3)
    q = cache.append_rotated([a, b], x, x, x, counts=[70, 3], **HOW)
    assert torch.equal(q, x)
    c = cache.fork(a)
    got = cache.append_rotated([c, b], rows([3, 4]), rows([3, 4]), rows([3, 4]), fetch=True, **HOW)
    assert len(got) == 3
    want = {a: [1] * 70, b: [2] * 3 + [4], c: [1] * 70 + [3]}
    check(cache, want)
    batch = cache.batch([a, b, c], rotates=True)
    q = batch.append_rotated(step([5, 6, 7], 2, 4), step([5, 6, 7], 2), step([5, 6, 7], 2), **HOW)
    assert q.shape == (3, 4, 2, D) and (q[:, 0, :, 0] == torch.tensor([[5], [6], [7]])).all()
    for s, t in zip((a, b, c), (5, 6, 7)):
        want[s] = want[s] + [t] * 2
    check(cache, want)
    assert batch._lens.tolist() == [72, 6, 73]


@pytest.mark.parametrize("what", ["paged_append_rotated", "_tables", "copy_pages"])
@pytest.mark.parametrize("through", ["append", "batch"])
def test_an_append_that_fails_leaves_the_session(rotating, monkeypatch, what, through):
    cache = PagedKVCache(12, H, device="cpu")
    a = cache.open()
    cache.append([a], rows([1] * 100), rows([1] * 100))
    keep = cache.fork(a)
    batch = cache.batch([a], rotates=True)
    fail_once(monkeypatch, PagedKVCache if what == "_tables" else paged, what)
    with pytest.raises(Lost):
        if through == "append":
            cache.append_rotated([a], rows([9] * 140), rows([9] * 140), rows([9] * 140), **HOW)
        else:
            batch.append_rotated(step([9], 140), step([9], 140), step([9], 140), **HOW)
    check(cache, {a: [1] * 100, keep: [1] * 100})
    batch.append_rotated(step([2], 1), step([2], 1), step([2], 1), **HOW)
    check(cache, {a: [1] * 100 + [2], keep: [1] * 100})


def test_refusals(rotating, monkeypatch):
    cache = PagedKVCache(3, H, device="cpu")
    a = cache.open()
    x = rows([1] * 70)
    cache.append([a], x, x)
    for bad in (dict(sessions=[]), dict(sessions=[a, a]), dict(sessions=[a + 1]), dict(k=x[:69]), dict(v=x[:, :1]),
                dict(k=x.float()), dict(counts=[69]), dict(counts=[71, -1])):
        with pytest.raises(ValueError):
            cache.append_rotated(**dict(dict(sessions=[a], q=x, k=x, v=x, **HOW), **bad))
    with pytest.raises(OutOfPages):
        cache.append_rotated([a], *[rows([1] * 140)] * 3, **HOW)
    check(cache, {a: [1] * 70})
    batch = cache.batch([a], rotates=True)
    y = step([1], 2)
    for bad in ((step([1, 1], 2),) * 3, (y[:, :1], y, y), (y, y, y[:, :1]), (y, y[:, :, :1], y[:, :, :1]),
                (y.float(), y, y), (y, y.float(), y.float())):
        with pytest.raises(ValueError):
            batch.append_rotated(*bad, **HOW)
    with pytest.raises(ValueError, match="window"):
        cache.batch([a], window=0)
    q = torch.zeros((71, 4, D), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="shorter"):
        cache.chunk_attention([a], q, 0.1)
    with pytest.raises(ValueError, match="counts"):
        cache.chunk_attention([a], q, 0.1, counts=[3, 4])
    check(cache, {a: [1] * 70})
    monkeypatch.setattr(paged._lib, "capturing", lambda dev: True)
    for call in (lambda: cache.append_rotated([a], x, x, x, **HOW), lambda: cache.chunk_attention([a], q[:2], 0.1),
                 lambda: batch.append_rotated(y, y, y, **HOW)):
        with pytest.raises(RuntimeError, match="captured"):
            call()


def test_attention_gets_the_sessions_tables(rotating, monkeypatch):
    """What the sessions' and the batch's attention hand on."""
    seen = []

    def attend(q, keys, values, table, lens, scale, counts=None, window=None):
        seen.append((q.shape, lens.tolist(), counts, window))
        return q
    monkeypatch.setattr(paged, "paged_chunk_attention", attend)
    monkeypatch.setattr(paged, "paged_decode_attention", lambda q, *a, shared: q + 1)
    cache = PagedKVCache(8, H, device="cpu")
    a, b = cache.open(), cache.open()
    cache.append([a, b], rows([1] * 73), rows([1] * 73), [70, 3])
    q = torch.zeros((6, 4, D), dtype=torch.bfloat16)
    assert cache.chunk_attention([b, a], q, 0.1).shape == q.shape
    cache.chunk_attention([a, b], q, 0.1, counts=[6, 0], window=5)
    assert seen == [((6, 4, D), [3, 70], [3, 3], None), ((6, 4, D), [70, 3], [6, 0], 5)]
    del seen[:]
    two, one = torch.arange(2 * 4 * 2 * D).view(2, 4, 2, D).to(torch.bfloat16), torch.zeros((2, 4, 1, D), dtype=torch.bfloat16)
    wide = cache.batch([a, b], rotates=True)
    assert torch.equal(wide.attend(two, 0.1), two) and (wide.attend(one, 0.1) == 1).all()
    many = torch.zeros((2, 17 * H, 1, D), dtype=torch.bfloat16)
    assert torch.equal(wide.attend(many, 0.1), many) and seen.pop()[0] == (2, 17 * H, D)
    slide = cache.batch([a, b], window=9)
    assert torch.equal(slide.attend(two, 0.1), two) and torch.equal(slide.attend(one, 0.1), one)
    assert seen == [((4, 4, D), [70, 3], [2, 2], None), ((4, 4, D), [70, 3], [2, 2], 9), ((2, 4, D), [70, 3], [1, 1], 9)]


def test_masks(rotating):
    cache = PagedKVCache(12, H, device="cpu")
    a, b = cache.open(), cache.open()
    cache.append([a, b], rows([1] * 140), rows([1] * 140))
    slide = cache.batch([a, b], window=50)
    m = slide.make_mask(3, window_size=50)
    assert m.shape == (3, 73) and m.sum(1).tolist() == [50] * 3 and m[0, 70] and not m[0, 71]
    for other in (None, 49, 51, 72):
        with pytest.raises(ValueError, match="window"):
            slide.make_mask(3, window_size=other)
    assert cache.batch([a, b], window=80).make_mask(3) == "causal"  # neither leaves a row out
    assert cache.batch([a, b], window=80).make_mask(1) is None
    with pytest.raises(ValueError, match="full-attention"):
        cache.batch([a, b]).make_mask(3, window_size=50)
    cache.trim(b, 69)
    with pytest.raises(ValueError, match="common offset"):
        slide.make_mask(3, window_size=50)
    both = cache.batch([a, b], window=50, rotates=True)
    assert both.make_mask(3, window_size=50) == "causal" and both.make_mask(1, window_size=50) is None
    with pytest.raises(ValueError, match="window"):
        both.make_mask(3)
    with pytest.raises(ValueError, match="common offset"):
        both.make_mask(3, return_array=True, window_size=50)
    wide = cache.batch([a, b], rotates=True)
    assert wide.make_mask(3) == "causal" and wide.make_mask(1) is None
    assert wide.make_mask(3, window_size=73) == "causal"
    with pytest.raises(ValueError, match="full-attention"):
        wide.make_mask(3, window_size=72)
