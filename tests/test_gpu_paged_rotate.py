"""``paged_append_rotated``: norm and rotation of projected rows and their way into the pages, against the formulas in
64 bits, and against the plain append where nothing is normed or turned."""
import pytest
import torch

from lagunalab_amd.paged import paged_append, paged_append_rotated, paged_gather
from lagunalab_amd.rotary import Rotary
from paged_util import D, PAGE, fill_pool, make_table, randn

pytestmark = pytest.mark.gpu
EPS = 1e-6
YARN = {"rope_type": "yarn", "rope_theta": 5e5, "factor": 32.0, "original_max_position_embeddings": 4096}


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def exact_rows(x, pos, w, rotary, eps=EPS):
    """Rows [T, H, 128] normed and turned, in 64 bits, on the CPU, and how far fp32 may be off: the sum of squares
    and the root 2^-20 relative, a product's or sum's roundings a few 2^-24, sines and cosines 2^-22."""
    x = x.double().cpu()
    if w is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w.double().cpu()
    size = x.abs()
    if rotary is not None and rotary.dims:
        f = rotary.inv_freq.double().cpu()
        n = len(f)
        a = torch.outer(pos.double(), f)[:, None]
        c, s = a.cos() * rotary.mscale, a.sin() * rotary.mscale
        i = torch.arange(n)
        one, two = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + n)
        p, q = x[..., one], x[..., two]
        x, size = x.clone(), size.clone()
        x[..., one], x[..., two] = p * c - q * s, p * s + q * c
        big = (p.abs() + q.abs()) * rotary.mscale
        size[..., one] = size[..., two] = big
    return x, size * 2.0 ** -18 + 1e-30


def positions(starts, counts):
    return torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)]) if sum(counts) else torch.zeros(0)


def rotary_of(kind, dims, dev):
    if kind is None:
        return None
    rope = dict(YARN if kind == "yarn" else {"rope_theta": 1e4}, partial_rotary_factor=dims / D)
    return Rotary.of(rope, dev, interleaved=kind == "pairs")


def case(g, hq, kv, starts, counts, dev, norm, std=1.0):
    T = sum(counts)
    table, pages = make_table(g, [s + c for s, c in zip(starts, counts)], 0)
    pool = fill_pool(g, pages, kv, dev)
    proj = randn(g, T, (hq + 2 * kv) * D + 8, std=std).to(dev)
    q, k, v = (x.unflatten(1, (-1, D)) for x in proj[:, :-8].split([hq * D, kv * D, kv * D], 1))
    ws = tuple((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(dev) for _ in range(2)) if norm else (None, None)
    return q, k, v, pool, table.to(dev), ws


def check(dev, hq, kv, starts, counts, rotary, norm, seed=0, std=1.0, eps=EPS):
    q, k, v, pool, table, (qw, kw) = case(gen(seed), hq, kv, starts, counts, dev, norm, std)
    before = [t.clone() for buf in pool for t in buf]
    s_d = ints(starts, dev)
    got_q, got_k, got_v = paged_append_rotated(q, k, v, *pool, table, s_d, rotary, counts, qw, kw, eps=eps, fetch=True)
    pos = positions(starts, counts)
    want, off = exact_rows(q, pos, qw, rotary, eps)
    # one rounding to bf16
    assert ((got_q.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2 * off).all()
    # values and what the pages hold
    other = fill_pool(gen(1), pool[0][0].shape[0], kv, dev)
    paged_append(v, v, *other, table, s_d, counts)
    rows_k, rows_v = paged_gather(*pool, table, s_d, counts)
    assert torch.equal(rows_v, paged_gather(*other, table, s_d, counts)[1]) and torch.equal(rows_v, got_v)
    assert torch.equal(rows_k, got_k)
    # keys: half a step of the codes, scale and bias rounded to bf16 (2^-8 of each), the value too
    want, off = exact_rows(k, pos, kw, rotary, eps)
    groups = want.unflatten(-1, (2, 64))
    span = (groups.amax(-1) - groups.amin(-1)).repeat_interleave(64, -1)
    edge = groups.abs().amax(-1).repeat_interleave(64, -1)
    # the scale is the edge over a whole number of steps: up to half a step of 127 longer than span / 255
    step = span / 255 * (1 + 1 / 254) + 1e-7
    bound = step / 2 + (255 * step + edge) * 2.0 ** -8 + want.abs() * 2.0 ** -8 + 4 * off
    assert ((got_k.double().cpu() - want).abs() <= bound).all()
    # and nothing else was written
    used = torch.zeros(pool[0][0].shape[0], PAGE, dtype=torch.bool)
    t = table.cpu()
    for b, (s, c) in enumerate(zip(starts, counts)):
        at = torch.arange(s, s + c)
        used[t[b, at // PAGE].long(), at % PAGE] = True
    free = (~used)[:, None].expand(-1, kv, -1).to(dev)
    for now, old in zip([t for buf in pool for t in buf], before):
        bits = (lambda x: x) if now.dtype == torch.uint8 else (lambda x: x.view(torch.int16))
        assert torch.equal(bits(now)[free], bits(old)[free])


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("kind,dims", [(None, 0), ("half", 128), ("half", 64), ("half", 32), ("half", 96), ("half", 20),
                                       ("half", 4), ("yarn", 64), ("yarn", 128), ("pairs", 128), ("pairs", 64), ("pairs", 6)])
def test_layouts(dev, kind, dims, norm):
    rotary = rotary_of(kind, dims, dev)
    for hq, kv, starts, counts in ((32, 8, [1037], [1]), (6, 2, [0, 63, 5, 128], [3, 2, 0, 70]), (1, 1, [64], [1]),
                                   (5, 3, [7, 8], [1, 1])):
        check(dev, hq, kv, starts, counts, rotary, norm, seed=dims + hq)


@pytest.mark.parametrize("kind", ["half", "pairs", "yarn"])
def test_many_rows(dev, kind):
    rotary = rotary_of(kind, 64, dev)
    check(dev, 48, 8, [700, 0, 9], [300, 1, 211], rotary, True)
    check(dev, 7, 3, [0], [1500], rotary, True)
    check(dev, 8, 2, [3 * i for i in range(90)], [i % 5 for i in range(90)], rotary, False)


def test_far_positions(dev):
    """Angles of positions where a product in 32 bits would be off by up to a radian: the table has the last page only
    for those, the others are not read."""
    g = gen(3)
    rotary = rotary_of("half", 128, dev)
    pool = fill_pool(g, 4, 2, dev)
    width = (1 << 24) // PAGE
    table = torch.zeros((1, width), dtype=torch.int32, device=dev)
    for start in (82671, 1 << 20, (1 << 24) - 2):
        q, k, v = (randn(g, 2, h, D).to(dev) for h in (4, 2, 2))
        got = paged_append_rotated(q, k, v, *pool, table, ints([start], dev), rotary, [2])
        want, off = exact_rows(q, torch.arange(start, start + 2), None, rotary)
        assert ((got.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2 * off).all()


@pytest.mark.parametrize("std,eps", [(1e-3, 1e-6), (100.0, 1e-6), (1e-12, 1e-6), (1.0, 0.0), (1e15, 1e-5)])
def test_magnitudes(dev, std, eps):
    check(dev, 4, 2, [5, 100], [3, 2], rotary_of("half", 64, dev), True, std=std, eps=eps)


def test_nothing_normed_or_turned_is_the_plain_append(dev):
    g = gen(4)
    starts, counts = [60, 3], [70, 9]
    q, k, v, pool, table, _ = case(g, 4, 2, starts, counts, dev, False)
    other = fill_pool(gen(9), pool[0][0].shape[0], 2, dev)
    for a, b in zip((t for buf in pool for t in buf), (t for buf in other for t in buf)):
        b.copy_(a)
    paged_append(k, v, *other, table, ints(starts, dev), counts)
    for rotary in (None, Rotary(torch.zeros(0, device=dev))):
        got = paged_append_rotated(q, k, v, *pool, table, ints(starts, dev), rotary, counts)
        assert torch.equal(got, q)
        for a, b in zip((t for buf in pool for t in buf), (t for buf in other for t in buf)):
            bits = torch.uint8 if a.dtype == torch.uint8 else torch.int16
            assert torch.equal(a.view(bits), b.view(bits))


def test_rows_that_are_not_stored_still_come_back(dev):
    g = gen(5)
    rotary = rotary_of("half", 64, dev)
    q, k, v, pool, table, (qw, kw) = case(g, 4, 2, [0, 0, 0], [3, 3, 3], dev, True)
    before = [t.clone() for buf in pool for t in buf]
    bad = table.clone()
    bad[1] = pool[0][0].shape[0]
    bad[2] = -1
    starts = ints([-2, 5, 7], dev)  # of the first, position 0 alone exists
    got = paged_append_rotated(q, k, v, *pool, bad, starts, rotary, [3, 3, 3], qw, kw, fetch=True)
    want, off = exact_rows(q, torch.tensor([-2, -1, 0, 5, 6, 7, 7, 8, 9]), qw, rotary)
    assert ((got[0].double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2 * off).all()
    assert torch.isfinite(got[1]).all() and torch.isfinite(got[2]).all()
    slot = (int(table[0, 0]), 0)
    for now, old in zip((t for buf in pool for t in buf), before):
        bits = (lambda x: x) if now.dtype == torch.uint8 else (lambda x: x.view(torch.int16))
        same = bits(now) == bits(old)
        same[slot[0], :, slot[1]] = True
        assert same.all()
    assert torch.equal(paged_gather(*pool, table, ints([0, 0, 0], dev), [1, 0, 0])[0], got[1][2:3])


def test_captured_appends_follow_positions(dev):
    g = gen(6)
    rotary = rotary_of("yarn", 64, dev)
    counts = [2, 1, 4]
    q, k, v, pool, table, (qw, kw) = case(g, 12, 2, [200, 300, 100], counts, dev, True)
    s_d = ints([0, 0, 0], dev)
    paged_append_rotated(q, k, v, *pool, table, s_d, rotary, counts, qw, kw, fetch=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_append_rotated(q, k, v, *pool, table, s_d, rotary, counts, qw, kw, fetch=True)
    for starts in ([5, 6, 7], [190, 63, 90], [62, 290, 0]):
        s_d.copy_(torch.tensor(starts, dtype=torch.int32))
        graph.replay()
        rows = paged_gather(*pool, table, s_d, counts)
        want = paged_append_rotated(q, k, v, *pool, table, s_d, rotary, counts, qw, kw, fetch=True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(rows[0], want[1]) and torch.equal(rows[1], want[2])


def test_no_rows_and_rows_of_odd_strides(dev):
    g = gen(7)
    rotary = rotary_of("half", 64, dev)
    q, k, v, pool, table, (qw, kw) = case(g, 4, 2, [3], [5], dev, True)
    want = paged_append_rotated(q, k, v, *pool, table, ints([3], dev), rotary, None, qw, kw, fetch=True)
    odd = [torch.empty(5, x.shape[1] * D + 1, dtype=torch.bfloat16, device=dev)[:, 1:].unflatten(1, (-1, D)) for x in (q, k, v)]
    for x, y in zip(odd, (q, k, v)):
        x.copy_(y)
    got = paged_append_rotated(*odd, *pool, table, ints([3], dev), rotary, None, qw, kw, fetch=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    none = paged_append_rotated(q[:0], k[:0], v[:0], *pool, table, ints([3], dev), rotary, [0], fetch=True)
    assert [t.shape[0] for t in none] == [0, 0, 0]
    keys_alone = paged_append_rotated(q[:, :0], k, v, *pool, table, ints([3], dev), rotary, None, None, kw)
    assert keys_alone.shape == (5, 0, D)
    assert torch.equal(paged_gather(*pool, table, ints([3], dev), [5])[0], want[1])
