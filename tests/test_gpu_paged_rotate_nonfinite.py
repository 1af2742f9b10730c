"""Infinities and NaN among the rows of ``paged_append_rotated``: they reach the dims that the formula takes them to, a
dim that is not turned no other one."""
import pytest
import torch

from lagunalab_amd.paged import paged_append_rotated
from paged_util import D, fill_pool, make_table, randn
from test_gpu_paged_rotate import gen, ints, rotary_of

pytestmark = pytest.mark.gpu

LAYOUTS = [("half", 64), ("half", 20), ("yarn", 96), ("pairs", 64), ("pairs", 6), ("pairs", 126), ("pairs", 100)]


def call(dev, rotary, q, k, ws):
    g = gen(2)
    table, pages = make_table(g, [60 + len(q)], 0)
    pool = fill_pool(g, pages, k.shape[1], dev, poison=False)
    v = randn(g, *k.shape).to(dev)
    return paged_append_rotated(q, k, v, *pool, table.to(dev), ints([60], dev), rotary, None, *ws, fetch=True)


@pytest.mark.parametrize("rows", [3, 700])  # a head per lane, and several
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("kind,dims", LAYOUTS)
def test_a_dim_that_stays_is_left_alone(dev, kind, dims, bad, rows):
    g = gen(dims)
    rotary = rotary_of(kind, dims, dev)
    hq, kv = 32, 8
    q, k = randn(g, rows, hq, D).to(dev), randn(g, rows, kv, D).to(dev)
    clean = call(dev, rotary, q, k, (None, None))
    for at in (dims, dims + 1, D - 2, D - 1):  # neighbours of each other, the first two of turned ones
        q2, k2 = q.clone(), k.clone()
        q2[-1, -1, at], k2[0, 1, at] = bad, bad
        got = call(dev, rotary, q2, k2, (None, None))
        want = clean[0].clone()
        want[-1, -1, at] = bad
        assert torch.equal(got[0].nan_to_num(7.0), want.nan_to_num(7.0)), at
        if at >= 64:  # the other group of the key, and every other key
            assert torch.equal(got[1][0, 1, :64], clean[1][0, 1, :64])
        hit = torch.zeros_like(clean[1], dtype=torch.bool)
        hit[0, 1] = True
        assert torch.equal(got[1].masked_fill(hit, 0.0), clean[1].masked_fill(hit, 0.0))
        assert torch.equal(got[2], clean[2])


@pytest.mark.parametrize("kind,dims", LAYOUTS)
def test_a_norm_weight_of_a_dim_that_stays(dev, kind, dims):
    g = gen(dims)
    rotary = rotary_of(kind, dims, dev)
    q, k = randn(g, 5, 4, D).to(dev), randn(g, 5, 2, D).to(dev)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(dev)
    clean = call(dev, rotary, q, k, (w, w))[0]
    for at in (dims, dims + 1, D - 1):
        w2 = w.clone()
        w2[at] = float("inf")
        got = call(dev, rotary, q, k, (w2, w))[0]
        assert not torch.isfinite(got[..., at]).any()
        got[..., at] = clean[..., at]
        assert torch.equal(got, clean), at


@pytest.mark.parametrize("kind,dims", LAYOUTS)
def test_a_turned_dim_reaches_its_pair_alone(dev, kind, dims):
    g = gen(dims)
    rotary = rotary_of(kind, dims, dev)
    q, k = randn(g, 5, 4, D).to(dev), randn(g, 5, 2, D).to(dev)
    clean = call(dev, rotary, q, k, (None, None))[0]
    for at in (0, 1, dims // 2, dims - 1):
        q2 = q.clone()
        q2[2, 1, at] = float("nan")
        got = call(dev, rotary, q2, k, (None, None))[0]
        pair = at ^ 1 if rotary.interleaved else (at + dims // 2) % dims
        assert got[2, 1, [at, pair]].isnan().all()
        got[2, 1, [at, pair]] = clean[2, 1, [at, pair]]
        assert torch.equal(got, clean), at
