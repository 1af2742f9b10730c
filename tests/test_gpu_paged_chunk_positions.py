"""Every position that a row of chunk attention sees, once and no other, at the lengths that serving reaches: equal
weights over V rows that name their key. A call has a pair of pages whose 128 keys are 1 in a dim each, another pair for
every KV head, all other rows being 0; over the calls every key of every sequence is named. A lost or doubled key shows as
such, where a bound on ordinary rows would let 32 of 30,000 keys pass."""
import ctypes as C

import pytest
import torch

from lagunalab_amd import _lib
from lagunalab_amd.paged import paged_chunk_attention
from paged_util import D, PAGE, make_table, randn
from test_gpu_paged_chunk import SCALE, assert_within, exact, sessions

NAMED = 2 * PAGE  # keys of a pair of pages


def share_of(first, n, c, window):
    """What the last c of n positions take of the named keys first .. first + 127 under equal weights: [c, 128]."""
    at, key = torch.arange(n - c, n)[:, None], first + torch.arange(NAMED)
    sees = (key <= at) & (key > at - (window or 1 << 40))
    seen = torch.clamp(at + 1, max=window or 1 << 40)
    return sees.double() / seen.clamp(min=1)


def assert_shares(got, want, what):
    """The weights are 1 and the sums whole numbers below 2^24, exact but for the reciprocal and the product (2^-24
    each, with room); the output is rounded to bf16 (2^-8)."""
    bad = ~((got.double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -20))
    assert not bad.any(), f"{what}: {int(bad.sum())} values, of dims {bad.nonzero()[:4, -1].tolist()}"


def test_a_missing_half_page_would_show():
    """Mistakes planted in what is expected: a key less or twice, one more position in the count of a short row, a row
    that sees one key too many or too few."""
    n, c = 82671, 5
    first = n - NAMED
    want = share_of(first, n, c, None)
    assert_shares(want.to(torch.bfloat16), want, "as it is")
    assert (want[-1] > 0).all() and (want[0] > 0).sum() == NAMED - 4
    for spoil in (lambda x: x[:, 32:64].zero_(), lambda x: x[0, 5].zero_(), lambda x: x[:, 7].mul_(2),
                  lambda x: x[0, -4].fill_(1 / n), lambda x: x[2, -3].zero_()):
        other = want.clone()
        spoil(other)
        with pytest.raises(AssertionError, match="values"):
            assert_shares(want.to(torch.bfloat16), other, "spoiled")
    # a window's edge, both sides
    want = share_of(n - 600, n, c, 512)
    assert (want[0] > 0).sum() == NAMED - (600 - 516) and want[0].max() == 1 / 512
    for window in (511, 513):
        with pytest.raises(AssertionError):
            assert_shares(want.to(torch.bfloat16), share_of(n - 600, n, c, window), "window")


# heads, lengths, rows, window, pages of a table's row beyond the longest
LONG = [
    (32, 8, [82671], [5], None, 0),           # one block of few rows, dealt out
    (32, 8, [42771], [1], None, 900),         # a table wider than the sequence
    (48, 8, [42771], [8], None, 0),           # two blocks of 32
    (48, 8, [82671], [16], None, 0),          # two of 64
    (4, 4, [30000], [2], 29000, 0),           # a long window
    (32, 8, [50003, 20011, 700], [1, 8, 2], None, 0),
    (48, 8, [8191] * 7 + [60], [1] * 8, 512, 0),  # short windows, taken whole
    (8, 8, [60001, 333], [100, 120], None, 0),    # blocks of 128 rows, in shares
    (48, 8, [82671], [40], None, 0),          # one of 256
    (32, 8, [42771, 5000], [300, 70], 40000, 0),
    (48, 8, [12000, 9000, 63], [257, 3, 2], None, 30),  # both kinds in a call
    (16, 16, [9000], [700], 1000, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,kv,lens,counts,window,spare", LONG)
def test_every_key_counts_once(dev, hq, kv, lens, counts, window, spare):
    g = torch.Generator().manual_seed(sum(lens))
    table, pages = make_table(g, lens, 0, width_spare=spare)
    codes = torch.randint(0, 256, (pages, kv, PAGE, D), generator=g, dtype=torch.uint8).to(dev)
    used = torch.zeros((pages, PAGE), dtype=torch.bool)
    for b, n in enumerate(lens):
        at = torch.arange(n)
        used[table[b, at // PAGE].long(), at % PAGE] = True
    scales, biases = (torch.where(used, x, float("nan"))[:, None, :, None].expand(-1, kv, -1, 2).to(torch.bfloat16).to(dev)
                      for x in (1.0, 0.0))
    named = torch.zeros_like(codes)
    keys, values = (codes, scales, biases), (named, scales, biases)
    q = randn(g, sum(counts), hq, D).to(dev)
    t_d, n_d = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    eye = torch.eye(NAMED, dtype=torch.uint8, device=dev).view(2, PAGE, D)
    calls = -(-max(-(-n // NAMED) for n in lens) // kv)
    for i in range(calls):
        named.zero_()
        for b, n in enumerate(lens):
            for h in range(kv):
                for half in range(2):
                    p = 2 * (kv * i + h) + half
                    if PAGE * p < n:
                        named[table[b, p].item(), h] = eye[half]
        out = paged_chunk_attention(q, keys, values, t_d, n_d, 0.0, counts, window).view(-1, kv, hq // kv, D)
        a = 0
        for b, (n, c) in enumerate(zip(lens, counts)):
            want = torch.stack([share_of(NAMED * (kv * i + h), n, c, window) for h in range(kv)], 1)
            assert_shares(out[a:a + c], want[:, :, None].to(dev), f"sequence {b}, call {i}")
            a += c


@pytest.mark.gpu
@pytest.mark.parametrize("heads,counts", [(200, [300, 140]), (300, [120, 97, 100])])
@pytest.mark.parametrize("window", [None, 200])
def test_more_kv_heads_than_shares(dev, heads, counts, window):
    """As many KV heads as workgroups or more, a table too wide for whole blocks: one share per KV head, which walks every
    block of every sequence and cuts none, so that there is nothing to merge."""
    g = torch.Generator().manual_seed(heads)
    lens = [500, 333, 120][:len(counts)]
    pool, table = sessions(g, heads, lens, dev, spare=60)
    need = _lib.load().lq_paged_chunk_workspace_bytes((C.c_int32 * len(counts))(*counts), len(counts), heads, heads,
                                                      table.shape[1], window or 0)
    assert need == 0
    q = randn(g, sum(counts), heads, D).to(dev)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = paged_chunk_attention(q, *pool, table.to(dev), n_d, SCALE, counts, window)
    assert_within(out, *exact(q, pool, table, lens, counts, window, SCALE))
