"""Every form of the paged decode kernel and every way of dealing out prompts, on values that name their page or
their key (one lost, doubled or taken from elsewhere shows at any length), at the scales and magnitudes where a
form's own arithmetic could go wrong, and on pages beyond 4 GB. Which form a call takes follows from its shape;
the tests check that the shapes here take the one they mean."""
import ctypes as C
import math

import pytest
import torch

from lagunalab_amd import _lib
from lagunalab_amd.paged import copy_pages, paged_append, paged_decode_attention, paged_gather
from lagunalab_amd.prompt_attn import prompt_attention
from paged_util import D, PAGE, assert_within, exact_attention, make_table, randn, read_rows, write_rows

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5

# (query heads, KV heads, sequences, shared positions): pages dealt out; the shared ones with them (9 query rows);
# shared parts for blocks of 32, 64 and 128 rows, for two blocks; parts of 32 pages, whose last ones are left
# to the workgroups of own pages
FORMS = {
    "dealt out": (8, 2, 9, 0), "dealt out, 16 rows": (32, 2, 9, 0), "shared dealt out": (16, 16, 9, 512),
    "blocks of 32": (32, 16, 9, 512), "blocks of 64": (64, 16, 9, 512), "blocks of 128": (64, 8, 9, 1024),
    "two blocks": (128, 8, 9, 1024), "late pages": (128, 64, 9, 8192),
}
SPARE = 17  # pages that a table row has beyond the longest: tables of up to 16 take whole sequences


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def workspace(B, hq, kv, pages):
    return _lib.load().lq_paged_decode_workspace_bytes(B, hq, kv, pages)


def lengths(B, shared, most=300):
    """Own positions from none to several pages, sequences that end before the shared part, with it, and in it."""
    g = gen(shared + B)
    lens = [shared + int(n) for n in torch.randint(1, most, (B,), generator=g)]
    if shared:
        lens[0], lens[1], lens[2], lens[3] = shared - 1, shared, 1, shared // 2 + 5
    else:
        lens[0], lens[1], lens[2], lens[3] = 63, 64, 1, 0
    return lens


def check_form(form, table):
    hq, kv, B, shared = FORMS[form]
    assert table.shape[1] > 16
    # read once: with rows of partial results for them
    once = workspace(B, hq, kv, shared // PAGE) > workspace(B, hq, kv, 0)
    assert once == (shared > 0)


def names(pages, kv, by):
    """The dim that names a pool's slot [pages, kv, 64]: by its page or by its key."""
    at, heads = torch.arange(pages)[:, None, None], torch.arange(kv)[:, None]
    return ((5 * at + 3 * heads + (37 * torch.arange(PAGE) if by == "key" else 0)) % D).expand(pages, kv, PAGE)


def wanted(dim, table, lens):
    """What every sequence and KV head gets of rows that are 1 in their dim, under equal weights."""
    kv = dim.shape[1]
    want = torch.zeros((len(lens), kv, D), dtype=torch.float64)
    for b, n in enumerate(lens):
        if n:
            p, slot = table[b, torch.arange(n) // PAGE].long(), torch.arange(n) % PAGE
            want[b].scatter_add_(1, dim[p, :, slot].T, torch.ones((kv, n), dtype=torch.float64))
            want[b] /= n
    return want


def named(seed, dim, table, lens, dev):
    """A pool whose V rows are 1 in their dim; slots that no sequence has hold NaN scales."""
    pages, kv, _ = dim.shape
    used = torch.zeros((pages, PAGE), dtype=torch.bool)
    for b, n in enumerate(lens):
        used[table[b, torch.arange(n) // PAGE].long(), torch.arange(n) % PAGE] = True
    v = torch.zeros((pages, kv, PAGE, D), dtype=torch.uint8).scatter_(3, dim[..., None], 1)
    k = torch.randint(0, 256, (pages, kv, PAGE, D), generator=gen(seed), dtype=torch.uint8)
    scales, biases = (torch.where(used, x, float("nan"))[:, None, :, None].expand(-1, kv, -1, 2)
                      .to(torch.bfloat16) for x in (1.0, 0.0))
    return [tuple(t.contiguous().to(dev) for t in (codes, scales, biases)) for codes in (k, v)]


def assert_named(out, want, what):
    """Equal weights: sums and their quotient of whole numbers below 2^24, exact but for the reciprocal and the
    product (2^-24 each, with room), rounded to bf16 (2^-8)."""
    got = out.double().cpu()
    off = (got - want).abs() - want * (2.0 ** -8 + 2.0 ** -20)
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} values, by up to {off.max().item():.3g}"


@pytest.mark.parametrize("by", ["page", "key"])
@pytest.mark.parametrize("form", FORMS)
def test_every_page_and_key_counts_once(dev, form, by):
    hq, kv, B, shared = FORMS[form]
    lens = lengths(B, shared)
    table, pages = make_table(gen(1), lens, shared, width_spare=SPARE)
    check_form(form, table)
    dim = names(pages, kv, by)
    pool = named(2, dim, table, lens, dev)
    q = randn(gen(3), B, hq, 1, D).to(dev)
    n_d = torch.zeros(B, dtype=torch.int32, device=dev)
    # shorter by up to two pages and a part: the shared part's end passes through the lengths
    for less in (0, 1, 64, 150):
        now = [max(0, n - less) for n in lens]
        n_d.copy_(torch.tensor(now, dtype=torch.int32))
        out = paged_decode_attention(q, *pool, table.to(dev), n_d, 0.0, shared=shared)
        want = wanted(dim, table, now).repeat_interleave(hq // kv, 1)[:, :, None]
        assert_named(out, want, f"{form}, {less} fewer")


@pytest.mark.parametrize("by", ["page", "key"])
@pytest.mark.parametrize("hq,kv,lens,spare", [
    (4, 1, [16390, 5], 0), (32, 8, [16001], 0), (16, 1, [1024, 1023, 577], 0), (32, 8, [130] * 33 + [1000], 0),
    (6, 2, list(range(0, 640, 7)), 9), (3, 3, [2, 9000, 1, 700], 0),
])
def test_every_page_and_key_of_single_sequences(dev, hq, kv, lens, spare, by):
    table, pages = make_table(gen(4), lens, 0, width_spare=spare)
    dim = names(pages, kv, by)
    pool, want = named(5, dim, table, lens, dev), wanted(dim, table, lens)
    q = randn(gen(6), len(lens), hq, 1, D).to(dev)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = paged_decode_attention(q, *pool, table.to(dev), n_d, 0.0)
    assert_named(out, want.repeat_interleave(hq // kv, 1)[:, :, None], "single")


def rows_case(form, dev, vstd=1.0, own=90):
    """Quantized rows of a form's sequences: (pool, table, lens)."""
    hq, kv, B, shared = FORMS[form]
    lens = lengths(B, shared, own if shared else 1500)
    g = gen(7)
    table, pages = make_table(g, lens, shared, width_spare=SPARE)
    check_form(form, table)
    pool = []
    for _ in range(2):  # what no sequence has: NaN
        codes = torch.randint(0, 256, (pages, kv, PAGE, D), generator=g, dtype=torch.uint8)
        words = torch.full((pages, kv, PAGE, 2), float("nan"), dtype=torch.bfloat16)
        pool.append((codes.to(dev), words.to(dev), words.to(dev)))
    if shared:
        longest = max(range(B), key=lambda b: lens[b])
        write_rows(pool, table[longest], randn(g, shared, kv, D), randn(g, shared, kv, D, std=vstd))
    for b, n in enumerate(lens):
        if n > shared:
            write_rows(pool, table[b], randn(g, n - shared, kv, D), randn(g, n - shared, kv, D, std=vstd), shared)
    return pool, table, lens


def check_rows(out, q, pool, table, lens, scale, rows):
    hq, kv = q.shape[1], pool[0][0].shape[1]
    G = hq // kv
    for b in rows:
        k, v = (read_rows(buf, table[b], lens[b]) for buf in pool)
        for h in range(kv):
            want, bound = exact_attention(q[b, h * G:(h + 1) * G, 0].double(), k[:, h], v[:, h],
                                          [lens[b] - 1] * G, scale)
            assert_within(out[b, h * G:(h + 1) * G, 0], want, bound, f"sequence {b} head {h}")


SMALLER = [f for f in FORMS if f != "late pages"]


@pytest.mark.parametrize("form", SMALLER)
def test_forms_at_other_scales(dev, form):
    hq, kv, B, shared = FORMS[form]
    pool, table, lens = rows_case(form, dev)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    for scale, std in ((-SCALE, 1.0), (0.0, 1.0), (1.0, 1.0), (SCALE, 30.0), (SCALE, 1e-6)):
        q = randn(gen(8), B, hq, 1, D, std=std)
        out = paged_decode_attention(q.to(dev), *pool, table.to(dev), n_d, scale, shared=shared)
        check_rows(out, q, pool, table, lens, scale, [0, 4, B - 1])


@pytest.mark.parametrize("vstd", [1e20, 1e-20])
@pytest.mark.parametrize("form", SMALLER)
def test_forms_at_large_and_tiny_values(dev, form, vstd):
    hq, kv, B, shared = FORMS[form]
    pool, table, lens = rows_case(form, dev, vstd=vstd)
    q = randn(gen(9), B, hq, 1, D)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = paged_decode_attention(q.to(dev), *pool, table.to(dev), n_d, SCALE, shared=shared)
    check_rows(out, q, pool, table, lens, SCALE, [0, 1, B - 1])


def test_late_pages_at_other_scales(dev):
    hq, kv, B, shared = FORMS["late pages"]
    pool, table, lens = rows_case("late pages", dev, own=30)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    for scale, std in ((-SCALE, 1.0), (SCALE, 30.0)):
        q = randn(gen(10), B, hq, 1, D, std=std)
        out = paged_decode_attention(q.to(dev), *pool, table.to(dev), n_d, scale, shared=shared)
        check_rows(out, q, pool, table, lens, scale, [B - 1])


@pytest.mark.parametrize("kv,pages,second", [
    (2, 16, 8),    # whole sequences, 8 waves: a wave takes every eighth page
    (300, 9, 4),   # 4 waves
    (64, 200, 4),  # dealt out in 8 shares of 26 pages, a wave's every fourth
])
def test_a_weight_counts_the_same_in_values_and_sum(dev, kv, pages, second):
    """Two keys that one wave meets in turn, the second's weight 128.4 times the first's (below the 2^8 at which
    a running maximum moves), the others' 2^-93. 128.4 rounds to 128 in bf16. In the values and in the sum alike
    that moves the result by 0.4 / 128.4 of 128.4 / 129.4^2 of the two values' difference, 2.4e-5; in one of
    them by 0.3%, which shows beside a bf16 result's half step in half of the dims."""
    g = gen(13)
    steps = 15
    scale = math.log(128.4) / steps
    k = torch.zeros((pages, kv, PAGE, D), dtype=torch.uint8)
    first, last = (0, 5), (second, 33)  # page, slot
    k[first[0], :, first[1], 0], k[last[0], :, last[1], 0] = 200, 200 + steps
    v = torch.randint(0, 256, (pages, kv, PAGE, D), generator=g, dtype=torch.uint8)
    word = lambda x: torch.full((pages, kv, PAGE, 2), x, dtype=torch.bfloat16, device=dev)  # noqa: E731
    pool = (k.to(dev), word(1.0), word(0.0)), (v.to(dev), word(2.0 ** -6), word(-2.0))
    q = torch.zeros((1, kv, 1, D), dtype=torch.bfloat16)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32)[None].to(dev)
    n_d = torch.tensor([64 * pages], dtype=torch.int32, device=dev)
    out = paged_decode_attention(q.to(dev), *pool, table, n_d, scale)
    a, b = (v[p, :, s].double() * 2.0 ** -6 - 2 for p, s in (first, last))
    want = (a + 128.4 * b) / 129.4
    # and fp32: the scale, scores of 93 log2 units, exp2, sums (2^-24 each, 100-fold through the exponential)
    slack = (a - b).abs() * 2.5e-5 + (a.abs() + b.abs()) * 200 * 2.0 ** -24
    # the other keys: 2^-93.4 of the first's weight each (200 codes of log2(128.4) / 15), values up to 2; where
    # both of the two are 0 they are what the row has (a first run showed 1e-29 there)
    slack = slack + 64 * pages * 2 * 2.0 ** -93
    half = torch.exp2(torch.floor(torch.log2(want.abs() + slack)) - 8)
    off = (out[0, :, 0].double().cpu() - want).abs() - half - slack
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()}, by up to {off.max().item():.3g}"


HUGE = [3e8, 1e10, 3e12, -1e10, 1e20]  # queries whose scores pass 2^31


@pytest.mark.parametrize("form", [*FORMS, "whole sequences"])
def test_huge_queries_take_the_key_of_the_largest_score(dev, form):
    """Scores of any finite size: a query along one dim, keys of small whole numbers in it, so that products are
    exact and a step between two keys is 2^22 and more; the row is the V of its one largest key, bit for bit."""
    hq, kv, B, shared = FORMS.get(form, (16, 2, 3, 0))
    spare = 0 if form == "whole sequences" else SPARE
    lens = [shared + 130 + 61 * b for b in range(B)]
    g = gen(14)
    table, pages = make_table(g, lens, shared, width_spare=spare)
    assert (table.shape[1] > 16) == (spare > 0)
    k = torch.randint(100, 120, (pages, kv, PAGE, D), generator=g, dtype=torch.uint8)
    v = torch.randint(0, 256, (pages, kv, PAGE, D), generator=g, dtype=torch.uint8)
    tops, lows = [], []  # positions of the largest and the smallest key: in the shared part and in the own one
    for b, n in enumerate(lens):
        tops.append((7 * b) % shared if shared and b % 2 else n - 1 - 5 * b)
        lows.append(n - 70 - b)
    if shared:  # one key of the shared part for all that have theirs there
        tops = [77 if b % 2 else t for b, t in enumerate(tops)]
    for b in range(B):
        for at, code in ((tops[b], 200 if b % 2 else 255), (lows[b], 3)):
            k[table[b, at // PAGE].long(), :, at % PAGE, 0] = code
    word = lambda x: torch.full((pages, kv, PAGE, 2), x, dtype=torch.bfloat16, device=dev)  # noqa: E731
    pool = (k.to(dev), word(1.0), word(0.0)), (v.to(dev), word(2.0 ** -6), word(-2.0))
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    for size in HUGE:
        q = torch.zeros((B, hq, 1, D), dtype=torch.bfloat16)
        q[..., 0] = size
        out = paged_decode_attention(q.to(dev), *pool, table.to(dev), n_d, SCALE, shared=shared)
        for b in range(B):
            at = tops[b] if size > 0 else lows[b]
            want = v[table[b, at // PAGE].long(), :, at % PAGE].double() * 2.0 ** -6 - 2
            want = want.repeat_interleave(hq // kv, 0)
            assert torch.equal(out[b, :, 0].double().cpu(), want), f"sequence {b}, queries of {size}"


@pytest.mark.parametrize("hq,kv,q_lens,k_lens", [
    (8, 2, [256, 100], [256, 256]),   # small blocks
    (8, 2, [256, 31], [9000, 4444]),  # shares that end inside blocks
    (256, 8, [256] * 64, [4400] * 64),  # large blocks, several rounds
])
def test_huge_queries_of_prompts(dev, hq, kv, q_lens, k_lens):
    """The last keys' numbers rise: every row takes the V of its own position, or with a negative query of the
    first key, whose number is the smallest."""
    g = gen(15)
    k = torch.zeros((sum(k_lens), kv, D), dtype=torch.bfloat16)
    at = 0
    for n, m in zip(q_lens, k_lens):
        k[at:at + m, :, 0] = (torch.arange(m) - (m - 256)).clamp(min=-1)[:, None].to(torch.bfloat16)
        k[at, :, 0] = -5
        at += m
    v = randn(g, sum(k_lens), kv, D)
    for size in HUGE:
        q = torch.zeros((sum(q_lens), hq, D), dtype=torch.bfloat16)
        q[..., 0] = size
        out = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens).cpu()
        a = c = 0
        for n, m in zip(q_lens, k_lens):
            own = v[c + m - n:c + m] if size > 0 else v[c:c + 1].expand(n, -1, -1)
            assert torch.equal(out[a:a + n], own.repeat_interleave(hq // kv, 1)), f"{n} on {m}, queries of {size}"
            a, c = a + n, c + m


FAR = {"dealt out": (16, 8, 3, 0), "shared dealt out": (8, 8, 9, 1024), "blocks of 32": (8, 8, 17, 512),
       "blocks of 64": (16, 8, 17, 512), "blocks of 128": (64, 8, 17, 512)}


def test_forms_on_pages_beyond_32_bit_offsets(dev):
    """Pages whose codes lie more than 4 GB into the pool, in the tables of every form: appended, attended to,
    copied and read back."""
    pages, kv = 67000, 8
    pool = [(torch.empty((pages, kv, PAGE, D), dtype=torch.uint8, device=dev),
             torch.empty((pages, kv, PAGE, 2), dtype=torch.bfloat16, device=dev),
             torch.empty((pages, kv, PAGE, 2), dtype=torch.bfloat16, device=dev)) for _ in range(2)]
    g = gen(11)
    for form, (hq, kv, B, shared) in FAR.items():
        lens = [(shared or 1000) + 10 + 37 * b for b in range(B)]
        low, count = make_table(g, lens, shared, spare=0, width_spare=SPARE)
        assert low.shape[1] > 16
        assert (workspace(B, hq, kv, shared // PAGE) > workspace(B, hq, kv, 0)) == (shared > 0), form
        ids = 66000 + torch.randperm(1000, generator=g)[:count].to(torch.int32)
        far = ids[low.long()]
        # the shared rows through the first sequence, its own and the others' behind them
        counts = [lens[0]] + [n - shared for n in lens[1:]]
        k, v = randn(g, sum(counts), kv, D).to(dev), randn(g, sum(counts), kv, D).to(dev)
        starts = torch.tensor([0] + [shared] * (B - 1), dtype=torch.int32, device=dev)
        paged_append(k, v, *pool, far.to(dev), starts, counts)
        near = [tuple(t[ids.long().to(dev)].cpu() for t in buf) for buf in pool]
        q = randn(g, B, hq, 1, D)
        n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
        out = paged_decode_attention(q.to(dev), *pool, far.to(dev), n_d, SCALE, shared=shared)
        check_rows(out, q, near, low, lens, SCALE, [0, B // 2, B - 1])
        rows = paged_gather(*pool, far.to(dev), torch.zeros_like(n_d), lens)
        for x, buf in zip(rows, near):
            want = torch.cat([read_rows(buf, low[b], lens[b]) for b in range(B)])
            assert torch.equal(x.cpu().double(), want), form
        there = 65000 + torch.arange(count)
        copy_pages(*pool, ids, there)
        for buf in pool:
            for t in buf:
                same = t[ids.long().to(dev)].view(torch.uint8) == t[there.to(dev)].view(torch.uint8)
                assert same.all(), form


# -------------------------------------------------------------------------------- packed prompts

@pytest.mark.parametrize("hq,kv,q_lens,k_lens,parts", [
    (8, 2, [700, 0, 1, 130, 64, 40], [700, 9, 1, 130, 190, 33], False),  # small blocks, all resident
    (64, 8, [900] * 3 + [77], [900] * 3 + [600], False),                  # small blocks, several rounds
    (8, 2, [260, 33], [9000, 4444], True),                                # shares that end inside blocks
    (12, 2, [512], [8193], True), (5, 1, [1000, 1, 700], [5001, 8000, 700], True),
    (256, 4, [1600], [7000], False),                                      # large blocks, several rounds
])
def test_every_key_of_a_prompt_counts_once(dev, hq, kv, q_lens, k_lens, parts):
    """Equal weights over V rows that are 1 in the dim of their key: row i gets the shares of the keys it sees."""
    lq, lk = ((C.c_int32 * len(x))(*x) for x in (q_lens, k_lens))
    assert (_lib.load().lq_prompt_workspace_bytes(lq, lk, len(q_lens), hq, kv) > 0) == parts
    g = gen(12)
    q, k = randn(g, sum(q_lens), hq, D), randn(g, sum(k_lens), kv, D)
    for by in (1, 64):  # every key, every tile of keys
        dim = (5 * (torch.arange(sum(k_lens))[:, None] // by) + 3 * torch.arange(kv)) % D
        v = torch.nn.functional.one_hot(dim, D)
        out = prompt_attention(q.to(dev), k.to(dev), v.to(torch.bfloat16).to(dev), q_lens, 0.0, k_lens=k_lens)
        a = c = 0
        for n, m in zip(q_lens, k_lens):
            seen = torch.arange(m - n, m).clamp(min=-1) + 1  # keys of each row
            upto = torch.cat([torch.zeros((1, kv, D)), v[c:c + m].double().cumsum(0)])  # [m + 1, kv, 128]
            want = upto[seen] / seen.clamp(min=1)[:, None, None]
            assert_named(out[a:a + n], want.repeat_interleave(hq // kv, 1), f"{n} rows on {m}")
            a, c = a + n, c + m
