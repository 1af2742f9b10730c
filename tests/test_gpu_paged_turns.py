"""The rotated append and chunk attention as they are used together: sessions that read prompts, go on by chunks,
verified blocks and tokens, are forked and trimmed, with and without a window; recorded steps; the attention block and
a model over sessions of different lengths and over sliding-window layers. And chunk attention at sizes at which its
blocks are taken whole or cut into shares."""
import ctypes as C

import pytest
import torch

from lagunalab_amd import _lib
from lagunalab_amd.attention import Attention
from lagunalab_amd.cache import DequantKVCache
from lagunalab_amd.paged import PagedKVCache, paged_append_rotated, paged_chunk_attention
from lagunalab_amd.rotary import Rotary
from paged_util import D, PAGE, fill_pool, make_table, randn
from test_gpu_paged_chunk import SCALE, assert_within, exact, sessions
from test_gpu_paged_rotate import exact_rows
from tiny_model import TinyArgs, TinyLM, _rms, _rope, sdpa

pytestmark = pytest.mark.gpu
ROPE = {"rope_theta": 1e4, "partial_rotary_factor": 0.5}


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("window", [None, 90])
@pytest.mark.parametrize("hq,kv", [(8, 2), (6, 6), (18, 1)])
def test_sessions_in_turns(dev, hq, kv, window):
    """Every step's rows against attention over all rows that the session was given, as they came back when they were
    stored, and its queries against the formula."""
    g = gen(1)
    cache = PagedKVCache(60, kv, dev)
    rotary = Rotary.of(ROPE, dev)
    norms = [(1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(dev) for _ in range(2)]
    a, b, c = (cache.open() for _ in range(3))
    given = {s: [torch.zeros((0, kv, D), dtype=torch.bfloat16, device=dev)] * 2 for s in (a, b, c)}

    def step(who, counts):
        T = sum(counts)
        proj = randn(g, T, (hq + 2 * kv) * D + 8).to(dev)
        x = [t.unflatten(1, (-1, D)) for t in proj[:, :-8].split([hq * D, kv * D, kv * D], 1)]
        pos = torch.cat([torch.arange(cache.length(s), cache.length(s) + n) for s, n in zip(who, counts)])
        q, *rows = cache.append_rotated(who, *x, rotary, counts, *norms, eps=1e-5, fetch=True)
        want, off = exact_rows(x[0], pos, norms[0], rotary, 1e-5)
        assert ((q.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2 * off).all()
        out = cache.chunk_attention(who, q, SCALE, counts, window)
        at = 0
        for s, n in zip(who, counts):
            given[s] = [torch.cat([old, new[at:at + n]]) for old, new in zip(given[s], rows)]
            k, v = cache.rows([s])
            assert torch.equal(k, given[s][0]) and torch.equal(v, given[s][1])
            table = torch.tensor([cache.pages(s)], dtype=torch.int32)
            if n:
                assert_within(out[at:at + n], *exact(q[at:at + n], (cache.keys, cache.values), table, [cache.length(s)], [n],
                                                     window, SCALE), f"session {s}, {n} rows")
            at += n

    step([a, b, c], [130, 1, 70])
    step([b, a], [200, 5])
    d = cache.fork(a)
    given[d] = list(given[a])
    step([a, d, c], [4, 4, 0])
    for s, n in ((a, 2), (b, 9)):
        assert cache.trim(s, n) == n
        given[s] = [t[:-n] for t in given[s]]
    step([a, b, c, d], [1, 1, 1, 1])
    cache.compact()
    step([d, b], [60, 3])
    step([c], [1])


@pytest.mark.parametrize("counts,window", [([1, 1, 1], None), ([1, 1, 1], 100), ([5, 40, 2], None), ([150, 1, 60], 200)])
def test_a_recorded_turn(dev, counts, window):
    """Both calls in one graph, positions and lengths moved on by it: every replay as the eager calls on a pool of its
    own."""
    g = gen(2)
    hq, kv, starts = 12, 2, [700, 61, 0]
    lens = [s + 4 * c for s, c in zip(starts, counts)]
    table, pages = make_table(g, lens, 0)
    first = fill_pool(g, pages, kv, dev, poison=False)
    pools = [[tuple(t.clone() for t in buf) for buf in first] for _ in range(2)]
    rotary, T = Rotary.of(ROPE, dev), sum(counts)
    table, more = table.to(dev), ints(counts, dev)
    x = [randn(g, T, h, D).to(dev) for h in (hq, kv, kv)]
    at = [ints(starts, dev) for _ in range(2)]

    def turn(i):
        q, k, v = paged_append_rotated(*x, *pools[i], table, at[i], rotary, counts, fetch=True)
        at[i].add_(more)
        return q, k, v, paged_chunk_attention(q, *pools[i], table, at[i], SCALE, counts, window)

    turn(0)  # both once, eagerly
    turn(1)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = turn(0)
    torch.cuda.current_stream(dev).wait_stream(stream)
    for i in range(3):
        for t in x:
            t.copy_(randn(g, *t.shape))
        graph.replay()
        want = turn(1)
        torch.cuda.synchronize(dev)
        assert torch.equal(at[0], at[1])
        for a, b in zip((*got, *pools[0][0], *pools[0][1]), (*want, *pools[1][0], *pools[1][1])):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def block_of(g, dev, hq=8, kv=2, C=256):
    w = lambda *s: randn(g, *s, std=0.06).to(dev)  # noqa: E731
    return Attention(w(hq * D, C), w(kv * D, C), w(kv * D, C), w(C, hq * D), w(hq, C), w(D) + 1, w(D) + 1, hq, kv, ROPE)


def near(got, want):
    """8-bit rows within half a step of a 255th of their range, queries, keys, weights and outputs rounded to bf16
    (2^-8 each) on either side: a few hundredths of the largest value, as for the block over its other caches."""
    assert (got.float() - want.float()).abs().max() < 3e-2 * want.float().abs().max()


def test_the_block_over_sessions_of_different_lengths(dev):
    g = gen(3)
    block = block_of(g, dev)
    pool = PagedKVCache(40, 2, dev)
    had = [150, 67, 0]
    who, plain = [pool.open() for _ in had], [DequantKVCache() for _ in had]
    for s, c, n in zip(who, plain, had):
        if n:
            x = randn(g, 1, n, 256).to(dev)
            near(block(x, "causal", pool.batch([s], rotates=True)), block(x, "causal", c))
    batch = pool.batch(who, rotates=True)
    for L in (1, 3, 40, 1):
        x = randn(g, 3, L, 256).to(dev)
        got = block(x, batch.make_mask(L), batch)
        for i, c in enumerate(plain):
            near(got[i:i + 1], block(x[i:i + 1], c.make_mask(L), c))
    assert [pool.length(s) for s in who] == [195, 112, 45]


@pytest.mark.parametrize("rotates", [False, True])
def test_the_block_as_a_sliding_layer(dev, rotates):
    g = gen(4)
    block = block_of(g, dev)
    pool = PagedKVCache(40, 2, dev)
    batch = pool.batch([pool.open(), pool.open()], window=50, rotates=rotates)
    plain = DequantKVCache()
    for L in (130, 1, 3, 20, 1):
        x = randn(g, 2, L, 256).to(dev)
        at = torch.arange(plain.offset + L)
        mask = (at[None, :] <= at[-L:, None]) & (at[None, :] > at[-L:, None] - 50)
        near(block(x, batch.make_mask(L, window_size=50), batch), block(x, mask, plain))


@torch.no_grad()
def test_a_model_with_sliding_layers(dev):
    """The tiny model with full and sliding layers, a prompt, chunks and tokens, forked on the way: logits as over the
    dequantizing caches with the layers' masks."""
    types = ["full_attention", "sliding_attention", "full_attention", "sliding_attention"]
    model = TinyLM(TinyArgs(layer_types=types), device="cuda", seed=3)
    W = model.args.sliding_window

    class Masked(DequantKVCache):
        def make_mask(self, N, return_array=False, window_size=None):
            from lagunalab_amd.cache import create_attention_mask
            return create_attention_mask(N, self.offset, return_array, window_size)

    pools = [PagedKVCache(20, 2, dev) for _ in types]
    windows = [W if t == "sliding_attention" else None for t in types]
    first = [p.open() for p in pools]
    paged = [p.batch([s], window=w) for p, s, w in zip(pools, first, windows)]
    plain = [Masked() for _ in types]
    ids = torch.randint(0, 1024, (1, 150), generator=gen(5)).to(dev)
    for part in ids.split([100, 1, 5, 43, 1], dim=1):
        got, want = model(part, cache=paged), model(part, cache=plain)
        assert (got - want).abs().max() < 5e-2 * want.abs().max()
    both = [p.batch([s, p.fork(s)], window=w) for p, s, w in zip(pools, first, windows)]
    wide = []
    for c in plain:
        w = Masked()
        w.state = tuple(tuple(t.expand(2, -1, -1, -1).contiguous() for t in x) for x in c.state)
        wide.append(w)
    for i in range(3):
        tok = torch.tensor([[i + 1], [i + 70]], device="cuda")
        got, want = model(tok, cache=both), model(tok, cache=wide)
        assert (got - want).abs().max() < 5e-2 * want.abs().max()


# heads, lengths, counts, window, and whether blocks of many rows are taken whole (no workspace) on 256 CUs
PLANS = [
    (32, 8, [300 + i for i in range(8)], [300] * 8, None, True),       # blocks of 256 rows
    (32, 8, [700, 3, 650, 0, 580], [400, 3, 650, 0, 400], 128, True),  # few of them, and a sequence of few rows
    (48, 8, [2300], [1500], 200, True),
    (32, 8, [2600], [2600], None, False),
    (48, 8, [200 + 9 * i for i in range(40)], [20] * 40, None, True),  # blocks of 128 rows
    (48, 8, [2000 + 9 * i for i in range(10)], [20] * 10, None, False),
    (48, 8, [900], [512], None, False),
]


@pytest.mark.parametrize("hq,kv,lens,counts,window,whole", PLANS)
def test_blocks_whole_and_in_shares(dev, hq, kv, lens, counts, window, whole):
    g = gen(6)
    pool, table = sessions(g, kv, lens, dev)
    q = randn(g, sum(counts), hq, D).to(dev)
    need = _lib.load().lq_paged_chunk_workspace_bytes((C.c_int32 * len(counts))(*counts), len(counts), hq, kv,
                                                      table.shape[1], window or 0)
    assert (need == 0) == whole
    out = paged_chunk_attention(q, *pool, table.to(dev), ints(lens, dev), SCALE, counts, window)
    assert_within(out, *exact(q, pool, table, lens, counts, window, SCALE))
    # shorter sequences than the table allows, some of them shorter than their rows, empty or not there at all
    now = [n if i % 4 == 3 else max(0, n - 97 * (i % 4 + 1)) for i, n in enumerate(lens)]
    now[-1] = [0, lens[-1] - 1][len(lens) > 1]
    out = paged_chunk_attention(q, *pool, table.to(dev), ints(now, dev), SCALE, counts, window)
    assert_within(out, *exact(q, pool, table, now, counts, window, SCALE))
    bad = list(lens)
    bad[0] = PAGE * table.shape[1] + 1
    out = paged_chunk_attention(q, *pool, table.to(dev), ints(bad, dev), SCALE, counts, window)
    assert out[:counts[0]].isnan().all()
    want, bound = exact(q, pool, table, lens, counts, window, SCALE)
    if len(lens) > 1:
        assert_within(out[counts[0]:], want[counts[0]:], bound[counts[0]:])


@pytest.mark.parametrize("spare", [0, 60])  # a short table, taken whole, and a long one, dealt out
@pytest.mark.parametrize("window", [None, 70])
@pytest.mark.parametrize("longest", [10, 16])  # of 6 query heads each: 60 rows, one block, and 96, two
def test_many_verified_blocks(dev, longest, window, spare):
    """More than 32 query rows of so many sequences that 64 go as one block, beside single tokens: values, a V row that
    some rows see and others do not, a page and a length that are not there."""
    g = gen(7)
    hq, kv, B = 48, 8, 64
    lens = [(37 * i * i) % 400 + 17 for i in range(B)]
    counts = [[6, 1, 8, longest, min(11, longest), 5][i % 6] for i in range(B)]
    lens[9], counts[9], counts[10] = 0, 3, 0
    pool, table = sessions(g, kv, lens, dev, spare=spare)
    q = randn(g, sum(counts), hq, D).to(dev)
    args = (ints(lens, dev), SCALE, counts, window)
    clean = paged_chunk_attention(q, *pool, table.to(dev), *args)
    want_all, bound = exact(q, pool, table, lens, counts, window, SCALE)
    assert_within(clean, want_all, bound)
    ends = torch.tensor(counts).cumsum(0).tolist()
    for b in (3, 2, 34):  # the longest, 48 rows of a KV head, the next longest
        first = ends[b] - counts[b]
        at = lens[b] - counts[b] // 2
        spoiled = [tuple(t.clone() for t in buf) for buf in pool]
        spoiled[1][1][int(table[b, at // PAGE]), 5, at % PAGE, 0] = float("inf")
        got = paged_chunk_attention(q, *spoiled, table.to(dev), *args)
        see = slice(ends[b] - counts[b] // 2, ends[b])
        assert not torch.isfinite(got[see][:, 30:36, :64]).any()
        want = clean.clone()
        want[see, 30:36, :64] = got[see, 30:36, :64] = 0
        assert torch.equal(got, want)
        bad = table.clone()
        bad[b, (lens[b] - 1) // PAGE] = pool[0][0].shape[0]
        got = paged_chunk_attention(q, *pool, bad.to(dev), *args)
        sees = (lens[b] - 1) // PAGE * PAGE - (lens[b] - counts[b])  # the first row that does
        assert got[first + max(0, sees):ends[b]].isnan().all()
        for part in (slice(0, first + max(0, sees)), slice(ends[b], None)):
            assert torch.equal(got[part], clean[part])
        for n in (-1, PAGE * table.shape[1] + 1):
            now = list(lens)
            now[b] = n
            got = paged_chunk_attention(q, *pool, table.to(dev), ints(now, dev), *args[1:])
            assert got[first:ends[b]].isnan().all()
            for part in (slice(0, first), slice(ends[b], None)):  # other lengths cut the others' keys elsewhere
                assert_within(got[part], want_all[part], bound[part])


def test_views_and_many_sequences(dev):
    """One sequence's pages under several lengths (a table of one expanded row), queries and keys expanded over heads,
    more sequences than a launch takes, a table far wider than the sequences, another stream."""
    g = gen(8)
    pool, table = sessions(g, 2, [700], dev)
    lens, counts = [700, 130, 1, 64, 699], [90, 1, 1, 64, 40]
    one = randn(g, sum(counts), 1, D).to(dev)
    q = one.expand(-1, 8, -1)
    wide = table.to(dev).expand(len(lens), -1)
    out = paged_chunk_attention(q, *pool, wide, ints(lens, dev), SCALE, counts, 100)
    assert_within(out, *exact(q, pool, wide.cpu(), lens, counts, 100, SCALE))
    far = torch.full((len(lens), 3000), -1, dtype=torch.int32, device=dev)
    far[:, :wide.shape[1]] = wide
    for window in (None, 100):
        out = paged_chunk_attention(q, *pool, far, ints(lens, dev), SCALE, counts, window)
        assert_within(out, *exact(q, pool, wide.cpu(), lens, counts, window, SCALE))

    starts = [(7 * i) % 200 for i in range(150)]
    counts = [i % 4 for i in range(150)]
    T = sum(counts)
    table, pages = make_table(g, [s + c for s, c in zip(starts, counts)], 0)
    rotary = Rotary.of(ROPE, dev)
    x, k, v = randn(g, T, 4, D).to(dev), randn(g, T, 1, D).to(dev).expand(-1, 2, -1), randn(g, T, 2, D).to(dev)
    pools = [[tuple(t.clone() for t in buf) for buf in p] for p in [fill_pool(g, pages, 2, dev, poison=False)] * 2]
    got = paged_append_rotated(x, k, v, *pools[0], table.to(dev), ints(starts, dev), rotary, counts, fetch=True)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):  # a sequence at a time
        at = 0
        for b, (s, c) in enumerate(zip(starts, counts)):
            part = paged_append_rotated(x[at:at + c], k[at:at + c], v[at:at + c], *pools[1], table[b:b + 1].to(dev),
                                        ints([s], dev), rotary, [c], fetch=True)
            for t, p in zip(got, part):
                assert torch.equal(t[at:at + c], p)
            at += c
    torch.cuda.current_stream(dev).wait_stream(stream)
    for a, b in zip((*pools[0][0], *pools[0][1]), (*pools[1][0], *pools[1][1])):
        assert torch.equal(a, b)
    want, off = exact_rows(x, torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)]), None, rotary)
    assert ((got[0].double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2 * off).all()


class RotatingLM(TinyLM):
    """The tiny model with its projections rounded to bf16, as the rows of a rotating batch are: over one its attention
    hands them on, norm and rotation are the append's."""

    def _attention(self, m, x, mask, cache):
        a, bf = self.args, torch.bfloat16
        B, L, _ = x.shape
        heads = (a.num_attention_heads, a.num_key_value_heads, a.num_key_value_heads)
        q, k, v = ((x @ w.T).to(bf).view(B, L, h, D) for w, h in zip((m.q_proj, m.k_proj, m.v_proj), heads))
        if cache.rotates:
            q = cache.append_rotated(q, k, v, Rotary.of({"rope_theta": a.rope_theta}, x.device), m.q_norm.to(bf),
                                     m.k_norm.to(bf), a.rms_norm_eps)
            out = cache.attend(q, SCALE)
        else:
            q, k = (_rope(_rms(t.float(), w, a.rms_norm_eps).transpose(1, 2), cache.offset, a.rope_theta).to(bf)
                    for t, w in ((q, m.q_norm), (k, m.k_norm)))
            k, v = cache.update_and_fetch(k.contiguous(), v.transpose(1, 2).contiguous())
            out = cache.attend(q.contiguous(), SCALE) if cache.fused_step else sdpa(q, k, v, mask, SCALE)
        gate = torch.nn.functional.softplus(x @ m.g_proj.T)[..., None]
        return (out.to(x.dtype).transpose(1, 2) * gate).reshape(B, L, -1) @ m.o_proj.T


@torch.no_grad()
def test_a_model_over_sessions_of_different_lengths(dev):
    """Full and sliding layers over rotating batches, a pool per layer: prompts of three lengths, a chunk, tokens, a
    session forked and one trimmed on the way; every session's logits as over dequantizing caches of its own with the
    layers' masks. The tolerance is the one of the model above: the bf16 rows, weights and outputs of either side are off
    by 2^-8 of their size, an 8-bit row by half a step."""
    types = ["full_attention", "sliding_attention", "full_attention", "sliding_attention"]
    model = RotatingLM(TinyArgs(layer_types=types), device="cuda", seed=4)
    for m in model.layers:
        for w in (m.q_norm, m.k_norm):
            w.copy_(w.to(torch.bfloat16))
    windows = [model.args.sliding_window if t == "sliding_attention" else None for t in types]

    class Masked(DequantKVCache):
        rotates = False

        def make_mask(self, N, return_array=False, window_size=None):
            from lagunalab_amd.cache import create_attention_mask
            return create_attention_mask(N, self.offset, return_array, window_size)

    g = gen(9)
    pools = [PagedKVCache(40, 2, dev) for _ in types]
    who, plain = [], []

    def near_logits(got, want):
        assert (got - want).abs().max() < 5e-2 * want.abs().max()

    for n in (150, 67, 3):
        s, own = [p.open() for p in pools], [Masked() for _ in types]
        ids = torch.randint(0, 1024, (1, n), generator=g).to(dev)
        near_logits(model(ids, cache=[p.batch([x], w, rotates=True) for p, x, w in zip(pools, s, windows)]),
                    model(ids, cache=own))
        who.append(s)
        plain.append(own)

    def steps(*lengths):
        batches = [p.batch([s[i] for s in who], w, rotates=True) for i, (p, w) in enumerate(zip(pools, windows))]
        for L in lengths:
            ids = torch.randint(0, 1024, (len(who), L), generator=g).to(dev)
            got = model(ids, cache=batches)
            for i, own in enumerate(plain):
                near_logits(got[i:i + 1], model(ids[i:i + 1], cache=own))

    steps(1, 40, 1, 5)
    who.append([p.fork(x) for p, x in zip(pools, who[0])])
    plain.append([Masked() for _ in types])
    for old, new in zip(plain[0], plain[-1]):
        new.state = tuple(tuple(t.clone() for t in x) for x in old.state)
    for p, x, own in zip(pools, who[1], plain[1]):
        assert p.trim(x, 3) == own.trim(3) == 3
    steps(1, 6, 1)
    assert [pools[0].length(s[0]) for s in who] == [205, 119, 58, 205]
