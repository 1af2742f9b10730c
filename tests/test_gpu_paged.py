"""The paged 8-bit cache and packed-prompt attention against plain computations in 64 bits."""
import pytest
import torch

from lagunalab_amd import _lib
from lagunalab_amd.paged import (copy_pages, page_pool, paged_append, paged_decode_attention,
                                 paged_gather)
from lagunalab_amd.prompt_attn import prompt_attention
from paged_util import (D, PAGE, assert_within, exact_attention, fill_pool, make_table, randn,
                        read_rows, write_rows)

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def bits(t):
    return t.view(torch.int16) if t.dtype == torch.bfloat16 else t


# ------------------------------------------------------------------------------- rows in and out

@pytest.mark.parametrize("kv,starts,counts", [
    (1, [0], [1]),
    (8, [5, 0, 63, 64, 130], [1, 1, 1, 1, 1]),
    (2, [0, 7, 64, 200, 3], [64, 130, 0, 1, 61]),
    (3, [1] * 70, [2] * 70),  # more sequences than one launch takes
])
def test_append_is_the_quantizer_at_the_tables_slots(dev, kv, starts, counts):
    from lagunalab_amd.quant import quantize
    g = gen(1)
    ends = [s + c for s, c in zip(starts, counts)]
    table, pages = make_table(g, ends, 0)
    pool = fill_pool(g, pages, kv, dev)
    before = [tuple(t.clone() for t in buf) for buf in pool]
    T = sum(counts)
    k, v = randn(g, T, kv, D).to(dev), randn(g, T, kv, D, std=3.0).to(dev)
    paged_append(k, v, *pool, table.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), counts)
    b = torch.cat([torch.full((c,), i) for i, c in enumerate(counts)])
    at = torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)])
    where = table[b, at // PAGE].long().to(dev), (at % PAGE).to(dev)
    for rows, buf, old in zip((k, v), pool, before):
        for t, x, o in zip(buf, quantize(rows), old):
            assert torch.equal(bits(t[where[0], :, where[1]]), bits(x))
            o[where[0], :, where[1]] = x
            assert torch.equal(bits(t), bits(o)), "a slot that no row goes to changed"


def test_append_special_rows_and_strides(dev):
    from lagunalab_amd.quant import quantize
    from gpu_util import special_rows
    rows = torch.from_numpy(special_rows()).to(torch.bfloat16)  # [n, 128]
    n = rows.shape[0]
    wide = torch.zeros((n, 5, 2, D + 8), dtype=torch.bfloat16)  # heads and rows apart
    wide[:, 1, :, :D] = rows[:, None]
    wide[:, 3, :, :D] = rows.flip(0)[:, None]
    wide = wide.to(dev)
    k, v = wide[:, 1, :, :D], wide[:, 3, :, :D]
    pool = page_pool(2, 2, dev)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
    paged_append(k, v, *pool, table, torch.tensor([60], dtype=torch.int32, device=dev))
    at = torch.arange(60, 60 + n)
    where = table[0].cpu()[at // PAGE].long().to(dev), (at % PAGE).to(dev)
    for x, buf in ((k, pool[0]), (v, pool[1])):
        for t, y in zip(buf, quantize(x.contiguous())):
            assert torch.equal(bits(t[where[0], :, where[1]]), bits(y))


def test_append_skips_positions_and_pages_that_do_not_exist(dev):
    g = gen(2)
    pool = fill_pool(g, 3, 2, dev)
    before = [tuple(t.clone() for t in buf) for buf in pool]
    k = randn(g, 12, 2, D).to(dev)
    # pages -1 and 3 do not exist, position 128 is beyond the row, negative positions are before it
    table = torch.tensor([[-1, 3], [3, 2], [0, -7]], dtype=torch.int32, device=dev)
    starts = torch.tensor([62, 126, -3], dtype=torch.int32, device=dev)
    paged_append(k, k, *pool, table, starts, [4, 4, 4])
    for buf, old in zip(pool, before):
        for t, o in zip(buf, old):
            changed = torch.zeros(t.shape[:3], dtype=torch.bool)
            changed[2, :, 62:64] = True  # rows 126, 127 of sequence 1
            changed[0, :, 0:1] = True    # row 0 of sequence 2
            same = (bits(t) == bits(o)).all(-1).cpu()
            assert same[~changed].all()
            assert not same[changed].any()


@pytest.mark.parametrize("kv,starts,counts", [
    (8, [0], [1]), (2, [0, 63, 64, 1], [64, 2, 65, 200]), (1, [100, 5, 0], [0, 59, 128]),
    (4, list(range(67)), [3] * 67),
])
def test_gather_is_the_dequantizer(dev, kv, starts, counts):
    g = gen(3)
    ends = [s + c for s, c in zip(starts, counts)]
    table, pages = make_table(g, ends, 0)
    pool = fill_pool(g, pages, kv, dev)
    rows = [(randn(g, n, kv, D), randn(g, n, kv, D)) for n in ends]
    for b, (k, v) in enumerate(rows):
        if ends[b]:
            write_rows(pool, table[b], k, v)
    got = paged_gather(*pool, table.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), counts)
    for x, buf in zip(got, pool):
        want = torch.cat([read_rows(buf, table[b], ends[b])[starts[b]:] for b in range(len(ends))])
        assert x.shape == want.shape and torch.equal(x.cpu().double(), want)


def test_gather_of_positions_that_do_not_exist_is_nan(dev):
    g = gen(4)
    pool = fill_pool(g, 2, 1, dev, poison=False)
    table = torch.tensor([[1, 5]], dtype=torch.int32, device=dev)
    k, v = paged_gather(*pool, table, torch.tensor([-2], dtype=torch.int32, device=dev), [140])
    for x in (k, v):
        lost = torch.isnan(x).all(-1).all(-1).cpu()
        assert lost.tolist() == [True] * 2 + [False] * 64 + [True] * 74


@pytest.mark.parametrize("kv,pages,n", [(8, 10, 1), (1, 2500, 1000), (3, 40, 17)])
def test_copy_pages(dev, kv, pages, n):
    g = gen(5)
    pool = fill_pool(g, pages, kv, dev, poison=False)
    for buf in pool:
        buf[1].copy_(torch.randn(buf[1].shape, generator=g))
        buf[2].copy_(torch.randn(buf[1].shape, generator=g))
    order = torch.randperm(pages, generator=g)
    src, dst = order[:n], order[n:2 * n]
    want = [[t.clone() for t in buf] for buf in pool]
    for buf in want:
        for t in buf:
            t[dst.to(dev)] = t[src.to(dev)]
    copy_pages(*pool, src, dst.tolist())
    copy_pages(*pool, [], [])
    for buf, w in zip(pool, want):
        for t, x in zip(buf, w):
            assert torch.equal(bits(t), bits(x))


def test_one_page_copied_to_several(dev):
    g = gen(6)
    pool = fill_pool(g, 6, 2, dev, poison=False)
    want = [[t.clone() for t in buf] for buf in pool]
    for buf in want:
        for t in buf:
            t[[0, 1, 5]] = t[3].clone()
    copy_pages(*pool, [3, 3, 3], [0, 5, 1])
    for buf, w in zip(pool, want):
        for t, x in zip(buf, w):
            assert torch.equal(bits(t), bits(x))


# ------------------------------------------------------------------------------------- decoding

def decode_case(seed, hq, kv, lens, shared, dev, std=1.0, width_spare=0):
    g = gen(seed)
    table, pages = make_table(g, lens, shared, width_spare=width_spare)
    pool = fill_pool(g, pages, kv, dev)
    common = shared // PAGE * PAGE
    if common:
        row = max(range(len(lens)), key=lambda b: lens[b])
        n = min(common, lens[row])
        write_rows(pool, table[row], randn(g, n, kv, D), randn(g, n, kv, D))
    for b, n in enumerate(lens):
        if n > common:
            write_rows(pool, table[b], randn(g, n - common, kv, D), randn(g, n - common, kv, D), common)
    q = randn(g, len(lens), hq, 1, D, std=std)
    return q, pool, table


def check_decode(out, q, pool, table, lens, scale=SCALE, rows=None):
    hq, kv = q.shape[1], pool[0][0].shape[1]
    G = hq // kv
    for b in rows if rows is not None else range(len(lens)):
        k, v = (read_rows(buf, table[b], lens[b]) for buf in pool)
        for h in range(kv):
            want, bound = exact_attention(q[b, h * G:(h + 1) * G, 0].double(), k[:, h], v[:, h],
                                          [lens[b] - 1] * G, scale)
            assert_within(out[b, h * G:(h + 1) * G, 0], want, bound, f"sequence {b} head {h}")


@pytest.mark.parametrize("hq,kv,lens", [
    (4, 1, [1]), (8, 8, [64]), (32, 8, [1037]), (6, 1, [63, 64, 65, 0, 1]), (16, 1, [300, 5]),
    (10, 2, [129, 1000, 2]), (48, 8, [4099]), (2, 2, [17] * 70), (3, 1, [20011, 1]),
])
def test_decode_without_a_shared_prefix(dev, hq, kv, lens):
    q, pool, table = decode_case(7, hq, kv, lens, 0, dev, width_spare=2)
    out = paged_decode_attention(q.to(dev), *pool, table.to(dev),
                                 torch.tensor(lens, dtype=torch.int32, device=dev), SCALE)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    check_decode(out, q, pool, table, lens)


@pytest.mark.parametrize("hq,kv,shared,own", [
    (4, 1, 64, [1]), (8, 2, 64, [0, 1, 64, 65]), (32, 8, 640, [3] * 16), (16, 1, 192, [5, 0, 70, 1000, 9]),
    (12, 2, 2048, list(range(1, 34))), (6, 6, 130, [62, 63, 64, 300]), (3, 1, 4096, [11] * 70),
])
def test_decode_with_a_shared_prefix(dev, hq, kv, shared, own):
    lens = [shared + n for n in own]
    q, pool, table = decode_case(8, hq, kv, lens, shared, dev)
    args = (q.to(dev), *pool, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), SCALE)
    out = paged_decode_attention(*args, shared=shared)
    rows = sorted({0, 1, len(lens) // 2, len(lens) - 1} & set(range(len(lens))))
    check_decode(out, q, pool, table, lens, rows=rows)
    # the same numbers whether the batch is told of the shared pages or not, to the roundings of both
    plain = paged_decode_attention(*args)
    assert (out.float() - plain.float()).abs().max() < 2 ** -5


def test_decode_of_sequences_shorter_than_the_shared_part(dev):
    """The longest is not the first; one ends inside the shared part, one is empty, one ends with it."""
    lens = [70, 0, 200, 128, 129, 1]
    q, pool, table = decode_case(9, 8, 2, lens, 128, dev)
    out = paged_decode_attention(q.to(dev), *pool, table.to(dev),
                                 torch.tensor(lens, dtype=torch.int32, device=dev), SCALE, shared=128)
    check_decode(out, q, pool, table, lens)
    assert (out[1] == 0).all()
    # no sequence as long as the shared part
    short = [70, 0, 100, 127, 64, 1]
    out = paged_decode_attention(q.to(dev), *pool, table.to(dev),
                                 torch.tensor(short, dtype=torch.int32, device=dev), SCALE, shared=128)
    check_decode(out, q, pool, table, short)


@pytest.mark.parametrize("shared", [0, 128])
@pytest.mark.parametrize("scale,std", [(-SCALE, 1.0), (0.0, 1.0), (1.0, 1.0), (SCALE, 30.0), (SCALE, 1e-6)])
def test_decode_scales(dev, scale, std, shared):
    lens = [200, 131]
    q, pool, table = decode_case(10, 8, 2, lens, shared, dev, std=std)
    out = paged_decode_attention(q.to(dev), *pool, table.to(dev),
                                 torch.tensor(lens, dtype=torch.int32, device=dev), scale, shared=shared)
    check_decode(out, q, pool, table, lens, scale=scale)


def test_decode_of_large_and_tiny_values(dev):
    """K and V far outside the fp16 range, as bf16 rows may be."""
    g = gen(11)
    lens = [150, 200]
    for vstd in (1e20, 1e-20):
        table, pages = make_table(g, lens, 128)
        pool = fill_pool(g, pages, 2, dev)
        write_rows(pool, table[0], randn(g, 128, 2, D), randn(g, 128, 2, D, std=vstd))
        for b, n in enumerate(lens):
            write_rows(pool, table[b], randn(g, n - 128, 2, D), randn(g, n - 128, 2, D, std=vstd), 128)
        q = randn(g, 2, 4, 1, D)
        args = (q.to(dev), *pool, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), SCALE)
        for shared in (0, 128):
            check_decode(paged_decode_attention(*args, shared=shared), q, pool, table, lens)


@pytest.mark.parametrize("shared", [0, 64])
def test_decode_of_bad_lengths_and_pages_is_nan_for_their_sequence_alone(dev, shared):
    lens = [100, 300, 150, 90, 128]
    q, pool, table = decode_case(12, 4, 2, lens, shared, dev)
    told = list(lens)
    told[0] = -1
    told[1] = 64 * table.shape[1] + 1
    bad = table.clone()
    bad[2, 2] = pool[0][0].shape[0]
    bad[3, 1] = -5
    out = paged_decode_attention(q.to(dev), *pool, bad.to(dev),
                                 torch.tensor(told, dtype=torch.int32, device=dev), SCALE, shared=shared)
    assert torch.isnan(out[:4]).all()
    check_decode(out, q, pool, table, lens, rows=[4])
    if shared:  # a bad page in the shared part: NaN for all that attend to it
        bad = table.clone()
        bad[:, 0] = 1 << 30
        out = paged_decode_attention(q.to(dev), *pool, bad.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev), SCALE, shared=shared)
        assert torch.isnan(out).all()


def test_decode_reads_table_rows_of_any_stride_and_no_row_behind_the_batch(dev):
    lens = [100, 200, 70]
    q, pool, table = decode_case(13, 8, 2, lens, 0, dev)
    wide = torch.full((5, table.shape[1] + 9), -1, dtype=torch.int32)
    wide[:3, :table.shape[1]] = table
    view = wide.to(dev)[:3, :table.shape[1]]
    out = paged_decode_attention(q.to(dev), *pool, view,
                                 torch.tensor(lens, dtype=torch.int32, device=dev), SCALE)
    check_decode(out, q, pool, table, lens)


# Head layouts, batches and shared positions whose shared pages are read once: dealt out with the own ones (up
# to 16 query rows), and in blocks of 64 and 128 rows.
SHARED = [(16, 16, 9, 512), (32, 16, 9, 512), (64, 8, 9, 1024), (6, 1, 23, 4096), (10, 2, 3, 16400)]


@pytest.mark.parametrize("hq,kv,B,shared", SHARED)
def test_shared_pages_read_once(dev, hq, kv, B, shared):
    """Own lengths from none to several pages; some sequences end before the shared part does or with it,
    one is empty, the first of all is short."""
    g = gen(33)
    lens = [shared + int(n) for n in torch.randint(0, 300, (B,), generator=g)]
    lens[0] = shared // PAGE * PAGE - 1
    lens[1] = shared // PAGE * PAGE
    if B > 3:
        lens[2], lens[3], lens[B - 1] = 0, 1, shared + 700
    q, pool, table = decode_case(33, hq, kv, lens, shared, dev)
    args = (q.to(dev), *pool, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev))
    out = paged_decode_attention(*args, SCALE, shared=shared)
    check_decode(out, q, pool, table, lens)
    assert (out.float() - paged_decode_attention(*args, SCALE).float()).abs().max() < 2 ** -5
    check_decode(paged_decode_attention(*args, -0.3, shared=shared), q, pool, table, lens, scale=-0.3,
                 rows=[0, 1, B - 1])
    # none as long as the shared part
    short = [min(n, shared // PAGE * PAGE - 1) for n in lens]
    args = (*args[:-1], torch.tensor(short, dtype=torch.int32, device=dev))
    check_decode(paged_decode_attention(*args, SCALE, shared=shared), q, pool, table, short)


@pytest.mark.parametrize("hq,kv,B,shared", SHARED[:4])
def test_shared_pages_that_are_bad(dev, hq, kv, B, shared):
    lens = [shared + 30 * b for b in range(B)]
    q, pool, table = decode_case(34, hq, kv, lens, shared, dev)
    args = (q.to(dev), *pool)
    n_d = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    told = list(lens)
    told[0], told[B - 1] = -5, 64 * table.shape[1] + 1
    own = table.clone()
    own[2, shared // PAGE] = -1  # sequence 2's first own page
    out = paged_decode_attention(*args, own.to(dev), n_d(told), SCALE, shared=shared)
    assert torch.isnan(out[[0, 2, B - 1]]).all()
    check_decode(out, q, pool, table, lens, rows=[1, 3])
    bad = table.clone()
    bad[:, 3] = pool[0][0].shape[0]
    told = list(lens)
    told[1] = 150  # ends before the bad page
    out = paged_decode_attention(*args, bad.to(dev), n_d(told), SCALE, shared=shared)
    assert torch.isnan(out[[b for b in range(B) if b != 1]]).all()
    check_decode(out, q, pool, table, told, rows=[1])


@pytest.mark.parametrize("hq,kv,B,shared", SHARED[:3])
def test_shared_pages_captured_and_on_two_streams(dev, hq, kv, B, shared):
    most = [shared + 200] * B
    q, pool, table = decode_case(35, hq, kv, most, shared, dev)
    q_d, t_d = q.to(dev), table.to(dev)
    n_d = torch.tensor(most, dtype=torch.int32, device=dev)
    call = lambda: paged_decode_attention(q_d, *pool, t_d, n_d, SCALE, shared=shared)  # noqa: E731
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    graphs, outs = [], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            call()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=st):
                outs.append(call())
    torch.cuda.synchronize(dev)
    for i in range(4):
        lens = [shared + (37 * b + 50 * i) % 201 for b in range(B)]
        lens[i] = 40 * i
        n_d.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize(dev)
        for st, graph in zip(streams, graphs):  # both at once
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize(dev)
        eager = call()
        for out in outs:
            assert torch.equal(bits(out), bits(eager))
        check_decode(eager, q, pool, table, lens, rows=[0, i, B - 1])


def test_decode_captured_follows_lengths_and_tables(dev):
    lens = [190, 130]
    q, pool, table = decode_case(14, 8, 2, [256, 256], 128, dev)
    q_d, t_d = q.to(dev), table.to(dev)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        paged_decode_attention(q_d, *pool, t_d, n_d, SCALE, shared=128)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = paged_decode_attention(q_d, *pool, t_d, n_d, SCALE, shared=128)
    torch.cuda.current_stream(dev).wait_stream(stream)
    for step in ([190, 130], [191, 131], [256, 1], [0, 129], [192, 256]):
        n_d.copy_(torch.tensor(step, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(dev)
        eager = paged_decode_attention(q_d, *pool, t_d, n_d, SCALE, shared=128)
        assert torch.equal(bits(out), bits(eager))
        check_decode(out, q, pool, table, step)


def test_decode_on_two_streams_at_once(dev):
    cases = [decode_case(s, 8, 2, [1500, 700], 512, dev) for s in (15, 16)]
    lens = torch.tensor([1500, 700], dtype=torch.int32, device=dev)
    args = [(q.to(dev), *pool, table.to(dev), lens, SCALE) for q, pool, table in cases]
    want = [paged_decode_attention(*a, shared=512) for a in args]
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for _ in range(10):
        got = []
        for st, a in zip(streams, args):
            with torch.cuda.stream(st):
                got.append(paged_decode_attention(*a, shared=512))
        torch.cuda.synchronize(dev)
        for x, y in zip(got, want):
            assert torch.equal(bits(x), bits(y))


@pytest.mark.parametrize("hq,B", [(128, 9), (256, 10), (512, 12), (1024, 10)])
@pytest.mark.parametrize("heavy", [False, True])
def test_long_shared_parts(dev, hq, B, heavy):
    """Shared parts of 32 pages and more, with few own pages (the parts' last pages are then taken by the workgroups
    of the own ones) and with many; row blocks of 32, 64 and 128 rows, one and two."""
    kv, shared = 64, 8192
    lens = [shared + (70 * b if heavy else b % 2) for b in range(B)]
    lens[2], lens[B - 1] = shared - 1, 0
    q, pool, table = decode_case(37, hq, kv, lens, shared, dev)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = (q.to(dev), *pool, table.to(dev), n_d, SCALE)
    out = paged_decode_attention(*args, shared=shared)
    check_decode(out, q, pool, table, lens, rows=[1, 2])
    assert (out[B - 1] == 0).all()
    assert (out.float() - paged_decode_attention(*args).float()).abs().max() < 2 ** -5
    assert torch.equal(bits(out), bits(paged_decode_attention(*args, shared=shared)))
    bad = table.clone()
    bad[:, shared // PAGE - 1] = -1  # the last shared page
    out = paged_decode_attention(q.to(dev), *pool, bad.to(dev), n_d, SCALE, shared=shared)
    assert torch.isnan(out[:B - 1]).all() and (out[B - 1] == 0).all()


@pytest.mark.parametrize("hq,kv,lens,shared", [
    (12, 4, [0, 1, 63, 64, 65, 300, 1024], 64), (32, 8, [130] * 33 + [1000], 128), (16, 1, [1024, 1023, 577], 0),
    (128, 16, [64, 1, 200] * 7, 64),
])
def test_decode_in_whole_sequences_and_dealt_out(dev, hq, kv, lens, shared):
    """Sequences of few pages, as a table of their width (a workgroup per sequence and head) and a wider one
    (pages dealt out) have them: the same to the roundings of both, bad lengths and pages NaN in both, captured
    calls that follow the lengths."""
    q, pool, table = decode_case(36, hq, kv, lens, shared, dev)
    wide = torch.full((len(lens), 40), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = [(q.to(dev), *pool, t.to(dev), n_d, SCALE, shared) for t in (table, wide)]
    outs = [paged_decode_attention(*a) for a in args]
    for out in outs:
        check_decode(out, q, pool, table, lens)
    assert (outs[0].float() - outs[1].float()).abs().max() < 2 ** -5
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = [paged_decode_attention(*a) for a in args]
    torch.cuda.synchronize(dev)
    for step in range(3):
        now = [max(0, n - 29 * step) for n in lens]
        now[0], now[1] = (-1, 64 * 40 + 1) if step == 2 else now[:2]
        n_d.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(dev)
        for out, a in zip(held, args):
            if step == 2:
                assert torch.isnan(out[:2]).all()
            check_decode(out, q, pool, table, now, rows=list(range(2 * (step == 2), len(lens))))
            assert torch.equal(bits(out), bits(paged_decode_attention(*a)))
    n_d.copy_(torch.tensor(lens, dtype=torch.int32))
    last = len(lens) - 1
    for t, a in zip((table, wide), args):
        bad = t.clone()
        bad[last, (lens[last] - 1) // PAGE] = pool[0][0].shape[0]
        out = paged_decode_attention(*a[:3], bad.to(dev), n_d, SCALE, 0)
        assert torch.isnan(out[last]).all()
        check_decode(out, q, pool, table, lens, rows=[0, 1, last - 1])


def test_pool_beyond_32_bit_offsets(dev):
    """Pages whose codes lie more than 4 GB into the pool: appended, attended, copied and read back."""
    pages, kv = 67000, 8
    pool = [(torch.empty((pages, kv, PAGE, D), dtype=torch.uint8, device=dev),
             torch.empty((pages, kv, PAGE, 2), dtype=torch.bfloat16, device=dev),
             torch.empty((pages, kv, PAGE, 2), dtype=torch.bfloat16, device=dev)) for _ in range(2)]
    g = gen(17)
    table = torch.tensor([[66999, 66001, 3]], dtype=torch.int32)
    k, v = randn(g, 150, kv, D), randn(g, 150, kv, D)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    paged_append(k.to(dev), v.to(dev), *pool, table.to(dev), zero)
    copy_pages(*pool, [66999, 3], [65999, 66500])
    moved = torch.tensor([[65999, 66001, 66500]], dtype=torch.int32)
    q = randn(g, 1, 16, 1, D)
    n = torch.tensor([150], dtype=torch.int32, device=dev)
    small = [tuple(t[[66999, 66001, 3]].cpu() for t in buf) for buf in pool]
    straight = torch.arange(3, dtype=torch.int32)[None]
    for t in (table, moved):
        out = paged_decode_attention(q.to(dev), *pool, t.to(dev), n, SCALE)
        check_decode(out, q, small, straight, [150])
        out = paged_decode_attention(q.to(dev), *pool, t.to(dev), n, SCALE, shared=128)
        check_decode(out, q, small, straight, [150])
        for x, buf in zip(paged_gather(*pool, t.to(dev), zero, [150]), small):
            assert torch.equal(x.cpu().double(), read_rows(buf, straight[0], 150))


# -------------------------------------------------------------------------------- packed prompts

def check_prompt(out, q, k, v, q_lens, k_lens, scale=SCALE, some=None):
    hq, kv = q.shape[1], k.shape[1]
    G = hq // kv
    a = c = 0
    q, k, v = (x.cpu().double() for x in (q, k, v))
    for s, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        rows = range(lq) if some is None or lq <= some else sorted(
            {0, 1, lq - 1, lq // 2} | {int(i) for i in torch.linspace(0, lq - 1, some)})
        for h in range(hq if lq else 0):
            if lk == 0:
                assert (out[a:a + lq, h] == 0).all()
                continue
            rows = list(rows)
            want, bound = exact_attention(q[a:a + lq, h][rows], k[c:c + lk, h // G], v[c:c + lk, h // G],
                                          [lk - lq + i for i in rows], scale)
            assert_within(out[a:a + lq, h][rows], want, bound, f"sequence {s} head {h}")
        a, c = a + lq, c + lk


@pytest.mark.parametrize("hq,kv,q_lens,k_lens", [
    (1, 1, [1], None), (4, 1, [64], None), (8, 2, [65, 1, 63, 128, 200], None), (6, 1, [43, 0, 86], None),
    (3, 3, [300], None), (16, 1, [33], None), (64, 1, [9, 5], None), (5, 1, [103], None),
    (8, 2, [1, 1, 1], [1, 64, 65]), (4, 2, [70, 5], [200, 5]), (48, 8, [17], [900]),
    (4, 1, [10, 7, 3], [4, 0, 3]), (2, 1, [700], [1500]), (32, 8, [12] * 66, None),
])
def test_prompts(dev, hq, kv, q_lens, k_lens):
    g = gen(20)
    k_lens = q_lens if k_lens is None else k_lens
    q = randn(g, sum(q_lens), hq, D)
    k, v = randn(g, sum(k_lens), kv, D), randn(g, sum(k_lens), kv, D)
    out = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    check_prompt(out, q, k, v, q_lens, k_lens, some=24)


@pytest.mark.parametrize("hq,kv,q_lens,k_lens", [
    (32, 8, [2048], [2048]), (6, 1, [3001, 900], [3001, 2500]), (8, 1, [20], [40000]), (12, 2, [512], [8193]),
])
def test_long_prompts(dev, hq, kv, q_lens, k_lens):
    g = gen(21)
    q = randn(g, sum(q_lens), hq, D)
    k, v = randn(g, sum(k_lens), kv, D), randn(g, sum(k_lens), kv, D)
    out = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    check_prompt(out, q, k, v, q_lens, k_lens, some=10)


def test_prompts_of_many_blocks(dev):
    """Enough blocks for every CU to take several whole ones, longest first: chunks, an empty sequence, rows
    without keys, a V row with an infinity."""
    g = gen(27)
    q_lens, k_lens = [3000, 0, 300, 1, 3107], [3000, 50, 100, 1, 3500]
    q = randn(g, sum(q_lens), 64, D)
    k, v = randn(g, sum(k_lens), 32, D), randn(g, sum(k_lens), 32, D)
    out = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    assert (out[3000:3200] == 0).all()  # of the sequence with more rows than keys
    check_prompt(out, q, k, v, q_lens, k_lens, some=4)
    v[1234, 5, 7] = float("inf")
    hit = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    same = torch.ones(hit.shape, dtype=torch.bool)
    same[1234:3000, 10:12, 7] = False
    assert (bits(hit) == bits(out)).cpu()[same].all()
    assert torch.isinf(hit[1234:3000, 10:12, 7]).all()


@pytest.mark.parametrize("scale,std", [(-SCALE, 1.0), (0.0, 1.0), (1.0, 1.0), (SCALE, 30.0)])
def test_prompt_scales(dev, scale, std):
    g = gen(22)
    q, k, v = randn(g, 150, 4, D, std=std), randn(g, 150, 2, D), randn(g, 150, 2, D)
    out = prompt_attention(q.to(dev), k.to(dev), v.to(dev), [150], scale)
    check_prompt(out, q, k, v, [150], [150], scale=scale)


def test_prompt_rows_of_a_fused_projection(dev):
    """q, k and v as views of one projection, and of rows that are not 16-byte aligned."""
    g = gen(23)
    T, hq, kv = 130, 8, 2
    for pad in (0, 1):
        proj = randn(g, T, (hq + 2 * kv) * D + 24 + pad)
        d = proj.to(dev)
        q, k, v = (d[:, a * D + pad:b * D + pad].unflatten(1, (b - a, D))
                   for a, b in ((0, hq), (hq, hq + kv), (hq + kv, hq + 2 * kv)))
        out = prompt_attention(q, k, v, [100, 30], SCALE)
        check_prompt(out, q, k, v, [100, 30], [100, 30], some=20)


def test_prompt_heads_first_layout(dev):
    g = gen(24)
    q, k, v = (randn(g, h, 90, D).to(dev).transpose(0, 1) for h in (6, 2, 2))
    check_prompt(prompt_attention(q, k, v, [90], SCALE), q, k, v, [90], [90])


@pytest.mark.parametrize("hq,kv,q_lens,k_lens,parts", [
    (8, 2, [700, 0, 1, 130, 64, 40], [700, 9, 1, 130, 190, 33], False),  # small blocks, all resident
    (64, 8, [900] * 3 + [77], [900] * 3 + [600], False),                  # small blocks, several rounds
    (8, 2, [260, 33], [9000, 4444], True),                                # shares that end inside blocks
    (256, 4, [1600], [7000], False),                                      # large blocks, several rounds
])
def test_prompt_ways_of_dealing_out(dev, hq, kv, q_lens, k_lens, parts):
    """Every way of dealing out the blocks, without and with an infinity in a V row that some rows see."""
    from array import array
    g = gen(31)
    lq, lk = array("i", q_lens), array("i", k_lens)
    need = _lib.load().lq_prompt_workspace_bytes(lq.buffer_info()[0], lk.buffer_info()[0], len(lq), hq, kv)
    assert (need > 0) == parts
    q = randn(g, sum(q_lens), hq, D)
    k, v = randn(g, sum(k_lens), kv, D), randn(g, sum(k_lens), kv, D)
    out = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    check_prompt(out, q, k, v, q_lens, k_lens, some=4)
    G, row = hq // kv, q_lens[0] // 2  # the first row of the first sequence that sees the key
    key = k_lens[0] - q_lens[0] + row
    v[key, 1, 7] = float("inf")
    hit = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    same = torch.ones(hit.shape, dtype=torch.bool)
    same[row:q_lens[0], G:2 * G, 7] = False
    assert (bits(hit) == bits(out)).cpu()[same].all()
    assert not hit[row:q_lens[0], G:2 * G, 7].isfinite().any()


@pytest.mark.parametrize("what", ["k nan", "k inf", "v nan", "v inf"])
@pytest.mark.parametrize("q_lens,k_lens,at", [([200], [200], 130), ([100], [164], 150), ([3, 60], [3, 60], 40)])
def test_prompt_keys_that_a_row_does_not_see_do_not_reach_it(dev, what, q_lens, k_lens, at):
    g = gen(25)
    q, k, v = randn(g, sum(q_lens), 8, D), randn(g, sum(k_lens), 2, D), randn(g, sum(k_lens), 2, D)
    seq = len(k_lens) - 1
    row = sum(k_lens[:seq]) + at
    clean = prompt_attention(q.to(dev), k.to(dev), v.to(dev), q_lens, SCALE, k_lens=k_lens)
    x = (k if what[0] == "k" else v)
    bad = x.clone()
    bad[row, 1, 7 if what[0] == "v" else slice(None)] = float(what[2:])
    args = (bad, v) if what[0] == "k" else (k, bad)
    out = prompt_attention(q.to(dev), *(t.to(dev) for t in args), q_lens, SCALE, k_lens=k_lens)
    first = sum(q_lens[:seq]) + max(0, at - (k_lens[seq] - q_lens[seq]))  # first row that sees it
    assert torch.equal(bits(out[:first]), bits(clean[:first]))
    assert torch.equal(bits(out[:, :4]), bits(clean[:, :4])), "heads of another KV head"
    if what[0] == "v":  # the rows that do see it: that dim alone
        dim = out[first:, 4:, 7].float()
        assert torch.isnan(dim).all() if "nan" in what else not torch.isfinite(dim).any()
        rest = [d for d in range(D) if d != 7]
        assert torch.equal(bits(out[first:, :, rest]), bits(clean[first:, :, rest]))
    elif "nan" in what:
        assert torch.isnan(out[first:, 4:]).all()


def test_prompt_captured(dev):
    g = gen(26)
    q_lens, k_lens = [65, 300], [65, 700]
    q, k, v = (randn(g, n, h, D).to(dev) for n, h in ((365, 8), (765, 2), (765, 2)))
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        prompt_attention(q, k, v, q_lens, SCALE, k_lens=k_lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = prompt_attention(q, k, v, q_lens, SCALE, k_lens=k_lens)
    torch.cuda.current_stream(dev).wait_stream(stream)
    for i in range(3):
        q.copy_(randn(g, 365, 8, D))
        graph.replay()
        torch.cuda.synchronize(dev)
        eager = prompt_attention(q, k, v, q_lens, SCALE, k_lens=k_lens)
        assert torch.equal(bits(out), bits(eager))
        check_prompt(out, q, k, v, q_lens, k_lens, some=12)


def test_a_step_captured(dev):
    """Rows appended, pages copied, rows read back and attended, all in one graph, replayed on new contents."""
    g = gen(28)
    lens = [100, 63]
    q, pool, table = decode_case(28, 8, 2, [n + 1 for n in lens], 0, dev)
    q_d, t_d = q.to(dev), table.to(dev)
    n_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    k, v = randn(g, 2, 2, D).to(dev), randn(g, 2, 2, D).to(dev)
    zero = torch.zeros_like(n_d)
    spare = [p for p in range(pool[0][0].shape[0]) if p not in table.flatten().tolist() + [0]][0]

    def step():
        paged_append(k, v, *pool, t_d, n_d)
        copy_pages(*pool, [int(table[0, 0])], [spare])
        rows = paged_gather(*pool, t_d, zero, [n + 1 for n in lens])
        out = paged_decode_attention(q_d, *pool, t_d, n_d + 1, SCALE)
        wide = prompt_attention(q_d.transpose(1, 2).reshape(2, 8, D), *rows, [1, 1], SCALE,
                                k_lens=[n + 1 for n in lens])
        return (*rows, out, wide)

    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    torch.cuda.current_stream(dev).wait_stream(stream)
    for i in range(4):
        k.copy_(randn(g, 2, 2, D))
        v.copy_(randn(g, 2, 2, D))
        q_d.copy_(randn(g, 2, 8, 1, D))
        torch.cuda.synchronize(dev)
        graph.replay()
        torch.cuda.synchronize(dev)
        held = [x.clone() for x in got]
        for x, y in zip(held, step()):
            assert torch.equal(bits(x), bits(y))
        check_decode(held[2], q_d.cpu(), pool, table, [n + 1 for n in lens])
        assert (held[2].float().flatten() - held[3].float().flatten()).abs().max() < 2 ** -5
        for buf in pool:
            for t in buf:
                assert torch.equal(bits(t[spare]), bits(t[int(table[0, 0])]))


def test_nothing_to_do(dev):
    pool = page_pool(2, 2, dev)
    e = torch.empty((0, 2, D), dtype=torch.bfloat16, device=dev)
    one = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    n = torch.zeros(1, dtype=torch.int32, device=dev)
    paged_append(e, e, *pool, one, n, [0])
    paged_append(e, e, *pool, one[:0], n[:0], [])
    assert paged_gather(*pool, one, n, [0])[0].shape == (0, 2, D)
    assert paged_gather(*pool, one[:0], n[:0], [])[1].shape == (0, 2, D)
    q = torch.ones((0, 4, 1, D), dtype=torch.bfloat16, device=dev)
    assert paged_decode_attention(q, *pool, one[:0], n[:0], SCALE).shape == (0, 4, 1, D)
    q = torch.ones((1, 4, 1, D), dtype=torch.bfloat16, device=dev)
    assert (paged_decode_attention(q, *pool, one, n, SCALE) == 0).all()


def test_prompt_of_no_rows(dev):
    e = torch.empty((0, 8, D), dtype=torch.bfloat16, device=dev)
    kv = torch.empty((0, 2, D), dtype=torch.bfloat16, device=dev)
    assert prompt_attention(e, kv, kv, [], SCALE).shape == (0, 8, D)
    assert prompt_attention(e, kv, kv, [0, 0], SCALE).shape == (0, 8, D)
    q = torch.ones((5, 8, D), dtype=torch.bfloat16, device=dev)
    assert (prompt_attention(q, kv, kv, [2, 3], SCALE, k_lens=[0, 0]) == 0).all()


# ------------------------------------------------------------------- a server's use of them together

def test_sessions_prompted_forked_decoded_and_compacted(dev):
    """Prompts attended packed and appended, one forked, tokens appended to all and attended, sessions closed
    and the pool compacted: every step against the contiguous cache of each session."""
    from lagunalab_amd.cache import DequantKVCache
    from lagunalab_amd.paged import PagedKVCache
    g = gen(30)
    hq, kv = 12, 2
    cache = PagedKVCache(60, kv, dev)
    prompts = [300, 64, 1, 130]
    k, v = randn(g, sum(prompts), kv, D).to(dev), randn(g, sum(prompts), kv, D).to(dev)
    q = randn(g, sum(prompts), hq, D).to(dev)
    check_prompt(prompt_attention(q, k, v, prompts, SCALE), q, k, v, prompts, prompts, some=8)
    ids = [cache.open() for _ in prompts]
    cache.append(ids, k, v, prompts)
    plain = {}
    for s, kk, vv in zip(ids, k.split(prompts), v.split(prompts)):
        plain[s] = DequantKVCache(fused_decode=True)
        plain[s].update_and_fetch(kk.transpose(0, 1)[None], vv.transpose(0, 1)[None])
        plain[s].state  # a short prompt's rows are pending until they are asked for
    forks = [cache.fork(ids[0]) for _ in range(5)]
    for s in forks:
        plain[s] = DequantKVCache(fused_decode=True)
        plain[s].update_and_fetch(k[:300].transpose(0, 1)[None], v[:300].transpose(0, 1)[None])

    def step(sessions, n=1):
        T = n * len(sessions)
        kk, vv = randn(g, T, kv, D).to(dev), randn(g, T, kv, D).to(dev)
        qq = randn(g, len(sessions), hq, 1, D).to(dev)
        cache.append(sessions, kk, vv)
        out = cache.attention(sessions, qq, SCALE)
        rows = cache.rows(sessions)[0].split([cache.length(s) for s in sessions])
        for i, s in enumerate(sessions):
            part = slice(i * n, (i + 1) * n)
            qk, qv = plain[s].q.update_and_fetch(kk[part].transpose(0, 1)[None], vv[part].transpose(0, 1)[None])
            assert plain[s].offset == cache.length(s)
            held = [tuple(t[0].cpu() for t in x) for x in (qk, qv)]  # [kv, rows, .]
            n_rows = plain[s].offset
            c, sc, bi = (t.double() for t in held[0])
            val = [(x[0].double() * x[1].double().repeat_interleave(64, -1)
                    + x[2].double().repeat_interleave(64, -1)).to(torch.bfloat16).double() for x in held]
            assert (rows[i].cpu().double() == val[0].transpose(0, 1)).all().item()
            for h in range(kv):
                G = hq // kv
                want, bound = exact_attention(qq[i, h * G:(h + 1) * G, 0].cpu().double(), val[0][h], val[1][h],
                                              [n_rows - 1] * G, SCALE)
                assert_within(out[i, h * G:(h + 1) * G, 0], want, bound, f"session {s} head {h}")
            # the contiguous cache's fused kernel, to both kernels' roundings
            fused = plain[s].attend(qq[i:i + 1], SCALE)
            assert (out[i].float() - fused[0].float()).abs().max() < 2e-2

    step(ids + forks)
    step([ids[0], *forks])
    step(forks, 40)
    for s in (ids[0], ids[2], forks[1]):
        cache.close(s)
        del plain[s]
    assert cache.trim(forks[0], 30) == 30
    plain[forks[0]].trim(30)
    used = cache.compact()
    assert used == 60 - cache.free_pages and max(max(cache.pages(s)) for s in plain) < used
    step(sorted(plain))
    cache.resize(used + 8)
    step(sorted(plain))
    step([forks[2], ids[3]], 3)


def test_adopted_session(dev):
    from lagunalab_amd.cache import DequantKVCache, QuantizedKVCache
    from lagunalab_amd.paged import PagedKVCache
    g = gen(31)
    for cls, n in ((DequantKVCache, 200), (QuantizedKVCache, 128), (DequantKVCache, 5), (DequantKVCache, 0)):
        src = cls()
        cache = PagedKVCache(6, 2, dev)
        cache.open()
        if n:
            src.update_and_fetch(randn(g, 1, 2, n, D).to(dev), randn(g, 1, 2, n, D).to(dev))
        s = cache.adopt(src)
        assert cache.length(s) == n
        if n:
            from lagunalab_amd.quant import dequantize
            for x, buf in zip(cache.rows([s]), src.state):
                assert torch.equal(bits(x), bits(dequantize(*buf)[0].transpose(0, 1)))
    four = DequantKVCache(bits=4)
    four.update_and_fetch(randn(g, 1, 2, 3, D).to(dev), randn(g, 1, 2, 3, D).to(dev))
    with pytest.raises(ValueError, match="8 bits"):
        cache.adopt(four)
    two = DequantKVCache()
    two.update_and_fetch(randn(g, 2, 2, 3, D).to(dev), randn(g, 2, 2, 3, D).to(dev))
    with pytest.raises(ValueError, match="one sequence"):
        cache.adopt(two)


@torch.no_grad()
def test_model_over_paged_batches(dev):
    """The tiny model's forward pass on PagedBatch caches: a prompt, forked into a batch, decoded; logits as
    over the dequantizing cache of the same rows."""
    from lagunalab_amd.cache import DequantKVCache
    from lagunalab_amd.paged import PagedKVCache
    from tiny_model import TinyArgs, TinyLM
    model = TinyLM(TinyArgs(layer_types=["full_attention"] * 2), device="cuda", seed=2)
    pools = [PagedKVCache(40, 2, dev) for _ in range(2)]
    first = [p.open() for p in pools]
    ids = torch.tensor([[5, 9, 2, 7, 1, 3, 8, 4] * 25], device="cuda")
    plain = [DequantKVCache() for _ in range(2)]
    one = [p.batch([s]) for p, s in zip(pools, first)]
    for part in ids.split(120, dim=1):  # two chunks
        got, want = model(part, cache=one), model(part, cache=plain)
        assert (got - want).abs().max() < 5e-2 * want.abs().max()
    forks = [[s] + [p.fork(s) for _ in range(2)] for p, s in zip(pools, first)]
    batch = [p.batch(f) for p, f in zip(pools, forks)]
    wide = []
    for c in plain:
        w = DequantKVCache()
        w.state = tuple(tuple(t.expand(3, -1, -1, -1).contiguous() for t in x) for x in c.state)
        wide.append(w)
    for i in range(3):
        tok = torch.tensor([[i + 1], [i + 70], [i + 300]], device="cuda")
        got, want = model(tok, cache=batch), model(tok, cache=wide)
        assert (got - want).abs().max() < 5e-2 * want.abs().max()
        assert batch[0].offset == 201 + i
    assert pools[0].free_pages == 40 - 3 - 3  # 3 shared whole pages, the fourth one for each
    for b in batch:
        assert b.trim(2) == 2


@torch.no_grad()
def test_lookup_generation_over_paged_caches(dev):
    from lagunalab_amd.generate import generate_greedy, generate_lookup
    from lagunalab_amd.paged import PagedKVCache
    from tiny_model import TinyArgs, TinyLM
    model = TinyLM(TinyArgs(layer_types=["full_attention"] * 2), device="cuda", seed=2)

    def make():
        pools = [PagedKVCache(8, 2, dev) for _ in range(2)]
        return [p.batch([p.open()]) for p in pools]
    prompt = [3, 1, 4, 1, 5, 9, 2, 6, 3, 1, 4, 1]
    want = generate_greedy(model, prompt, 24, cache=make())
    got, stats = generate_lookup(model, prompt, 24, g=2, n_draft=5, make_cache=make)
    assert got == want


def test_attention_block_over_a_paged_batch(dev):
    """The attention block of a layer on sessions of one prompt, beside the same block on the dequantizing
    cache."""
    from lagunalab_amd.attention import Attention
    from lagunalab_amd.cache import DequantKVCache
    from lagunalab_amd.paged import PagedKVCache
    g = gen(32)
    C, hq, kv = 256, 8, 2
    w = lambda *s: randn(g, *s, std=0.06).to(dev)  # noqa: E731
    block = Attention(w(hq * D, C), w(kv * D, C), w(kv * D, C), w(C, hq * D), w(hq, C), w(D) + 1, w(D) + 1, hq, kv,
                      {"rope_theta": 5e5, "partial_rotary_factor": 0.5})
    pool = PagedKVCache(20, kv, dev)
    s = pool.open()
    x = randn(g, 1, 150, C).to(dev)
    plain = DequantKVCache()
    got, want = block(x, "causal", pool.batch([s])), block(x, "causal", plain)
    assert (got.float() - want.float()).abs().max() < 3e-2 * want.float().abs().max()
    wide = DequantKVCache()
    wide.state = tuple(tuple(t.expand(4, -1, -1, -1).contiguous() for t in y) for y in plain.state)
    batch = pool.batch([s] + [pool.fork(s) for _ in range(3)])
    for L in (1, 3, 1):
        x = randn(g, 4, L, C).to(dev)
        mask = None if L == 1 else "causal"
        got, want = block(x, mask, batch), block(x, mask, wide)
        assert (got.float() - want.float()).abs().max() < 3e-2 * want.float().abs().max()


def test_prompt_rows_far_apart(dev):
    """Keys, values and queries 2^24 values apart, as rows of a wide buffer are."""
    g = gen(38)
    q, k, v = randn(g, 3, 4, D), randn(g, 5, 2, D), randn(g, 5, 2, D)
    wide = torch.zeros((5, 1 << 24), dtype=torch.bfloat16, device=dev)
    views = []
    for at, x in ((0, q), (1024, k), (2048, v)):
        views.append(wide[:x.shape[0], at:at + x[0].numel()].unflatten(1, x.shape[1:]))
        views[-1].copy_(x)
    check_prompt(prompt_attention(*views, [1, 2], SCALE, k_lens=[3, 2]), q, k, v, [1, 2], [3, 2])


def test_sessions_are_not_captured(dev):
    """A step of a batch inside a capture is refused before anything is recorded or moved; the graph goes on
    without it, and the sessions step outside."""
    from lagunalab_amd.paged import PagedKVCache
    g = gen(39)
    cache = PagedKVCache(8, 2, dev)
    batch = cache.batch([cache.open(), cache.open()])
    rows = lambda L: randn(g, 2, 2, L, D).to(dev)  # noqa: E731
    batch.update_and_fetch(rows(70), rows(70))
    k, q = rows(1), randn(g, 2, 4, 1, D).to(dev)
    batch.attend(q, SCALE)
    before = [t.clone() for t in (*cache.keys, *cache.values)]
    x = torch.zeros(4, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x += 1
            for call in (lambda: batch.update_and_fetch(k, k), lambda: batch.attend(q, SCALE),
                         lambda: cache.attention(batch.sessions, q, SCALE)):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
    torch.cuda.current_stream(dev).wait_stream(stream)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize(dev)
        assert (x == i + 1).all() and batch.offset == 70
        for t, o in zip((*cache.keys, *cache.values), before):
            assert torch.equal(bits(t), bits(o))
    batch.update_and_fetch(k, k)
    assert batch.offset == 71 and batch.attend(q, SCALE).isfinite().all()
