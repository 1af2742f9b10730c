"""Refusals of the rotated append and of chunk attention on the CPU: the C ABI returns LQ_EINVAL before any launch, the
Python functions raise."""
import ctypes as C

import pytest
import torch

from lagunalab_amd import _lib, paged
from lagunalab_amd.rotary import Rotary


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from lagunalab_amd import build
        build.build()
    return _lib.load()


def ints(*x):
    return (C.c_int32 * len(x))(*x)


POOL = (256,) * 6  # pointers that pass the alignment checks and are never followed


def rotate(lib, **kw):
    a = dict(q=256, k=256, v=256, q_tok=1024, q_head=128, k_tok=256, k_head=128, v_tok=256, v_head=128, qw=256, kw=256,
             eps=1e-6, freq=256, dims=128, mscale=1.0, pairs=0, pool=POOL, pages=4, hq=8, kv=2, D=128, table=256, stride=4,
             width=4, starts=256, counts=ints(1, 2), n=2, q_out=256, k_out=None, v_out=None)
    a.update(kw)
    return lib.lq_paged_append_rotated(
        a["q"], a["k"], a["v"], a["q_tok"], a["q_head"], a["k_tok"], a["k_head"], a["v_tok"], a["v_head"], a["qw"], a["kw"],
        a["eps"], a["freq"], a["dims"], a["mscale"], a["pairs"], *a["pool"], a["pages"], a["hq"], a["kv"], a["D"],
        a["table"], a["stride"], a["width"], a["starts"], a["counts"], a["n"], a["q_out"], a["k_out"], a["v_out"], None)


@pytest.mark.parametrize("bad,word", [
    (dict(D=64), b"head_dim"), (dict(kv=0), b"KV heads"), (dict(kv=1025), b"KV heads"), (dict(pages=0), b"pages"),
    (dict(pages=1 << 26), b"pages"), (dict(width=0), b"table row"), (dict(width=1 << 19), b"table row"),
    (dict(table=None), b"null"), (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(v=None), b"null"),
    (dict(starts=None), b"null"), (dict(q_out=None), b"null"), (dict(pool=(256, None, 256, 256, 256, 256)), b"null"),
    (dict(pool=(257,) * 6), b"aligned"), (dict(q=264), b"aligned"), (dict(k=260), b"aligned"), (dict(v=8), b"aligned"),
    (dict(q_out=8), b"aligned"), (dict(qw=264), b"aligned"), (dict(kw=2), b"aligned"), (dict(q_tok=1028), b"aligned"),
    (dict(k_head=4), b"aligned"), (dict(v_tok=130), b"aligned"), (dict(k_out=264, v_out=256), b"aligned"),
    (dict(k_out=256), b"alone"), (dict(v_out=256), b"alone"), (dict(hq=-1), b"query heads"),
    (dict(hq=(1 << 16) + 1), b"query heads"), (dict(dims=130), b"rotated"), (dict(dims=-4), b"rotated"),
    (dict(dims=66), b"rotated"), (dict(dims=65, pairs=1), b"rotated"), (dict(dims=132, pairs=1), b"rotated"),
    (dict(freq=None), b"frequencies"), (dict(mscale=float("inf")), b"mscale"), (dict(eps=-1e-6), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(counts=ints(1, -2)), b"count"), (dict(counts=None), b"counts"),
    (dict(n=0), b"sequences"), (dict(n=65, counts=ints(*[1] * 65)), b"sequences"),
    (dict(counts=ints(1 << 29, 1 << 29)), b"count"), (dict(counts=ints(1 << 28, 1)), b"too large"),
])
def test_rotate_refusals(lib, bad, word):
    assert rotate(lib, **bad) == _lib.LQ_EINVAL
    assert word in lib.lq_last_error()


def test_no_rows_are_no_launch(lib):
    assert rotate(lib, counts=ints(0, 0), q=None, k=None, v=None, q_out=None, starts=None) == _lib.LQ_OK
    assert attend(lib, counts=ints(0, 0), q=None, out=None, lens=None, ws=None, wsb=0) == _lib.LQ_OK


def attend(lib, **kw):
    a = dict(q=256, q_tok=1024, q_head=128, pool=POOL, pages=4, hq=8, kv=2, D=128, table=256, stride=4, width=4, lens=256,
             counts=ints(1, 200), n=2, window=0, scale=0.1, out=256, ws=256, wsb=1 << 40)
    a.update(kw)
    return lib.lq_paged_chunk_attn(a["q"], a["q_tok"], a["q_head"], *a["pool"], a["pages"], a["hq"], a["kv"], a["D"],
                                   a["table"], a["stride"], a["width"], a["lens"], a["counts"], a["n"], a["window"],
                                   a["scale"], a["out"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("bad,word", [
    (dict(D=64), b"head_dim"), (dict(kv=0), b"KV heads"), (dict(pages=0), b"pages"), (dict(width=0), b"table row"),
    (dict(width=1 << 19), b"table row"), (dict(stride=-1), b"table row"), (dict(table=None), b"null"),
    (dict(pool=(256, 256, 256, 256, 256, None)), b"null"), (dict(pool=(264,) * 6), b"aligned"),
    (dict(hq=9), b"Hq"), (dict(hq=0), b"Hq"), (dict(hq=130), b"Hq"), (dict(q=None), b"null"), (dict(out=None), b"null"),
    (dict(lens=None), b"null"), (dict(q=264), b"aligned"), (dict(out=8), b"aligned"), (dict(q_tok=1028), b"aligned"),
    (dict(q_head=4), b"aligned"), (dict(counts=None), b"counts"), (dict(n=0), b"sequences"),
    (dict(n=65, counts=ints(*[1] * 65)), b"sequences"), (dict(counts=ints(-1, 2)), b"count"),
    (dict(counts=ints((1 << 24) + 1, 2)), b"count"), (dict(hq=128, counts=ints(1 << 24, 2)), b"count"),
    (dict(window=-1), b"window"), (dict(window=1 << 40), b"window"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(ws=264), b"aligned"),
    # more rows than all the workgroups of a launch, or costs than 32 bits
    (dict(hq=1024, kv=1024, counts=ints(1 << 24, 1 << 24), q_tok=1 << 17), b"too many rows"),
    (dict(hq=2, counts=ints(1 << 23, 2), width=1 << 18, stride=1 << 18), b"too many rows"),
    (dict(hq=2, counts=ints(1 << 20, 2), width=1 << 18, stride=1 << 18), b"too many rows"),
])
def test_chunk_refusals(lib, bad, word):
    assert attend(lib, **bad) == _lib.LQ_EINVAL
    assert word in lib.lq_last_error()


def test_a_workspace_that_is_too_small(lib):
    counts = ints(1, 200)
    need = lib.lq_paged_chunk_workspace_bytes(counts, 2, 8, 2, 100, 0)
    assert need > 0
    for bad in (dict(ws=None), dict(wsb=need - 1), dict(wsb=0)):
        assert attend(lib, **dict(dict(counts=counts, width=100, stride=100, wsb=need), **bad)) == _lib.LQ_EWORKSPACE
        assert b"workspace" in lib.lq_last_error()


def test_workspace_sizes(lib):
    need = lib.lq_paged_chunk_workspace_bytes
    assert need(ints(0), 1, 8, 2, 4, 0) == 0
    assert need(ints(1), 1, 8, 2, 4, 0) == 0  # a short table: one launch
    for bad in ((None, 1, 8, 2, 4, 0), (ints(1), 0, 8, 2, 4, 0), (ints(1), 65, 8, 2, 4, 0), (ints(-1), 1, 8, 2, 4, 0),
                (ints(1), 1, 7, 2, 4, 0), (ints(1), 1, 8, 2, 0, 0), (ints(1), 1, 8, 2, 4, -1)):
        assert need(*bad) < 0, bad
    # a share per KV head is not cut
    assert need(ints(5000), 1, 512, 512, 1 << 18, 0) == 0
    # partial rows, whatever the lengths: below 128 MiB up to 64 KV heads
    for hq, kv in ((8, 1), (32, 8), (48, 8), (64, 64), (512, 8)):
        for counts in ([1], [1] * 64, [500] * 64, [4096], [5, 4096]):
            assert 0 <= need(ints(*counts), len(counts), hq, kv, 1 << 18, 0) < 1 << 27, (hq, kv, counts)


def test_there_is_no_cpu_path():
    keys, values = paged.page_pool(4, 2, device="cpu")
    x = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    table = torch.zeros((2, 2), dtype=torch.int32)
    n = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm"):
        paged.paged_append_rotated(x, x, x, keys, values, table, n, None)
    with pytest.raises(ValueError, match="ROCm"):
        paged.paged_chunk_attention(x, keys, values, table, n, 0.1)


@pytest.fixture
def anywhere(monkeypatch):
    """Tensors pass for the GPU's, and a launch is a failure."""
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(paged, "_pool", lambda keys, values: (*keys[0].shape[:2], keys[0].device, [256] * 6))

    def launched(*a):
        raise AssertionError("launched")
    monkeypatch.setattr(_lib, "load", launched)


X = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
N = torch.ones(2, dtype=torch.int32)
TABLE = torch.zeros((2, 3), dtype=torch.int32)


@pytest.mark.parametrize("bad,word", [
    (dict(q=X[:3]), "q must be"), (dict(q=X.float()), "q must be"), (dict(q=X[0]), "q must be"), (dict(q=X[..., :64]), "q must"),
    (dict(k=X[:, :1]), "k must be"), (dict(k=X.half()), "k must be"), (dict(v=X[:3]), "v must be"),
    (dict(k=X[:3]), "the same number"), (dict(counts=[1, 2]), "add up"), (dict(counts=[4]), "counts for"),
    (dict(counts=[5, -1]), "negative"), (dict(table=TABLE[0]), "table"), (dict(table=TABLE.long()), "table"),
    (dict(table=TABLE[:, :0]), "no pages"), (dict(starts=N[:1]), "starts"), (dict(starts=N.long()), "starts"),
    (dict(starts=[1, 2]), "starts"), (dict(q_norm=X[0, 0, :64]), "q_norm"), (dict(k_norm=X[0, 0].float()), "k_norm"),
    (dict(k_norm=X[0]), "k_norm"),
])
def test_rotate_arguments_that_do_not_fit(anywhere, bad, word):
    keys, values = paged.page_pool(4, 2, device="cpu")
    a = dict(dict(q=X, k=X, v=X, keys=keys, values=values, table=TABLE, starts=N, rotary=None), **bad)
    with pytest.raises(ValueError, match=word):
        paged.paged_append_rotated(**a)


@pytest.mark.parametrize("bad,word", [
    (dict(q=X[0]), "q must be"), (dict(q=X.float()), "q must be"), (dict(q=X[..., :64]), "q must be"),
    (dict(q=X[:3]), "the same number"), (dict(q=X[:, :1]), "query heads"), (dict(q=X.repeat(1, 65, 1)), "query heads"),
    (dict(q=torch.cat([X, X[:, :1]], 1)), "query heads"), (dict(counts=[1, 2]), "add up"), (dict(counts=[4]), "counts for"),
    (dict(counts=[5, -1]), "negative"), (dict(window=0), "window"), (dict(window=-3), "window"), (dict(table=TABLE[0]), "table"),
    (dict(table=TABLE[:, :0]), "no pages"), (dict(lens=N.long()), "lens"), (dict(lens=N[:1]), "lens"),
    (dict(lens=torch.ones((2, 1), dtype=torch.int32)), "lens"),
])
def test_chunk_arguments_that_do_not_fit(anywhere, bad, word):
    keys, values = paged.page_pool(4, 2, device="cpu")
    a = dict(dict(q=X, keys=keys, values=values, table=TABLE, lens=N, scale=0.1), **bad)
    with pytest.raises(ValueError, match=word):
        paged.paged_chunk_attention(**a)


def test_rows_that_want_a_gradient(anywhere):
    keys, values = paged.page_pool(4, 2, device="cpu")
    x, w, f = X.clone().requires_grad_(), X[0, 0].clone().requires_grad_(), torch.ones(4).requires_grad_()
    with pytest.raises(ValueError, match="attention has no backward"):
        paged.paged_chunk_attention(x, keys, values, TABLE, N, 0.1)
    for a in (dict(q=x), dict(k=x), dict(v=x), dict(q_norm=w), dict(k_norm=w), dict(rotary=Rotary(f))):
        with pytest.raises(ValueError, match="append has no backward"):
            paged.paged_append_rotated(**dict(dict(q=X, k=X, v=X, keys=keys, values=values, table=TABLE, starts=N,
                                                   rotary=None), **a))


def test_rotaries_that_cannot_be():
    f = torch.ones(4)
    for bad in (f.double(), f[None], f.long()):
        with pytest.raises(ValueError, match="frequencies"):
            Rotary(bad)
    for m in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="factor"):
            Rotary(f, m)
    r = Rotary(torch.arange(8.0)[::2], 2)
    assert r.dims == 8 and r.inv_freq.is_contiguous() and r.mscale == 2.0 and not r.interleaved
