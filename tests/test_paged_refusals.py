"""Refusals of the paged cache and packed-prompt entry points, on the CPU: the C ABI returns LQ_EINVAL
before any launch, the Python functions raise."""
import ctypes as C

import pytest
import torch

from lagunalab_amd import _lib, paged, prompt_attn


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from lagunalab_amd import build
        build.build()
    return _lib.load()


def ints(*x):
    return (C.c_int32 * len(x))(*x)


POOL = (256,) * 6  # pointers that pass the alignment checks and are never followed


def append(lib, **kw):
    a = dict(k=256, v=256, k_tok=256, k_head=128, v_tok=256, v_head=128, pool=POOL, pages=4, kv=2, D=128,
             table=256, stride=4, width=4, starts=256, counts=ints(1, 2), n=2)
    a.update(kw)
    return lib.lq_paged_append(a["k"], a["v"], a["k_tok"], a["k_head"], a["v_tok"], a["v_head"], *a["pool"],
                               a["pages"], a["kv"], a["D"], a["table"], a["stride"], a["width"],
                               a["starts"], a["counts"], a["n"], None)


@pytest.mark.parametrize("bad,word", [
    (dict(D=64), b"head_dim"), (dict(kv=0), b"KV heads"), (dict(pages=0), b"pages"),
    (dict(pages=1 << 26), b"pages"), (dict(width=0), b"table row"), (dict(width=1 << 19), b"table row"),
    (dict(table=None), b"null"), (dict(k=None), b"null"), (dict(starts=None), b"null"),
    (dict(pool=(256, 256, None, 256, 256, 256)), b"null"), (dict(pool=(257,) * 6), b"aligned"),
    (dict(k=260), b"aligned"), (dict(k_tok=130), b"aligned"), (dict(v_head=4), b"aligned"),
    (dict(counts=ints(1, -2)), b"count"), (dict(counts=None), b"counts"), (dict(n=0), b"sequences"),
    (dict(n=65, counts=ints(*[1] * 65)), b"sequences"), (dict(counts=ints(1 << 29, 1 << 29)), b"count"),
    (dict(kv=8, counts=ints(1 << 25, 1)), b"too large"),
])
def test_append_refusals(lib, bad, word):
    assert append(lib, **bad) == _lib.LQ_EINVAL
    assert word in lib.lq_last_error()


def test_no_rows_are_no_launch(lib):
    assert append(lib, counts=ints(0, 0), k=None, v=None) == _lib.LQ_OK
    assert lib.lq_paged_gather(*POOL, 4, 2, 128, 256, 4, 4, 256, ints(0, 0), 2, None, None, None) == _lib.LQ_OK
    assert lib.lq_prompt_attn(None, None, None, 128, 128, 128, 128, 128, 128, ints(0), ints(5), 1, 4, 2, 128, 0.1,
                              None, None, 0, None) == _lib.LQ_OK


def test_gather_refusals(lib):
    ok = [*POOL, 4, 2, 128, 256, 4, 4, 256, ints(1, 2), 2, 256, 256, None]
    for i, x, word in ((0, None, b"null"), (8, 96, b"head_dim"), (9, None, b"null"), (13, None, b"counts"),
                       (14, 65, b"sequences"), (15, None, b"null"), (16, 264, b"aligned")):
        args = list(ok)
        args[i] = x
        assert lib.lq_paged_gather(*args) == _lib.LQ_EINVAL, i
        assert word in lib.lq_last_error()


@pytest.mark.parametrize("src,dst,word", [
    ([0], [4], b"pool"), ([-1], [0], b"pool"), ([0, 1], [2, 2], b"twice"), ([0, 1], [1, 2], b"twice"),
    ([2], [2], b"twice"), ([0, 0, 0, 0, 0], [1, 2, 3, 1, 2], b"pages to copy"),
])
def test_copy_refusals(lib, src, dst, word):
    st = lib.lq_copy_pages(*POOL, 4, 2, 128, ints(*src), ints(*dst), len(src), None)
    assert st == _lib.LQ_EINVAL and word in lib.lq_last_error()


def test_copy_of_no_pages_is_no_launch(lib):
    assert lib.lq_copy_pages(*POOL, 4, 2, 128, None, None, 0, None) == _lib.LQ_OK
    assert lib.lq_copy_pages(*POOL, 4, 2, 128, None, None, 1, None) == _lib.LQ_EINVAL
    assert lib.lq_copy_pages(*POOL, 4, 2, 128, None, None, -1, None) == _lib.LQ_EINVAL


@pytest.mark.parametrize("bad,word", [
    (dict(q=None), b"null"), (dict(q=264), b"aligned"), (dict(lens=None), b"null"), (dict(D=96), b"head_dim"),
    (dict(hq=9), b"Hq"), (dict(hq=34), b"Hq"), (dict(kv=1024, hq=16384, B=512), b"too many"), (dict(B=0), b"batch"), (dict(B=4097), b"batch"),
    (dict(shared=5), b"shared"), (dict(shared=-1), b"shared"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(wsb=1000), b"workspace"), (dict(ws=None), b"workspace"),
])
def test_decode_refusals(lib, bad, word):
    a = dict(q=256, pages=4, B=2, hq=8, kv=2, D=128, table=256, stride=4, width=4, lens=256, shared=1,
             scale=0.1, out=256, ws=256, wsb=1 << 40)
    a.update(bad)
    st = lib.lq_paged_decode_attn(a["q"], *POOL, a["pages"], a["B"], a["hq"], a["kv"], a["D"], a["table"],
                                  a["stride"], a["width"], a["lens"], a["shared"], a["scale"], a["out"],
                                  a["ws"], a["wsb"], None)
    assert st in (_lib.LQ_EINVAL, _lib.LQ_EWORKSPACE) and word in lib.lq_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(q=264), b"aligned"), (dict(k_tok=100), b"aligned"),
    (dict(D=64), b"head_dim"), (dict(hq=7), b"Hq"), (dict(hq=130), b"Hq"), (dict(n=65), b"sequences"),
    (dict(n=0), b"sequences"), (dict(ql=ints(-1, 2)), b"rows"), (dict(kl=ints(3, (1 << 24) + 1)), b"keys"),
    (dict(ql=None), b"null"), (dict(scale=float("inf")), b"scale"),
    (dict(ql=ints(20, 3), kl=ints(40000, 3)), b"workspace"),
])
def test_prompt_refusals(lib, bad, word):
    a = dict(q=256, k=256, v=256, q_tok=1024, q_head=128, k_tok=256, k_head=128, v_tok=256, v_head=128,
             ql=ints(4, 3), kl=ints(4, 3), n=2, hq=8, kv=2, D=128, scale=0.1, out=256, ws=None, wsb=0)
    a.update(bad)
    st = lib.lq_prompt_attn(a["q"], a["k"], a["v"], a["q_tok"], a["q_head"], a["k_tok"], a["k_head"],
                            a["v_tok"], a["v_head"], a["ql"], a["kl"], a["n"], a["hq"], a["kv"], a["D"],
                            a["scale"], a["out"], a["ws"], a["wsb"], None)
    assert st in (_lib.LQ_EINVAL, _lib.LQ_EWORKSPACE) and word in lib.lq_last_error()


def test_workspace_sizes(lib):
    assert lib.lq_paged_decode_workspace_bytes(0, 8, 2, 0) < 0
    assert lib.lq_paged_decode_workspace_bytes(1, 8, 3, 0) < 0
    small = lib.lq_paged_decode_workspace_bytes(1, 8, 2, 0)
    assert 0 < small < lib.lq_paged_decode_workspace_bytes(16, 8, 2, 512) < 1 << 27
    assert lib.lq_paged_decode_workspace_bytes(4096, 128, 8, 1 << 18) < 1 << 32
    assert lib.lq_prompt_workspace_bytes(ints(0), ints(0), 1, 8, 2) == 0
    assert lib.lq_prompt_workspace_bytes(ints(1), ints(70000), 1, 8, 2) > 0
    assert lib.lq_prompt_workspace_bytes(ints(1), ints(-1), 1, 8, 2) < 0


def test_there_is_no_cpu_path():
    keys, values = paged.page_pool(4, 2, device="cpu")
    x = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    table = torch.zeros((2, 2), dtype=torch.int32)
    n = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm"):
        paged.paged_append(x, x, keys, values, table, n)
    with pytest.raises(ValueError, match="ROCm"):
        paged.paged_gather(keys, values, table, n, [1, 1])
    with pytest.raises(ValueError, match="ROCm"):
        paged.paged_decode_attention(x.unsqueeze(2), keys, values, table, n, 0.1)
    with pytest.raises(ValueError, match="ROCm"):
        paged.copy_pages(keys, values, [0], [1])
    with pytest.raises(ValueError, match="ROCm"):
        prompt_attn.prompt_attention(x, x, x, [2], 0.1)


def test_arguments_that_do_not_fit():
    x = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="negative"):
        prompt_attn.prompt_attention(x, x, x, [3, -1], 0.1)
    with pytest.raises(ValueError, match="q_lens"):
        prompt_attn.prompt_attention(x, x, x, [2], 0.1, k_lens=[1, 1])
    with pytest.raises(ValueError):
        paged.page_pool(0, 2, device="cpu")
    keys, values = paged.page_pool(4, 2, device="cpu")
    with pytest.raises(ValueError, match="values are"):
        paged.paged_gather(keys[:2], values, torch.zeros(1, 1), None, [1])
    with pytest.raises(ValueError, match="contiguous"):
        paged.paged_gather((keys[0].transpose(0, 1), *keys[1:]), values, torch.zeros(1, 1), None, [1])
    with pytest.raises(ValueError, match="contiguous"):
        paged.paged_gather((keys[0].int(), *keys[1:]), values, torch.zeros(1, 1), None, [1])


def test_gradients_and_tangents_are_refused(monkeypatch):
    """Neither attention has a backward or a forward derivative: a call that would need one raises, before any
    work (what follows the check is left out here)."""
    from torch.autograd import forward_ad
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    x = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    grad = x.clone().requires_grad_()
    for args in ((grad, x, x), (x, grad, x), (x, x, grad)):
        with pytest.raises(ValueError, match="backward"):
            prompt_attn.prompt_attention(*args, [2], 0.1)
    monkeypatch.setattr(paged, "_pool", lambda k, v: (4, 2, x.device, [0] * 6))
    keys, values = paged.page_pool(4, 2, device="cpu")
    decode = lambda q: paged.paged_decode_attention(q.unsqueeze(2), keys, values, None, None, 0.1)  # noqa: E731
    with pytest.raises(ValueError, match="backward"):
        decode(grad)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for no_grad in (False, True):  # which does not stop forward mode
            with torch.set_grad_enabled(not no_grad):
                for args in ((dual, x, x), (x, dual, x), (x, x, dual)):
                    with pytest.raises(ValueError, match="tangent"):
                        prompt_attn.prompt_attention(*args, [2], 0.1)
                with pytest.raises(ValueError, match="tangent"):
                    decode(dual)
        with pytest.raises(ValueError, match="table"):  # plain tensors beside it go on
            decode(x)


def test_prompt_rows_far_apart_are_copied():
    """Any token and head strides: the kernel takes rows less than 2^24 values apart as they lie, others are
    copied, and so is a single row whatever its stride."""
    far = 1 << 24
    store = torch.zeros(far + 300, dtype=torch.bfloat16)
    for rows, stride, copied in ((2, far, True), (2, far - 8, False), (1, 1 << 40, True), (1, 256, False)):
        x = store.as_strided((rows, 2, 128), (stride, 128, 1))
        got, tok, head = prompt_attn._rows(x, 2, rows, "k")
        assert (got is not x) == copied and (tok, head) == ((256 if copied else stride), 128)


def test_appends_of_a_full_grid_are_refused(lib):
    """16 rows per workgroup of 256 threads: 2^32 threads are more than a launch may have."""
    for kv, rows in ((8, (1 << 25) - 1), (1, (1 << 28) - 14)):
        assert append(lib, kv=kv, counts=ints(rows), n=1) == _lib.LQ_EINVAL
        assert b"too large" in lib.lq_last_error()
