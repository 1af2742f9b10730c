"""Causal attention of packed prompts on plain bf16 rows (``lq_prompt_attn``): sequences of different
lengths one behind the other, grouped heads, no padding and no score matrix. The counterpart, for rows
that are not in a cache yet or were read back from one, of the SDPA that ``laguna_mlx/laguna.py:107``
runs with the causal mask."""
from __future__ import annotations

from array import array

import torch
from torch.autograd import forward_ad

from . import _lib

HEAD_DIM = 128


def _refuse_grad(*tensors, what="attention"):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"this {what} has no backward pass: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"this {what} has no forward derivative: its inputs have tangents")


def _lens(lens, what):
    lens = array("i", lens.tolist() if torch.is_tensor(lens) else lens)
    if lens and min(lens) < 0:
        raise ValueError(f"negative length in {what}")
    return lens


def _rows(x, heads, total, what):
    if x.dim() != 3 or x.shape[2] != HEAD_DIM or x.dtype != torch.bfloat16:
        raise ValueError(f"{what} must be bfloat16 [rows, heads, {HEAD_DIM}], got {tuple(x.shape)} {x.dtype}")
    if x.shape[0] != total or (heads and x.shape[1] != heads):
        raise ValueError(f"{what} {tuple(x.shape)} does not have {total} rows"
                         + (f" of {heads} heads" if heads else ""))
    st = x.stride()
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or st[0] >= 1 << 24 or x.data_ptr() % 16:  # the kernel's limits
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
    return x, st[0], st[1]


def prompt_attention(q, k, v, q_lens, scale, k_lens=None):
    """``q`` bf16 ``[sum(q_lens), Hq, 128]`` over ``k``, ``v`` bf16 ``[sum(k_lens), Hkv, 128]`` (any token
    and head strides): row ``i`` of sequence ``s`` sees its keys ``0 .. k_lens[s] - q_lens[s] + i``.
    ``q_lens`` and ``k_lens`` are host integers, ``k_lens`` None where every sequence has as many keys as
    rows; a chunk of a prompt has more. Returns ``[sum(q_lens), Hq, 128]``; rows that see no key are 0."""
    q_lens = _lens(q_lens, "q_lens")
    k_lens = q_lens if k_lens is None else _lens(k_lens, "k_lens")
    if len(q_lens) != len(k_lens):
        raise ValueError(f"{len(q_lens)} q_lens and {len(k_lens)} k_lens")
    dev = _lib.require_device(q, k, v)
    _refuse_grad(q, k, v)
    q, qt, qh = _rows(q, 0, sum(q_lens), "q")
    k, kt, kh = _rows(k, 0, sum(k_lens), "k")
    Hq, Hkv = q.shape[1], k.shape[1]
    v, vt, vh = _rows(v, Hkv, sum(k_lens), "v")
    if Hkv < 1 or Hq % Hkv or not 1 <= Hq // Hkv <= 64:
        raise ValueError(f"{Hq} query heads are not 1 to 64 per KV head ({Hkv})")
    lib = _lib.load()
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
    qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    lq, lk = q_lens.buffer_info()[0], k_lens.buffer_info()[0]
    with _lib.on_device(dev):
        qa = ka = 0
        for a in range(0, len(q_lens), _lib.LQ_MAX_SEQS):  # sequences per launch
            n = min(len(q_lens) - a, _lib.LQ_MAX_SEQS)
            need = lib.lq_prompt_workspace_bytes(lq + 4 * a, lk + 4 * a, n, Hq, Hkv)
            if need < 0:
                _lib.check(_lib.LQ_EINVAL, "lq_prompt_workspace_bytes")
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            _lib.check(lib.lq_prompt_attn(qp + 2 * qa * qt, kp + 2 * ka * kt, vp + 2 * ka * vt, qt, qh, kt, kh,
                                          vt, vh, lq + 4 * a, lk + 4 * a, n, Hq, Hkv, HEAD_DIM, scale,
                                          op + 2 * qa * Hq * HEAD_DIM, _lib.ptr(ws), need,
                                          _lib.raw_stream(dev)), "lq_prompt_attn")
            qa, ka = qa + sum(q_lens[a:a + n]), ka + sum(k_lens[a:a + n])
    return out
