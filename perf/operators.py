"""Performance cases of the operators that serve several sessions from one paged 8-bit cache.

A pool holds the K/V of one layer in pages of 64 positions: codes ``uint8 [pages, Hkv, 64, 128]``,
scales and biases ``bf16 [pages, Hkv, 64, 2]`` (8-bit affine codes, groups of 64), for keys and for
values. Row ``b`` of an int32 table lists the pages of sequence ``b`` in order; sequences that were
forked from one prompt list the same pages. The operations (``op``):

* ``decode``: attention of one new token per sequence over its pages, the pages that all sequences
  share read once for the batch.
* ``prompt``: causal attention of packed prompts of different lengths, plain bf16 rows; a chunk of a
  prompt has fewer query rows than keys.
* ``chunk``: new rows quantized into the pages, and all rows of the sequences read back as bf16 for
  the chunk's attention.
* ``copy``: pages copied within the pool, when forked sequences part or the pool is compacted.

An attended value is what dequantizing the page gives: ``bf16(scale * code + bias)``. Head layouts
are query heads / KV heads of head_dim 128; 48/8 is Laguna's, 32/8 the benchmark's.
"""
import math
import random

import torch

own = False

D = 128
PAGE = 64
GROUP = 64
SCALE = D ** -0.5
ROW_BYTES = 2 * (D + 2 * 2 * (D // GROUP))  # K and V codes, scales and biases of a row of one head


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token of one session early in a chat: latency
        {"name": "decode 1k", "op": "decode", "heads": 32, "kv": 8, "seqs": 1, "shared": 0,
         "shortest": 1037, "longest": 1037},
        # a token of each of eight long sessions that share nothing (the ragged lengths of the benchmark)
        {"name": "decode ragged 8", "op": "decode", "heads": 32, "kv": 8, "seqs": 8, "shared": 0,
         "shortest": 42771, "longest": 82671},
        # sixteen answers sampled from one long prompt
        {"name": "decode 16 of 32k", "op": "decode", "heads": 32, "kv": 8, "seqs": 16,
         "shared": 32768, "shortest": 1, "longest": 1023},
        # a serving batch behind one long system prompt, Laguna's head layout
        {"name": "decode 48 of 16k", "op": "decode", "heads": 48, "kv": 8, "seqs": 48,
         "shared": 16384, "shortest": 97, "longest": 2011},
        # one ordinary prompt
        {"name": "prompt 2k", "op": "prompt", "heads": 32, "kv": 8, "seqs": 1, "shortest": 2048,
         "longest": 2048, "past": 0},
        # a batch of new requests of very different lengths
        {"name": "prompts packed 48q", "op": "prompt", "heads": 48, "kv": 8, "seqs": 7, "shortest": 1,
         "longest": 4099, "past": 0},
        # a new user turn behind an existing session
        {"name": "prompt 512 on 8k", "op": "prompt", "heads": 48, "kv": 8, "seqs": 1, "shortest": 512,
         "longest": 512, "past": 7681},
        # one long prompt in a single call
        {"name": "prompt 16k", "op": "prompt", "heads": 32, "kv": 8, "seqs": 1, "shortest": 16384,
         "longest": 16384, "past": 0},
        # one new row for each of a batch of short sessions
        {"name": "chunk 8 rows", "op": "chunk", "kv": 8, "seqs": 8, "rows": 1, "shortest": 5,
         "longest": 199},
        # a prompt chunk behind a long session
        {"name": "chunk 2048 on 32k", "op": "chunk", "kv": 8, "seqs": 1, "rows": 2048,
         "shortest": 32771, "longest": 32771},
        # the last page of a prompt copied for each of its forks
        {"name": "fork 15", "op": "copy", "kv": 8, "pages": 15, "sources": 1, "pool": 640},
        # a pool of ended sessions compacted
        {"name": "compact 1500", "op": "copy", "kv": 8, "pages": 1500, "sources": 1500, "pool": 4096},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    return rng.choice([(32, 8), (32, 8), (48, 8), (48, 8), (64, 8), (16, 8), (16, 2), (8, 8)])


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "prompt", "chunk", "copy"])
    hq, kv = _heads(rng)
    if op == "decode":
        seqs = _log(rng, 1, 64)
        if rng.random() < 0.5:  # nothing shared: up to the longest listed batch
            longest = _log(rng, 2, min(82671, 8 * 62721 * 32 // (seqs * hq)))
            return {"op": op, "heads": hq, "kv": kv, "seqs": seqs, "shared": 0,
                    "shortest": rng.randint(1 + longest // 20, longest), "longest": longest}
        shared = PAGE * _log(rng, 1, min(1024, max(1, 48 * 270 * 48 // (seqs * hq))))
        longest = _log(rng, 2, 4096)
        return {"op": op, "heads": hq, "kv": kv, "seqs": seqs, "shared": shared,
                "shortest": rng.randint(0, longest // 2), "longest": longest}
    if op == "prompt":
        seqs = rng.choice([1, 1, 2, 3, 5, 9, 17])
        longest = _log(rng, 2, 8192 if seqs == 1 else 2048)
        past = rng.choice([0, 0, _log(rng, 1, 16384)]) if longest * seqs <= 4096 else 0
        return {"op": op, "heads": hq, "kv": kv, "seqs": seqs,
                "shortest": longest if seqs == 1 else rng.randint(0, longest // 2), "longest": longest,
                "past": past}
    if op == "chunk":
        seqs = rng.choice([1, 2, 5, 8, 31])
        longest = _log(rng, 1, 32768 // seqs)
        return {"op": op, "kv": kv, "seqs": seqs, "rows": _log(rng, 1, max(2, 2048 // seqs)),
                "shortest": rng.randint(0, longest), "longest": longest}
    pages = _log(rng, 1, 1500)
    return {"op": op, "kv": kv, "pages": pages, "sources": rng.choice([1, pages]),
            "pool": 2 * pages + rng.randint(1, 64)}


def _spread(case):
    """The lengths of a case's sequences: from shortest to longest, in mixed order."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lens = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(lens)
    return lens


# ----------------------------------------------------------------------------------------- inputs

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)


def _pool(gen, pages, kv):
    """K and V pools that hold N(0, 1) rows in 8 bits, filled in slabs."""
    made = []
    for _ in range(2):
        codes = torch.empty((pages, kv, PAGE, D), dtype=torch.uint8, device="cuda")
        scales = torch.empty((pages, kv, PAGE, D // GROUP), dtype=torch.bfloat16, device="cuda")
        biases = torch.empty_like(scales)
        for p in range(0, pages, 512):
            q = min(pages, p + 512)
            codes[p:q], scales[p:q], biases[p:q] = _quantize(_randn(gen, q - p, kv, PAGE, D))
        made.append((codes, scales, biases))
    return made


def _table(gen, lens, shared):
    """Pages for sequences of these lengths whose first ``shared`` positions are one another's, in
    random order over a pool with some pages to spare: (table, pages of the pool)."""
    need = [-(-n // PAGE) for n in lens]
    common = shared // PAGE
    total = common + sum(max(0, n - common) for n in need)
    pages = total + total // 16 + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(need + [1])), dtype=torch.int32, device="cuda")
    at = common
    for b, n in enumerate(need):
        k = min(n, common)
        table[b, :k] = order[:k]
        if n > common:
            table[b, common:n] = order[at:at + n - common]
            at += n - common
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"op": op}
    if op == "decode":
        lens = [case["shared"] + n for n in _spread(case)]
        s["table"], pages = _table(gen, lens, case["shared"])
        s["keys"], s["values"] = _pool(gen, pages, case["kv"])
        s["q"] = _randn(gen, case["seqs"], case["heads"], 1, D)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["shared"] = case["shared"]
    elif op == "prompt":
        s["q_lens"] = _spread(case)
        s["k_lens"] = [n + case["past"] for n in s["q_lens"]]
        rows, keys = sum(s["q_lens"]), sum(s["k_lens"])
        s["q"] = _randn(gen, rows, case["heads"], D)
        s["k"], s["v"] = _randn(gen, keys, case["kv"], D), _randn(gen, keys, case["kv"], D)
    elif op == "chunk":
        starts = _spread(case)
        s["counts"] = [case["rows"]] * case["seqs"]
        s["ends"] = [n + case["rows"] for n in starts]
        s["table"], pages = _table(gen, s["ends"], 0)
        s["keys"], s["values"] = _pool(gen, pages, case["kv"])
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["zeros"] = torch.zeros_like(s["starts"])
        rows = sum(s["counts"])
        s["k"], s["v"] = _randn(gen, rows, case["kv"], D), _randn(gen, rows, case["kv"], D)
    else:
        s["keys"], s["values"] = _pool(gen, case["pool"], case["kv"])
        order = torch.randperm(case["pool"], generator=gen, device="cuda").tolist()
        s["dst"] = sorted(order[:case["pages"]])
        s["src"] = (sorted(order[case["pages"]:2 * case["pages"]]) if case["sources"] > 1
                    else order[-1:] * case["pages"])
    return s


# ------------------------------------------------------------------------------- the plain forms

def _round(x):
    """Nearest whole number, halves away from zero."""
    t = torch.trunc(x)
    return t + torch.where((x - t).abs() >= 0.5, torch.sign(x), torch.zeros_like(x))


def _quantize(x):
    """8-bit affine codes, bf16 scales and biases of rows [..., 128], in groups of 64: the scale is the
    group's range over 255, signed so that codes count from the edge of larger magnitude, and made
    to divide that edge."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    delta = ((hi - lo) / 255.0).clamp_min(1e-7)
    low = lo.abs() > hi.abs()
    scale, edge = torch.where(low, delta, -delta), torch.where(low, lo, hi)
    steps = _round(edge / scale)
    zero = steps == 0
    scale = torch.where(zero, scale, edge / torch.where(zero, torch.ones_like(steps), steps))
    bias = torch.where(zero, torch.zeros_like(edge), edge)
    codes = _round((g - bias) / scale).clamp(0, 255)
    return (codes.flatten(-2).to(torch.uint8), scale.squeeze(-1).to(torch.bfloat16),
            bias.squeeze(-1).to(torch.bfloat16))


def _values(buf, pages, slots):
    """Rows (page, slot) of a pool as bf16 [rows, Hkv, 128]."""
    codes, scales, biases = (t[pages, :, slots] for t in buf)
    g = codes.float().unflatten(-1, (-1, GROUP))
    return (g * scales.float().unsqueeze(-1) + biases.float().unsqueeze(-1)).flatten(-2).to(torch.bfloat16)


def _places(table, b, start, end):
    at = torch.arange(start, end, device=table.device)
    return table[b].long()[at // PAGE], at % PAGE


def _attend(q, k, v, first):
    """Softmax attention of rows q [L, Hq, 128] over k, v [n, Hkv, 128]: row i sees keys 0 .. first + i.
    A row without keys is zero. In slabs of rows, a KV head at a time."""
    rows, hq, _ = q.shape
    keys, kv, _ = k.shape
    group = hq // kv
    out = torch.zeros((rows, hq, D), dtype=torch.float32, device=q.device)
    if keys == 0:
        return out.to(torch.bfloat16)
    slab = max(1, (1 << 28) // (group * keys))
    at = torch.arange(keys, device=q.device)
    for h in range(kv):
        kh, vh = k[:, h].float(), v[:, h].float()
        for a in range(0, rows, slab):
            e = min(rows, a + slab)
            x = q[a:e, h * group:(h + 1) * group].float().reshape(-1, D) @ kh.t().contiguous() * SCALE
            last = first + torch.arange(a, e, device=q.device).repeat_interleave(group)
            x = x.masked_fill(at[None, :] > last[:, None], float("-inf"))
            m = x.amax(-1, keepdim=True)
            w = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
            total = w.sum(-1, keepdim=True)
            o = (w @ vh) / torch.where(total == 0, torch.ones_like(total), total)
            out[a:e, h * group:(h + 1) * group] = o.reshape(e - a, group, D)
    return out.to(torch.bfloat16)


def _plain(s):
    if s["op"] == "decode":
        outs = []
        for b, n in enumerate(s["lens"].tolist()):
            pages, slots = _places(s["table"], b, 0, n)
            k, v = _values(s["keys"], pages, slots), _values(s["values"], pages, slots)
            outs.append(_attend(s["q"][b].transpose(0, 1), k, v, n - 1).transpose(0, 1))
        return torch.stack(outs)
    if s["op"] == "prompt":
        outs, a, c = [], 0, 0
        for lq, lk in zip(s["q_lens"], s["k_lens"]):
            outs.append(_attend(s["q"][a:a + lq], s["k"][c:c + lk], s["v"][c:c + lk], lk - lq))
            a, c = a + lq, c + lk
        return torch.cat(outs)
    if s["op"] == "chunk":
        at = 0
        for b, (start, count) in enumerate(zip(s["starts"].tolist(), s["counts"])):
            pages, slots = _places(s["table"], b, start, start + count)
            for rows, buf in ((s["k"], s["keys"]), (s["v"], s["values"])):
                for t, x in zip(buf, _quantize(rows[at:at + count])):
                    t[pages, :, slots] = x
            at += count
        places = [_places(s["table"], b, 0, n) for b, n in enumerate(s["ends"])]
        pages, slots = (torch.cat(x) for x in zip(*places))
        return _values(s["keys"], pages, slots), _values(s["values"], pages, slots)
    src, dst = (torch.tensor(s[x], device="cuda") for x in ("src", "dst"))
    for t in (*s["keys"], *s["values"]):
        t[dst] = t[src]
    return *s["keys"], *s["values"]


def run(state):
    s = state
    if own:
        from lagunalab_amd import paged, prompt_attn
        if s["op"] == "decode":
            return paged.paged_decode_attention(s["q"], s["keys"], s["values"], s["table"], s["lens"],
                                                SCALE, shared=s["shared"])
        if s["op"] == "prompt":
            return prompt_attn.prompt_attention(s["q"], s["k"], s["v"], s["q_lens"], SCALE,
                                                k_lens=s["k_lens"])
        if s["op"] == "chunk":
            paged.paged_append(s["k"], s["v"], s["keys"], s["values"], s["table"], s["starts"],
                               s["counts"])
            return paged.paged_gather(s["keys"], s["values"], s["table"], s["zeros"], s["ends"])
        paged.copy_pages(s["keys"], s["values"], s["src"], s["dst"])
        return *s["keys"], *s["values"]
    return _plain(s)


# ------------------------------------------------------------------------------------------- work

def work(case):
    op, kv = case["op"], case["kv"]
    lens = _spread(case) if op != "copy" else []
    if op == "decode":
        rows = case["shared"] + sum(lens)
        seen = case["seqs"] * case["shared"] + sum(lens)
        return {"bytes": rows * kv * ROW_BYTES + 4 * case["seqs"] * case["heads"] * D,
                "flops": 4 * D * case["heads"] * seen}
    if op == "prompt":
        rows, past = sum(lens), case["past"]
        seen = sum(n * past + n * (n + 1) // 2 for n in lens)
        keys = rows + past * case["seqs"]
        return {"bytes": 4 * rows * case["heads"] * D + 4 * keys * kv * D,
                "flops": 4 * D * case["heads"] * seen}
    if op == "chunk":
        new, past = case["rows"] * case["seqs"], sum(lens)
        # new rows read and written, all rows read as codes and written as bf16 (the new ones' codes
        # are not read again)
        return {"bytes": kv * (new * (4 * D + ROW_BYTES) + past * ROW_BYTES + (new + past) * 4 * D),
                "flops": 0}
    return {"bytes": (case["sources"] + case["pages"]) * kv * PAGE * ROW_BYTES, "flops": 0}


# ---------------------------------------------------------------------------------- in 64 bits

def _exact_rows(buf):
    """A pool's values in 64 bits, [pages, Hkv, 64, 128], as bf16 holds them."""
    codes, scales, biases = (t.double() for t in buf)
    wide = [x.repeat_interleave(GROUP, dim=-1) for x in (scales, biases)]
    return torch.addcmul(wide[1], codes, wide[0]).to(torch.bfloat16).double()


def _exact_softmax(q, k, v, visible):
    """q [R, 128], k and v [n, 128], visible [R, n] or None, in 64 bits."""
    x = torch.mm(q, k.t()).mul_(SCALE)
    if visible is not None:
        x.masked_fill_(~visible, float("-inf"))
    return torch.mm(torch.softmax(x, dim=1), v).nan_to_num(0.0)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        kv, group = case["kv"], case["heads"] // case["kv"]
        for b, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            pages = s["table"][b, :-(-n // PAGE)].long()
            k, v = (_exact_rows([t[pages] for t in buf]) for buf in (s["keys"], s["values"]))
            for h in range(kv):
                rows = slice(h * group, (h + 1) * group)
                out[b, rows, 0] = _exact_softmax(s["q"][b, rows, 0].double(),
                                                 k[:, h].reshape(-1, D)[:n],
                                                 v[:, h].reshape(-1, D)[:n], None)
        return out
    if s["op"] == "prompt":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        out = torch.zeros_like(q)
        group = case["heads"] // case["kv"]
        a = c = 0
        for lq, lk in zip(s["q_lens"], s["k_lens"]):
            for h in range(case["heads"]):
                for i in range(0, lq, 4096):
                    j = min(lq, i + 4096)
                    visible = torch.ones((j - i, lk), dtype=torch.bool, device="cuda").tril(lk - lq + i)
                    out[a + i:a + j, h] = _exact_softmax(q[a + i:a + j, h], k[c:c + lk, h // group],
                                                         v[c:c + lk, h // group], visible)
            a, c = a + lq, c + lk
        return out
    if s["op"] == "chunk":
        outs = []
        for rows, buf in ((s["k"], s["keys"]), (s["v"], s["values"])):
            old, at = _exact_rows(buf), 0
            x = rows.double().reshape(*rows.shape[:-1], D // GROUP, GROUP)
            lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            below = lo.abs() > hi.abs()
            edge = torch.where(below, lo, hi)
            step = torch.clamp((hi - lo) / 255, min=1e-7) * torch.where(below, 1.0, -1.0)
            n = torch.floor((edge / step).abs() + 0.5) * torch.sign(edge / step)
            step = torch.where(n != 0, edge / n.masked_fill(n == 0, 1.0), step)
            edge = edge.masked_fill(n == 0, 0.0)
            code = torch.floor((x - edge) / step + 0.5).clamp_(0, 255)
            new = code * step.to(torch.bfloat16).double() + edge.to(torch.bfloat16).double()
            new, parts = new.reshape(rows.shape), []
            for b, (start, count) in enumerate(zip(s["starts"].tolist(), s["counts"])):
                pages = s["table"][b, :-(-start // PAGE)].long()
                parts.append(old[pages].transpose(1, 2).reshape(-1, old.shape[1], D)[:start])
                parts.append(new[at:at + count])
                at += count
            outs.append(torch.cat(parts))
        return tuple(outs)
    outs = [t.clone() for t in (*s["keys"], *s["values"])]
    for t, old in zip(outs, (*s["keys"], *s["values"])):
        for a, b in zip(s["src"], s["dst"]):
            t[b].copy_(old[a])
    return tuple(t if t.dtype == torch.uint8 else t.double() for t in outs)
