"""Performance cases of the operators that take a model's step straight to and from a paged 8-bit cache.

A pool holds the K/V of one layer in pages of 64 positions: codes ``uint8 [pages, Hkv, 64, 128]``,
scales and biases ``bf16 [pages, Hkv, 64, 2]`` (8-bit affine codes, groups of 64), for keys and for
values. Row ``b`` of an int32 table lists the pages of sequence ``b`` in order. The operations (``op``):

* ``rotate``: projected rows of several sequences, each at its own positions: RMSNorm of every query and
  key head (or none), rotary embedding (half or interleaved pairs, some or all dims, default or YaRN
  frequencies), keys and values quantized into the pages. The stored rows come back as they read.
* ``attend``: attention of the last rows of each sequence -- one token, a verified block, a chunk --
  over its pages, causal, over everything or within a window.
* ``step``: both, as a layer of a model call runs them.

An attended value is what dequantizing the page gives: ``bf16(scale * code + bias)``. Head layouts are
query heads / KV heads of head_dim 128; 48/8 is Laguna's, 32/8 the benchmark's. 512 is Laguna's window.
"""
import math
import random

import torch

own = False

D = 128
PAGE = 64
GROUP = 64
SCALE = D ** -0.5
EPS = 1e-6
ROW_BYTES = 2 * (D + 2 * 2 * (D // GROUP))  # K and V codes, scales and biases of a row of one head
# rotary embeddings: YaRN frequencies for contexts of 32 times 4,096 positions, or plain ones
YARN_BASE, YARN_FACTOR, YARN_LENGTH, YARN_FAST, YARN_SLOW = 5e5, 32.0, 4096, 32.0, 1.0
BASE = 1e4


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token of one session early in a chat: latency
        {"name": "token step", "op": "step", "heads": 32, "kv": 8, "seqs": 1, "least": 1, "most": 1,
         "shortest": 1037, "longest": 1037, "window": 0, "dims": 64, "yarn": True, "pairs": "half",
         "norm": True},
        # a token of each of a serving batch in a sliding-window layer, Laguna's head layout
        {"name": "window step 64", "op": "step", "heads": 48, "kv": 8, "seqs": 64, "least": 1, "most": 1,
         "shortest": 42, "longest": 8191, "window": 512, "dims": 128, "yarn": False, "pairs": "half",
         "norm": True},
        # new user turns behind four sessions
        {"name": "turns step 4", "op": "step", "heads": 32, "kv": 8, "seqs": 4, "least": 37, "most": 211,
         "shortest": 299, "longest": 5003, "window": 0, "dims": 64, "yarn": True, "pairs": "half",
         "norm": True},
        # one ordinary prompt chunk behind a long session
        {"name": "rotate 2k", "op": "rotate", "heads": 48, "kv": 8, "seqs": 1, "least": 2048,
         "most": 2048, "shortest": 32771, "longest": 32771, "dims": 64, "yarn": True, "pairs": "half",
         "norm": True},
        # a batch of new requests of very different lengths, interleaved pairs, heads without a norm
        {"name": "rotate packed", "op": "rotate", "heads": 32, "kv": 8, "seqs": 7, "least": 1,
         "most": 4099, "shortest": 0, "longest": 0, "dims": 128, "yarn": False, "pairs": "interleaved",
         "norm": False},
        # a block of four drafts verified behind a long session
        {"name": "verify 5 on 64k", "op": "attend", "heads": 32, "kv": 8, "seqs": 1, "least": 5, "most": 5,
         "shortest": 65536, "longest": 65536, "window": 0},
        # seven drafts of each of sixteen sessions
        {"name": "verify 8 of 16", "op": "attend", "heads": 48, "kv": 8, "seqs": 16, "least": 8, "most": 8,
         "shortest": 97, "longest": 4099, "window": 0},
        # a new user turn behind an existing session
        {"name": "chunk 512 on 8k", "op": "attend", "heads": 48, "kv": 8, "seqs": 1, "least": 512,
         "most": 512, "shortest": 7681, "longest": 7681, "window": 0},
        # a prompt chunk behind a long session
        {"name": "chunk 2048 on 32k", "op": "attend", "heads": 32, "kv": 8, "seqs": 1, "least": 2048,
         "most": 2048, "shortest": 32771, "longest": 32771, "window": 0},
        # the same chunk in a sliding-window layer
        {"name": "window 2048 on 32k", "op": "attend", "heads": 48, "kv": 8, "seqs": 1, "least": 2048,
         "most": 2048, "shortest": 32771, "longest": 32771, "window": 512},
        # tokens, drafts and chunks of a serving batch in one call
        {"name": "mixed 24", "op": "attend", "heads": 48, "kv": 8, "seqs": 24, "least": 1, "most": 301,
         "shortest": 5, "longest": 6007, "window": 0},
        # a batch of first prompts
        {"name": "prompts 5", "op": "attend", "heads": 32, "kv": 8, "seqs": 5, "least": 1, "most": 2049,
         "shortest": 0, "longest": 0, "window": 0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotate", "attend", "attend", "attend", "step", "step"])
    hq, kv = rng.choice([(32, 8), (32, 8), (48, 8), (48, 8), (64, 8), (16, 8), (16, 2), (8, 8)])
    c = {"op": op, "heads": hq, "kv": kv, "seqs": _log(rng, 1, 64)}
    if op == "rotate":
        c["most"] = _log(rng, 1, max(1, 16384 // c["seqs"]))
        c["longest"] = rng.choice([0, _log(rng, 1, max(1, 131072 // c["seqs"]))])
    else:
        c["most"] = rng.choice([1, _log(rng, 2, 16), _log(rng, 16, max(16, 2048 // c["seqs"]))])
        # as many scores as the longest listed chunk has at most, a million positions in the pool
        rows = c["seqs"] * c["most"] * hq
        c["longest"] = _log(rng, 1, max(1, min(82671, 2 ** 31 // rows, 2 ** 20 // c["seqs"])))
        c["window"] = rng.choice([0, 0, 512, _log(rng, 1, 4096)])
    c["least"] = c["most"] if c["seqs"] == 1 else rng.randint(0, c["most"])
    c["shortest"] = c["longest"] if c["seqs"] == 1 else rng.randint(0, c["longest"])
    if op != "attend":
        c["dims"] = rng.choice([64, 128, 128, 32, 96])
        c["yarn"] = rng.random() < 0.5
        c["pairs"] = rng.choice(["half", "half", "interleaved"])
        c["norm"] = rng.random() < 0.7
    return c


def _spread(n, lo, hi, salt):
    """n lengths from lo to hi, in mixed order."""
    lens = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(7 * n + salt).shuffle(lens)
    return lens


def _counts(case):
    """New rows of each sequence, and rows before them."""
    n = case["seqs"]
    return _spread(n, case["least"], case["most"], 0), _spread(n, case["shortest"], case["longest"], 1)


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
            codes[p:q], scales[p:q], biases[p:q] = _quantize(_randn(gen, q - p, kv, PAGE, D).float())
        made.append((codes, scales, biases))
    return made


def _frequencies(case):
    """Rotary frequencies (radians per position) of the case's dims, and the factor on rotated dims."""
    dims = case["dims"]
    i = torch.arange(dims // 2, dtype=torch.float64)
    if not case["yarn"]:
        return (BASE ** (-2 * i / dims)).float().cuda(), 1.0
    freq = YARN_BASE ** (-2 * i / dims)
    # between the pairs that turn YARN_FAST and YARN_SLOW times over the original length, from kept to divided
    low, high = (dims * math.log(YARN_LENGTH / (2 * math.pi * turns)) / (2 * math.log(YARN_BASE))
                 for turns in (YARN_FAST, YARN_SLOW))
    low, high = max(math.floor(low), 0), min(math.ceil(high), dims - 1)
    divided = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return (freq * (1 - divided + divided / YARN_FACTOR)).float().cuda(), 0.1 * math.log(YARN_FACTOR) + 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hq, kv = case["heads"], case["kv"]
    counts, past = _counts(case)
    ends = [n + c for n, c in zip(past, counts)]
    need = [-(-n // PAGE) for n in ends]
    pages = sum(need) + sum(need) // 16 + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(ends), max(need + [1])), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"op": case["op"], "counts": counts, "table": table, "window": case.get("window") or None,
         "starts": torch.tensor(past, dtype=torch.int32, device="cuda"),
         "lens": torch.tensor(ends, dtype=torch.int32, device="cuda")}
    s["keys"], s["values"] = _pool(gen, pages, kv)
    rows = sum(counts)
    if case["op"] == "attend":
        s["q"] = _randn(gen, rows, hq, D)
        return s
    # the rows of a block's projection: query heads, key heads, value heads, a gate logit per query head
    proj = _randn(gen, rows, (hq + 2 * kv) * D + hq)
    q, k, v, _ = proj.split([hq * D, kv * D, kv * D, hq], dim=1)
    s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, D)) for x in (q, k, v))
    s["freq"], s["factor"] = _frequencies(case)
    s["interleaved"] = case["pairs"] == "interleaved"
    s["norms"] = (None, None)
    if case["norm"]:
        s["norms"] = tuple((1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(torch.bfloat16)
                           for _ in range(2))
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
    g = x.unflatten(-1, (-1, GROUP))
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


def _values(codes, scales, biases):
    """What codes, scales and biases stand for, bf16 [..., 128]."""
    g = codes.float().unflatten(-1, (-1, GROUP))
    return (g * scales.float().unsqueeze(-1) + biases.float().unsqueeze(-1)).flatten(-2).to(torch.bfloat16)


def _row_index(s):
    """Sequence, number within it and position of every row."""
    counts = torch.tensor(s["counts"], device="cuda")
    b = torch.repeat_interleave(torch.arange(len(s["counts"]), device="cuda"), counts)
    i = torch.arange(len(b), device="cuda") - (counts.cumsum(0) - counts)[b]
    return b, i, s["starts"].long()[b] + i


def _places(table, b, at):
    """Page and slot of positions."""
    return table[b, at // PAGE].long(), at % PAGE


def _norm_rotate(x, weight, s, pos):
    """RMSNorm and rotation of x [rows, heads, 128] in 32 bits, the angles in 64."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    dims = 2 * len(s["freq"])
    angle = pos.double()[:, None, None] * s["freq"].double()
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    r = x[..., :dims]
    a, c = (r[..., 0::2], r[..., 1::2]) if s["interleaved"] else r.chunk(2, dim=-1)
    a, c = a * cos - c * sin, a * sin + c * cos
    r = torch.stack([a, c], -1).flatten(-2) if s["interleaved"] else torch.cat([a, c], -1)
    return torch.cat([r, x[..., dims:]], -1)


def _plain_rotate(s):
    b, _, pos = _row_index(s)
    pages, slots = _places(s["table"], b, pos)
    q = _norm_rotate(s["q"], s["norms"][0], s, pos).to(torch.bfloat16)
    k = _quantize(_norm_rotate(s["k"], s["norms"][1], s, pos))
    v = _quantize(s["v"].float())
    s["keys"][0][pages, :, slots], s["keys"][1][pages, :, slots], s["keys"][2][pages, :, slots] = k
    s["values"][0][pages, :, slots], s["values"][1][pages, :, slots], s["values"][2][pages, :, slots] = v
    return q, _values(*k), _values(*v)


def _plain_attend(s, q):
    """Softmax attention of the packed rows q, all sequences at once, padded to the longest."""
    hq, kv, n = q.shape[1], s["keys"][0].shape[1], len(s["counts"])
    b, i, pos = _row_index(s)
    most = max(s["counts"])
    lens, counts = s["lens"].long(), torch.tensor(s["counts"], device="cuda")
    first = torch.zeros_like(lens) if s["window"] is None else (lens - counts - s["window"] + 1).clamp_min(0)
    at = first[:, None] + torch.arange(int((lens - first).max()), device="cuda")
    pages, slots = _places(s["table"], torch.arange(n, device="cuda")[:, None],
                           at.clamp_max(PAGE * s["table"].shape[1] - 1))
    k = _values(*(t[pages, :, slots] for t in s["keys"])).float().permute(0, 2, 3, 1).contiguous()
    v = _values(*(t[pages, :, slots] for t in s["values"])).float().transpose(1, 2).contiguous()
    x = torch.zeros((n, most, hq, D), device="cuda")
    x[b, i] = q.float()
    x = x.view(n, most, kv, hq // kv, D).transpose(1, 2).reshape(n, kv, most * (hq // kv), D)
    x = (x @ k).mul_(SCALE).view(n, kv, most, hq // kv, -1)
    row = (lens - counts)[:, None] + torch.arange(most, device="cuda")
    hidden = at[:, None, :] > row[:, :, None]
    if s["window"] is not None:
        hidden |= at[:, None, :] <= row[:, :, None] - s["window"]
    x.masked_fill_(hidden[:, None, :, None, :], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(n, kv, most * (hq // kv), -1) @ v).view(n, kv, most, hq // kv, D)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.transpose(1, 2).reshape(n, most, hq, D)[b, i].to(torch.bfloat16)


def run(state):
    s = state
    if own:
        from lagunalab_amd import paged
        from lagunalab_amd.rotary import Rotary
        if s["op"] == "attend":
            return paged.paged_chunk_attention(s["q"], s["keys"], s["values"], s["table"], s["lens"], SCALE,
                                               s["counts"], window=s["window"])
        rotary = Rotary(s["freq"], s["factor"], s["interleaved"])
        got = paged.paged_append_rotated(s["q"], s["k"], s["v"], s["keys"], s["values"], s["table"],
                                         s["starts"], rotary, s["counts"], *s["norms"], eps=EPS,
                                         fetch=s["op"] == "rotate")
        if s["op"] == "rotate":
            return got
        return got, paged.paged_chunk_attention(got, s["keys"], s["values"], s["table"], s["lens"], SCALE,
                                                s["counts"], window=s["window"])
    if s["op"] == "attend":
        return _plain_attend(s, s["q"])
    got = _plain_rotate(s)
    return got if s["op"] == "rotate" else (got[0], _plain_attend(s, got[0]))


# ------------------------------------------------------------------------------------------- work

def work(case):
    hq, kv = case["heads"], case["kv"]
    counts, past = _counts(case)
    window = case.get("window") or 1 << 30
    nbytes, flops, rows = 0, 0, sum(counts)
    if case["op"] != "attend":
        # projections read, rotated queries and stored rows written (and the rows as they read)
        nbytes += 2 * D * rows * (2 * hq + 2 * kv) + rows * kv * ROW_BYTES
        nbytes += 4 * D * rows * kv if case["op"] == "rotate" else 0
    if case["op"] != "rotate":
        new = 0 if case["op"] == "attend" else 1
        for n, c in zip(past, counts):
            if c:
                # the pages' rows (those of a step's own are not read again), queries in, outputs out
                nbytes += kv * ROW_BYTES * (min(n, window - 1) + (0 if new else c))
                nbytes += 2 * D * c * hq * (1 if new else 2)
                short = max(0, min(c, window - n))  # rows that see everything before them
                seen = short * n + short * (short + 1) // 2 + (c - short) * min(window, n + c)
                flops += 4 * D * hq * seen
    return {"bytes": max(nbytes, 1), "flops": flops}


# ---------------------------------------------------------------------------------- in 64 bits

def _exact_codes(x):
    """Rows [..., 128] in 64 bits through 8 bits and back."""
    x = x.reshape(*x.shape[:-1], D // GROUP, GROUP)
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    below = lo.abs() > hi.abs()
    edge = torch.where(below, lo, hi)
    step = torch.clamp((hi - lo) / 255, min=1e-7) * torch.where(below, 1.0, -1.0)
    n = torch.floor((edge / step).abs() + 0.5) * torch.sign(edge / step)
    step = torch.where(n != 0, edge / n.masked_fill(n == 0, 1.0), step)
    edge = edge.masked_fill(n == 0, 0.0)
    code = torch.floor((x - edge) / step + 0.5).clamp_(0, 255)
    x = code * step.to(torch.bfloat16).double() + edge.to(torch.bfloat16).double()
    return x.to(torch.bfloat16).double().flatten(-2)


def _exact_turn(x, weight, s, pos):
    """Rows x [rows, heads, 128] normed and turned, as complex numbers, in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x * weight.double() / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
    r = len(s["freq"])
    turn = torch.polar(torch.full_like(s["freq"].double(), s["factor"]).expand(len(pos), r),
                       torch.outer(pos.double(), s["freq"].double()))[:, None]
    first = slice(0, 2 * r, 2) if s["interleaved"] else slice(0, r)
    second = slice(1, 2 * r, 2) if s["interleaved"] else slice(r, 2 * r)
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_pages(buf, pages):
    """Pages' values in 64 bits, [positions, Hkv, 128], as bf16 holds them."""
    codes, scales, biases = (t[pages].double() for t in buf)
    wide = [x.repeat_interleave(GROUP, dim=-1) for x in (scales, biases)]
    rows = torch.addcmul(wide[1], codes, wide[0]).to(torch.bfloat16).double()
    return rows.transpose(1, 2).reshape(-1, rows.shape[1], D)


def exact(case, seed):
    s = prepare(case, seed)
    hq, kv = case["heads"], case["kv"]
    counts, past = _counts(case)
    q, k, v = s["q"].double(), None, None
    if case["op"] != "attend":
        pos = torch.cat([torch.arange(n, n + c, device="cuda") for n, c in zip(past, counts)])
        q = _exact_turn(s["q"], s["norms"][0], s, pos)
        k = _exact_codes(_exact_turn(s["k"], s["norms"][1], s, pos))
        v = _exact_codes(s["v"].double())
        if case["op"] == "rotate":
            return q, k, v
    asked = q if case["op"] == "attend" else q.to(torch.bfloat16).double()
    out, a = torch.zeros_like(q), 0
    for b, (n, c) in enumerate(zip(past, counts)):
        if c == 0:
            continue
        low = max(0, n - s["window"] + 1) if s["window"] else 0
        ids = s["table"][b, low // PAGE:-(-(n + c) // PAGE)].long()
        base = low // PAGE * PAGE
        rows = [_exact_pages(buf, ids)[:n + c - base] for buf in (s["keys"], s["values"])]
        if k is not None:
            rows[0][n - base:], rows[1][n - base:] = k[a:a + c], v[a:a + c]
        for i in range(0, c, 1024):  # rows n + i .. n + j - 1
            j = min(c, i + 1024)
            far = torch.arange(n + i, n + j, device="cuda")[:, None] - torch.arange(base, n + c, device="cuda")
            seen = (far >= 0) & (far < (s["window"] or 1 << 40))
            for h in range(hq):
                x = torch.mm(asked[a + i:a + j, h], rows[0][:, h // (hq // kv)].t()) * SCALE
                x = torch.softmax(x.masked_fill_(~seen, float("-inf")), dim=1)
                out[a + i:a + j, h] = torch.mm(x, rows[1][:, h // (hq // kv)])
        a += c
    return out if case["op"] == "attend" else (q, out)
