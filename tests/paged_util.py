"""Helpers of the paged-cache tests: pools filled with quantized rows, and attention in 64 bits with the
error that the kernels' roundings can cause."""
import torch

PAGE, D = 64, 128


def randn(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float32) * std).to(torch.bfloat16)


def fill_pool(gen, pages, kv, dev, poison=True):
    """A pool whose slots hold what no test may read: NaN scales and biases, random codes."""
    made = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pages, kv, PAGE, D), generator=gen, dtype=torch.uint8)
        words = [torch.full((pages, kv, PAGE, 2), float("nan") if poison else 0.0, dtype=torch.bfloat16)
                 for _ in range(2)]
        made.append(tuple(t.to(dev) for t in (codes, *words)))
    return made


def make_table(gen, lens, shared, spare=3, width_spare=0):
    """(table, pages): distinct pages in random order; the first ``shared`` positions' are common."""
    common = shared // PAGE
    need = [-(-n // PAGE) for n in lens]
    total = common + sum(max(0, n - common) for n in need) + spare
    order = torch.randperm(total, generator=gen)
    table = torch.zeros((len(lens), max(need + [common, 1]) + width_spare), dtype=torch.int32)
    at = common
    for b, n in enumerate(need):
        table[b, :min(n, common)] = order[:min(n, common)]
        if n > common:
            table[b, common:n] = order[at:at + n - common]
            at += n - common
    return table, total


def write_rows(pool, table_row, rows_k, rows_v, start=0):
    """Quantizes rows into a sequence's pages with the contiguous quantizer (on the GPU)."""
    from lagunalab_amd.quant import quantize
    for buf, rows in zip(pool, (rows_k, rows_v)):
        dev = buf[0].device
        at = torch.arange(start, start + rows.shape[0])
        pages = table_row[at // PAGE].long().to(dev)
        slots = (at % PAGE).to(dev)
        for t, x in zip(buf, quantize(rows.to(dev))):
            t[pages, :, slots] = x


def read_rows(buf, table_row, n):
    """The first n positions of a sequence in 64 bits [n, Hkv, 128], as bf16 holds them (on the CPU)."""
    at = torch.arange(n)
    pages, slots = table_row[at // PAGE].long(), at % PAGE
    c, s, b = (t.cpu()[pages, :, slots] for t in buf)
    s, b = (x.double().repeat_interleave(64, dim=-1) for x in (s, b))
    return (c.double() * s + b).to(torch.bfloat16).double()


def exact_attention(q, k, v, lim, scale):
    """Rows q [R, 128] over k, v [n, 128] (64 bits), row r seeing keys <= lim[r]: (out, bound).

    bound is how far a kernel may be off that rounds the weights to bf16 (2^-8 relative each, once in
    the weighted values and once in their sum), the output to bf16 (2^-8), and sums scores of 128
    products in fp32 (128 2^-24 of the sum of magnitudes each, through the exponential, in weights and
    sum; the hardware's exp2 and the sums over keys are within the factor)."""
    n = k.shape[0]
    out = torch.zeros_like(q)
    bound = torch.full_like(q, 1e-30)  # a row without keys is 0
    for r in range(q.shape[0]):
        m = min(n, int(lim[r]) + 1)
        if m <= 0:
            continue
        x = (k[:m] @ q[r]) * scale
        p = torch.softmax(x, 0)
        out[r] = p @ v[:m]
        size = p @ v[:m].abs()
        mag = float((k[:m].abs() @ q[r].abs()).max()) * abs(scale)
        slack = 2 * 2.0 ** -8 + 4 * (128 * 2.0 ** -24 * mag + 2.0 ** -18)
        bound[r] = size * slack + out[r].abs() * 2.0 ** -8 + 1e-30
    return out, bound


def assert_within(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = ((got - want).abs() / bound).max().item()
    assert off <= 1.0, f"{what}: {off:.3f} times the bound"
