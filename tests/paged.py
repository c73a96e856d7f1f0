"""Plain statements, in 64 bits on the CPU, of the operators of a batch of sequences in HBM, written token by token
or pair by pair from their definitions, and inputs for their tests."""

import math

import torch

# half a rounding step of each type, relative to the value
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24,
             torch.float8_e4m3fn: 2.0 ** -4}
# half a step of the smallest numbers
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150,
            torch.float8_e4m3fn: 2.0 ** -10}


def turned(x, positions, freqs, layout, factor=1.0):
    """x (..., tokens, heads, D), positions (..., tokens); float64."""
    x, freqs = x.detach().cpu().double(), freqs.cpu()
    angle = positions.cpu().double()[..., None, None] * freqs
    out = x.clone()
    n = freqs.numel()
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        c, s = factor * angle[..., i].cos(), factor * angle[..., i].sin()
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def turned_bound(x, dtype, factor=1.0, rotary=None, layout="interleaved"):
    """How far a turned x may be from `turned`: cosine and sine in fp32 (angle, polynomial and factor: four half
    steps of one, times the pair's size), two products and a sum in fp32, one rounding to the type."""
    x = x.detach().cpu().double()
    n = (x.shape[-1] if rotary is None else rotary) // 2
    size = x.abs().clone()
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        pair = (x[..., a].square() + x[..., b].square()).sqrt() * factor
        size[..., a] = size[..., b] = pair
    # (a pair's |x cos| + |y sin| is at most its size; what the roundings ahead of the last come to is 8 * 2^-24 of it)
    return size * (HALF_STEP[dtype] * (1 + 1e-6) + 8 * 2.0 ** -24) + SMALLEST[dtype]


def attention(q, k_pages, v_pages, table, lengths, scale=None, k_scale=None, v_scale=None):
    """(out, lse, size, reach) in float64, sequence by sequence and head by head: size is sum_t w_t |v_t|, reach (B, Hq)
    the largest sum of |q_i k_i| scale over a sequence's tokens."""
    q, table, lengths = q.cpu().double(), table.cpu(), lengths.cpu()
    kp, vp = (x.cpu().float().double() for x in (k_pages, v_pages))
    B, Hq, D = q.shape
    pages, page, H, _ = kp.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, lse, size = torch.zeros(B, Hq, D).double(), torch.full((B, Hq), -math.inf).double(), torch.zeros(B, Hq, D).double()
    reach = torch.zeros(B, Hq).double()
    for b in range(B):
        n = max(0, min(int(lengths[b]), table.shape[1] * page))
        at = torch.arange(n)
        numbers = table[b].long()[at // page] if n else at
        fine = (numbers >= 0) & (numbers < pages)
        at, numbers = at[fine], numbers[fine]
        if not len(at):
            continue
        for j in range(Hq):
            h = j // (Hq // H)
            k, v = kp[numbers, at % page, h], vp[numbers, at % page, h]
            if k_scale is not None:
                k, v = k * k_scale[h].cpu().double(), v * v_scale[h].cpu().double()
            s = (k @ q[b, j]) * scale
            reach[b, j] = (k.abs() @ q[b, j].abs()).max() * abs(scale)
            lse[b, j] = torch.logsumexp(s, 0)
            w = torch.exp(s - lse[b, j])
            out[b, j], size[b, j] = w @ v, w @ v.abs()
    return out, lse, size, reach


def attention_bounds(out, size, reach, lengths, dtype):
    """(bound on the output, bound on lse), worst cases.  A score is a sum of D products in fp32, off by at most
    (D + 8) * 2^-24 of the sum of their sizes (the scale, the subtraction of the maximum and the exponential in the 8;
    another 8 * 2^-24 for the exponential's own relative error); a weight is off by that relatively.  Weights of 16-bit
    products are two numbers each, the second (at most 2^-7 or 1.5 * 2^-10 of a weight) rounded to nearest: off by at
    most 2^-15 of a weight for bf16, 1.5 * 2^-21 for fp16; sums over n tokens in fp32 are off by n * 2^-24 of the
    sum of sizes.  All of it counts for the sum and for the denominator; the output is rounded once."""
    D, n = out.shape[-1], lengths.cpu().clamp(min=0).double()[:, None]
    weight = (D + 8) * 2.0 ** -24 * reach + 8 * 2.0 ** -24
    rounded = {torch.bfloat16: 2.0 ** -15, torch.float16: 1.5 * 2.0 ** -21, torch.float32: 0.0}[dtype]
    relative = weight + rounded + (n + 8) * 2.0 ** -24
    # (fp16 weights below 2^-36 of the largest are 0)
    lost = n * 2.0 ** -36 if dtype == torch.float16 else 0.0
    bound = 2.02 * (relative + lost)[..., None] * size + HALF_STEP[dtype] * out.abs() * (1 + 1e-6) + SMALLEST[dtype]
    return bound, relative + 2.0 ** -22 + 2.0 ** -23 * reach


def pool(n_pages, page, heads, head_dim, dtype, device, g, layout="pages"):
    """Pages of N(0, 1) rows, as kv_pages lays them out or (pages, page, heads, D) contiguous ones."""
    if layout == "pages":
        x = torch.randn(n_pages, heads, page, 2, head_dim, generator=g).to(dtype).to(device)
        return x[:, :, :, 0].transpose(1, 2), x[:, :, :, 1].transpose(1, 2)
    return tuple(torch.randn(n_pages, page, heads, head_dim, generator=g).to(dtype).to(device) for _ in range(2))


def table_of(lengths, page, n_pages, g, width=None, dtype=torch.int32):
    """Page numbers in no order, each used once; -1 behind a sequence's last."""
    counts = [-(-n // page) for n in lengths]
    width = max(counts + [1]) if width is None else width
    order = torch.randperm(n_pages, generator=g)
    assert sum(counts) <= n_pages
    table, at = torch.full((len(lengths), width), -1, dtype=dtype), 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at: at + n]
        at += n
    return table


def outside(got, want, bound):
    """The entry that is furthest over its bound, as a message; '' if none is."""
    got, want = got.detach().cpu().float().double(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    over = torch.where(same, torch.zeros_like(want), (got - want).abs() - bound)
    over = torch.where(over.isnan(), torch.full_like(over, math.inf), over)
    if not over.numel() or over.max() <= 0:
        return ""
    at = divmod_index(int(over.argmax()), over.shape)
    return f"{int((over > 0).sum())} of {over.numel()} off; at {at}: {got[at]} instead of {want[at]}, bound {torch.as_tensor(bound).expand_as(want)[at]}"


def divmod_index(i, shape):
    at = []
    for n in reversed(shape):
        at.append(i % n)
        i //= n
    return tuple(reversed(at))
