"""The work by which the operators of a batch of sequences in HBM are judged: turning queries and keys by their
positions, storing a step's keys and values in pages, and attention of one new token of every sequence over its pages.
Each is computed in its plain form, or (``own``) by the framework's call.

Every case is a dict of plain values; ``kind`` says which operator:

  "rotate"  rotate(xq, xk, positions, freqs, layout=, factor=): a model's queries and keys, (B, S, heads, D); with
            ``train`` the gradients of both too
  "append"  append_kv_pages_(xk, xv, k_pages, v_pages, page_table, positions, ...): (tokens, kv heads, D) into pages,
            keys turned on the way and the queries beside them
  "attend"  paged_decode_attention(xq, k_pages, v_pages, page_table, lengths, ...): (B, heads, D)
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0
THETA = 500000.0


# ---- cases ---------------------------------------------------------------------------

def rotate(dtype, batch, tokens, heads, kv_heads, head_dim, rotary, layout, scaling, start, train):
    """``rotary``: channels of a head that turn; ``start``: position of the first token."""
    return dict(kind="rotate", dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, rotary=rotary, layout=layout, scaling=scaling, start=start, train=train)


def append(dtype, cache, seqs, tokens, longest, heads, kv_heads, head_dim, page, rotary, layout, scaling):
    """``tokens`` new ones of each sequence at the most (ragged from a quarter up, each sequence's behind what it has),
    in a cache of sequences of up to ``longest``; ``cache``: the pages' type, "e4m3" or the operands'."""
    return dict(kind="append", dtype=dtype, cache=cache, seqs=seqs, tokens=tokens, longest=longest, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, rotary=rotary, layout=layout, scaling=scaling)


def attend(dtype, cache, seqs, shortest, longest, heads, kv_heads, head_dim, page):
    """``seqs`` sequences of ``shortest`` to ``longest`` tokens, one of each length at least."""
    return dict(kind="attend", dtype=dtype, cache=cache, seqs=seqs, shortest=shortest, longest=longest, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page)


def listed():
    return [
        # One token of a chat far into its context: launch latency alone.
        dict(rotate("bf16", 1, 1, 32, 8, 128, 128, "interleaved", "llama3", 131072, False), name="rotate one token"),
        # A training step's queries and keys in the half layout, stretched to a longer context.
        dict(rotate("bf16", 4, 4096, 32, 8, 128, 128, "half", "yarn", 0, True), name="rotate train 4 x 4k"),
        # A part of each head, in fp32, an odd number of tokens: both ways too.
        dict(rotate("fp32", 3, 1777, 16, 4, 64, 32, "interleaved", "linear", 0, True), name="rotate fp32 partial"),
        # A decode step of a small batch: each sequence's new token.
        dict(append("bf16", "bf16", 8, 1, 32768, 32, 8, 128, 16, 128, "interleaved", "llama3"), name="append 8 tokens"),
        # A decode step of a large batch over a cache in 8 bits.
        dict(append("bf16", "e4m3", 256, 1, 4096, 28, 4, 128, 16, 128, "half", "yarn"), name="append 256 tokens e4m3"),
        # Prompts of several sequences at once.
        dict(append("bf16", "bf16", 6, 8192, 16384, 32, 8, 128, 16, 128, "interleaved", "llama3"),
             name="append prompts"),
        # Short prompts of small fp16 heads, part of each turned, in pages that are no power of two.
        dict(append("fp16", "fp16", 37, 211, 1000, 16, 16, 64, 24, 32, "half", "none"), name="append fp16 partial"),
        # One short sequence of the fp32 layer: latency of the launches.
        dict(attend("fp32", "fp32", 1, 777, 777, 8, 2, 64, 16), name="attend fp32 one short"),
        # Many short sequences, a kv head for every query head.
        dict(attend("fp16", "fp16", 192, 1, 1000, 16, 16, 64, 16), name="attend 192 short fp16"),
        # One long sequence: the work has to be split over its length.
        dict(attend("bf16", "bf16", 1, 131072, 131072, 32, 8, 128, 16), name="attend one 128k"),
        # A batch in 8 bits, seven query heads to a kv head.
        dict(attend("bf16", "e4m3", 48, 500, 32768, 28, 4, 128, 32), name="attend 48 e4m3 32k"),
        # The largest: a batch of long sequences of unlike lengths.
        dict(attend("bf16", "bf16", 16, 2000, 131072, 64, 8, 128, 16), name="attend 16 to 128k"),
    ]


def log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 2, 64), (16, 4, 64), (32, 8, 128), (24, 8, 128), (28, 4, 128), (64, 8, 128), (40, 10, 128), (16, 16, 64),
         (32, 4, 96), (8, 1, 256), (12, 12, 128)]


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "attend", "attend", "attend"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    cache = rng.choice([dtype, dtype, "e4m3"]) if dtype != "fp32" else dtype
    rotary = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
    layout, scaling = rng.choice(["interleaved", "half"]), rng.choice(["none", "linear", "ntk", "llama3", "yarn"])
    page = rng.choice([16, 16, 16, 32, 64, 24, 100])
    if kind == "rotate":
        tokens = log_uniform(rng, 1, 20000)
        batch = rng.randint(1, max(1, min(32, 20000 // tokens)))
        return rotate(dtype, batch, tokens, heads, kv_heads, head_dim, rotary, layout, scaling,
                      rng.choice([0, 1000, 100003, 1000003]), rng.random() < 0.4)
    if kind == "append":
        tokens = rng.choice([1, 1, log_uniform(rng, 2, 8192)])
        seqs = log_uniform(rng, 1, max(1, min(512, 50000 // tokens)))
        longest = max(tokens + 1, log_uniform(rng, 500, max(1000, min(32768, 262144 // seqs))))
        return append(dtype, cache, seqs, tokens, longest, heads, kv_heads, head_dim, page, rotary, layout, scaling)
    longest = log_uniform(rng, 200, 131072)
    # (keys and values of up to 2 GiB: the largest listed case has twice as much)
    room = (1 << 31) // (longest * kv_heads * 2 * head_dim * (1 if cache == "e4m3" else ESIZE[dtype]))
    seqs = log_uniform(rng, 1, max(1, min(512, room)))
    return attend(dtype, cache, seqs, 1 if rng.random() < 0.3 else max(1, longest // rng.choice([1, 4, 50])), longest,
                  heads, kv_heads, head_dim, page)


# ---- inputs --------------------------------------------------------------------------

def frequencies(rotary, scaling):
    """Radians per position of every pair of channels (float64, on the GPU) and the factor on cosine and sine."""
    i = np.arange(rotary // 2, dtype=np.float64)
    theta, factor, by = THETA, 1.0, 8.0
    if scaling == "ntk":
        theta *= by ** (rotary / (rotary - 2))
    f = theta ** (-2.0 * i / rotary)
    if scaling == "linear":
        f = f / by
    elif scaling == "llama3":       # wavelengths above 8192 slowed, below 2048 kept, blended between
        smooth = np.clip((8192.0 * f / (2 * np.pi) - 1.0) / 3.0, 0.0, 1.0)
        f = (1 - smooth) * f / by + smooth * f
    elif scaling == "yarn":         # pairs that turn over 32 times in 8192 positions kept, below once slowed
        turns = lambda n: rotary * math.log(8192.0 / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(0, math.floor(turns(32.0))), min(rotary - 1, math.ceil(turns(1.0)))
        slowed = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        f, factor = (1 - slowed) * f + slowed * f / by, 0.1 * math.log(by) + 1.0
    return torch.from_numpy(f).cuda(), factor


def normal(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def outlier_channels(g, kv_heads, head_dim, dtype):
    """Keys have channels that are larger than others, the same for all tokens."""
    return torch.exp(0.5 * normal(g, kv_heads, head_dim, dtype=torch.float32)).to(dtype)


def page_pool(case, g, lengths, filled):
    """Keys' and values' pages, (pages, page, kv heads, D) views of one tensor that holds a head's page in one piece,
    and the table of the sequences' page numbers, which are in no order; -1 where a sequence has no page."""
    page, H, D = case["page"], case["kv_heads"], case["head_dim"]
    counts = [-(-n // page) for n in lengths]
    pages, width = sum(counts) + 3, max(counts)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    starts = np.concatenate([[0], np.cumsum(counts)[:-1]])
    column = np.arange(width)
    where = torch.from_numpy(np.where(column < np.array(counts)[:, None], starts[:, None] + column, -1)).cuda()
    table = torch.where(where >= 0, order[where.clamp(min=0)], torch.full_like(where, -1, dtype=torch.int32))
    made = DTYPES[case["dtype"]]
    pool = torch.empty(pages, H, page, 2, D, dtype=torch.float8_e4m3fn if case["cache"] == "e4m3" else made,
                       device="cuda")
    scales = None
    if case["cache"] == "e4m3":     # what a head's largest values need
        scales = torch.exp(0.3 * normal(g, 2, H, dtype=torch.float32)) * 0.02
    if filled:
        outlier = outlier_channels(g, H, D, made)
        for i in range(0, pages, 4096):
            rows = normal(g, *pool[i: i + 4096].shape, dtype=made)
            rows[:, :, :, 0] *= outlier[:, None]
            pool[i: i + 4096] = rows if scales is None else (
                rows / scales.T[:, None, :, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(pool.dtype)
    else:
        pool.view(torch.uint8).zero_()
    views = [pool[:, :, :, i].transpose(1, 2) for i in range(2)]
    return views, table, (None, None) if scales is None else (scales[0].contiguous(), scales[1].contiguous())


def prepare(case, seed):
    g, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.RandomState(seed % (1 << 32))
    Hq, H, D, dtype = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] != "attend":
        s["freqs"], s["factor"] = frequencies(case["rotary"], case["scaling"])
    if case["kind"] == "rotate":
        B, S = case["batch"], case["tokens"]
        s["q"], s["k"] = normal(g, B, S, Hq, D, dtype=dtype), normal(g, B, S, H, D, dtype=dtype)
        s["positions"] = torch.arange(S, device="cuda", dtype=torch.int32) + case["start"]
        if case["train"]:
            s["dq"], s["dk"] = normal(g, B, S, Hq, D, dtype=dtype), normal(g, B, S, H, D, dtype=dtype)
        return s
    B, longest = case["seqs"], case["longest"]
    if case["kind"] == "append":
        shapes = np.random.RandomState(case["tokens"] * 1009 + longest)     # (lengths are the case's, values the seed's)
        new = shapes.randint(max(1, case["tokens"] // 4), case["tokens"] + 1, size=B)
        has = shapes.randint(0, longest - new + 1)
        sequences = np.repeat(np.arange(B), new)
        within = np.arange(new.sum()) - np.repeat(np.cumsum(new) - new, new)
        T = int(new.sum())
        (s["k_pages"], s["v_pages"]), s["table"], (s["k_scale"], s["v_scale"]) = page_pool(
            case, g, (has + new).tolist(), False)
        s["q"], s["k"], s["v"] = (normal(g, T, h, D, dtype=dtype) for h in (Hq, H, H))
        s["positions"] = torch.from_numpy((has[sequences] + within).astype(np.int32)).cuda()
        s["sequences"] = torch.from_numpy(sequences.astype(np.int32)).cuda()
        return s
    lengths = rng.randint(case["shortest"], longest + 1, size=B)
    lengths[rng.randint(B)] = longest
    (s["k_pages"], s["v_pages"]), s["table"], (s["k_scale"], s["v_scale"]) = page_pool(case, g, lengths.tolist(), True)
    s["lengths"] = torch.from_numpy(lengths.astype(np.int32)).cuda()
    s["q"] = normal(g, B, Hq, D, dtype=dtype)
    return s


# ---- the plain forms -----------------------------------------------------------------

def plain_turned(x, positions, freqs, layout, factor):
    """x (..., heads, D) with its first channels turned, in 32 bits; angles in 64."""
    angle = positions.double()[..., None] * freqs
    cos, sin = (angle.cos().float() * factor)[..., None, :], (angle.sin().float() * factor)[..., None, :]
    r = 2 * freqs.numel()
    x = x.float()
    if layout == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def plain_append(s):
    case, page = s["case"], s["case"]["page"]
    k = plain_turned(s["k"], s["positions"], s["freqs"], case["layout"], s["factor"])
    q = plain_turned(s["q"], s["positions"], s["freqs"], case["layout"], s["factor"]).to(s["q"].dtype)
    positions = s["positions"].long()
    at = (s["table"][s["sequences"].long(), positions // page].long(), positions % page)

    def store(pages, rows, scale):
        if scale is not None:
            rows = (rows / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(pages.dtype)
            pages.view(torch.uint8)[at] = rows.view(torch.uint8)
        else:
            pages[at] = rows.to(pages.dtype)

    store(s["k_pages"], k, s["k_scale"])
    store(s["v_pages"], s["v"].float(), s["v_scale"])
    return q


def plain_attention(s):
    q, table, lengths = s["q"], s["table"].long().clamp(min=0), s["lengths"].long()
    B, Hq, D = q.shape
    H = s["k_pages"].shape[2]

    def rows(pages, scale):     # (B * kv heads, tokens, D)
        if scale is not None:
            x = pages.view(torch.uint8)[table].view(pages.dtype).float()
        else:
            x = pages[table].float()
        x = x.flatten(1, 2).transpose(1, 2).reshape(B * H, -1, D)
        return x if scale is None else x * scale.repeat(B)[:, None, None]

    k = rows(s["k_pages"], s["k_scale"])
    scores = torch.bmm(q.float().reshape(B * H, Hq // H, D), k.transpose(1, 2)) * D ** -0.5
    del k
    dead = torch.arange(scores.shape[-1], device=q.device) >= lengths.repeat_interleave(H)[:, None, None]
    scores = scores.masked_fill_(dead, -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp_()
    total = weights.sum(-1, keepdim=True)
    return (torch.bmm(weights, rows(s["v_pages"], s["v_scale"])) / total).reshape(B, Hq, D).to(q.dtype)


# ---- one pass ------------------------------------------------------------------------

def run(s):
    if own:
        from dram_attention_amd import append_kv_pages_, paged_decode_attention
        from dram_attention_amd import rotate as rotate_both
    case = s["case"]
    if case["kind"] == "rotate":
        q, k = s["q"], s["k"]
        if case["train"]:
            q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        if own:
            yq, yk = rotate_both(q, k, s["positions"], s["freqs"], layout=case["layout"], factor=s["factor"])
        else:
            yq, yk = (plain_turned(x, s["positions"], s["freqs"], case["layout"], s["factor"]).to(x.dtype)
                      for x in (q, k))
        if not case["train"]:
            return {"q": yq, "k": yk}
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (s["dq"], s["dk"]))
        return {"q": yq.detach(), "k": yk.detach(), "dq": dq, "dk": dk}
    if case["kind"] == "append":
        if own:
            q = append_kv_pages_(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["positions"],
                                 sequences=s["sequences"], xq=s["q"], freqs=s["freqs"], layout=case["layout"],
                                 factor=s["factor"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        else:
            q = plain_append(s)
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if own:
        out = paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"])
    else:
        out = plain_attention(s)
    return {"out": out}


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    e, Hq, H, D = ESIZE[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
    c = 1 if case.get("cache") == "e4m3" else e
    if case["kind"] == "rotate":
        n = case["batch"] * case["tokens"] * (Hq + H) * (2 if case["train"] else 1)
        return {"bytes": 2 * n * D * e, "flops": 3 * n * case["rotary"]}
    B = case["seqs"]
    if case["kind"] == "append":
        n = B * (max(1, case["tokens"] // 4) + case["tokens"]) // 2
        return {"bytes": n * D * (2 * Hq * e + 2 * H * (e + c)), "flops": 3 * n * (Hq + H) * case["rotary"]}
    n = case["longest"] + (B - 1) * (case["shortest"] + case["longest"]) // 2
    return {"bytes": n * H * 2 * D * c + 2 * B * Hq * D * e, "flops": 4 * n * Hq * D}


# ---- in 64 bits, from the definitions ------------------------------------------------

def exact_turned(x, positions, freqs, layout, factor):
    """Pairs of channels as complex numbers, times factor * e^(i position frequency)."""
    x, half = x.double().clone(), freqs.numel()
    turn = torch.polar(torch.full_like(freqs, factor).expand(*positions.shape, half),
                       positions.double().unsqueeze(-1) * freqs.double()).unsqueeze(-2)
    first, second = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (
        slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact_attention(s, b):
    """The sequence's tokens, one after the other out of its pages; (heads, D)."""
    n, page = int(s["lengths"][b]), s["case"]["page"]
    at = torch.arange(n, device="cuda")
    pages, q = s["table"][b].long()[at // page], s["q"][b].double()
    out = []
    for h in range(s["k_pages"].shape[2]):
        k, v = (x[:, :, h].view(torch.uint8)[pages, at % page].view(x.dtype).double() if s["k_scale"] is not None
                else x[pages, at % page, h].double() for x in (s["k_pages"], s["v_pages"]))
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
        rep = q.shape[0] // s["k_pages"].shape[2]
        p = torch.softmax(q[h * rep: (h + 1) * rep] @ k.T / math.sqrt(q.shape[1]), dim=-1)
        out.append(p @ v)
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        if case["seqs"] * case["kv_heads"] > 4096:
            return None
        return {"out": torch.stack([exact_attention(s, b) for b in range(case["seqs"])])}
    turned = {x: exact_turned(s[x], s["positions"], s["freqs"], case["layout"], s["factor"]) for x in ("q", "k")}
    if case["kind"] == "rotate":
        if case["train"]:       # the inverse turn: the same matrix transposed
            turned.update({d: exact_turned(s[d], -s["positions"], s["freqs"], case["layout"], s["factor"])
                           for d in ("dq", "dk")})
        return turned
    pools = []
    for pages, rows, scale in ((s["k_pages"], turned["k"], s["k_scale"]), (s["v_pages"], s["v"].double(), s["v_scale"])):
        pool = torch.zeros(pages.shape, dtype=torch.float64, device="cuda")
        if scale is not None:
            rows = (rows / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        where = s["table"][s["sequences"].long(), s["positions"].long() // case["page"]].long()
        pool[where, s["positions"].long() % case["page"]] = rows
        pools.append(pool)
    return {"q": turned["q"], "k_pages": pools[0], "v_pages": pools[1]}
