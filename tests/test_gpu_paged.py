"""Keys and values of a batch of sequences in pages, and attention over them, on the GPU against their definitions in
64 bits (tests/paged.py)."""

import math

import pytest
import torch

from dram_attention_amd import append_kv_pages_, kv_pages, paged_decode_attention, rotary_frequencies, rotate

from . import paged as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def bits(x):
    return x.contiguous().view(torch.uint8)


# ---- append --------------------------------------------------------------------------

def expected_append(k_pages, v_pages, table, sequences, positions, k, v, fk, fv):
    """Pools in float64 and their bounds (0 where nothing is stored), token by token."""
    want = [x.cpu().float().double() for x in (k_pages, v_pages)]
    far = [torch.zeros_like(x) for x in want]
    page, pages = k_pages.shape[1], k_pages.shape[0]
    for t, (s, p) in enumerate(zip(sequences.tolist(), positions.tolist())):
        if not (0 <= s < table.shape[0] and 0 <= p < table.shape[1] * page):
            continue
        number = int(table[s, p // page])
        if not 0 <= number < pages:
            continue
        for i, (rows, bound) in enumerate(((k, fk), (v, fv))):
            want[i][number, p % page] = rows[t]
            far[i][number, p % page] = bound[t]
    return want, far


CASES = [   # dtype, cache, kv heads, heads, head_dim, page, rotary, layout, pool
    (torch.bfloat16, None, 8, 32, 128, 16, 128, "interleaved", "pages"),
    (torch.bfloat16, E4M3, 4, 28, 128, 16, 128, "half", "pages"),
    (torch.bfloat16, E4M3, 2, 6, 96, 7, 32, "interleaved", "pages"),
    (torch.float16, E4M3, 1, 1, 66, 5, 22, "half", "rows"),
    (torch.float16, None, 3, 9, 64, 1, 20, "interleaved", "rows"),
    (torch.float16, None, 16, 16, 64, 24, 32, "half", "pages"),
    (torch.float32, None, 2, 8, 64, 16, 64, "interleaved", "pages"),
    (torch.float32, None, 2, 2, 5, 3, 4, "half", "rows"),
    (torch.bfloat16, None, 5, 0, 256, 100, 64, "half", "pages"),
    # (rows taken 4 and 2 elements a load)
    (torch.float16, E4M3, 3, 3, 96, 16, 24, "half", "pages"),
    (torch.bfloat16, E4M3, 2, 4, 80, 16, 20, "half", "rows"),
    (torch.bfloat16, None, 2, 4, 80, 16, 20, "interleaved", "pages"),
    (torch.float32, None, 2, 4, 80, 16, 20, "half", "pages"),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append_against_the_definition(case, wide):
    dtype, cache, H, Hq, D, page, rotary, layout, pool = case
    g = gen(H * D + page)
    kp, vp = P.pool(40, page, H, D, cache or dtype, DEV, g, pool)
    whole = torch.int64 if wide else torch.int32
    new = [1, 3, page, 2 * page + 1, 1]
    has = [0, page - 1, 1, 2, 5 * page]
    table = P.table_of([h + n for h, n in zip(has, new)], page, 40, g, dtype=whole)
    sequences = torch.tensor([s for s, n in enumerate(new) for _ in range(n)])
    positions = torch.cat([torch.arange(n) + h for h, n in zip(has, new)])
    # padding, positions and sequences beyond the table, pages beyond the pool: nothing is stored
    table[4, 5] = 40
    table[0, 0] = -1
    more_s, more_p = torch.tensor([1, 1, -1, 5, 2]), torch.tensor([-1, table.shape[1] * page, 0, 0, -(2 ** 31)])
    sequences, positions = torch.cat([more_s, sequences]), torch.cat([more_p, positions])
    order = torch.randperm(len(positions), generator=g)
    sequences, positions = sequences[order], positions[order]
    T = len(positions)
    q = randn(g, T, Hq, D, dtype=dtype) if Hq else None
    k, v = randn(g, T, H, D, dtype=dtype), randn(g, T, H, D, dtype=dtype)
    freqs, factor = rotary_frequencies(rotary, scaling={"type": "yarn", "factor": 4.0, "original_length": 32}, device=DEV)
    scales = {}
    if cache:
        scales = {"k_scale": torch.rand(H, generator=g).add(0.01).mul(0.3).to(DEV),
                  "v_scale": torch.rand(H, generator=g).add(0.001).mul(0.02).to(DEV)}     # (some values are clamped)
    k64, v64 = P.turned(k, positions, freqs, layout, factor), v.cpu().double()
    fk = P.turned_bound(k, dtype, factor, rotary, layout)
    fv = torch.zeros_like(v64)
    if cache:
        # in fp32: what the turn is off by and the division's half step; then one rounding to 8 bits
        ks, vs = (scales[n].cpu().double()[:, None] for n in ("k_scale", "v_scale"))
        exact = (fk - P.SMALLEST[dtype]) / P.HALF_STEP[dtype] * 12 * 2.0 ** -24 / ks
        k64, v64 = (k64 / ks).clamp(-448, 448), (v64 / vs).clamp(-448, 448)
        fk = P.HALF_STEP[E4M3] * (k64.abs() + exact) + exact + P.SMALLEST[E4M3]
        fv = P.HALF_STEP[E4M3] * v64.abs() * (1 + 2.0 ** -20) + P.SMALLEST[E4M3]
    want, far = expected_append(kp, vp, table, sequences, positions, k64, v64, fk, fv)
    before = [bits(kp.clone()), bits(vp.clone())]
    got = append_kv_pages_(k, v, kp, vp, table.to(DEV), positions.to(whole).to(DEV), sequences=sequences.to(whole).to(DEV),
                           xq=q, freqs=freqs, layout=layout, factor=factor, **scales)
    for pages, x, y, old in zip((kp, vp), want, far, before):
        wrong = P.outside(pages, x, y)
        assert not wrong, wrong
        kept = (y == 0).all(-1)
        e = old.shape[-1] // x.shape[-1]
        assert torch.equal(bits(pages).cpu()[kept[..., None].expand(*kept.shape, e * D)],
                           old.cpu()[kept[..., None].expand(*kept.shape, e * D)]) or not cache and bool((y == 0).all())
    if Hq:
        plain, _ = rotate(q, None, positions.to(DEV), freqs, layout=layout, factor=factor)
        assert torch.equal(got, plain)
    else:
        assert got is None


def test_append_without_sequences_frequencies_or_tokens():
    g = gen(1)
    kp, vp = P.pool(8, 16, 2, 64, torch.bfloat16, DEV, g)
    table = P.table_of([16, 32, 1], 16, 8, g).to(DEV)
    k, v, q = (randn(g, 3, h, 64, dtype=torch.bfloat16) for h in (2, 2, 4))
    positions = torch.tensor([3, 17, 0], device=DEV)
    assert torch.equal(append_kv_pages_(k, v, kp, vp, table, positions, xq=q), q)
    for t, p in enumerate(positions.tolist()):
        at = int(table[t, p // 16])
        assert torch.equal(kp[at, p % 16], k[t]) and torch.equal(vp[at, p % 16], v[t])
    none = k[:0]
    assert append_kv_pages_(none, none, kp, vp, table, positions[:0], sequences=positions[:0]) is None
    empty = kp[:0]
    before = kp.clone()
    append_kv_pages_(k, v, empty, vp[:0], table, positions)         # a pool without pages stores nothing
    append_kv_pages_(k, v, kp, vp, table[:, :0], positions)         # nor does a table without columns
    assert torch.equal(kp, before)


def test_append_of_views_and_nan():
    """A fused projection's parts, as they lie; NaN stays NaN in 8 bits, infinities are clamped."""
    g = gen(2)
    fused = randn(g, 5, 8 + 2 + 2, 128, dtype=torch.bfloat16)
    fused[0, 11, 3], fused[0, 11, 4], fused[0, 11, 5] = float("nan"), float("inf"), -float("inf")
    freqs, _ = rotary_frequencies(128, device=DEV)
    table = torch.arange(5, dtype=torch.int32, device=DEV)[:, None]
    positions = torch.tensor([0, 4, 8, 15, 1], dtype=torch.int32, device=DEV)
    pools = [kv_pages(5, 16, 2, 128, dtype=t, device=DEV) for t in (torch.bfloat16, E4M3)]
    for kp, vp in pools:
        q = append_kv_pages_(fused[:, 8:10], fused[:, 10:], kp, vp, table, positions, xq=fused[:, :8], freqs=freqs)
        wq, wk = rotate(fused[:, :8].contiguous(), fused[:, 8:10].contiguous(), positions, freqs)
        assert torch.equal(q, wq)
        at = positions.long()
        if kp.dtype == torch.bfloat16:
            assert torch.equal(kp[torch.arange(5), at], wk)
    v = pools[1][1][0, 0, 1].float()
    assert v[3].isnan() and v[4] == 448 and v[5] == -448 and not v[6:].isnan().any()
    misaligned = torch.empty(5 * 2 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(5, 2, 128).copy_(fused[:, 8:10])
    kp, vp = kv_pages(5, 16, 2, 128, device=DEV)
    append_kv_pages_(misaligned, misaligned, kp, vp, table, positions, freqs=freqs)
    assert torch.equal(kp[torch.arange(5), at], wk)


# ---- attention -----------------------------------------------------------------------

def attention_case(g, lengths, Hq, H, D, dtype, cache=None, page=16, layout="pages", spare=3, whole=torch.int32, width=None):
    n_pages = sum(-(-n // page) for n in lengths) + spare
    kp, vp = P.pool(n_pages, page, H, D, cache or dtype, DEV, g, layout)
    table = P.table_of(lengths, page, n_pages, g, width, whole).to(DEV)
    q = randn(g, len(lengths), Hq, D, dtype=dtype)
    scales = {}
    if cache:
        scales = {"k_scale": torch.rand(H, generator=g).add(0.5).to(DEV), "v_scale": torch.rand(H, generator=g).add(0.5).to(DEV)}
    return (q, kp, vp, table, torch.tensor(lengths, dtype=whole, device=DEV)), scales


def check_attention(args, scales, scale=None, **more):
    q, lengths = args[0], args[4]
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = paged_decode_attention(*args, scale=scale, lse=lse, **scales, **more)
    out, want_lse, size, reach = P.attention(*args, scale, scales.get("k_scale"), scales.get("v_scale"))
    bound, lse_bound = P.attention_bounds(out, size, reach, lengths, q.dtype)
    far = P.outside(got, out, bound)
    assert not far, far
    far = P.outside(lse, want_lse, lse_bound + 2.0 ** -23 * want_lse.abs().nan_to_num(posinf=0.0))
    assert not far, "lse: " + far
    return got


BORDERS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 0, 255, 256, 257, 300, 511, 512, 513, 700, 0]
TYPES = [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None), (torch.bfloat16, E4M3), (torch.float16, E4M3)]


@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 8, 128), (7, 1, 96), (6, 3, 256)], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_attention_at_the_borders_of_tiles_and_units(types, heads):
    dtype, cache = types
    Hq, H, D = heads
    args, scales = attention_case(gen(D), BORDERS, Hq, H, D, dtype, cache, page=16)
    check_attention(args, scales)


@pytest.mark.parametrize("page", [1, 3, 7, 16, 24, 64, 100, 1000])
@pytest.mark.parametrize("layout", ["pages", "rows"])
def test_attention_over_pages_of_any_size(page, layout):
    args, scales = attention_case(gen(page), [1, 5, 999, 0, 130, 33], 8, 4, 64, torch.bfloat16, page=page, layout=layout,
                                  whole=torch.int64 if page % 2 else torch.int32)
    check_attention(args, scales)


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (15, 1), (16, 1), (17, 1), (40, 2), (71, 1), (64, 8)], ids=str)
@pytest.mark.parametrize("types", TYPES[:4], ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_attention_of_groups_of_any_size(types, heads):
    dtype, cache = types
    args, scales = attention_case(gen(heads[0]), [40, 600, 3], heads[0], heads[1], 64, dtype, cache)
    check_attention(args, scales)


@pytest.mark.parametrize("heads", [(17, 1, 128), (64, 2, 96), (100, 2, 128), (33, 1, 256)], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_attention_of_large_groups_at_every_head_size(types, heads):
    dtype, cache = types
    Hq, H, D = heads
    args, scales = attention_case(gen(Hq), [0, 31, 1100, 129, 400], Hq, H, D, dtype, cache)
    check_attention(args, scales)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
@pytest.mark.parametrize("lengths", [[20000], [3001, 1], [1, 9000, 2, 0, 5000], [0, 0, 12345, 0]], ids=str)
def test_attention_split_over_long_sequences(types, lengths):
    dtype, cache = types
    args, scales = attention_case(gen(len(lengths)), lengths, 6, 2, 128, dtype, cache)
    check_attention(args, scales)


def test_attention_of_many_ragged_sequences():
    """More sequences than shares and than a workgroup has threads: several in a share, some across a border."""
    g = gen(11)
    lengths = torch.randint(0, 300, (700,), generator=g).tolist()
    for i in (0, 5, 255, 256, 400, 699):
        lengths[i] = 0
    lengths[333] = 2500
    args, scales = attention_case(g, lengths, 2, 1, 64, torch.bfloat16, page=8)
    check_attention(args, scales)


@pytest.mark.parametrize("dtype, heads, n", [(torch.float16, (1, 1, 64), 131072), (torch.bfloat16, (3, 1, 128), 131072),
                                             (torch.bfloat16, (1, 1, 64), 200001)])
def test_attention_of_one_sequence_in_as_many_shares_as_there_are(dtype, heads, n):
    args, _ = attention_case(gen(26), [n], *heads, dtype, page=64)
    check_attention(args, {})


@pytest.mark.parametrize("width", [1, 64])
def test_attention_of_more_sequences_than_16_bits_count(width):
    """70000 sequences of 0 to 3 tokens, a workgroup each or in shares."""
    g = gen(27)
    B, n_pages = 70000, 500
    kp, vp = P.pool(n_pages, 16, 1, 64, torch.float32, DEV, g)
    table = torch.zeros(B, width, dtype=torch.int32)
    table[:, 0] = torch.randint(0, n_pages, (B,), generator=g)
    table, lengths = table.to(DEV), torch.randint(0, 4, (B,), generator=g).to(DEV)
    q = randn(g, B, 1, 64, dtype=torch.float32)
    got = paged_decode_attention(q, kp, vp, table, lengths)
    k, v = (x[table[:, 0].long(), :3, 0].double() for x in (kp, vp))
    scores = torch.einsum("bd,btd->bt", q[:, 0].double(), k) / 8
    weights = torch.where(torch.arange(3, device=DEV) < lengths[:, None], (scores - scores.amax(1, keepdim=True)).exp(), 0.0)
    want = torch.einsum("bt,btd->bd", weights / weights.sum(1, keepdim=True).clamp(min=1e-300), v)
    size = v.abs().amax(1)
    # (scores of up to 64 * 5 * 5 / 8 in fp32: off by (64 + 8) * 2^-24 of their products' sizes)
    reach = torch.einsum("bd,btd->bt", q[:, 0].double().abs(), k.abs()).amax(1, keepdim=True) / 8
    far = P.outside(got[:, 0], want.cpu(), (2.02 * (72 * 2.0 ** -24 * reach + 20 * 2.0 ** -24) * size).cpu() + 2.0 ** -24 * want.abs().cpu())
    assert not far, far


def test_operands_that_do_not_lie_in_a_row():
    """Lengths, positions and sequences with gaps; one layer of a pool of several; page tables wider than they are used."""
    g = gen(28)
    args, _ = attention_case(g, [100, 1000, 7], 4, 2, 64, torch.bfloat16)
    q, kp, vp, table, lengths = args
    want = paged_decode_attention(*args)
    spread = torch.zeros(6, dtype=torch.int64, device=DEV)
    spread[::2] = lengths
    layers = torch.full((3, *kp.shape), float("nan"), dtype=kp.dtype, device=DEV), torch.full((3, *kp.shape), float("nan"), dtype=kp.dtype, device=DEV)
    layers[0][1], layers[1][1] = kp, vp
    wide = torch.full((3, 2 * table.shape[1]), -1, dtype=torch.int64, device=DEV)
    wide[:, : table.shape[1]] = table
    assert torch.equal(paged_decode_attention(q, layers[0][1], layers[1][1], wide[:, : table.shape[1]], spread[::2]), want)
    k, v = (randn(g, 3, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    at = torch.tensor([3, 0, 40, 0, 5, 0], device=DEV)[::2]
    of = torch.tensor([2, 9, 0, 9, 1, 9], dtype=torch.int32, device=DEV)[::2]
    append_kv_pages_(k, v, layers[0][1], layers[1][1], wide, at, sequences=of)
    for t, (b, p) in enumerate(zip(of.tolist(), at.tolist())):
        number = int(table[b, p // 16])
        assert torch.equal(layers[0][1][number, p % 16], k[t]) and torch.equal(layers[1][1][number, p % 16], v[t])
    assert layers[0][0].isnan().all() and layers[1][2].isnan().all()


def test_eight_bit_pages_with_one_scale_or_none():
    args, scales = attention_case(gen(29), [50, 700], 4, 2, 64, torch.bfloat16, E4M3)
    q, kp, vp, table, lengths = args
    ones = torch.ones(2, device=DEV)
    for k_scale, v_scale in ((None, None), (scales["k_scale"], None), (None, scales["v_scale"])):
        want = paged_decode_attention(*args, k_scale=ones if k_scale is None else k_scale,
                                      v_scale=ones if v_scale is None else v_scale)
        assert torch.equal(paged_decode_attention(*args, k_scale=k_scale, v_scale=v_scale), want)
    k, v = (randn(gen(30), 2, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    append_kv_pages_(k, v, kp, vp, table, lengths - 1, v_scale=scales["v_scale"])
    at = table[torch.arange(2), (lengths.cpu() - 1).long() // 16].long(), (lengths.long() - 1) % 16
    assert torch.equal(bits(kp[at]), bits(k.to(E4M3)))
    assert torch.equal(bits(vp[at]), bits((v.float() / scales["v_scale"][:, None]).to(E4M3)))


def test_attention_of_empty_batches_tables_and_pools():
    args, _ = attention_case(gen(12), [5, 700], 4, 2, 64, torch.bfloat16)
    q, kp, vp, table, lengths = args
    assert paged_decode_attention(q[:0], kp, vp, table[:0], lengths[:0]).shape == (0, 4, 64)
    for a in ((q, kp, vp, table[:, :0], lengths), (q, kp[:0], vp[:0], table, lengths), (q, kp, vp, table, lengths * 0),
              (q, kp, vp, table, lengths * 0 - 5), (q, kp, vp, table * 0 - 1, lengths), (q, kp, vp, table * 0 + kp.shape[0], lengths)):
        lse = torch.zeros(2, 4, device=DEV)
        out = torch.full_like(q, float("nan"))
        assert paged_decode_attention(*a, out=out, lse=lse) is out
        assert not out.any() and (lse == -math.inf).all()


def test_lengths_beyond_the_table_are_clamped():
    args, _ = attention_case(gen(13), [64, 640], 4, 2, 64, torch.bfloat16)
    q, kp, vp, table, lengths = args
    long = torch.tensor([2 ** 40, 2 ** 31 + 5], device=DEV)
    table[0] = table[1].flip(0)
    want = paged_decode_attention(q, kp, vp, table, torch.tensor([640, 640], device=DEV))
    assert torch.equal(paged_decode_attention(q, kp, vp, table, long), want)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_what_does_not_count_is_not_seen(types):
    """NaN and infinities in spare pages, behind sequences' ends and in page 0, where addresses of tokens that do not
    count point; page numbers out of the pool in the middle of a sequence."""
    dtype, cache = types
    g = gen(14)
    lengths = [33, 100, 1300, 1]
    args, scales = attention_case(g, lengths, 6, 2, 64, dtype, cache, page=16, spare=5)
    q, kp, vp, table, lens = args
    used = torch.zeros(kp.shape[0], 16, dtype=torch.bool)
    table[2, 3], table[2, 40], table[1, 1] = -7, kp.shape[0], 2 ** 31 - 1
    cpu = table.cpu()
    for b, n in enumerate(lengths):
        for t in range(n):
            if 0 <= cpu[b, t // 16] < kp.shape[0]:
                used[cpu[b, t // 16], t % 16] = True
    want = check_attention(args, scales)
    bad = torch.tensor(float("nan")).to(kp.dtype).to(DEV)
    for pages in (kp, vp):
        pages.view(torch.uint8 if cache else dtype)[~used.to(DEV)] = bad.view(torch.uint8) if cache else bad
    assert torch.equal(paged_decode_attention(*args, **scales), want)


def test_infinite_and_missing_values_stay_with_their_sequence_and_head():
    args, _ = attention_case(gen(15), [200, 200, 700, 700], 4, 2, 64, torch.bfloat16)
    q, kp, vp, table, lengths = args
    clean = paged_decode_attention(*args)
    vp[int(table[0, 3]), 5, 1, 7] = float("inf")
    kp[int(table[3, 40]), 2, 0, 9] = float("nan")
    got = paged_decode_attention(*args)
    assert (got[0, 2:, 7] == float("inf")).all() and got[3, :2].isnan().all()
    got[0, 2:, 7], got[3, :2] = clean[0, 2:, 7], clean[3, :2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scores_of_any_size(dtype):
    """Weights that underflow, one token that takes all, scores far below zero and rising along the sequence."""
    g = gen(16)
    args, _ = attention_case(g, [1000, 1500, 300], 4, 2, 64, dtype)
    q, kp, vp, table, lengths = args
    check_attention(args, {}, scale=30.0)
    check_attention(args, {}, scale=-4.0)
    check_attention(args, {}, scale=0.0)
    ramp = torch.linspace(-40, 40, 1500)
    q[1] = 0
    q[1, :, 0] = 1
    for t in range(1500):
        kp[int(table[1, t // 16]), t % 16, :, 0] = ramp[t]
    check_attention(args, {}, scale=1.0)
    q[1, :, 0] = -1
    check_attention(args, {}, scale=1.0)
    if dtype != torch.float16:       # scores near the type's lowest value, all of them
        q[2], kp[table[2, :19].long()] = 2.0 ** 60, -(2.0 ** 60)
        out = paged_decode_attention(*args, scale=1.0)
        mean = torch.stack([vp[int(table[2, t // 16]), t % 16].float() for t in range(300)]).double().mean(0)
        want = mean.repeat_interleave(2, 0).cpu()
        # (equal scores: the mean, in fp32 sums of 300 tokens and one rounding)
        far = P.outside(out[2], want, 2 * 308 * 2.0 ** -24 * 4 + 2.0 ** -15 + P.HALF_STEP[dtype] * want.abs())
        assert not far, far


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_values_near_the_largest_of_their_type(dtype):
    """Scores that rise a little from tile to tile, and large values under the largest weight: no sum is above it."""
    n = 400
    args, _ = attention_case(gen(25), [n], 1, 1, 64, dtype)
    q, kp, vp, table, lengths = args
    q.zero_(), kp.zero_()
    q[0, 0, 0] = 1
    large = {torch.bfloat16: 2.0 ** 127, torch.float16: 60000.0, torch.float32: 2.0 ** 127}[dtype]
    for t in range(n):
        kp[int(table[0, t // 16]), t % 16, 0, 0] = (t // 32) * 0.5
    kp[int(table[0, (n - 1) // 16]), (n - 1) % 16, 0, 0] = 9.0          # (6.0 is the largest of the others)
    vp[int(table[0, (n - 1) // 16]), (n - 1) % 16, 0] = large
    check_attention(args, {}, scale=1.0)


def test_fp16_weights_of_many_small_scores_are_not_lost():
    """One token far above 60000 others that together weigh as much."""
    n = 60001
    args, _ = attention_case(gen(17), [n], 1, 1, 64, torch.float16)
    q, kp, vp, table, lengths = args
    q.zero_()
    q[0, 0, 0] = 1
    kp.zero_()
    kp[int(table[0, 0]), 0, 0, 0] = math.log(n - 1)
    vp.fill_(1.0)
    vp[int(table[0, 0]), 0, 0] = -1.0
    check_attention(args, {}, scale=1.0)


def test_offsets_beyond_32_bits():
    """Pages of a pool of 4.6 GB: byte and element offsets above 2^31 and 2^32."""
    n_pages, page, H, D = 70001, 16, 8, 128
    kp, vp = kv_pages(n_pages, page, H, D, device=DEV)
    assert kp.stride(0) * n_pages > 2 ** 31
    g = gen(18)
    numbers = [n_pages - 1, 32769, 65537, 0, 50000]
    table = torch.tensor([numbers, numbers[::-1]], dtype=torch.int32, device=DEV)
    positions = torch.arange(80, device=DEV).repeat(2)
    sequences = torch.arange(2, device=DEV).repeat_interleave(80)
    keep = (sequences == 0)
    k, v = randn(g, 160, H, D, dtype=torch.bfloat16), randn(g, 160, H, D, dtype=torch.bfloat16)
    append_kv_pages_(k[keep], v[keep], kp, vp, table, positions[keep], sequences=sequences[keep])
    q = randn(g, 2, 32, D, dtype=torch.bfloat16)
    got = paged_decode_attention(q, kp, vp, table, torch.tensor([80, 80], device=DEV))
    small = torch.stack([kp[i] for i in numbers]), torch.stack([vp[i] for i in numbers])
    order = torch.tensor([[0, 1, 2, 3, 4], [4, 3, 2, 1, 0]], dtype=torch.int32, device=DEV)
    want = paged_decode_attention(q, *small, order, torch.tensor([80, 80], device=DEV))
    assert torch.equal(got, want)
    assert torch.equal(torch.cat([kp[i] for i in numbers]), k[keep])


def test_queries_of_any_strides_and_outputs_given():
    args, _ = attention_case(gen(19), [100, 1000], 4, 2, 64, torch.bfloat16)
    q, rest = args[0], args[1:]
    want = check_attention(args, {})
    wide = torch.zeros(2, 8, 64, dtype=q.dtype, device=DEV)
    wide[:, ::2] = q
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=q.dtype, device=DEV)[1:].view(2, 4, 64).copy_(q)
    spread = torch.zeros(2, 4, 128, dtype=q.dtype, device=DEV)
    spread[..., ::2] = q
    for view in (wide[:, ::2], odd, q.transpose(0, 1).contiguous().transpose(0, 1), spread[..., ::2]):
        assert torch.equal(paged_decode_attention(view, *rest), want)
    out = torch.empty_like(q)
    assert paged_decode_attention(q, *rest, out=out) is out and torch.equal(out, want)
    table = torch.full((2, 200), -1, dtype=torch.int32, device=DEV)[:, ::1]
    table[:, : args[3].shape[1]] = args[3]
    assert torch.equal(paged_decode_attention(q, *rest[:2], table[:, : args[3].shape[1]], rest[3]), want)
    with pytest.raises(ValueError, match="out must be"):
        paged_decode_attention(q, *rest, out=wide[:, ::2])
    with pytest.raises(RuntimeError, match="lengths is on cpu"):
        paged_decode_attention(q, *rest[:3], rest[3].cpu())
    unaligned = [torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape) for x in rest[:2]]
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        paged_decode_attention(q, *unaligned, *rest[2:])


def test_the_same_call_gives_the_same_bits_and_streams_do_not_meet():
    g = gen(20)
    cases = [attention_case(g, lengths, 8, 2, 128, torch.bfloat16)[0] for lengths in ([9000], [5000, 1, 800], [300] * 40)]
    want = [paged_decode_attention(*a) for a in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for i, (a, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(paged_decode_attention(*a))
    torch.cuda.synchronize()
    for x, ys in zip(want, got):
        assert all(torch.equal(x, y) for y in ys)


def test_two_graphs_of_one_pool_do_not_share_their_workspaces():
    """Captured calls of unlike shapes, replayed in turn and with eager calls and other allocations between."""
    g = gen(22)
    long, _ = attention_case(g, [6000, 900], 8, 2, 128, torch.bfloat16)
    q, kp, vp, table, lengths = long
    short = (q[:1].clone(), kp, vp, table[:1], lengths[:1].clone())
    want = paged_decode_attention(*long), paged_decode_attention(*short)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for args in (long, short):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_decode_attention(*args))
        graphs.append(graph)
    for turn in range(4):
        for i in (turn % 2, 1 - turn % 2):
            outs[i].fill_(float("nan"))
            graphs[i].replay()
            junk = torch.full((1 << 22,), float("nan"), device=DEV)
            assert torch.equal(paged_decode_attention(*long), want[0])
            del junk
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    lengths.fill_(17)           # the lengths are the device's: a replay sees them
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], paged_decode_attention(*long))


def test_calls_from_several_threads():
    import threading

    g = gen(23)
    cases = [attention_case(g, lengths, 4, 2, 64, torch.bfloat16)[0] for lengths in ([3000], [40] * 30, [700, 2], [1])]
    want = [paged_decode_attention(*a) for a in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = paged_decode_attention(*cases[i])
                stream.synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_pages_shared_by_sequences():
    """A common beginning: the same page numbers in several rows of the table."""
    args, _ = attention_case(gen(24), [320, 64, 1000], 4, 2, 64, torch.float16)
    q, kp, vp, table, lengths = args
    table[1, :4] = table[0, :4]
    table[2, :20] = table[0, :20]
    check_attention(args, {})


# ---- a run of them -------------------------------------------------------------------

@pytest.mark.parametrize("types", [(torch.bfloat16, None), (torch.float32, None), (torch.bfloat16, E4M3)],
                         ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_decoding_a_batch_against_attention_over_its_history(types):
    """Prompts into the pages, then steps of one token for every sequence that is still running, captured once and
    replayed, against attention in 64 bits over the turned keys that each sequence has had."""
    dtype, cache = types
    g = gen(21)
    Hq, H, D, page, prompts, steps = 8, 2, 64, 16, [40, 1, 900, 7], 6
    freqs, factor = rotary_frequencies(D, 500000.0, {"type": "llama3"}, device=DEV)
    n_pages = sum(-(-(n + steps) // page) for n in prompts) + 2
    kp, vp = kv_pages(n_pages, page, H, D, dtype=cache or dtype, device=DEV)
    kp.view(torch.uint8).fill_(0xff if cache else 0x7f), vp.view(torch.uint8).fill_(0xff if cache else 0x7f)
    table = P.table_of([n + steps for n in prompts], page, n_pages, g).to(DEV)
    scales = {}
    if cache:
        scales = {"k_scale": torch.full((H,), 0.01, device=DEV), "v_scale": torch.full((H,), 0.02, device=DEV)}
    T = sum(prompts)
    k, v = randn(g, T, H, D, dtype=dtype), randn(g, T, H, D, dtype=dtype)
    sequences = torch.arange(4).repeat_interleave(torch.tensor(prompts)).to(DEV)
    positions = torch.cat([torch.arange(n) for n in prompts]).to(DEV)
    append_kv_pages_(k, v, kp, vp, table, positions, sequences=sequences, freqs=freqs, factor=factor, **scales)

    # static buffers of the captured step; a sequence that has ended has position -1
    q1, k1, v1 = (torch.zeros(4, h, D, dtype=dtype, device=DEV) for h in (Hq, H, H))
    at = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    running = torch.ones(4, dtype=torch.bool, device=DEV)

    def step():
        here = torch.where(running, at, -1)
        turned = append_kv_pages_(k1, v1, kp, vp, table, here, xq=q1, freqs=freqs, factor=factor, **scales)
        return turned, paged_decode_attention(turned, kp, vp, table, torch.where(running, at + 1, 0), **scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = step()

    history = [[(k[sequences == b][i], v[sequences == b][i], i) for i in range(n)] for b, n in enumerate(prompts)]
    for s in range(steps):
        for x in (q1, k1, v1):
            x.copy_(randn(g, *x.shape, dtype=dtype))
        if s == 3:
            running[1] = False
        graph.replay()
        torch.cuda.synchronize()
        here = at.tolist()
        for b in range(4):
            if not running[b]:
                assert not out[b].any()
                continue
            history[b].append((k1[b].clone(), v1[b].clone(), here[b]))
            keys, values = (torch.stack([h[i] for h in history[b]]) for i in (0, 1))
            where = torch.tensor([h[2] for h in history[b]])
            k64 = P.turned(keys, where, freqs, "interleaved", factor)
            v64 = values.cpu().double()
            q64 = P.turned(q1[b:b + 1], at[b:b + 1], freqs, "interleaved", factor)[0]
            n = len(history[b])
            assert where.tolist() == list(range(n))
            kh, vh = (x.repeat_interleave(Hq // H, 1) for x in (k64, v64))
            scores = torch.einsum("hd,thd->ht", q64, kh) / math.sqrt(D)
            w = scores.softmax(-1)
            want = torch.einsum("ht,thd->hd", w, vh)
            # queries and keys are rounded once to their types: a score is off by the two roundings times its products'
            # sizes, a weight by that relatively; values are rounded to the pages' type
            kt, vt = P.HALF_STEP[cache or dtype], P.HALF_STEP[cache] if cache else 0.0
            small = (P.SMALLEST[E4M3] * 0.02 if cache else 0.0)
            reach = torch.einsum("hd,thd->ht", q64.abs(), kh.abs()).amax(-1) / math.sqrt(D)
            ks = (P.SMALLEST[E4M3] * 0.01 * q64.abs().sum(-1) / math.sqrt(D)) if cache else 0.0
            d = (kt + P.HALF_STEP[dtype]) * 1.01 * reach * math.sqrt(2) + ks
            size = torch.einsum("ht,thd->hd", w, vh.abs())
            relative = torch.expm1(2 * d)[:, None] + (n + 2 * D + 64) * 2.0 ** -24 * (1 + reach[:, None]) + 2.0 ** -15
            far = P.outside(out[b], want, size * (relative * (1 + vt) + vt) + small + P.HALF_STEP[dtype] * (want.abs() + size * relative) + 1e-30)
            assert not far, (s, b, far)
            # and, much closer, against the same pages read back
            o, _, sz, rc = P.attention(turned[b:b + 1], kp, vp, table[b:b + 1], at[b:b + 1] + 1, None, scales.get("k_scale"),
                                       scales.get("v_scale"))
            bound, _ = P.attention_bounds(o, sz, rc, at[b:b + 1] + 1, dtype)
            far = P.outside(out[b:b + 1], o, bound)
            assert not far, (s, b, far)
        at.add_(1)


@pytest.mark.parametrize("n", [15, 30, 60])
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_weights_keep_their_bits(types, n):
    """One token against n that weigh 1/n each: what is left of the sum shows what a weight has lost."""
    dtype, cache = types
    args, scales = attention_case(gen(31), [n + 1], 2, 1, 64, dtype, cache)
    q, kp, vp, table, _ = args
    q.zero_()
    q[:, :, 0] = 1
    key, value = torch.zeros(n + 1, 64), torch.full((n + 1, 64), -1.0)
    key[1:, 0], value[0] = 1, 1
    for t in range(n + 1):
        at = int(table[0, t // 16])
        kp[at, t % 16, 0], vp[at, t % 16, 0] = key[t].to(kp.dtype).to(DEV), value[t].to(vp.dtype).to(DEV)
    ones = {name: torch.ones_like(x) for name, x in scales.items()}
    scale = float(torch.tensor(-math.log(n)))
    out, _, size, reach = P.attention(*args, scale)
    got = paged_decode_attention(*args, scale=scale, **ones)
    # a score is one product times the scale times log2 e: four half steps of it, the exponential eight of the weight;
    # n + 1 weights and values are added up in fp32; fp16 weights are two numbers, off by 1.5 * 2^-21.  (The quotient's
    # own errors are those of a number that is nearly nothing.)
    relative = 2.0 ** -24 * (4 * reach + 8 + n + 8) + (1.5 * 2.0 ** -21 if dtype == torch.float16 else 0.0)
    far = P.outside(got, out, (relative[..., None] * (size + 2 * out.abs())) + P.HALF_STEP[dtype] * out.abs() + P.SMALLEST[dtype])
    assert not far, far


@pytest.mark.parametrize("dtype, below", [(torch.float16, 28), (torch.bfloat16, 28), (torch.bfloat16, 90), (torch.float32, 90)])
@pytest.mark.parametrize("n", [200, 3000])
def test_infinite_values_under_small_weights(dtype, below, n):
    """An infinite value is one whatever its token weighs, as far as its weight has all its parts."""
    args, _ = attention_case(gen(32), [n, n], 4, 2, 64, dtype)
    q, kp, vp, table, _ = args
    q.zero_()
    q[:, :, 0] = 1
    kp[..., 0] = 0
    scale = below * math.log(2.0)
    for t in range(n):      # (the largest weight is at the end of sequence 0 and at the beginning of sequence 1)
        for b, top in ((0, n - 1), (1, 0)):
            kp[int(table[b, t // 16]), t % 16, :, 0] = 1.0 if t == top else -0.01 * (t % 2)
    clean = check_attention(args, {}, scale=scale)
    last = (n - 1) // 32 * 32
    # (beside the largest weight in its wave's tile of 32, in that wave's tile before or behind, in other waves')
    for b, t in ((0, last + 1), (0, last - 126), (0, 3), (1, 1), (1, 130), (1, n - 2)):
        vp[int(table[b, t // 16]), t % 16, 0, 5] = float("inf")
        vp[int(table[b, t // 16]), t % 16, 1, 9] = -float("inf")
    got = paged_decode_attention(*args, scale=scale)
    assert (got[:, :2, 5] == float("inf")).all() and (got[:, 2:, 9] == -float("inf")).all()
    got[:, :2, 5], got[:, 2:, 9] = clean[:, :2, 5], clean[:, 2:, 9]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("types", [(torch.bfloat16, E4M3), (torch.float16, E4M3), (torch.float16, None)],
                         ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_missing_values_stay_with_their_sequence_and_head(types):
    dtype, cache = types
    args, scales = attention_case(gen(33), [200, 200, 700, 700], 4, 2, 64, dtype, cache)
    q, kp, vp, table, _ = args
    clean = paged_decode_attention(*args, **scales)
    nan = torch.tensor(float("nan")).to(kp.dtype).to(DEV)
    whole = torch.uint8 if cache else dtype
    vp.view(whole)[int(table[0, 3]), 5, 1, 7] = nan.view(whole)
    kp.view(whole)[int(table[3, 40]), 2, 0, 9] = nan.view(whole)
    got = paged_decode_attention(*args, **scales)
    assert got[0, 2:, 7].isnan().all() and got[3, :2].isnan().all()
    got[0, 2:, 7], got[3, :2] = clean[0, 2:, 7], clean[3, :2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("heads", [(4, 2, 64), (6, 2, 128), (40, 1, 128)], ids=str)
@pytest.mark.parametrize("types", TYPES[:3], ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_scores_of_minus_infinity(types, heads):
    """A sequence of which every token scores -inf has the definition's 0 / 0 and a denominator of 0; where others do not,
    its tokens weigh nothing, as if they were not there.  A sequence without tokens has zeros."""
    dtype, _ = types
    lengths = [40, 40, 3000, 3000, 0, 700, 20]
    args, _ = attention_case(gen(34), lengths, *heads, dtype)
    q, kp, vp, table, lens = args
    q[..., 0] = 1
    rep = heads[0] // heads[1]
    for b in (0, 2):                                            # all tokens, of kv head 0
        kp[table[b, : -(-lengths[b] // 16)].long(), :, 0, 0] = -float("inf")
    without = table.clone()
    for b, pages in ((1, [0, 1]), (3, range(3, 150)), (5, [43]), (6, [])):     # whole pages, of all kv heads
        for i in pages:
            kp[int(table[b, i]), :, :, 0] = -float("inf")
            without[b, i] = -1
    lse, want_lse = torch.zeros(q.shape[:2], device=DEV), torch.zeros(q.shape[:2], device=DEV)
    got = paged_decode_attention(*args, lse=lse)
    want = paged_decode_attention(q, kp, vp, without, lens, lse=want_lse)
    for b in (0, 2):
        assert got[b, :rep].isnan().all() and (lse[b, :rep] == -math.inf).all()
        assert not got[b, rep:].isnan().any() and lse[b, rep:].isfinite().all()
    assert not got[4].any() and (lse[4] == -math.inf).all()
    assert torch.equal(got[[1, 3, 4, 5, 6]], want[[1, 3, 4, 5, 6]]) and torch.equal(lse, want_lse)
    assert torch.equal(got[:, rep:], want[:, rep:])
    assert not got[[1, 3, 5, 6]].isnan().any()


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
@pytest.mark.parametrize("lengths", [[40, 0, 300, 512], [3000, 1, 0, 700, 128, 5000, 17, 2]], ids=str)
def test_the_output_may_be_the_queries(types, lengths):
    dtype, cache = types
    for heads in ((4, 2, 64), (33, 1, 128), (24, 8, 256)):
        args, scales = attention_case(gen(35), lengths, *heads, dtype, cache)
        want = paged_decode_attention(*args, **scales)
        q = args[0].clone()
        assert paged_decode_attention(q, *args[1:], **scales, out=q) is q and torch.equal(q, want)
