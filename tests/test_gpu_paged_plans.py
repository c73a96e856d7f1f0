"""Attention over pages in every form its launches take: shares of many units and of several sequences, sequences over
two, three and many shares, one workgroup a sequence, at every pair of types, head size and number of query rows that
share keys and values.  Which form a case takes is asserted from the workspace that it asks for, so that a change of the
rules cannot empty a case unseen."""

import ctypes
import functools
import math

import pytest
import torch

from dram_attention_amd import _lib, paged_decode_attention

from . import paged as P
from .test_paged_cpu import AttentionArgs

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
TYPES = [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None), (torch.bfloat16, E4M3), (torch.float16, E4M3)]
name_of = lambda t: "-".join(str(x).replace("torch.", "") for x in t)  # noqa: E731


def shares_of(B, width, page, Hq, H, D, dtype, cache):
    """Workgroups that a kv head's sequences are shared out to; 0: one a sequence."""
    a = AttentionArgs(n_pages=4, page_size=page, n_sequences=B, pages_per_sequence=width, n_q_heads=Hq, n_kv_heads=H,
                      head_dim=D, dtype=_lib.dtype_code(dtype), page_dtype=_lib.DA_E4M3 if cache else _lib.dtype_code(dtype))
    need = _lib.load().da_paged_attention_workspace_bytes(bytes(a), ctypes.sizeof(a))
    if not need:
        return 0
    rep = Hq // H
    rows = 32 if rep > 16 and D <= 128 and dtype != torch.float32 else 16       # that a share's sums are kept for
    head_groups = H * -(-rep // rows)
    prefix = -(-(B + 1) * 4 // 16) * 16
    shares, rest = divmod(need - prefix, 16 + head_groups * 2 * rows * (8 + 4 * D))
    assert rest == 0, "the workspace is laid out otherwise"
    return shares


def case_of(seed, lengths, Hq, H, D, dtype, cache, page, width):
    """As tests/test_gpu_paged.py makes them, on the GPU."""
    g, cpu = torch.Generator(device=DEV).manual_seed(seed), torch.Generator().manual_seed(seed)
    n_pages = sum(-(-n // page) for n in lengths) + 3
    pool = torch.empty(n_pages, H, page, 2, D, dtype=cache or dtype, device=DEV)
    for i in range(0, n_pages, 64):
        rows = pool[i: i + 64]
        pool[i: i + 64] = torch.randn(rows.shape, generator=g, device=DEV).to(pool.dtype)
    kp, vp = pool[:, :, :, 0].transpose(1, 2), pool[:, :, :, 1].transpose(1, 2)
    q = torch.randn(len(lengths), Hq, D, generator=g, device=DEV).to(dtype)
    table = P.table_of(lengths, page, n_pages, cpu, width).to(DEV)
    scales = {}
    if cache:
        scales = {n: torch.rand(H, generator=cpu).add(0.5).to(DEV) for n in ("k_scale", "v_scale")}
    return (q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)), scales


def attention64(q, k_pages, v_pages, table, lengths, k_scale=None, v_scale=None):
    """tests/paged.py's attention, all heads of a sequence at a time, in float64 on the GPU."""
    B, Hq, D = q.shape
    page, H = k_pages.shape[1:3]
    out, lse = torch.zeros(B, Hq, D).double(), torch.full((B, Hq), -math.inf).double()
    size, reach = torch.zeros(B, Hq, D).double(), torch.zeros(B, Hq).double()
    for b in range(B):
        n = int(lengths[b])
        if n == 0:
            continue
        numbers = table[b, : -(-n // page)].long()

        def rows(pages, scale):
            raw = pages.view(torch.uint8)[numbers].view(pages.dtype) if pages.dtype == E4M3 else pages[numbers]
            x = raw.float().double().flatten(0, 1)[:n].transpose(0, 1)       # (H, n, D)
            return (x if scale is None else x * scale.double()[:, None, None]).contiguous()

        k, v = rows(k_pages, k_scale), rows(v_pages, v_scale)
        x = q[b].double().view(H, Hq // H, D)
        s = torch.bmm(x, k.transpose(1, 2).contiguous()) / math.sqrt(D)
        top = torch.logsumexp(s, -1)
        w = torch.exp(s - top[..., None])
        out[b], size[b] = torch.bmm(w, v).view(Hq, D).cpu(), torch.bmm(w, v.abs()).view(Hq, D).cpu()
        lse[b] = top.view(Hq).cpu()
        reach[b] = (torch.bmm(x.abs(), k.abs().transpose(1, 2).contiguous()).amax(-1) / math.sqrt(D)).view(Hq).cpu()
    return out, lse, size, reach


def check(args, scales):
    q, lengths = args[0], args[4]
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = paged_decode_attention(*args, lse=lse, **scales)
    out, want_lse, size, reach = attention64(*args, **scales)
    bound, lse_bound = P.attention_bounds(out, size, reach, lengths, q.dtype)
    far = P.outside(got, out, bound)
    assert not far, far
    far = P.outside(lse, want_lse, lse_bound + 2.0 ** -23 * want_lse.abs().nan_to_num(posinf=0.0))
    assert not far, "lse: " + far
    assert torch.equal(paged_decode_attention(*args, **scales), got)


UNITS = {torch.float32: 64}         # tokens that are shared out together; 128 in 16 bits


@functools.lru_cache(None)
def kv_heads_for(B, width, page, rep, D, dtype, cache, most):
    """The least kv heads that leave no more than `most` shares."""
    for H in (1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256):
        if rep * H <= 4096 and shares_of(B, width, page, rep * H, H, D, dtype, cache) <= most:
            return H
    raise AssertionError("no such number of kv heads")


# sequences shorter, as long as, and longer than a unit; without tokens; of one token; ones over several shares
RAGGED = [0, 1, 127, 128, 129, 1500, 0, 255, 256, 257, 700, 3, 1100, 0, 64, 65, 63, 1]
EVEN = [512] * 16                                               # borders on the sequences' ends
LONG = [0, 2600, 5, 130, 0, 1900, 1, 0, 300, 17, 1]             # over two, three and many shares


@pytest.mark.parametrize("lengths", [RAGGED, EVEN, LONG, [4000, 1, 3300], [5000]], ids=["ragged", "even", "long", "three", "one"])
@pytest.mark.parametrize("rep", [2, 17])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("types", TYPES, ids=name_of)
def test_shares_of_many_units(types, D, rep, lengths):
    dtype, cache = types
    page, B = 16, len(lengths)
    width = -(-max(lengths + [1100]) // page) + 2               # (more than a workgroup a sequence is for)
    H = kv_heads_for(B, width, page, rep, D, dtype, cache, 8)
    shares = shares_of(B, width, page, rep * H, H, D, dtype, cache)
    unit = UNITS.get(dtype, 128)
    assert 2 <= shares <= 8 and sum(-(-n // unit) for n in lengths) >= 4 * shares
    assert (shares <= B) == (B >= 8)                            # (both forms of the join)
    args, scales = case_of(D + rep, lengths, rep * H, H, D, dtype, cache, page, width)
    check(args, scales)


@pytest.mark.parametrize("rep", [1, 4, 33])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("types", TYPES, ids=name_of)
def test_a_workgroup_a_sequence(types, D, rep):
    dtype, cache = types
    lengths, page, width, H = [512, 511, 0, 1, 300, 257, 256, 129, 128, 127, 31, 33, 500], 16, 32, 3
    assert shares_of(len(lengths), width, page, rep * H, H, D, dtype, cache) == 0
    args, scales = case_of(D + rep, lengths, rep * H, H, D, dtype, cache, page, width)
    check(args, scales)


@pytest.mark.parametrize("types", TYPES, ids=name_of)
def test_many_sequences_of_all_lengths_in_few_shares(types):
    """Several sequences a share, some over several, none or many tokens: 100 of them in pages that are no power of two."""
    dtype, cache = types
    g = torch.Generator().manual_seed(40)
    lengths = torch.randint(0, 3000, (100,), generator=g).tolist()
    for i in (0, 1, 20, 21, 22, 60, 99):
        lengths[i] = 0
    for i in (5, 6, 7, 50):
        lengths[i] = i % 2 + 1
    page, H, rep, D = 24, 16, 2, 64
    width = 3000 // page + 1
    shares = shares_of(100, width, page, rep * H, H, D, dtype, cache)
    assert 32 <= shares <= 100
    args, scales = case_of(41, lengths, rep * H, H, D, dtype, cache, page, width)
    check(args, scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shares_of_more_sequences_than_16_bits_count(dtype):
    """70000 sequences, most of them of no tokens, some of a few, some over several shares."""
    g = torch.Generator().manual_seed(42)
    B, page, width, D = 70000, 16, 80, 64
    few = torch.randperm(B, generator=g)[:3000]
    lengths = torch.zeros(B, dtype=torch.int64)
    lengths[few] = torch.randint(1, 4, (3000,), generator=g)
    long = few[:9].tolist() + [0, B - 1, 255, 256, 65535, 65536]
    lengths[long] = torch.randint(900, width * page + 1, (len(long),), generator=g)
    shares = shares_of(B, width, page, 2, 2, D, dtype, None)
    unit = UNITS.get(dtype, 128)
    units = (lengths + unit - 1) // unit
    each = -(-int(units.sum()) // shares)
    assert shares > 100 and int(units.max()) > each             # (some are over several shares)
    n_pages = 500
    kp, vp = (x.to(DEV) for x in P.pool(n_pages, page, 2, D, dtype, "cpu", g))
    table = torch.randint(0, n_pages, (B, width), generator=g, dtype=torch.int32).to(DEV)
    q = torch.randn(B, 2, D, generator=g).to(dtype).to(DEV)
    lens = lengths.to(DEV)
    lse = torch.zeros(B, 2, device=DEV)
    got = paged_decode_attention(q, kp, vp, table, lens, lse=lse)
    assert not got[(lens == 0)].any() and (lse[lens == 0] == -math.inf).all()
    some = lens.nonzero()[:, 0]
    out, want_lse, size, reach = attention64(q[some], kp, vp, table[some], lens[some])
    bound, lse_bound = P.attention_bounds(out, size, reach, lens[some], dtype)
    far = P.outside(got[some], out, bound)
    assert not far, far
    far = P.outside(lse[some], want_lse, lse_bound + 2.0 ** -23 * want_lse.abs())
    assert not far, "lse: " + far
