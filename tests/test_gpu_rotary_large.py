"""Rotary rows and the append where a workgroup has several tokens, and where rows come and go by streaming: bit for bit
what the same tokens give in small calls, which tests/test_gpu_rotary.py and tests/test_gpu_paged.py hold to the definition."""

import pytest
import torch

from dram_attention_amd import append_kv_pages_, kv_pages, rotary_frequencies, rotate, rotate_

from . import paged as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
STREAMED = 256 << 20        # bytes read and written from which calls stream


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def bits(x):
    return x.contiguous().view(torch.uint8)


def in_pieces(call, tokens, piece=900):
    return torch.cat([call(slice(i, min(i + piece, tokens))) for i in range(0, tokens, piece)])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("D, rotary, dtype", [(64, 16, torch.bfloat16), (64, 64, torch.float32), (80, 20, torch.float16),
                                              (96, 2, torch.bfloat16), (5, 4, torch.float32)])
def test_workgroups_across_batches(D, rotary, dtype, layout):
    """Several tokens a workgroup, the last one with fewer, of two sequences with positions of their own."""
    g = gen(D + rotary)
    freqs, _ = rotary_frequencies(rotary, 10000.0, device=DEV)
    for B, S in ((3, 1001), (1367, 3), (2, 9001)):
        q, k = randn(g, B, S, 3, D, dtype=dtype), randn(g, B, S, 1, D, dtype=dtype)
        positions = torch.randint(-5, 200000, (B, S), generator=g, device=DEV)
        for at in (positions, positions.int().t().contiguous().t(), positions[:1].expand(B, S), positions[0]):
            yq, yk = rotate(q, k, at, freqs, layout=layout, factor=1.25)
            flat = at.expand(B, S).reshape(-1)
            for x, y in ((q, yq), (k, yk)):
                x = x.flatten(0, 1)
                want = in_pieces(lambda i: rotate(x[i], None, flat[i], freqs, layout=layout, factor=1.25)[0], B * S)
                assert torch.equal(y.flatten(0, 1), want)
        wide = torch.stack((q, q), 3)[:, :, :, 0]           # (rows with gaps)
        assert torch.equal(rotate(wide, None, positions, freqs, layout=layout, factor=1.25)[0],
                           rotate(q, None, positions, freqs, layout=layout, factor=1.25)[0])
    some = torch.arange(0, 2 * 9001, 997, device=DEV)
    rows, where = q.flatten(0, 1)[some], positions.reshape(-1)[some]
    got = rotate(q, None, positions, freqs, layout=layout)[0].flatten(0, 1)[some]
    far = P.outside(got, P.turned(rows, where, freqs, layout), P.turned_bound(rows, dtype, 1.0, rotary, layout))
    assert not far, far


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("types", [(torch.bfloat16, None), (torch.float16, E4M3), (torch.float32, None), (torch.bfloat16, E4M3)],
                         ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
@pytest.mark.parametrize("D, rotary, T", [(64, 16, 8203), (64, 64, 2051), (80, 20, 4099), (66, 22, 17001)])
def test_appends_of_several_tokens_a_workgroup(D, rotary, T, types, layout):
    """Tokens that are stored beside ones that are not: padding, sequences and positions beyond the table, pages beyond
    the pool."""
    dtype, cache = types
    g = gen(T)
    H, page, B = 2, 16, 7
    freqs, factor = rotary_frequencies(rotary, scaling={"type": "yarn", "factor": 4.0, "original_length": 32}, device=DEV)
    width = -(-T // (B * page)) + 3
    n_pages = B * width
    table = torch.randperm(n_pages, generator=g, device=DEV).view(B, width).int()
    table[2, 1], table[3, 2], table[4, 0] = -1, n_pages, 2 ** 31 - 1
    order = torch.randperm(B * width * page, generator=g, device=DEV)[:T]           # places of their own
    sequences, positions = order // (width * page), order % (width * page)
    odd = torch.rand(T, generator=g, device=DEV)
    sequences = torch.where(odd < 0.05, torch.where(odd < 0.02, -1, B), sequences)
    positions = torch.where(odd > 0.95, torch.where(odd > 0.98, -1 - positions, width * page), positions)
    q, k, v = (randn(g, T, h, D, dtype=dtype) for h in (3, H, H))
    scales = {}
    if cache:
        scales = {"k_scale": torch.tensor([0.3, 0.02], device=DEV), "v_scale": torch.tensor([0.01, 1.0], device=DEV)}
    pools = [kv_pages(n_pages, page, H, D, dtype=cache or dtype, device=DEV) for _ in range(2)]
    for pool in pools:
        for x in pool:
            x.view(torch.uint8).fill_(0x55)

    def call(pool, i):
        return append_kv_pages_(k[i], v[i], *pool, table, positions[i], sequences=sequences[i], xq=q[i], freqs=freqs,
                                layout=layout, factor=factor, **scales)

    got, want = call(pools[0], slice(0, T)), in_pieces(lambda i: call(pools[1], i), T)
    assert torch.equal(got, want)
    for x, y in zip(*pools):
        assert torch.equal(bits(x), bits(y))
    stored = ((bits(pools[0][0]).view(n_pages, page, -1) != 0x55).any(-1)).sum()
    good = (sequences >= 0) & (sequences < B) & (positions >= 0) & (positions < width * page)
    number = table[sequences.clamp(0, B - 1), (positions // page).clamp(0, width - 1)]
    assert stored == (good & (number >= 0) & (number < n_pages)).sum() and stored < T


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_calls_that_stream(dtype, layout):
    g = gen(7)
    e = torch.empty(0, dtype=dtype).element_size()
    Hq, H, D, page = 32, 8, 128, 16
    freqs, _ = rotary_frequencies(D, device=DEV)
    T = STREAMED // (2 * e * (Hq + H) * D) + 101
    assert 2 * T * (Hq + H) * D * e >= STREAMED > 2 * 900 * (Hq + 2 * H) * D * e
    q, k, v = (randn(g, T, h, D, dtype=dtype) for h in (Hq, H, H))
    positions = torch.randint(0, 200000, (T,), generator=g, device=DEV)
    want = [in_pieces(lambda i: rotate(x[i], None, positions[i], freqs, layout=layout)[0], T) for x in (q, k)]
    yq, yk = rotate(q, k, positions, freqs, layout=layout)
    assert torch.equal(yq, want[0]) and torch.equal(yk, want[1])
    a, b = q.clone(), k.clone()
    rotate_(a, b, positions, freqs, layout=layout)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    del a, b
    half = freqs[: D // 4].contiguous()                     # (a part of the head)
    yq, yk = rotate(q, k, positions, half, layout=layout)
    for x, y in ((q, yq), (k, yk)):
        assert torch.equal(y, in_pieces(lambda i: rotate(x[i], None, positions[i], half, layout=layout)[0], T))
    for cache in (dtype, E4M3)[: 1 if dtype == torch.float32 else 2]:
        width = -(-T // page)
        table = torch.randperm(width, generator=g, device=DEV).view(1, width)
        at = torch.randperm(T, generator=g, device=DEV)
        of = torch.zeros_like(at)
        pools = [kv_pages(width, page, H, D, dtype=cache, device=DEV) for _ in range(2)]
        for pool in pools:
            for x in pool:
                x.view(torch.uint8).zero_()

        def call(pool, i):
            return append_kv_pages_(k[i], v[i], *pool, table, at[i], sequences=of[i], xq=q[i], freqs=freqs, layout=layout)

        got, want = call(pools[0], slice(0, T)), in_pieces(lambda i: call(pools[1], i), T)
        assert torch.equal(got, want)
        for x, y in zip(*pools):
            assert torch.equal(bits(x), bits(y))
