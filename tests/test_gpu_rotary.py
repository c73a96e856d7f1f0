"""Rotary positions on the GPU against their definition in 64 bits (tests/paged.py), forward and backward."""

import pytest
import torch

from dram_attention_amd import rotary_frequencies, rotate, rotate_

from . import paged as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def check(got, x, positions, freqs, layout, factor=1.0):
    want = P.turned(x, positions, freqs, layout, factor)
    far = P.outside(got, want, P.turned_bound(x, x.dtype, factor, 2 * freqs.numel(), layout))
    assert not far, far


# (tokens, heads, kv heads, head_dim, rotary_dim)
SHAPES = [(1, 32, 8, 128, 128), (1, 1, 1, 8, 2), (257, 5, 3, 80, 20), (64, 7, 1, 64, 64), (33, 4, 2, 128, 32),
          (19, 3, 3, 96, 96), (10, 2, 1, 256, 256), (5, 3, 1, 512, 512), (9, 2, 2, 66, 66), (7, 40, 2, 24, 8),
          (3, 2, 1, 5, 4), (300, 70, 10, 16, 16), (65, 4, 1, 96, 24), (31, 3, 2, 20, 12)]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotate_against_the_definition(shape, dtype, layout):
    T, Hq, H, D, R = shape
    g = gen(T + D)
    q, k = randn(g, T, Hq, D, dtype=dtype), randn(g, T, H, D, dtype=dtype)
    freqs, _ = rotary_frequencies(R, 10000.0, device=DEV)
    positions = torch.randint(-5, 200000, (T,), generator=g).to(torch.int32).to(DEV)
    yq, yk = rotate(q, k, positions, freqs, layout=layout, factor=1.25)
    check(yq, q, positions, freqs, layout, 1.25)
    check(yk, k, positions, freqs, layout, 1.25)
    assert torch.equal(yq[..., R:], q[..., R:]) and torch.equal(yk[..., R:], k[..., R:])
    alone, none = rotate(q, None, positions.long(), freqs, layout=layout, factor=1.25)
    assert none is None and torch.equal(alone, yq)
    a, b = q.clone(), k.clone()
    assert rotate_(a, b, positions, freqs, layout=layout, factor=1.25) == (a, b)
    assert torch.equal(a, yq) and torch.equal(b, yk)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_far_positions_keep_their_angles(layout):
    """2^27 positions: an angle is off by what two roundings in 64 bits are, 2^-52 * 2^27 rad, below fp32's."""
    positions = torch.tensor([0, 1, 131071, 999_983, 16_777_217, 2 ** 27 - 1, -(2 ** 27 - 1)], dtype=torch.int64, device=DEV)
    freqs, _ = rotary_frequencies(64, 500000.0, device=DEV)
    x = randn(gen(0), 7, 2, 64, dtype=torch.float32)
    check(rotate(x, None, positions, freqs, layout=layout)[0], x, positions, freqs, layout)


def test_no_channel_turns():
    x = randn(gen(1), 4, 2, 64, dtype=torch.bfloat16)
    none = torch.empty(0, dtype=torch.float64, device=DEV)
    assert torch.equal(rotate(x, None, torch.arange(4, device=DEV), none)[0], x)


def test_empty_operands():
    freqs, _ = rotary_frequencies(64, device=DEV)
    for shape in ((0, 4, 64), (3, 0, 64), (2, 0, 4, 64), (0, 5, 4, 64)):
        x = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        positions = torch.zeros(shape[:-2], dtype=torch.int32, device=DEV)
        assert rotate(x, x, positions, freqs)[1].shape == x.shape


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_any_strides(dtype, layout):
    g = gen(2)
    B, S, H, D = 3, 21, 4, 64
    freqs, _ = rotary_frequencies(D, device=DEV)
    positions = torch.randint(0, 5000, (B, S), generator=g).to(torch.int32).to(DEV)
    fused = randn(g, B, S, 3 * H + 1, D, dtype=dtype)
    odd = randn(g, B * S * H * D + 1, dtype=dtype)[1:].view(B, S, H, D)                 # unaligned rows
    for q, k in ((fused[:, :, :H], fused[:, :, H: 2 * H + 1]), (odd, odd[:, :, :1]),
                 (randn(g, B, H, S, D, dtype=dtype).transpose(1, 2), fused[:, :, 1:2]),
                 (randn(g, 1, S, H, D, dtype=dtype).expand(B, S, H, D), randn(g, B, S, 1, D, dtype=dtype).expand(B, S, H, D)),
                 (randn(g, B, S, D, H, dtype=dtype).transpose(2, 3), randn(g, B, S, H, 2 * D, dtype=dtype)[..., ::2])):
        yq, yk = rotate(q, k, positions, freqs, layout=layout)
        check(yq, q, positions, freqs, layout)
        check(yk, k, positions, freqs, layout)
        wide = positions.t().contiguous().t().long()
        assert torch.equal(rotate(q, k, wide, freqs, layout=layout)[0], yq)
    both = fused.clone()
    rotate_(both[:, :, :H], both[:, :, H: 2 * H], positions, freqs, layout=layout)
    check(both[:, :, : 2 * H], fused[:, :, : 2 * H], positions, freqs, layout)
    assert torch.equal(both[:, :, 2 * H:], fused[:, :, 2 * H:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(dtype, layout):
    g = gen(3)
    B, S, Hq, H, D, R = 2, 13, 6, 2, 64, 48
    freqs, factor = rotary_frequencies(R, scaling={"type": "yarn", "factor": 8.0, "original_length": 64}, device=DEV)
    positions = torch.arange(100, 100 + S, device=DEV)
    q, k = randn(g, B, S, Hq, D, dtype=dtype).requires_grad_(), randn(g, B, S, H, D, dtype=dtype).requires_grad_()
    gq, gk = randn(g, B, S, Hq, D, dtype=dtype), randn(g, B, H, S, D, dtype=dtype).transpose(1, 2)
    both = positions.expand(B, S)
    yq, yk = rotate(q, k, positions, freqs, layout=layout, factor=factor)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for got, gr in ((dq, gq), (dk, gk)):     # the transpose of the turn is the turn back
        check(got, gr, -both, freqs, layout, factor)
    # against differences of the (linear) function itself, summed in 64 bits
    for y, x, gr, dx in ((yq, q, gq, dq), (yk, k, gk, dk)):
        want = (y.detach().double() * gr.double()).sum()
        got = (dx.double() * x.detach().double()).sum()
        size = (y.detach().double() * gr.double()).abs().sum() + (dx.double() * x.detach().double()).abs().sum()
        assert abs(got - want) <= 2 * P.HALF_STEP[dtype] * size
    # one output used, one input that wants a gradient, and neither tensor's graph holding the other
    dq1, = torch.autograd.grad(rotate(q, k, positions, freqs, layout=layout, factor=factor)[0], (q,), gq)
    assert torch.equal(dq1, dq)
    dk1, = torch.autograd.grad(rotate(q.detach(), k, positions, freqs, layout=layout, factor=factor)[1], (k,), gk)
    assert torch.equal(dk1, dk)
    dq2, = torch.autograd.grad(rotate(q, None, positions, freqs, layout=layout, factor=factor)[0], (q,), gq)
    assert torch.equal(dq2, dq)


def test_gradients_of_broadcast_rows_and_gradients_add_up():
    g = gen(4)
    S, H, D = 9, 6, 64
    freqs, _ = rotary_frequencies(D, device=DEV)
    positions = torch.arange(S, device=DEV)
    one = randn(g, S, 1, D, dtype=torch.float32).requires_grad_()
    y, _ = rotate(one.expand(S, H, D), None, positions, freqs)
    gr = randn(g, S, 1, D, dtype=torch.float32)
    got, = torch.autograd.grad(y, (one,), gr.expand(S, H, D))
    want = P.turned(gr, -positions, freqs, "interleaved") * H
    far = P.outside(got, want, (H + 1) * P.turned_bound(gr, torch.float32) + H * H * 2.0 ** -24 * want.abs())
    assert not far, far


def test_gradients_that_are_lazy_views():
    """What autograd hands over may be the negative, or nothing, of what its memory holds."""
    g = gen(9)
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(5, device=DEV)
    q = randn(g, 5, 2, 64, dtype=torch.float32).requires_grad_()
    y, _ = rotate(q, None, positions, freqs)
    negative = torch.randn(5, 2, 64, dtype=torch.complex64, generator=g).to(DEV).conj().imag
    assert negative.is_neg()
    dq, = torch.autograd.grad(y, (q,), negative)
    check(dq, negative.resolve_neg().contiguous(), -positions, freqs, "interleaved")


def test_the_gradient_has_a_gradient():
    g = gen(5)
    q = randn(g, 5, 2, 64, dtype=torch.float32).requires_grad_()
    gr = randn(g, 5, 2, 64, dtype=torch.float32).requires_grad_()
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(5, device=DEV)
    y, _ = rotate(q, None, positions, freqs, layout="half")
    dq, = torch.autograd.grad(y, (q,), gr, create_graph=True)
    v = randn(g, 5, 2, 64, dtype=torch.float32)
    back, = torch.autograd.grad(dq, (gr,), v)
    check(back, v, positions, freqs, "half")


def test_rotating_back_and_forth_through_a_graph_and_on_another_stream():
    g = gen(6)
    S, D = 50, 128
    freqs, _ = rotary_frequencies(D, device=DEV)
    q, k = randn(g, S, 8, D, dtype=torch.bfloat16), randn(g, S, 2, D, dtype=torch.bfloat16)
    positions = torch.arange(S, device=DEV, dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotate(q, k, positions, freqs)
        ql, kl = q.clone().requires_grad_(), k.clone().requires_grad_()
        gq, gk = torch.ones_like(q), torch.ones_like(k)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = rotate(ql, kl, positions, freqs)
        dq, dk = torch.autograd.grad((yq, yk), (ql, kl), (gq, gk))
    for step in range(3):
        with torch.no_grad():
            ql.copy_(randn(g, S, 8, D, dtype=torch.bfloat16))
            gq.copy_(randn(g, S, 8, D, dtype=torch.bfloat16))
            positions.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        check(yq, ql, positions, freqs, "interleaved")
        check(yk, kl, positions, freqs, "interleaved")
        check(dq, gq, -positions, freqs, "interleaved")
        with torch.no_grad():
            assert torch.equal(rotate(ql, kl, positions, freqs)[0], yq)


def test_gradients_on_another_stream_and_under_autocast():
    g = gen(8)
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(300, device=DEV)
    q, gr = randn(g, 300, 4, 64, dtype=torch.bfloat16), randn(g, 300, 4, 64, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.autocast("cuda", dtype=torch.float16):
        leaf = q.clone().requires_grad_()
        y, _ = rotate(leaf, None, positions, freqs)
        y.backward(gr)
    side.synchronize()
    assert y.dtype == torch.bfloat16
    check(y, q, positions, freqs, "interleaved")
    check(leaf.grad, gr, -positions, freqs, "interleaved")


def test_positions_changed_before_the_backward_pass_are_noticed():
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(4, device=DEV)
    x = torch.ones(4, 2, 64, device=DEV, requires_grad=True)
    y, _ = rotate(x, None, positions, freqs)
    positions.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_what_is_turned_in_place_is_noticed_by_a_graph_that_needs_it():
    freqs, _ = rotary_frequencies(64, device=DEV)
    x, w = torch.ones(4, 2, 64, device=DEV), torch.ones(4, 2, 64, device=DEV, requires_grad=True)
    y = (x * w).sum()
    rotate_(x, None, torch.arange(4, device=DEV), freqs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_captured_call_refuses_leaves_that_an_eager_graph_holds():
    """(Refused ahead of the first launch; the same leaves are taken once the eager graph is gone.)"""
    g = gen(10)
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(6, device=DEV)
    x, gr = randn(g, 6, 2, 64, dtype=torch.bfloat16).requires_grad_(), randn(g, 6, 2, 64, dtype=torch.bfloat16)
    eager, _ = rotate(x, None, positions, freqs)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="held by an eager graph"):
            rotate(x, None, positions, freqs)
        with torch.no_grad():
            rotate(x, None, positions, freqs)       # (without gradients nothing leads there)
    want = eager.detach().clone()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = rotate(x, None, positions, freqs)
        again, _ = rotate(x, None, positions, freqs)
        dx, = torch.autograd.grad((y, again), (x,), (gr, gr))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(again, want)
        back = rotate(gr, None, -positions, freqs)[0]
        assert torch.equal(dx, back + back)


def test_many_waves():
    """More waves than a grid's first dimension has threads in one workgroup, heads in several windows."""
    T, H, D = 20011, 9, 64
    g = gen(7)
    q = randn(g, T, H, D, dtype=torch.bfloat16)
    freqs, _ = rotary_frequencies(32, device=DEV)
    positions = torch.arange(T, device=DEV)
    check(rotate(q, None, positions, freqs, layout="half")[0], q, positions, freqs, "half")


def test_infinite_and_missing_values_stay_in_their_pairs():
    x = torch.ones(1, 2, 64, dtype=torch.float32, device=DEV)
    x[0, 0, 4] = float("nan")
    freqs, _ = rotary_frequencies(64, device=DEV)
    y = rotate(x, None, torch.tensor([3], device=DEV), freqs)[0].cpu()
    assert y[0, 0, 4:6].isnan().all() and y[0, 0].isnan().sum() == 2 and not y[0, 1].isnan().any()


def test_refusals_that_need_a_gpu():
    x = torch.zeros(4, 2, 64, device=DEV)
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(4, device=DEV)
    with pytest.raises(RuntimeError, match="freqs is on cpu"):
        rotate(x, None, positions, freqs.cpu())
    with pytest.raises(ValueError, match="share memory"):
        rotate_(x[:, :1].expand(4, 2, 64), None, positions, freqs)
    with pytest.raises(ValueError, match="share memory"):
        rotate_(x, x, positions, freqs)
    with pytest.raises(ValueError, match="dense rows"):
        rotate_(torch.zeros(4, 2, 128, device=DEV)[..., ::2], None, positions, freqs)
    with pytest.raises(RuntimeError, match="no gradient"):
        rotate_(x.clone().requires_grad_(), None, positions, freqs)


def test_the_gradient_drops_no_tangent_and_is_not_traced():
    """A backward pass of an eager graph under forward mode or a tracer; the same graph is taken without them."""
    import torch.autograd.forward_ad as fwad
    from torch.fx.experimental.proxy_tensor import make_fx

    g = gen(11)
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(5, device=DEV)
    q = randn(g, 5, 2, 64, dtype=torch.float32).requires_grad_()
    gr = randn(g, 5, 2, 64, dtype=torch.float32)
    y, _ = rotate(q, None, positions, freqs)

    def back(x):
        return torch.autograd.grad(y, (q,), x, retain_graph=True)[0]

    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        back(fwad.make_dual(gr, torch.ones_like(gr)))
    with fwad.dual_level():
        check(back(gr), gr, -positions, freqs, "interleaved")
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(back)(gr)
    check(back(gr), gr, -positions, freqs, "interleaved")


def test_transforms_are_refused():
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions, x = torch.arange(5, device=DEV), torch.ones(3, 5, 2, 64, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: rotate(q, None, positions, freqs)[0])(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda q: rotate(q, None, positions, freqs)[0].sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: rotate(q, None, positions, freqs)[0], (x,), (x,))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_an_output_wants_a_gradient_if_its_input_does(layout):
    g = gen(12)
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(5, device=DEV)
    q, k = randn(g, 5, 4, 64, dtype=torch.float32), randn(g, 5, 2, 64, dtype=torch.float32)
    want = rotate(q, k, positions, freqs, layout=layout)
    for wants in ((True, False), (False, True), (True, True)):
        x = [t.clone().requires_grad_(w) for t, w in zip((q, k), wants)]
        y = rotate(*x, positions, freqs, layout=layout)
        assert [t.requires_grad for t in y] == list(wants) and [t.is_leaf for t in y] == [not w for w in wants]
        assert all(torch.equal(a, b) for a, b in zip(y, want))
        gr = [randn(g, *t.shape, dtype=t.dtype).requires_grad_() for t in y]
        leaves, outs = [t for t in x if t.requires_grad], [t for t in y if t.requires_grad]
        back = torch.autograd.grad(outs, leaves, [r for r, t in zip(gr, y) if t.requires_grad], create_graph=True)
        for d, r in zip(back, [r for r, t in zip(gr, y) if t.requires_grad]):
            check(d, r, -positions, freqs, layout)
            v = randn(g, *d.shape, dtype=d.dtype)
            again, = torch.autograd.grad(d, (r,), v, retain_graph=True)
            check(again, v, positions, freqs, layout)


def test_rows_in_place_that_share_memory_are_found_whatever_their_strides():
    """Parts of a fused projection with a head in common, windows over one another; parts that only lie between each other
    are turned."""
    freqs, _ = rotary_frequencies(64, device=DEV)
    positions = torch.arange(5, device=DEV)
    fused = torch.zeros(5, 12, 64, device=DEV)
    flat = torch.zeros(5000, device=DEV)
    for q, k in ((fused[:, :8], fused[:, 7:10]), (fused[:, 7:], fused[:, :8]), (fused[:, ::2], fused[:, 4:5]),
                 (fused[:, :4], fused[:, :4]), (fused[:, :4], fused[:, :4, :]), (fused, fused),
                 (flat.as_strided((5, 4, 64), (256, 64, 1)), flat.as_strided((5, 2, 64), (300, 64, 1), 1270))):
        with pytest.raises(ValueError, match="xq and xk share memory"):
            rotate_(q, k, positions, freqs)
    for q in (flat.as_strided((5, 4, 64), (64, 64, 1)), flat.as_strided((5, 4, 64), (250, 64, 1)), flat.as_strided((5, 4, 64), (256, 60, 1)),
              fused[:, :1].expand(5, 4, 64)):
        with pytest.raises(ValueError, match="do not share memory"):
            rotate_(q, None, positions, freqs)
    g = gen(13)
    base = randn(g, 5, 12, 64, dtype=torch.float32)
    strided = randn(g, 5000, dtype=torch.float32)
    for q, k in ((base[:, :8], base[:, 8:]), (base[:, ::2], base[:, 1::2]), (base[:, 4:5], base[:, 5:]), (base[:, :0], base),
                 (strided.as_strided((5, 2, 64), (320, 64, 1)), strided.as_strided((5, 3, 64), (320, 64, 1), 128)),
                 (strided.as_strided((5, 4, 64), (64, 320, 1)), strided.as_strided((5, 2, 64), (128, 64, 1), 1600))):
        q0, k0 = q.clone(), k.clone()
        rotate_(q, k, positions, freqs)
        check(q, q0, positions, freqs, "interleaved")
        check(k, k0, positions, freqs, "interleaved")


def test_rows_in_place_that_share_memory_are_found_exactly():
    """Against the sets of elements, over views of any strides of one buffer."""
    import random

    rng = random.Random(5)
    freqs, _ = rotary_frequencies(2, device=DEV)
    buffer, numbers, met = torch.zeros(3000, device=DEV), torch.arange(3000), [0, 0]
    for _ in range(300):
        views = []
        T = rng.randint(1, 4)
        for _ in range(2):
            shape = (T, rng.randint(1, 4), 4)
            views.append((shape, (rng.choice([2, 4, 7, 16, 24, 100]), rng.choice([3, 4, 8, 16, 60]), 1), rng.randint(0, 120)))
        q, k = (buffer.as_strided(*v) for v in views)
        places = [numbers.as_strided(*v).flatten().tolist() for v in views]
        folds, meets = any(len(set(p)) < len(p) for p in places), bool(set(places[0]) & set(places[1]))
        met[0] += folds
        met[1] += meets and not folds
        at = torch.zeros(T, dtype=torch.int32, device=DEV)
        if folds or meets:
            with pytest.raises(ValueError, match="do not share memory" if folds else "xq and xk share memory"):
                rotate_(q, k, at, freqs)
        else:
            rotate_(q, k, at, freqs)
    assert met == [190, 33]     # (of each kind enough)
