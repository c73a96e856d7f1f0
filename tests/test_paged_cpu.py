"""Batches of sequences in HBM without a GPU: frequencies, refusals, the kernels' host side and its arithmetic."""

import ctypes
import math

import pytest
import torch

from dram_attention_amd import (append_kv_pages_, kv_pages, paged_decode_attention, rotary_frequencies, rotate,
                                rotate_)
from dram_attention_amd.llama import rope_frequencies


def freqs_of(n, *args, **more):
    return rotary_frequencies(n, *args, device="cpu", **more)


def test_frequencies_unscaled_and_llama3_are_the_models():
    for scaled in (False, True):
        freqs, factor = freqs_of(128, 500000.0, scaling={"type": "llama3"} if scaled else None)
        assert factor == 1.0 and freqs.dtype == torch.float64 and freqs.shape == (64,)
        # (the model's are formed in fp32: a power, a division and the blend)
        assert torch.allclose(freqs.float(), rope_frequencies(128, 500000.0, scaled), rtol=1e-5, atol=0)


def test_frequencies_by_their_formulas():
    plain, _ = freqs_of(8, 10000.0)
    assert torch.allclose(plain, torch.tensor([1.0, 0.1, 0.01, 0.001]).double(), rtol=1e-12)
    assert torch.equal(freqs_of(8, 10000.0, {"type": "linear", "factor": 4.0})[0], plain / 4)
    ntk, _ = freqs_of(8, 10000.0, {"type": "ntk", "factor": 16.0})
    assert math.isclose(ntk[0], 1.0) and math.isclose(ntk[3], plain[3] / 16)        # slowest by the factor
    yarn, factor = freqs_of(128, 10000.0, {"type": "yarn", "factor": 4.0, "original_length": 2048})
    base, _ = freqs_of(128, 10000.0)
    assert math.isclose(factor, 0.1 * math.log(4) + 1)
    turns = 2048 * base / (2 * math.pi)
    assert torch.allclose(yarn[turns > 40], base[turns > 40], rtol=1e-12)
    assert torch.allclose(yarn[turns < 0.8], base[turns < 0.8] / 4, rtol=1e-12)
    assert (yarn <= base).all() and (yarn >= base / 4 * (1 - 1e-12)).all() and (yarn[1:] < yarn[:-1]).all()
    assert freqs_of(128, 10000.0, {"type": "yarn", "factor": 4.0, "original_length": 2048, "attention_factor": 1.5})[1] == 1.5
    assert freqs_of(0)[0].numel() == 0


@pytest.mark.parametrize("n, theta, scaling, match", [
    (7, 1e4, None, "pairs"), (8, 1.0, None, "theta"), (8, 1e4, {"type": "linear"}, "factor"),
    (8, 1e4, {"type": "linear", "factor": -1}, "factor"), (2, 1e4, {"type": "ntk", "factor": 2}, "two pairs"),
    (8, 1e4, {"type": "yarn", "factor": 2}, "original_length"), (8, 1e4, {"type": "cubic"}, "unknown"),
    (8, 1e4, {"type": "linear", "factor": 2, "beta": 1}, "beta"),
    (8, 1e4, {"type": "llama3", "low_freq_factor": 4, "high_freq_factor": 1}, "high_freq_factor")])
def test_frequencies_refuse(n, theta, scaling, match):
    with pytest.raises(ValueError, match=match):
        freqs_of(n, theta, scaling)


def rotate_operands(**other):
    a = dict(xq=torch.zeros(2, 3, 4, 64), xk=torch.zeros(2, 3, 1, 64), positions=torch.arange(3),
             freqs=torch.zeros(32, dtype=torch.float64))
    a.update(other)
    return a


@pytest.mark.parametrize("other, kind, match", [
    ({}, RuntimeError, "GPU"),
    ({"xq": torch.zeros(3, 64)}, ValueError, "xq must be"),
    ({"xq": torch.zeros(2, 3, 4, 64, dtype=torch.float64)}, TypeError, "float32, float16 or bfloat16"),
    ({"xk": torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)}, TypeError, "xk is"),
    ({"xk": torch.zeros(2, 4, 1, 64)}, ValueError, "does not go with"),
    ({"positions": torch.arange(4)}, ValueError, "positions"),
    ({"positions": torch.zeros(3, 2, dtype=torch.int32)}, ValueError, "positions"),
    ({"positions": torch.zeros(3)}, TypeError, "int32 or int64"),
    ({"freqs": torch.zeros(32)}, TypeError, "float64"),
    ({"freqs": torch.zeros(33, dtype=torch.float64)}, ValueError, "channels"),
    ({"freqs": torch.zeros(64, dtype=torch.float64)[::2]}, ValueError, "contiguous"),
    ({"freqs": None}, TypeError, "freqs"),
    ({"freqs": torch.zeros(32, dtype=torch.float64, requires_grad=True)}, RuntimeError, "no gradient"),
    ({"layout": "both"}, ValueError, "layout"),
])
def test_rotate_refuses(other, kind, match):
    with pytest.raises(kind, match=match):
        rotate(**rotate_operands(**other))
    with pytest.raises(kind, match=match):
        rotate_(**rotate_operands(**other))


def test_rotate_refuses_lazy_negatives_and_sizes_that_32_bits_do_not_hold():
    x = torch.zeros(2, 3, 4, 64, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    with pytest.raises(ValueError, match="lazy"):
        rotate(**rotate_operands(xq=x))
    with pytest.raises(ValueError, match="too large"):
        rotate(**rotate_operands(xq=torch.zeros(1, 1, 1, 64).expand(2, 3, 2 ** 32 + 4, 64)))


def test_rotate_refuses_subclasses():
    class Kind(torch.Tensor):
        pass

    with pytest.raises(TypeError, match="plain"):
        rotate(**rotate_operands(xq=torch.zeros(2, 3, 4, 64).as_subclass(Kind)))


def test_rotate_refuses_forward_mode():
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        rotate(**rotate_operands())


def pages_on_cpu(dtype=torch.float32, **other):
    k, v = kv_pages(6, 16, 2, 64, dtype=dtype, device="cpu")
    a = dict(k_pages=k, v_pages=v, page_table=torch.zeros(3, 2, dtype=torch.int32))
    a.update(other)
    return a


def test_pool_layout():
    k, v = kv_pages(6, 16, 2, 64, device="cpu")
    assert k.shape == v.shape == (6, 16, 2, 64) and k.dtype == torch.bfloat16 and k.stride() == v.stride()
    assert k.stride() == (2 * 16 * 2 * 64, 128, 16 * 2 * 64, 1) and v.data_ptr() - k.data_ptr() == 128
    for bad in (dict(dtype=torch.float64), dict(dtype=torch.int8)):
        with pytest.raises(TypeError):
            kv_pages(6, 16, 2, 64, device="cpu", **bad)
    with pytest.raises(ValueError):
        kv_pages(6, 0, 2, 64, device="cpu")


X, I = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
APPEND = [
    ({}, RuntimeError, "GPU"),
    ({"xk": torch.zeros(3, 2, 32)}, ValueError, "as the pages are"),
    ({"xv": torch.zeros(3, 1, 64)}, ValueError, "as the pages are"),
    ({"xv": X.bfloat16()}, TypeError, "xv is"),
    ({"xk": X.half(), "xv": X.half()}, TypeError, "do not go with"),
    ({"positions": I[:2]}, ValueError, "positions"),
    ({"positions": X}, TypeError, "positions"),
    ({"sequences": I[:2]}, ValueError, "sequences"),
    ({"page_table": torch.zeros(4, 2, dtype=torch.int32)}, ValueError, "sequences="),
    ({"page_table": torch.zeros(3, 2)}, TypeError, "page_table"),
    ({"page_table": I}, ValueError, "page_table"),
    ({"v_pages": torch.zeros(6, 16, 2, 64)}, ValueError, "same strides"),
    ({"v_pages": torch.zeros(5, 16, 2, 64)}, ValueError, "must both be"),
    ({"xq": torch.zeros(2, 4, 64)}, ValueError, "xq"),
    ({"xq": torch.zeros(3, 4, 64, dtype=torch.half)}, TypeError, "xq is"),
    ({"k_scale": torch.ones(2)}, ValueError, "8-bit"),
    ({"freqs": torch.zeros(40, dtype=torch.float64)}, ValueError, "channels"),
    ({"layout": None}, ValueError, "layout"),
    ({"xk": X.clone().requires_grad_()}, RuntimeError, "no gradient"),
]


@pytest.mark.parametrize("other, kind, match", APPEND)
def test_append_refuses(other, kind, match):
    a = pages_on_cpu()
    a.update(xk=X, xv=X, positions=I)
    a.update(other)
    with pytest.raises(kind, match=match):
        append_kv_pages_(**a)


def test_eight_bit_pages_refuse():
    a = pages_on_cpu(torch.float8_e4m3fn)
    with pytest.raises(TypeError, match="16-bit"):
        append_kv_pages_(X, X, positions=I, **a)
    with pytest.raises(TypeError, match="16-bit"):
        paged_decode_attention(X, lengths=I, **a)
    h = X.bfloat16()
    for scale, kind in ((torch.ones(3), ValueError), (torch.ones(2).double(), TypeError), (torch.ones(4)[::2], ValueError)):
        with pytest.raises(kind, match="k_scale"):
            append_kv_pages_(h, h, positions=I, k_scale=scale, **a)
        with pytest.raises(kind, match="v_scale"):
            paged_decode_attention(h, lengths=I, v_scale=scale, **a)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_decode_attention(h, lengths=I, k_scale=torch.ones(2), v_scale=torch.ones(2), **a)


@pytest.mark.parametrize("other, kind, match", [
    ({}, RuntimeError, "GPU"),
    ({"xq": torch.zeros(3, 3, 64)}, ValueError, "multiple of 2 heads"),
    ({"xq": torch.zeros(3, 0, 64)}, ValueError, "multiple of 2 heads"),
    ({"xq": torch.zeros(2, 4, 64)}, ValueError, "3 sequences"),
    ({"xq": torch.zeros(3, 1, 4, 64)}, ValueError, "xq"),
    ({"xq": torch.zeros(3, 4, 64, dtype=torch.half)}, TypeError, "do not go with"),
    ({"lengths": I[:2]}, ValueError, "lengths"),
    ({"lengths": X}, TypeError, "lengths"),
    ({"scale": math.inf}, ValueError, "finite"),
    ({"scale": "1"}, TypeError, None),
    ({"out": torch.zeros(3, 4, 32)}, ValueError, "out"),
    ({"out": torch.zeros(3, 4, 64, dtype=torch.half)}, ValueError, "out"),
    ({"lse": torch.zeros(3, 2)}, ValueError, "lse"),
    ({"lse": torch.zeros(3, 4, dtype=torch.half)}, ValueError, "lse"),
    ({"v_scale": torch.ones(2)}, ValueError, "8-bit"),
    ({"xq": torch.zeros(3, 4, 64).requires_grad_()}, RuntimeError, "no gradient"),
])
def test_attention_refuses(other, kind, match):
    a = pages_on_cpu()
    a.update(xq=torch.zeros(3, 4, 64), lengths=I)
    a.update(other)
    with pytest.raises(kind, match=match):
        paged_decode_attention(**a)


class RotateArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "q_out", "k_out", "freqs", "positions")] + [
        ("strides", ctypes.c_int64 * 14), ("batch", ctypes.c_int64), ("tokens", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("n_q_heads", "n_k_heads", "head_dim", "rotary_dim", "layout", "inverse", "dtype",
                                      "position_type")] + [("factor", ctypes.c_float), ("reserved", ctypes.c_int32)]


class AppendArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "q_out", "k_pages", "v_pages", "freqs", "page_table",
                                               "positions", "sequences", "k_scale", "v_scale")] + [
        ("strides", ctypes.c_int64 * 11), ("table_stride", ctypes.c_int64), ("n_tokens", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("n_pages", "page_size", "n_sequences", "pages_per_sequence", "n_q_heads",
                                      "n_kv_heads", "head_dim", "rotary_dim", "layout", "dtype", "page_dtype",
                                      "table_type", "position_type", "sequence_type")] + [
        ("factor", ctypes.c_float), ("reserved", ctypes.c_int32)]


class AttentionArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k_pages", "v_pages", "page_table", "lengths", "k_scale", "v_scale",
                                               "out", "lse", "workspace")] + [
        ("q_strides", ctypes.c_int64 * 2), ("page_strides", ctypes.c_int64 * 3), ("table_stride", ctypes.c_int64),
        ("workspace_bytes", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("n_pages", "page_size", "n_sequences", "pages_per_sequence", "n_q_heads",
                                      "n_kv_heads", "head_dim", "dtype", "page_dtype", "table_type", "length_type")] + [
        ("scale", ctypes.c_float)]


def call(lib, name, a):
    return getattr(lib, name)(bytes(a), ctypes.sizeof(a), None)


def test_c_entry_points_check_before_any_launch(lib):
    for name in ("da_rotate", "da_paged_append", "da_paged_attention"):
        assert getattr(lib, name)(None, 0, None) == -1
        assert getattr(lib, name)(b"abc", 3, None) == -1 and b"argument block" in lib.da_last_error_string()
    rot = dict(batch=1, tokens=4, n_q_heads=2, n_k_heads=1, head_dim=64, rotary_dim=64, dtype=2, factor=1.0)
    for bad, code in (({}, -1), ({"dtype": 3}, -1), ({"rotary_dim": 63}, -1), ({"rotary_dim": 66}, -1), ({"layout": 2}, -1),
                      ({"tokens": -1}, -1), ({"position_type": 5}, -1), ({"head_dim": 1024, "rotary_dim": 1024, "freqs": 16}, -2),
                      ({"tokens": 1 << 40, "q": 16, "k": 16, "q_out": 16, "k_out": 16, "freqs": 16, "positions": 16}, -2),
                      ({"tokens": (1 << 31) - 300, "head_dim": 512, "rotary_dim": 512, "q": 16, "k": 16, "q_out": 16, "k_out": 16,
                        "freqs": 16, "positions": 16}, -2),
                      ({"tokens": 0, "freqs": 16}, 0)):
        assert call(lib, "da_rotate", RotateArgs(**{**rot, **bad})) == code, bad
    app = dict(n_pages=4, page_size=16, n_sequences=2, pages_per_sequence=3, n_kv_heads=2, head_dim=64, dtype=2,
               page_dtype=2, n_tokens=2, k=16, v=16, k_pages=16, v_pages=16, page_table=16, positions=16)
    for bad, code in (({"k": None}, -1), ({"n_tokens": 3}, -1), ({"page_dtype": 1}, -1), ({"dtype": 0, "page_dtype": 3}, -2),
                      ({"page_size": 0}, -1), ({"n_q_heads": 2}, -1), ({"k_scale": 16}, -1), ({"sequence_type": 2}, -1),
                      ({"page_size": 1 << 30}, -2), ({"rotary_dim": 64}, -1), ({"n_tokens": 0}, 0)):
        assert call(lib, "da_paged_append", AppendArgs(**{**app, **bad})) == code, bad
    att = dict(n_pages=4, page_size=16, n_sequences=2, pages_per_sequence=300, n_q_heads=4, n_kv_heads=2, head_dim=64,
               dtype=2, page_dtype=2, q=16, k_pages=16, v_pages=16, page_table=16, lengths=16, out=16, scale=1.0)
    for bad, code in (({"q": None}, -1), ({"head_dim": 80}, -2), ({"n_q_heads": 3}, -1), ({"page_dtype": 0}, -1),
                      ({"dtype": 0, "page_dtype": 3}, -2), ({"v_scale": 16}, -1), ({"q": 8}, -1), ({}, -1),
                      ({"workspace": 16, "workspace_bytes": 64}, -1), ({"page_size": 1 << 28}, -2), ({"length_type": 7}, -1),
                      ({"n_q_heads": 8192}, -2), ({"n_sequences": 1 << 23}, -2),
                      ({"q_strides": (ctypes.c_int64 * 2)(4, 64)}, -1), ({"n_sequences": 0}, 0)):
        assert call(lib, "da_paged_attention", AttentionArgs(**{**att, **bad})) == code, bad
    need = lib.da_paged_attention_workspace_bytes(bytes(AttentionArgs(**att)), ctypes.sizeof(AttentionArgs))
    assert need > 0
    assert lib.da_paged_attention_workspace_bytes(bytes(AttentionArgs(**{**att, "head_dim": 80})),
                                                  ctypes.sizeof(AttentionArgs)) == 0
    # (a batch that one workgroup a sequence finishes needs none)
    assert lib.da_paged_attention_workspace_bytes(bytes(AttentionArgs(**{**att, "pages_per_sequence": 1})),
                                                  ctypes.sizeof(AttentionArgs)) == 0


def test_division_by_multiplication():
    """The quotient that the kernels form for a token's page (csrc/paged_math.hpp), in its own integers."""
    import random

    rng = random.Random(0)
    for d in [1, 2, 3, 5, 7, 16, 24, 100, 641, 65535, 65536, 65537, (1 << 30) - 1, 1 << 30] + [rng.randint(1, 1 << 30) for _ in range(300)]:
        l = (d - 1).bit_length()
        m = ((1 << l) - d << 32) // d + 1
        assert m < 1 << 32
        for n in [0, 1, d - 1, d, d + 1, (1 << 31) - 1, (1 << 31) - d if d < 1 << 31 else 0] + [rng.randrange(1 << 31) for _ in range(50)]:
            assert ((m * n >> 32) + n) >> l == n // d, (n, d)


def calls_of_a_batch():
    """Every call as it would be made, on the CPU, where all that is wrong with it is the device."""
    x = torch.zeros(3, 4, 64)
    return {
        "rotate": lambda x=x: rotate(**rotate_operands(xq=x[None].expand(2, 3, 4, 64))),
        "rotate_": lambda x=x: rotate_(x, None, torch.arange(3), torch.zeros(32, dtype=torch.float64)),
        "append_kv_pages_": lambda x=X: append_kv_pages_(x, X, positions=I, **pages_on_cpu()),
        "paged_decode_attention": lambda x=x: paged_decode_attention(x, lengths=I, **pages_on_cpu()),
    }


@pytest.mark.parametrize("name", list(calls_of_a_batch()))
def test_no_call_drops_a_tangent(name):
    """Under torch.no_grad too, which leaves forward mode on."""
    import torch.autograd.forward_ad as fwad

    call = calls_of_a_batch()[name]
    with fwad.dual_level():
        x = X if name == "append_kv_pages_" else torch.zeros(3, 4, 64)
        dual = fwad.make_dual(x.clone(), torch.ones_like(x))
        for operand in (dual, x):
            with pytest.raises(RuntimeError, match=f"^{name} has no forward-mode"):
                call(operand)
            with torch.no_grad(), pytest.raises(RuntimeError, match=f"^{name} has no forward-mode"):
                call(operand)
    with pytest.raises(RuntimeError, match="GPU"):
        call()


@pytest.mark.parametrize("name", list(calls_of_a_batch()))
def test_no_call_is_traced(name):
    """What a tracer would keep of a call is its output's allocation; modes that only watch are no tracers."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    call = calls_of_a_batch()[name]
    x = X if name == "append_kv_pages_" else torch.zeros(3, 4, 64)

    def traced(x):
        with pytest.raises(RuntimeError, match=f"^{name} cannot be traced"):
            call(x)
        return x + 1

    make_fx(traced)(x)
    make_fx(traced, pre_dispatch=True)(x)
    torch.jit.trace(traced, x, check_trace=False)
    with FlopCounterMode(display=False), pytest.raises(RuntimeError, match="GPU"):
        call(x)
    with torch.device("cpu"), pytest.raises(RuntimeError, match="GPU"):
        call(x)


def append_into(k, v):
    d, heads = k.shape[-1], k.shape[2]
    x = torch.zeros(3, heads, d, dtype=k.dtype)
    append_kv_pages_(x, x, k, v, torch.zeros(3, 2, dtype=torch.int32), I)


def test_append_refuses_pools_that_share_memory():
    """Keys and values would race for the same bytes; pools that only lie between each other are taken."""
    base = torch.zeros(13, 32, 4, 64)
    k, v = kv_pages(6, 16, 2, 64, dtype=torch.float32, device="cpu")
    for a, b in ((k, k), (k, k[:]), (v, v.view(v.shape)), (base[:6], base[5:11]), (base[:6], base[:6]),
                 (base[:6, :16], base[:6, 15:31]), (base[:6, :, :2], base[:6, :, 1:3]),
                 (base[:6, :, :, :32], base[:6, :, :, 16:48]), (base[::2], base[::2])):
        with pytest.raises(ValueError, match="share memory"):
            append_into(a, b)
    for a, b in ((k, v), (v, k), (base[:6], base[6:12]), (base[6:12], base[:6]), (base[:12:2], base[1:13:2]),
                 (base[:6, :16], base[:6, 16:]), (base[:6, ::2], base[:6, 1::2]), (base[:6, :, ::2], base[:6, :, 1::2]),
                 (base[:6, :, :, :32], base[:6, :, :, 32:]), (base[:0], base[:0]), (base[:6], base.clone()[:6])):
        with pytest.raises(RuntimeError, match="GPU"):
            append_into(a, b)


def test_pools_that_share_memory_are_found_exactly():
    """Against the sets of elements, over views of any strides of one buffer."""
    import random

    rng = random.Random(3)
    buffer = torch.zeros(4000, dtype=torch.bfloat16)
    met = [0, 0]
    for _ in range(400):
        sizes = [rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 3), rng.choice([2, 3, 8])]
        strides = [rng.choice([1, 3, 8, 12, 16, 40, 64, 200]) for _ in range(3)] + [1]
        offsets = [rng.randint(0, 200), rng.randint(0, 200)]
        pools = [buffer.as_strided(sizes, strides, at) for at in offsets]
        sets = [set(torch.arange(4000).as_strided(sizes, strides, at).flatten().tolist()) for at in offsets]
        folds, shared = len(sets[0]) < math.prod(sizes), bool(sets[0] & sets[1])
        met[0] += folds
        met[1] += shared and not folds
        with pytest.raises(ValueError if folds or shared else RuntimeError,
                           match="pages must not share" if folds else "k_pages and v_pages share" if shared else "GPU"):
            append_into(*pools)
    assert all(40 < n < 300 for n in met)


def test_attention_refuses_to_write_over_what_it_reads():
    buffer = torch.zeros(1 << 16)
    k, v = buffer[: 6 * 16 * 2 * 64 * 2].view(6, 2, 16, 2, 64).permute(0, 2, 1, 3, 4).unbind(3)
    free = buffer[6 * 16 * 2 * 64 * 2:]
    q, lse, out = free[:768].view(3, 4, 64), free[768:780].view(3, 4), free[1024:1792].view(3, 4, 64)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)

    def call(**more):
        paged_decode_attention(**{**dict(xq=q, k_pages=k, v_pages=v, page_table=table, lengths=lengths), **more})

    as_ints = free[768:780].view(torch.int32)
    for more, what in (({"out": free[16:784].view(3, 4, 64)}, "out"), ({"out": buffer[64:832].view(3, 4, 64)}, "out"),
                       ({"out": out, "lse": free[1790:1802].view(3, 4)}, "out"), ({"lse": free[767:779].view(3, 4)}, "lse"),
                       ({"lse": lse, "lengths": as_ints[9:12]}, "lse"), ({"lse": lse, "page_table": as_ints[:6].view(3, 2)}, "lse"),
                       ({"lse": buffer[:12].view(3, 4)}, "lse"),
                       # (the same rows in another order)
                       ({"xq": q.flip(0), "out": out}, None), ({"xq": free[:768].view(3, 64, 4).transpose(1, 2), "out": q}, "out"),
                       ({"out": q}, None), ({"out": q[:]}, None), ({"out": out, "lse": lse}, None),
                       ({"xq": free[: 2 * 768].view(3, 8, 64)[:, ::2], "out": free[2 * 768: 3 * 768].view(3, 4, 64)}, None)):
        with pytest.raises(ValueError if what else RuntimeError, match=f"^{what} shares memory" if what else "GPU"):
            call(**more)


def test_memory_that_rows_reach_into_is_found_exactly():
    """Against the sets of elements: logarithms in one buffer with queries of any strides, many with gaps that hold them."""
    import random

    rng = random.Random(4)
    k, v = kv_pages(6, 16, 1, 2, dtype=torch.float32, device="cpu")
    table, lengths, buffer, met = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4000), 0
    for _ in range(400):
        strides, at, lse_at = [rng.choice([2, 5, 8, 16, 40, 200]) for _ in range(2)] + [1], rng.randint(0, 300), rng.randint(0, 400)
        heads = rng.randint(1, 5)
        rows = set(torch.arange(4000).as_strided((3, heads, 2), strides, at).flatten().tolist())
        shared = bool(rows & set(range(lse_at, lse_at + 3 * heads)))
        met += shared
        with pytest.raises(ValueError if shared else RuntimeError, match="lse shares memory" if shared else "GPU"):
            paged_decode_attention(buffer.as_strided((3, heads, 2), strides, at), k, v, table, lengths,
                                   lse=buffer[lse_at: lse_at + 3 * heads].view(3, heads))
    assert 40 < met < 360       # (both kinds)


@pytest.mark.parametrize("scale, fits", [(1e39, False), (-1e39, False), (3e38, False), (math.nan, False), (2.3e38, True),
                                         (1e-60, True), (0.0, True), (-2.0, True)])
def test_scales_that_fp32_does_not_hold_are_refused(scale, fits):
    a = pages_on_cpu()
    with pytest.raises(RuntimeError if fits else ValueError, match="GPU" if fits else "scale must be finite"):
        paged_decode_attention(torch.zeros(3, 4, 64), lengths=I, scale=scale, **a)


def test_scales_and_logarithms_that_want_gradients_are_refused():
    a, h = pages_on_cpu(torch.float8_e4m3fn), X.bfloat16()
    for name in ("k_scale", "v_scale"):
        scale = torch.ones(2, requires_grad=True)
        for call in (lambda: append_kv_pages_(h, h, positions=I, **{name: scale}, **a),
                     lambda: paged_decode_attention(h, lengths=I, **{name: scale}, **a)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
                call()
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_decode_attention(h, lengths=I, lse=torch.zeros(3, 2, requires_grad=True), **a)


def test_a_scaling_without_a_type_is_refused():
    with pytest.raises(ValueError, match="factor"):
        freqs_of(8, 1e4, {"factor": 2.0})
    given = {"type": "linear", "factor": 2.0}
    freqs_of(8, 1e4, given)
    assert given == {"type": "linear", "factor": 2.0}
