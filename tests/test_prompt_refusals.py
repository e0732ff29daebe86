"""What the operators around a prompt refuse, on the host: nothing is launched."""
import ctypes
import math
import os

import pytest
import torch

import pypto_amd
from pypto_amd import _C

BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pypto_amd", "libpypto_amd_sfa.so")


def refused(kind, text, op, args, **kw):
    with pytest.raises(kind, match=text):
        op(*args, **kw)


def changed(args, at, value):
    out = list(args)
    out[at] = value
    return out


# ---------------------------------------------------------------- rotary positions

def tables():
    return [torch.zeros(5, dtype=torch.int64), pypto_amd.rotary_frequencies(64), torch.zeros(5, 64, dtype=BF), torch.zeros(5, 64, dtype=BF)]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, torch.zeros(5), TypeError, "positions"), (0, [1, 2], TypeError, "not currently supported"), (0, torch.zeros(5, 1, dtype=torch.int64), ValueError, "1-dim"),
    (0, torch.zeros(10, dtype=torch.int64)[::2], RuntimeError, "contiguous"),
    (1, torch.zeros(32), TypeError, "frequencies"), (1, torch.zeros(6, dtype=torch.float64), ValueError, "multiple of 4"),
    (1, torch.zeros(132, dtype=torch.float64), ValueError, "up to 128"), (1, torch.zeros(0, dtype=torch.float64), ValueError, "multiple"),
    (2, torch.zeros(5, 64, dtype=torch.float64), TypeError, "cos_out"), (3, torch.zeros(5, 64), TypeError, "sin_out"),
    (2, torch.zeros(4, 64, dtype=BF), ValueError, "cos_out"), (3, torch.zeros(5, 32, dtype=BF), ValueError, "sin_out")])
def test_tables(at, value, kind, text):
    refused(kind, text, pypto_amd.rotary_tables, changed(tables(), at, value))


def test_tables_on_the_host_and_in_one_memory():
    refused(RuntimeError, "GPU", pypto_amd.rotary_tables, tables())
    args = tables()
    refused(ValueError, "overlap", pypto_amd.rotary_tables, changed(args, 3, args[2]))


def rotation():
    return [torch.zeros(5, 4, 80, dtype=BF), torch.zeros(5, 1, 64, dtype=BF), torch.zeros(5, dtype=torch.int64), pypto_amd.rotary_frequencies(64),
            torch.zeros(5, 4, 80, dtype=BF), torch.zeros(5, 1, 64, dtype=BF)]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, torch.zeros(5, 4, 80, dtype=torch.int8), TypeError, "query"), (1, torch.zeros(5, 1, 64), TypeError, "key"), (1, None, ValueError, "come together"),
    (5, None, ValueError, "come together"), (0, torch.zeros(4, 4, 80, dtype=BF), ValueError, "query"), (4, torch.zeros(5, 4, 64, dtype=BF), ValueError, "query"),
    (0, torch.zeros(5, 80, 4, dtype=BF).transpose(1, 2), RuntimeError, "last dimension"), (3, torch.zeros(12, dtype=torch.float64), ValueError, "multiple of 8"),
    (5, torch.zeros(1, 1, 64, dtype=BF).expand(5, 1, 64), ValueError, "share memory"), (2, torch.zeros(6, dtype=torch.int64), ValueError, "query")])
def test_rotation(at, value, kind, text):
    refused(kind, text, pypto_amd.rotary_embedding, changed(rotation(), at, value))


def test_rotation_s_scalars_overlaps_and_device():
    args = rotation()
    refused(ValueError, "layout", pypto_amd.rotary_embedding, args, layout="halves")
    refused(ValueError, "layout", pypto_amd.rotary_embedding, args, layout=1)
    refused(ValueError, "do not fit", pypto_amd.rotary_embedding, args, query_offset=17)
    refused(ValueError, "do not fit", pypto_amd.rotary_embedding, args, key_offset=-1)
    refused(RuntimeError, "GPU", pypto_amd.rotary_embedding, args, query_offset=16)
    both = torch.zeros(6, 4, 80, dtype=BF)
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, changed(changed(args, 0, both[:5]), 4, both[1:]))
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, changed(args, 5, args[4][:, :1, :64]))
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, changed(args, 1, args[4][:, :1, :64]))
    wide = torch.zeros(5, 5, 80, dtype=BF)                  # columns of one tensor, queries and then the key, do not meet
    refused(RuntimeError, "GPU", pypto_amd.rotary_embedding, changed(changed(args, 4, wide[:, :4]), 5, wide[:, 4:, :64]))
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, changed(changed(args, 4, wide[:, :4]), 5, wide[:, 3:4, :64]))


def test_rotation_of_one_tensor_as_queries_and_keys():
    """In place or not, no memory may be queries and keys at once; channels of the same heads that do not meet may."""
    pos, freq = torch.zeros(5, dtype=torch.int64), pypto_amd.rotary_frequencies(64)
    x = torch.zeros(5, 4, 160, dtype=BF)
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, [x, x, pos, freq, x, x])
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, [x[:, :3], x[:, 2:], pos, freq, x[:, :3], x[:, 2:]])
    refused(ValueError, "overlap", pypto_amd.rotary_embedding, [x[..., :96], x[..., 64:], pos, freq, x[..., :96], x[..., 64:]])
    q, k = x[..., :80], x[..., 80:]
    refused(RuntimeError, "GPU", pypto_amd.rotary_embedding, [q, k, pos, freq, q, k])
    refused(RuntimeError, "GPU", pypto_amd.rotary_embedding, [x[:, :3], x[:, 3:], pos, freq, x[:, :3], x[:, 3:]])
    odd = torch.zeros(1600, dtype=BF).as_strided((5, 3, 80), (200, 160, 1))          # heads run into the next row's
    other = torch.zeros(1600, dtype=BF)
    refused(ValueError, "overlap|share", pypto_amd.rotary_embedding,
            [odd, other.as_strided((5, 3, 80), (200, 160, 1)), pos, freq, odd, odd[:, :, :80]])


def test_frequencies():
    plain = pypto_amd.rotary_frequencies(64)
    assert plain.dtype == torch.float64 and float(plain[0]) == 1.0 and float(plain[16]) == pytest.approx(0.01, rel=1e-14)
    long = pypto_amd.rotary_frequencies(64, scaling=pypto_amd.RotaryScaling(factor=40.0))
    assert torch.equal(long[:10], plain[:10]) and torch.allclose(long[24:], plain[24:] / 40, rtol=1e-14) and bool((long <= plain).all())
    assert bool((long.diff() < 0).all())
    assert torch.equal(pypto_amd.rotary_frequencies(64, scaling=pypto_amd.RotaryScaling()), plain)
    assert pypto_amd.rotary_magnitude(1.0) == 1.0 and pypto_amd.rotary_magnitude(40.0) == pytest.approx(0.1 * math.log(40) + 1)
    for bad in (dict(dim=63), dict(dim=0), dict(dim=64, theta=1.0), dict(dim=64, scaling=pypto_amd.RotaryScaling(factor=-2.0))):
        with pytest.raises(ValueError):
            pypto_amd.rotary_frequencies(**bad)


# ---------------------------------------------------------------- the latent cache

def write():
    return [torch.zeros(3, 512, dtype=BF), torch.zeros(3, 64, dtype=BF), torch.zeros(3, dtype=torch.int64), torch.zeros(256, 512, dtype=torch.int8),
            torch.zeros(256, 64, dtype=BF), torch.zeros(256, 4), torch.zeros(3, 512, dtype=BF)]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, torch.zeros(3, 512, dtype=torch.int8), TypeError, "latent"), (0, torch.zeros(3, 500, dtype=BF), ValueError, "latent"), (1, torch.zeros(3, 64), TypeError, "key_rope"),
    (1, torch.zeros(4, 64, dtype=BF), ValueError, "key_rope"), (2, torch.zeros(3, dtype=torch.int32), TypeError, "cache_index"), (2, torch.zeros(4, dtype=torch.int64), ValueError, "cache_index"),
    (3, torch.zeros(256, 512, dtype=BF), TypeError, "kv_cache"), (3, torch.zeros(256, 656, dtype=torch.int8), ValueError, "kv_cache"), (4, torch.zeros(255, 64, dtype=BF), ValueError, "kr_cache"),
    (5, torch.zeros(256, 4, dtype=HALF), TypeError, "k_scale_cache"), (5, torch.zeros(256, 8)[:, :4], RuntimeError, "contiguous"), (6, torch.zeros(3, 512), TypeError, "latent_out"),
    (6, torch.zeros(1, 512, dtype=BF).expand(3, 512), ValueError, "share memory"), (0, torch.zeros(512, 3, dtype=BF).T, RuntimeError, "last dimension")])
def test_write(at, value, kind, text):
    refused(kind, text, pypto_amd.latent_cache_write, changed(write(), at, value))


def test_write_s_overlaps_and_device():
    args = write()
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_write, args)
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_write, changed(args, 6, args[0]))
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_write_packed, args[:3] + [torch.zeros(256, 656, dtype=torch.int8)])
    refused(ValueError, "656", pypto_amd.latent_cache_write_packed, args[:3] + [torch.zeros(256, 512, dtype=torch.int8)])
    both = torch.zeros(4, 512, dtype=BF)
    refused(ValueError, "overlap", pypto_amd.latent_cache_write, changed(changed(args, 0, both[:3]), 6, both[1:]))
    inside = args[3].view(BF)[:6].reshape(3, 512)
    refused(ValueError, "overlap", pypto_amd.latent_cache_write, changed(args, 0, inside))


def read():
    return [torch.zeros(256, 512, dtype=torch.int8), torch.zeros(256, 64, dtype=BF), torch.zeros(256, 4), torch.zeros(2, 3, dtype=torch.int32),
            torch.zeros(3, dtype=torch.int32), torch.zeros(9, 512, dtype=BF), torch.zeros(9, 64, dtype=BF), 128]


@pytest.mark.parametrize("at,value,kind,text", [
    (3, torch.zeros(2, 3, dtype=torch.int64), TypeError, "block_table"), (3, torch.zeros(3, dtype=torch.int32), ValueError, "block_table"), (4, torch.zeros(2, dtype=torch.int32), ValueError, "cu_seqlens"),
    (4, torch.zeros(3, dtype=torch.int64), TypeError, "cu_seqlens"), (5, torch.zeros(9, 512), TypeError, "latent_out"), (6, torch.zeros(8, 64, dtype=BF), ValueError, "key_rope_out"),
    (6, torch.zeros(1, 64, dtype=BF).expand(9, 64), ValueError, "share memory"), (0, torch.zeros(256, 512), TypeError, "kv_cache")])
def test_read(at, value, kind, text):
    refused(kind, text, pypto_amd.latent_cache_read, changed(read(), at, value))


def test_read_s_first_positions_and_device():
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_read, read())
    refused(ValueError, "first", pypto_amd.latent_cache_read, read(), first=torch.zeros(3, dtype=torch.int32))
    refused(TypeError, "first", pypto_amd.latent_cache_read, read(), first=torch.zeros(2, dtype=torch.int64))
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_read_packed, [torch.zeros(256, 656, dtype=torch.int8)] + read()[3:], first=torch.zeros(2, dtype=torch.int32))


def test_write_with_the_prolog_s_steps_refuses_what_the_other_does():
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_write, write(), prolog_steps=True)
    refused(TypeError, "cache_index", pypto_amd.latent_cache_write, changed(write(), 2, torch.zeros(3, dtype=torch.int32)), prolog_steps=True)
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_write_packed, write()[:3] + [torch.zeros(256, 656, dtype=torch.int8)], prolog_steps=1)


# ---------------------------------------------------------------- prompt attention

def attention():
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype)  # noqa: E731
    return [z(6, 4, 128), z(9, 2, 128), z(9, 2, 128), torch.tensor([0, 6], dtype=torch.int32), torch.tensor([0, 9], dtype=torch.int32), z(6, 4, 128), 0.1]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, torch.zeros(6, 4, 128), TypeError, "query"), (1, torch.zeros(9, 2, 128, dtype=HALF), TypeError, "key"), (0, torch.zeros(6, 512, dtype=BF), ValueError, "query"),
    (1, torch.zeros(9, 3, 128, dtype=BF), ValueError, "key"), (2, torch.zeros(8, 2, 128, dtype=BF), ValueError, "key"), (3, torch.tensor([0, 6]), TypeError, "cu_seqlens_q"),
    (4, torch.tensor([0, 3, 9], dtype=torch.int32), ValueError, "cu_seqlens"), (5, torch.zeros(6, 4, 64, dtype=BF), ValueError, "attention_out"),
    (5, torch.zeros(1, 4, 128, dtype=BF).expand(6, 4, 128), ValueError, "share memory"), (6, math.nan, ValueError, "finite"), (6, math.inf, ValueError, "finite")])
def test_attention(at, value, kind, text):
    refused(kind, text, pypto_amd.prompt_attention, changed(attention(), at, value))


def test_attention_s_heads_parts_overlaps_and_device():
    args = attention()
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype)  # noqa: E731
    op = pypto_amd.prompt_attention
    refused(RuntimeError, "GPU", op, args)
    refused(RuntimeError, "GPU", op, args, query_rope=z(6, 4, 64), key_rope=z(9, 64), softmax_lse=z(6, 4, dtype=F32), causal=False)
    refused(ValueError, "come together", op, args, query_rope=z(6, 4, 64))
    refused(ValueError, "query_rope", op, args, query_rope=z(6, 2, 64), key_rope=z(9, 64))
    refused(ValueError, "key_rope", op, args, query_rope=z(6, 4, 64), key_rope=z(9, 4, 64))
    refused(TypeError, "softmax_lse", op, args, softmax_lse=z(6, 4))
    refused(ValueError, "softmax_lse", op, args, softmax_lse=z(4, 6, dtype=F32))
    refused(ValueError, "overlap", op, changed(args, 5, args[0]))
    three = changed(changed(args, 1, z(9, 3, 128)), 2, z(9, 3, 128))
    refused(ValueError, "multiple", op, three)
    for d in (32, 96, 192, 256):
        wide = [z(6, 4, d), z(9, 2, d), z(9, 2, d), args[3], args[4], z(6, 4, d), 0.1]
        refused(ValueError, "not supported", op, wide)
    narrow = [z(6, 4, 64), z(9, 2, 64), z(9, 2, 64), args[3], args[4], z(6, 4, 64), 0.1]
    refused(ValueError, "128", op, narrow, query_rope=z(6, 4, 64), key_rope=z(9, 64))


def items_of(lens_q, lens_k, group, plan):
    """(row tile, piece) pairs of a key head, as the kernel counts them."""
    n = 0
    for q, k in zip(lens_q, lens_k):
        pieces = min(max(-(-k // plan["split_keys"]), 1), plan["key_splits"])
        n += -(-q * group // plan["rows_per_workgroup"]) * pieces
    return n


@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 16), (64, 8), (128, 128), (56, 8), (128, 1)])
def test_plans_hold_every_division_of_the_rows_over_sequences(heads, kv):
    """However the rows and keys are dealt out to the sequences: a launch that divides no keys has a workgroup for every row tile, one that
    does has no more pieces than its workspace holds, and workgroups for all or for four rounds."""
    g = torch.Generator().manual_seed(heads)
    rnd = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    for _ in range(300):
        b = rnd(1, 40)
        most_q, most_k = rnd(1, 12) ** rnd(1, 3), rnd(1, 20) ** rnd(1, 4)
        lens_q, lens_k = [rnd(0, most_q) for _ in range(b)], [rnd(0, most_k) for _ in range(b)]
        if rnd(0, 3) == 0:
            lens_k[rnd(0, b - 1)] = 100000
        if rnd(0, 3) == 0:
            lens_q[rnd(0, b - 1)] = 3000
        plan = _C.prompt_attention_plan(b, sum(lens_q), sum(lens_k), heads, kv, 128, True, rnd(0, 1) == 1)
        items = items_of(lens_q, lens_k, heads // kv, plan) * kv
        assert plan["workgroups"] % 8 == 0 and plan["workgroups"] >= (items if plan["key_splits"] == 1 else min(items, 1024)), (lens_q, lens_k, plan)
        assert 1 <= plan["key_splits"] <= 128 and plan["split_keys"] % 64 == 0
        need = sum(lens_q) * heads * plan["key_splits"] * (128 + 2) * 4 if plan["key_splits"] > 1 else 0
        assert plan["workspace_bytes"] == need <= 260 << 20, plan


def test_large_calls_are_not_divided_and_small_ones_are():
    assert _C.prompt_attention_plan(1, 4096, 4096, 128, 128, 128, True, True)["key_splits"] == 1
    assert _C.prompt_attention_plan(1, 1, 65536, 16, 1, 128, False, True)["key_splits"] > 16


# ---------------------------------------------------------------- the C entries

class Attention(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("query", "key", "value", "query_rope", "key_rope", "cu_seqlens_q", "cu_seqlens_k", "out", "lse", "workspace")] + \
               [("workspace_bytes", ctypes.c_size_t)] + [(n, ctypes.c_int64) for n in (
                   "b", "total_q", "total_k", "heads", "kv_heads", "d", "q_t", "q_h", "k_t", "k_h", "v_t", "v_h", "qr_t", "qr_h", "kr_t", "kr_h", "o_t", "o_h")] + \
               [("softmax_scale", ctypes.c_float), ("causal", ctypes.c_int32), ("fp16", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def test_c_entries_say_what_they_refuse():
    lib = ctypes.CDLL(LIB)
    lib.pto_last_error.restype = ctypes.c_char_p
    for name in ("pto_rotary_tables_launch", "pto_rotary_launch", "pto_cache_write_launch", "pto_cache_read_launch", "pto_prompt_attention_launch"):
        assert getattr(lib, name)(None, None) == -1 and b"NULL" in lib.pto_last_error(), name
    a = Attention(*([4096] * 3), None, None, *([4096] * 3), None, None, 0, 1, 100, 100, 8, 8, 128, 1024, 128, 1024, 128, 1024, 128, 0, 0, 0, 0, 1024, 128, 0.1, 1, 0, 0)
    for field, value, text in (("d", 96, b"d must be"), ("heads", 9, b"multiple"), ("b", 0, b"range"), ("total_q", -1, b"range"), ("query", None, b"NULL"),
                               ("key", 4104, b"16-byte"), ("k_t", 1028, b"multiples of 8"), ("v_t", 1 << 26, b"token strides"), ("k_t", -1024, b"token strides"),
                               ("softmax_scale", math.inf, b"finite"), ("query_rope", 4096, b"come together"), ("out", 4097, b"aligned")):
        b = Attention.from_buffer_copy(a)
        setattr(b, field, value)
        assert lib.pto_prompt_attention_launch(ctypes.byref(b), None) == -1, field
        assert text in lib.pto_last_error(), (field, lib.pto_last_error())
    n = ctypes.c_size_t(1)
    assert lib.pto_prompt_attention_workspace_bytes(ctypes.byref(a), None) == -1
    assert lib.pto_prompt_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value % 4 == 0
    a.total_q = 0
    assert lib.pto_prompt_attention_launch(ctypes.byref(a), None) == 0                 # an empty call does nothing


# ---------------------------------------------------------------- outputs in the memory of what says where and how much

def inside(t, dtype, *shape):
    """A tensor in the first bytes of another one."""
    n = math.prod(shape)
    return t.reshape(-1).view(dtype)[:n].view(shape)


@pytest.mark.parametrize("at", [2, 3])
def test_tables_over_positions_or_frequencies(at):
    args = tables()
    refused(ValueError, "positions overlap", pypto_amd.rotary_tables, changed(args, 0, inside(args[at], torch.int64, 5)))
    refused(ValueError, "frequencies overlap", pypto_amd.rotary_tables, changed(args, 1, inside(args[at], torch.float64, 32)))


@pytest.mark.parametrize("at", [4, 5])
def test_rotation_over_positions_or_frequencies(at):
    args = rotation()
    refused(ValueError, "positions overlap", pypto_amd.rotary_embedding, changed(args, 2, inside(args[at], torch.int64, 5)))
    refused(ValueError, "frequencies overlap", pypto_amd.rotary_embedding, changed(args, 3, inside(args[at], torch.float64, 32)))
    args[at - 4] = args[at]                                        # (in place too)
    refused(ValueError, "positions overlap", pypto_amd.rotary_embedding, changed(args, 2, inside(args[at], torch.int64, 5)))


@pytest.mark.parametrize("at", [3, 4, 5, 6])
def test_write_over_the_cache_index(at):
    args = write()
    refused(ValueError, "cache_index overlap", pypto_amd.latent_cache_write, changed(args, 2, inside(args[at], torch.int64, 3)))
    if at in (3, 6):
        packed = [torch.zeros(256, 656, dtype=torch.int8), args[6]]
        refused(ValueError, "cache_index overlap", pypto_amd.latent_cache_write_packed, args[:2] + [inside(packed[at // 6], torch.int64, 3)] + packed)


def test_write_to_arrays_of_a_cache_in_one_memory():
    one = torch.zeros(256 * (512 + 128 + 16), dtype=torch.int8)
    cut = lambda at, width, dtype: one[at:at + 256 * width].view(dtype).view(256, -1)  # noqa: E731
    parts = [cut(0, 512, torch.int8), cut(256 * 512, 128, BF), cut(256 * 640, 16, F32)]
    args = write()
    refused(RuntimeError, "GPU", pypto_amd.latent_cache_write, args[:3] + parts)           # side by side they do not meet
    for i, (at, width, dtype) in enumerate(((1024, 512, torch.int8), (256 * 512 - 128, 128, BF), (256 * 640 - 16, 16, F32))):
        refused(ValueError, "overlap", pypto_amd.latent_cache_write, changed(args[:3] + parts, 3 + i, cut(at, width, dtype)))


@pytest.mark.parametrize("at", [5, 6])
def test_read_over_the_tables(at):
    args = read()
    refused(ValueError, "block_table overlap", pypto_amd.latent_cache_read, changed(args, 3, inside(args[at], torch.int32, 2, 3)))
    refused(ValueError, "cu_seqlens overlap", pypto_amd.latent_cache_read, changed(args, 4, inside(args[at], torch.int32, 3)))
    refused(ValueError, "first overlap", pypto_amd.latent_cache_read, args, first=inside(args[at], torch.int32, 2))
    refused(ValueError, "first overlap", pypto_amd.latent_cache_read_packed, [torch.zeros(256, 656, dtype=torch.int8)] + args[3:],
            first=inside(args[at], torch.int32, 2))


def test_attention_over_the_beginnings_of_sequences():
    args = attention()
    lse = torch.zeros(6, 4)
    refused(ValueError, "cu_seqlens_q overlap", pypto_amd.prompt_attention, changed(args, 3, inside(args[5], torch.int32, 2)))
    refused(ValueError, "cu_seqlens_k overlap", pypto_amd.prompt_attention, changed(args, 4, inside(args[5], torch.int32, 2)))
    refused(ValueError, "cu_seqlens_q overlap", pypto_amd.prompt_attention, changed(args, 3, inside(lse, torch.int32, 2)), softmax_lse=lse)
    refused(ValueError, "cu_seqlens_k overlap", pypto_amd.prompt_attention, changed(args, 4, inside(lse, torch.int32, 2)), softmax_lse=lse)
