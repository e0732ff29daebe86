"""What a serving step's operators refuse, on the host: nothing is launched."""
import ctypes
import math

import pytest
import torch

import pypto_amd
from tests.test_prompt_refusals import LIB, Attention, attention, changed, inside, refused

BF, I32, I64 = torch.bfloat16, torch.int32, torch.int64


def z(*s, dtype=I32):
    return torch.zeros(s, dtype=dtype)


# ---------------------------------------------------------------- pages

def pages():
    return [z(3), z(3), z(3, 5), z(20), z(1), z(1), 128]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, z(3, dtype=I64), TypeError, "lens_before"), (0, z(4), ValueError, "lens_|block_table"), (1, z(2), ValueError, "lens_after"), (0, z(3, 1), ValueError, "1 dim"),
    (1, [1, 2, 3], TypeError, "not currently supported"), (2, z(3, 5, dtype=I64), TypeError, "block_table"), (2, z(15), ValueError, "2 dim"), (2, z(4, 5), ValueError, "block_table"),
    (2, z(3, 0), ValueError, "block_table"), (2, z(5, 3).T, RuntimeError, "contiguous"), (3, z(20, dtype=I64), TypeError, "free_pages"), (3, z(4, 5), ValueError, "free_pages"),
    (3, z(40)[::2], RuntimeError, "contiguous"), (4, z(1, dtype=I64), TypeError, "free_count"), (4, z(2), ValueError, "free_count"), (5, z(0), ValueError, "free_left"),
    (5, z(1).float(), TypeError, "free_left")])
def test_pages(at, value, kind, text):
    refused(kind, text, pypto_amd.cache_pages, changed(pages(), at, value))


def test_pages_overlaps_and_device():
    args = pages()
    refused(RuntimeError, "GPU", pypto_amd.cache_pages, args)
    refused(RuntimeError, "GPU", pypto_amd.cache_pages, changed(args, 5, args[4]))
    for at in (0, 1):
        refused(ValueError, "overlap", pypto_amd.cache_pages, changed(args, at, inside(args[2], I32, 3)))
        refused(ValueError, "overlap", pypto_amd.cache_pages, changed(args, at, inside(args[3], I32, 3)))
        refused(ValueError, "overlap", pypto_amd.cache_pages, changed(args, 5, args[at][1:2]))
    refused(ValueError, "overlap", pypto_amd.cache_pages, changed(args, 3, args[2].view(-1)[3:]))
    for at in (4, 5):
        refused(ValueError, "overlap", pypto_amd.cache_pages, changed(args, at, args[2].view(-1)[:1]))
        refused(ValueError, "overlap", pypto_amd.cache_pages, changed(args, at, args[3][19:]))
    same = changed(args, 1, args[0])                               # nothing changes: no fault
    refused(RuntimeError, "GPU", pypto_amd.cache_pages, same)


# ---------------------------------------------------------------- slots

def slots():
    return [z(3), z(3), z(3, 5), z(4), z(4), z(9, dtype=I64), z(9, dtype=I64), 128]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, z(3, dtype=I64), TypeError, "query_lens"), (0, z(4), ValueError, "block_table|seq_lens"), (1, z(2), ValueError, "seq_lens"), (2, z(3), ValueError, "block_table"),
    (3, z(3), ValueError, "cu_seqlens_q"), (3, z(4, dtype=I64), TypeError, "cu_seqlens_q"), (3, None, TypeError, "cu_seqlens_q|None|not currently"), (4, z(5), ValueError, "cu_seqlens_k"), (4, z(4).float(), TypeError, "cu_seqlens_k"),
    (5, z(9), TypeError, "positions"), (5, z(8, dtype=I64), ValueError, "cache_index"), (6, z(10, dtype=I64), ValueError, "cache_index"), (6, z(9), TypeError, "cache_index"),
    (6, z(18, dtype=I64)[::2], RuntimeError, "contiguous"), (5, z(9, 1, dtype=I64), ValueError, "positions")])
def test_slots(at, value, kind, text):
    refused(kind, text, pypto_amd.cache_slots, changed(slots(), at, value))


def test_slots_trees_overlaps_and_device():
    args, op = slots(), pypto_amd.cache_slots
    refused(RuntimeError, "GPU", op, args)
    refused(RuntimeError, "GPU", op, changed(args, 4, None))
    mask, up = z(9, 2, dtype=I64), z(9)
    refused(RuntimeError, "GPU", op, args, parents=up, tree_mask=mask)
    refused(ValueError, "come together", op, args, parents=up)
    refused(ValueError, "come together", op, args, tree_mask=mask)
    refused(TypeError, "parents", op, args, parents=up.long(), tree_mask=mask)
    refused(ValueError, "parents", op, args, parents=up[:8], tree_mask=mask)
    refused(TypeError, "tree_mask", op, args, parents=up, tree_mask=mask.int())
    for bad in (z(8, 2, dtype=I64), z(9, 17, dtype=I64), z(9, 0, dtype=I64), z(9, dtype=I64)):
        refused(ValueError, "tree_mask", op, args, parents=up, tree_mask=bad)
    for out in (3, 4, 5, 6):
        for at in (0, 1):
            refused(ValueError, "overlap", op, changed(args, at, inside(args[out], I32, 3)))
        wide = changed(args, 2, inside(z(64), I32, 3, 5))
        refused(ValueError, "overlap", op, changed(wide, out, inside(wide[2], args[out].dtype, *args[out].shape)) if out < 5 else
                changed(changed(wide, 2, inside(args[out], I32, 3, 5)), out, args[out]))
    refused(ValueError, "overlap", op, changed(args, 6, args[5]))
    refused(ValueError, "overlap", op, changed(args, 4, args[3]))
    refused(ValueError, "overlap", op, args, parents=inside(mask, I32, 9), tree_mask=mask)
    refused(ValueError, "overlap", op, args, parents=inside(args[5], I32, 9), tree_mask=mask)
    refused(ValueError, "overlap", op, args, parents=up, tree_mask=args[6].view(9, 1))


# ---------------------------------------------------------------- attention over the cached latents

def latent():
    return [z(6, 4, 512, dtype=BF), z(6, 4, 64, dtype=BF), z(256, 512, dtype=torch.int8), z(256, 64, dtype=BF), z(256, 4, dtype=torch.float32), z(2, 3), z(3), z(2),
            z(6, 4, 512, dtype=BF), 0.1, 128]


@pytest.mark.parametrize("at,value,kind,text", [
    (0, z(6, 4, 512).float(), TypeError, "query_nope"), (0, z(24, 512, dtype=BF), ValueError, "query_nope"), (0, z(6, 4, 500, dtype=BF), ValueError, "query_nope"),
    (0, z(6, 0, 512, dtype=BF), ValueError, "query_nope|query_rope"), (1, z(6, 4, 64, dtype=torch.float16), TypeError, "query_rope"), (1, z(6, 2, 64, dtype=BF), ValueError, "query_rope"),
    (0, z(6, 512, 4, dtype=BF).transpose(1, 2), RuntimeError, "last dimension"), (2, z(256, 512, dtype=BF), TypeError, "kv_cache"), (2, z(256, 656, dtype=torch.int8), ValueError, "kv_cache"),
    (3, z(255, 64, dtype=BF), ValueError, "kr_cache"), (4, z(256, 4, dtype=torch.float16), TypeError, "k_scale_cache"), (4, z(256, 8).float()[:, :4], RuntimeError, "contiguous"),
    (5, z(2, 3, dtype=I64), TypeError, "block_table"), (5, z(3, 3), ValueError, "block_table"), (5, z(2, 0), ValueError, "block_table"), (6, z(2), ValueError, "cu_seqlens_q"), (6, z(3, dtype=I64), TypeError, "cu_seqlens_q"),
    (7, z(3), ValueError, "block_table|seq_lens"), (7, z(2).float(), TypeError, "seq_lens"), (8, z(6, 4, 512).float(), TypeError, "attention_out"),
    (8, z(1, 4, 512, dtype=BF).expand(6, 4, 512), ValueError, "share memory"), (8, z(6, 4, 64, dtype=BF), ValueError, "attention_out"), (9, math.nan, ValueError, "finite"),
    (9, -math.inf, ValueError, "finite")])
def test_latent_attention(at, value, kind, text):
    refused(kind, text, pypto_amd.latent_attention, changed(latent(), at, value))


def test_latent_attention_s_masks_windows_overlaps_and_device():
    args, op = latent(), pypto_amd.latent_attention
    refused(RuntimeError, "GPU", op, args)
    refused(RuntimeError, "GPU", op, args, window=5, sinks=2, softmax_lse=z(6, 4, dtype=torch.float32))
    refused(RuntimeError, "GPU", op, args, tree_mask=z(6, 1, dtype=I64))
    refused(RuntimeError, "GPU", pypto_amd.latent_attention_packed, args[:2] + [z(256, 656, dtype=torch.int8)] + args[5:])
    refused(ValueError, "656", pypto_amd.latent_attention_packed, args[:2] + [z(256, 512, dtype=torch.int8)] + args[5:])
    for kw in (dict(window=0), dict(window=-3), dict(window=(1 << 30) + 1), dict(window=5, sinks=-1), dict(sinks=4), dict(window=5, sinks=1 << 31)):
        refused(ValueError, "window|sinks", op, args, **kw)
    for kw in (dict(window=5.0), dict(window=True), dict(window=5, sinks=1.5)):
        refused(ValueError, "window|sinks", op, args, **kw)
    refused(ValueError, "exclude", op, args, window=5, tree_mask=z(6, 1, dtype=I64))
    refused(TypeError, "tree_mask", op, args, tree_mask=z(6, 1))
    for bad in (z(5, 1, dtype=I64), z(6, 17, dtype=I64), z(6, 0, dtype=I64), z(6, dtype=I64)):
        refused(ValueError, "tree_mask", op, args, tree_mask=bad)
    refused(TypeError, "softmax_lse", op, args, softmax_lse=z(6, 4))
    refused(ValueError, "softmax_lse", op, args, softmax_lse=z(4, 6, dtype=torch.float32))
    refused(ValueError, "overlap", op, changed(args, 8, args[0]))
    for at, shape, dtype in ((1, (6, 4, 64), BF), (2, (12, 512), torch.int8), (5, (2, 3), I32), (6, (3,), I32), (7, (2,), I32)):
        given = changed(args, at, inside(args[8], dtype, *shape))
        if at == 2:
            given[3], given[4] = z(12, 64, dtype=BF), z(12, 4, dtype=torch.float32)
        refused(ValueError, "overlap", op, given)
    refused(ValueError, "overlap", op, args, tree_mask=inside(args[8], I64, 6, 1))
    refused(ValueError, "overlap", op, args, softmax_lse=inside(args[8], torch.float32, 6, 4))
    refused(ValueError, "overlap", op, args, softmax_lse=inside(args[0], torch.float32, 6, 4))
    mask = z(6, 4, dtype=I64)
    refused(ValueError, "overlap", op, args, tree_mask=mask, softmax_lse=inside(mask, torch.float32, 6, 4))


# ---------------------------------------------------------------- windows of prompts

def test_prompt_windows():
    args, op = attention(), pypto_amd.prompt_window_attention
    refused(RuntimeError, "GPU", op, args + [5])
    refused(RuntimeError, "GPU", op, args + [1 << 30], sinks=1 << 30, softmax_lse=z(6, 4, dtype=torch.float32))
    for kw in (dict(window=0), dict(window=-1), dict(window=(1 << 30) + 1), dict(window=5, sinks=-1), dict(window=5, sinks=(1 << 30) + 1)):
        refused(ValueError, "window|sinks", op, args, **kw)
    for kw in (dict(window=5.0), dict(window=True), dict(window=None), dict(window=5, sinks=None)):
        refused(ValueError, "window|sinks", op, args, **kw)
    refused(ValueError, "key", op, changed(args, 1, z(9, 3, 128, dtype=BF)) + [5])
    refused(ValueError, "overlap", op, changed(args, 5, args[0]) + [5])
    refused(ValueError, "come together", op, args + [5], query_rope=z(6, 4, 64, dtype=BF))
    refused(TypeError, "softmax_lse", op, args + [5], softmax_lse=z(6, 4))
    refused(ValueError, "finite", op, changed(args, 6, math.nan) + [5])


# ---------------------------------------------------------------- the C entries

def structure(pointers, numbers, tail=(), head=()):
    fields = list(head) + [(n, ctypes.c_size_t if n == "workspace_bytes" else ctypes.c_void_p) for n in pointers] + [(n, ctypes.c_int64) for n in numbers] + list(tail)
    return type("Args", (ctypes.Structure,), {"_fields_": fields})


Pages = structure(("lens_before", "lens_after", "block_table", "free_pages", "free_count", "free_left"), ("b", "max_blocknum_perbatch", "block_size", "room"))
Slots = structure(("query_lens", "seq_lens", "block_table", "cu_seqlens_q", "cu_seqlens_k", "positions", "cache_index", "parents", "tree_mask"),
                  ("b", "t", "max_blocknum_perbatch", "block_size", "mask_words"))
Latent = structure(("query_nope", "query_rope", "nope", "rope_cache", "scales", "block_table", "cu_seqlens_q", "seq_lens", "tree_mask", "out", "lse", "workspace", "workspace_bytes"),
                   ("b", "total_q", "heads", "cache_rows", "block_size", "max_blocknum_perbatch", "qn_t", "qn_h", "qr_t", "qr_h", "o_t", "o_h", "window", "sinks", "mask_words"),
                   [("softmax_scale", ctypes.c_float), ("packed", ctypes.c_int32)])
Window = type("Window", (ctypes.Structure,), {"_fields_": [("prompt", Attention), ("window", ctypes.c_int64), ("sinks", ctypes.c_int64)]})


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.pto_last_error.restype = ctypes.c_char_p
    return lib


def refusals(lib, entry, args, changes):
    for fields, text in changes:
        a = type(args).from_buffer_copy(args)
        for name, value in fields.items():
            at = a.prompt if name.startswith("prompt_") else a
            setattr(at, name.removeprefix("prompt_"), value)
        assert getattr(lib, entry)(ctypes.byref(a), None) == -1, fields
        assert text in lib.pto_last_error(), (fields, lib.pto_last_error())


def test_c_entries_without_arguments(lib):
    for name in ("pto_cache_pages_launch", "pto_cache_slots_launch", "pto_latent_attention_launch", "pto_prompt_window_launch"):
        assert getattr(lib, name)(None, None) == -1 and b"NULL" in lib.pto_last_error(), name
    n = ctypes.c_size_t()
    for name in ("pto_latent_attention_workspace_bytes", "pto_prompt_window_workspace_bytes"):
        assert getattr(lib, name)(None, ctypes.byref(n)) == -1 and b"NULL" in lib.pto_last_error(), name


def test_c_pages(lib):
    refusals(lib, "pto_cache_pages_launch", Pages(*([4096] * 6), 3, 5, 128, 20), [
        (dict(b=0), b"range"), (dict(b=(1 << 24) + 1), b"range"), (dict(max_blocknum_perbatch=0), b"max_blocknum"), (dict(block_size=0), b"block_size"),
        (dict(block_size=1 << 31), b"block_size"), (dict(b=1 << 20, max_blocknum_perbatch=1 << 20), b"entries"), (dict(room=-1), b"room"), (dict(room=1 << 31), b"room"),
        (dict(lens_before=None), b"NULL"), (dict(lens_after=None), b"NULL"), (dict(block_table=None), b"NULL"), (dict(free_pages=None), b"NULL"), (dict(free_left=None), b"NULL"),
        (dict(free_count=None), b"NULL"), (dict(block_table=4098), b"aligned"), (dict(free_left=4097), b"aligned")])


def test_c_slots(lib):
    refusals(lib, "pto_cache_slots_launch", Slots(*([4096] * 9), 3, 9, 5, 128, 1), [
        (dict(b=0), b"range"), (dict(t=-1), b"range"), (dict(t=(1 << 30) + 1), b"range"), (dict(max_blocknum_perbatch=0), b"max_blocknum"), (dict(block_size=-5), b"block_size"),
        (dict(parents=None), b"together"), (dict(tree_mask=None), b"together"), (dict(mask_words=0), b"mask_words"), (dict(mask_words=17), b"mask_words"),
        (dict(query_lens=None), b"NULL"), (dict(seq_lens=None), b"NULL"), (dict(cu_seqlens_q=None), b"NULL"), (dict(positions=None), b"NULL"), (dict(cache_index=None), b"NULL"),
        (dict(positions=4100), b"aligned"), (dict(tree_mask=4100), b"aligned"), (dict(cu_seqlens_k=4098), b"aligned")])


def latent_args():
    return Latent(*([4096] * 8), None, 4096, None, 4096, 1 << 40, 3, 9, 16, 1000, 128, 5, 16 * 512, 512, 16 * 64, 64, 16 * 512, 512, 0, 0, 0, 0.1, 0)


def test_c_latent_attention(lib):
    a = latent_args()
    refusals(lib, "pto_latent_attention_launch", a, [
        (dict(b=0), b"range"), (dict(total_q=-1), b"range"), (dict(heads=0), b"range"), (dict(heads=65537), b"range"), (dict(total_q=1 << 20, heads=65536), b"range"),
        (dict(block_size=0), b"block_size"), (dict(max_blocknum_perbatch=0), b"max_blocknum"), (dict(max_blocknum_perbatch=1 << 25, block_size=128), b"keys"),
        (dict(window=-1), b"window"), (dict(window=(1 << 30) + 1), b"window"), (dict(window=4, sinks=-1), b"sinks"), (dict(sinks=4), b"sinks"),
        (dict(tree_mask=4096, mask_words=1, window=4), b"exclude"), (dict(tree_mask=4096), b"mask_words"), (dict(tree_mask=4096, mask_words=17), b"mask_words"),
        (dict(softmax_scale=math.nan), b"finite"), (dict(softmax_scale=3e38), b"finite"), (dict(cache_rows=0), b"cache_rows"), (dict(cache_rows=1 << 31), b"cache_rows"),
        (dict(packed=1), b"packed"), (dict(rope_cache=None), b"arrays"), (dict(nope=None), b"cache"), (dict(query_nope=None), b"NULL"), (dict(out=None), b"NULL"),
        (dict(seq_lens=None), b"NULL"), (dict(nope=4104), b"16-byte"), (dict(scales=4100), b"16-byte"), (dict(query_rope=4104), b"16-byte"), (dict(qn_t=8196), b"multiples of 8"),
        (dict(qr_h=68), b"multiples of 8"), (dict(out=4097), b"aligned"), (dict(lse=4098), b"aligned"), (dict(tree_mask=4100, mask_words=1), b"aligned")])
    n = ctypes.c_size_t()
    assert lib.pto_latent_attention_workspace_bytes(ctypes.byref(a), None) == -1
    assert lib.pto_latent_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value % 4 == 0
    a.total_q = 0
    assert lib.pto_latent_attention_launch(ctypes.byref(a), None) == 0                     # an empty call does nothing


def workspace(lib, b, total_q, heads, keys, window=0, sinks=0):
    a = latent_args()
    a.b, a.total_q, a.heads, a.max_blocknum_perbatch, a.window, a.sinks = b, total_q, heads, -(-keys // 128), window, sinks
    n = ctypes.c_size_t()
    assert lib.pto_latent_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    return n.value


def test_workspaces_stay_small_and_follow_the_form(lib):
    """Two pieces of 64 rows to each compute unit, of 128 where sequences fill them and keys are many; a few for small calls."""
    small, large = 2 * 256 * 64 * 514 * 4, 2 * 256 * 128 * 514 * 4
    tables = 4096                                                  # (and the table of what is to be joined)
    assert workspace(lib, 1, 1, 16, 100) < small / 8
    assert small < workspace(lib, 32, 32, 128, 12000, 2048, 4) <= small + tables
    assert large < workspace(lib, 24, 1000, 128, 9000) <= large + tables
    assert large < workspace(lib, 1, 30000, 128, 1 << 20) <= large + tables
    assert workspace(lib, 1000, 1000, 8, 1 << 17) <= small + tables


def test_c_prompt_windows(lib):
    a = Window()
    a.prompt = Attention(*([4096] * 3), None, None, *([4096] * 3), None, None, 0, 1, 100, 100, 8, 8, 128, 1024, 128, 1024, 128, 1024, 128, 0, 0, 0, 0, 1024, 128, 0.1, 1, 0, 0)
    a.window = 5
    refusals(lib, "pto_prompt_window_launch", a, [
        (dict(window=0), b"window"), (dict(window=(1 << 30) + 1), b"window"), (dict(sinks=-1), b"sinks"), (dict(sinks=(1 << 30) + 1), b"sinks"), (dict(prompt_causal=0), b"causal"),
        (dict(prompt_d=96), b"d must be"), (dict(prompt_query=None), b"NULL"), (dict(prompt_key=4104), b"16-byte"), (dict(prompt_softmax_scale=math.inf), b"finite")])
    n = ctypes.c_size_t()
    assert lib.pto_prompt_window_workspace_bytes(ctypes.byref(a), None) == -1
    assert lib.pto_prompt_window_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    a.prompt.total_q = 0
    assert lib.pto_prompt_window_launch(ctypes.byref(a), None) == 0
