"""Refusals of the 8-bit paged K/V cache's entry points (CPU only: every one
is made before the context is touched)."""
import ctypes as C

import pytest

import mslim_attn

# Never dereferenced: a refused call reads its arguments alone.
CTX = C.addressof(C.create_string_buffer(1 << 16))
KEEP = []
A = 1 << 20  # an aligned address


def cache(**changes):
    fields = dict(k_pool=A, v_pool=2 * A, scales=3 * A, page_table=4 * A, pool_pages=10, pages_per_seq=4,
                  page_tokens=16, kv_heads=2, head_dim=64, format=mslim_attn.FORMAT_E4M3)
    fields.update(changes)
    return mslim_attn.Kv8Cache(**fields)


def refused(name, *args):
    lib = mslim_attn.library()
    rc = getattr(lib, name)(CTX, *args)
    assert rc == -1, (name, rc)
    return lib.mslim_attn_last_error().decode()


def lens(*x):
    return (C.c_int32 * len(x))(*x)


BAD_CACHE = [dict(k_pool=0), dict(v_pool=0), dict(scales=0), dict(page_table=0), dict(pool_pages=0),
             dict(pool_pages=1 << 31), dict(pages_per_seq=0), dict(page_tokens=8), dict(page_tokens=24),
             dict(page_tokens=8192), dict(kv_heads=0), dict(kv_heads=16385), dict(head_dim=8), dict(head_dim=72),
             dict(head_dim=272), dict(format=3), dict(format=6), dict(k_pool=A + 8), dict(v_pool=A + 4),
             dict(scales=A + 4), dict(pages_per_seq=1 << 27),
             dict(pages_per_seq=(1 << 27) - 256)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_cache(bad):
    c = C.byref(cache(**bad))
    assert refused("mslim_attn_decode_kv8", c, 5 * A, 6 * A, 1, lens(3), 4, 0.1)
    assert refused("mslim_attn_prefill_kv8", c, 5 * A, 6 * A, 1, 2, lens(3), 4, 0.1)
    assert refused("mslim_attn_pages_gather_kv8", c, 1, 3, None, 5 * A, 6 * A)
    assert refused("mslim_attn_rope_append_kv8", c, 5 * A, 6 * A, 7 * A, 8 * A, 1, 1, 9 * A, 4, 1e4, 0, 1, 1, 2, 1)


def test_null_context_and_cache():
    lib = mslim_attn.library()
    assert lib.mslim_attn_decode_kv8(None, C.byref(cache()), A, 2 * A, 1, lens(3), 4, 0.1) == -1
    assert b"null context" in lib.mslim_attn_last_error()
    assert lib.mslim_attn_rope_append_kv8(None, C.byref(cache()), A, A, A, A, 1, 1, A, 4, 1e4, 0, 1, 1, 2, 1) == -1
    assert lib.mslim_attn_pages_gather_kv8(None, C.byref(cache()), 1, 3, None, A, 2 * A) == -1
    assert refused("mslim_attn_decode_kv8", None, 5 * A, 6 * A, 1, lens(3), 4, 0.1)
    c = cache()
    c.reserved = 1
    assert "reserved" in refused("mslim_attn_decode_kv8", C.byref(c), 5 * A, 6 * A, 1, lens(3), 4, 0.1)


@pytest.mark.parametrize("change,says", [
    (dict(q=0), "non-null"), (dict(out=0), "non-null"), (dict(lens=None), "non-null"), (dict(q=A + 2), "aligned"),
    (dict(out=A + 8), "aligned"), (dict(q_heads=0), "q_heads"), (dict(q_heads=3), "q_heads"),
    (dict(out=5 * A), "alias"), (dict(out=A), "alias"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(batch=0), "batch"), (dict(batch=4097), "batch"),
    (dict(lens=lens(-1)), "length"), (dict(lens=lens(65)), "length")], ids=str)
def test_bad_attention(change, says):
    a = dict(q=5 * A, out=6 * A, batch=1, lens=lens(3), q_heads=4, scale=0.1)
    a.update(change)
    c = C.byref(cache())
    assert says in refused("mslim_attn_decode_kv8", c, a["q"], a["out"], a["batch"], a["lens"], a["q_heads"],
                           a["scale"])
    assert says in refused("mslim_attn_prefill_kv8", c, a["q"], a["out"], a["batch"], 1, a["lens"], a["q_heads"],
                           a["scale"])


def test_bad_prefill_rows():
    c = C.byref(cache())
    assert refused("mslim_attn_prefill_kv8", c, 5 * A, 6 * A, 1, 0, lens(3), 4, 0.1)
    assert "length" in refused("mslim_attn_prefill_kv8", c, 5 * A, 6 * A, 1, 62, lens(3), 4, 0.1)
    assert "rows" in refused("mslim_attn_prefill_kv8", c, 5 * A, 6 * A, 1, 1 << 30, lens(3), 4, 0.1)


@pytest.mark.parametrize("change,says", [
    (dict(q=0), "non-null"), (dict(k=0), "non-null"), (dict(v=0), "non-null"), (dict(out=0), "non-null"),
    (dict(positions=0), "non-null"), (dict(k=A + 2), "aligned"), (dict(q=A + 2), "aligned"), (dict(out=A + 8), "aligned"),
    (dict(out=5 * A), "alias"), (dict(out=6 * A), "alias"), (dict(out=2 * A), "alias"), (dict(batch=0), "batch"),
    (dict(tokens=0), "rows"), (dict(tokens=(1 << 22) + 1), "rows"), (dict(batch=4096, tokens=1025), "rows"),
    (dict(q_heads=3), "q_heads"), (dict(theta=-1.0), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(theta=float("inf")), "theta"), (dict(scaled=1, low=4.0, high=1.0), "llama3"),
    (dict(scaled=1, factor=0.0, low=1.0, high=4.0), "llama3")], ids=str)
def test_bad_append(change, says):
    a = dict(q=5 * A, k=6 * A, v=7 * A, out=8 * A, batch=1, tokens=1, positions=9 * A, q_heads=4, theta=1e4, scaled=0,
             factor=1.0, low=1.0, high=2.0)
    a.update(change)
    assert says in refused("mslim_attn_rope_append_kv8", C.byref(cache()), a["q"], a["k"], a["v"], a["out"], a["batch"],
                           a["tokens"], a["positions"], a["q_heads"], a["theta"], a["scaled"], a["factor"], a["low"],
                           a["high"], 8192.0)


def test_append_too_many_heads():
    assert "one call" in refused("mslim_attn_rope_append_kv8", C.byref(cache(kv_heads=16384)), 5 * A, 6 * A, 7 * A,
                                 8 * A, 4096, 2, 9 * A, 16384, 1e4, 0, 1, 1, 2, 1)


@pytest.mark.parametrize("args", [(0, 3, 5, 6), (1, 0, 5, 6), (1, 3, 0, 6), (1, 3, 5, 0), (1, 3, 5, 5), (1, 3, 1, 6),
                                  (1, 3, 5, 2)], ids=str)
def test_bad_gather(args):
    batch, tokens, k, v = args
    assert refused("mslim_attn_pages_gather_kv8", C.byref(cache()), batch, tokens, None, k * A, v * A)


def test_unaligned_gather():
    assert "aligned" in refused("mslim_attn_pages_gather_kv8", C.byref(cache()), 1, 3, None, 5 * A + 8, 6 * A)
