"""CPU tests of the attention entry points: the argument struct, and what the library rejects before a launch."""
from __future__ import annotations

import ctypes

import pytest

from gtx16_fp16 import _clib, attn

NAMES = (["q", "k", "v", "shared_k", "shared_v", "out", "q_offsets", "k_offsets", "visible", "lengths", "pages", "slopes"]
         + ["q_seq", "q_token", "q_head", "k_seq", "k_token", "k_head", "v_seq", "v_token", "v_head",
            "shared_k_token", "shared_k_head", "shared_v_token", "shared_v_head"]
         + ["seqs", "q_len", "k_len", "hq", "hkv", "d", "shared", "causal", "page", "max_pages", "num_pages", "is_f32", "num_cus"]
         + ["scale", "softcap", "reserved"])


def head(**changes) -> bytes:
    v = dict.fromkeys(NAMES, 0)
    v.update(q=4096, k=4096, v=4096, out=4096, lengths=4096, q_seq=512, q_token=128, q_head=64, k_seq=512, k_token=64, k_head=64,
             v_seq=512, v_token=64, v_head=64, seqs=2, q_len=4, k_len=8, hq=2, hkv=1, d=64, num_cus=256, scale=1.0, softcap=0.0)
    v.update(changes)
    return attn._ARGS.pack(*(v[n] for n in NAMES))


def call(name, **changes):
    # (every call here is rejected, so nothing is launched)
    return _clib.fast().args_call(_clib.address(name), head(**changes), None, 0, 0)


def size(name, **changes):
    return _clib.fast().args_size(_clib.address(name + "_workspace_bytes"), head(**changes))


SHAPE, ALIGN, NULL, WORKSPACE, DTYPE = -1, -2, -3, -4, -6


@pytest.mark.parametrize("name", ["g16_attention", "g16_attention_decode"])
@pytest.mark.parametrize("changes,status", [
    (dict(d=60), SHAPE), (dict(d=136), SHAPE), (dict(d=0), SHAPE), (dict(seqs=-1), SHAPE), (dict(hkv=0), SHAPE), (dict(hq=3, hkv=2), SHAPE),
    (dict(k_len=-1), SHAPE), (dict(shared=-1), SHAPE), (dict(softcap=-1.0), SHAPE), (dict(softcap=float("nan")), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(k_len=1 << 30, shared=1), SHAPE), (dict(is_f32=2), DTYPE),
    (dict(q=0), NULL), (dict(out=0), NULL), (dict(k=0), NULL), (dict(v=0), NULL), (dict(shared=3), NULL),
    (dict(q=4098), ALIGN), (dict(k=4104), ALIGN), (dict(out=4100), ALIGN), (dict(q_head=3), ALIGN), (dict(k_seq=3), ALIGN),
    (dict(k_token=56), SHAPE), (dict(v_token=1 << 23), SHAPE), (dict(k_token=65), SHAPE),
    (dict(shared=3, shared_k=4096, shared_v=4096, shared_k_token=8, shared_v_token=64), SHAPE),
])
def test_rejected_before_a_launch(name, changes, status):
    assert call(name, **changes) == status


def test_each_entry_points_own_rules():
    assert call("g16_attention", q_len=-1) == SHAPE
    assert call("g16_attention", q_offsets=4096) == NULL
    assert call("g16_attention", q_token=3) == ALIGN
    assert call("g16_attention_decode", lengths=0) == NULL
    assert call("g16_attention_decode", pages=4096) == SHAPE
    assert call("g16_attention_decode", pages=4096, page=4, max_pages=1) == SHAPE
    assert _clib.load().g16_attention(None, None) == NULL
    assert _clib.load().g16_attention_decode(None, None) == NULL


def test_nothing_to_do_is_no_error():
    assert call("g16_attention", seqs=0) == 0
    assert call("g16_attention", q_len=0) == 0
    assert call("g16_attention_decode", seqs=0) == 0


def test_workspace_is_asked_for_and_checked():
    long = dict(k_len=8000, q_len=4, k_seq=8000 * 64, v_seq=8000 * 64)
    assert size("g16_attention") == 0
    assert size("g16_attention", **long) > 0
    assert call("g16_attention", **long) == WORKSPACE
    shared = dict(shared=64, shared_k=4096, shared_v=4096, shared_k_token=64, shared_v_token=64)
    assert size("g16_attention_decode") == 0
    assert size("g16_attention_decode", **shared) > 0
    assert call("g16_attention_decode", **shared) == WORKSPACE
    assert size("g16_attention", d=60) == 0  # a rejected call needs none


def test_struct_size_is_checked_by_the_binding():
    fast = _clib.fast()
    with pytest.raises(ValueError):
        fast.args_call(_clib.address("g16_attention"), b"1234", None, 0, 0)
    with pytest.raises(TypeError):
        fast.args_size(_clib.address("g16_attention"))
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def plan(**changes):
    """(status, rows of a workgroup, splits) of g16_attention for these arguments."""
    args = ctypes.create_string_buffer(head(**changes) + bytes(16))
    rows, splits = ctypes.c_int(-1), ctypes.c_int(-1)
    st = _clib.load().g16_attention_plan(args, ctypes.byref(rows), ctypes.byref(splits))
    return st, rows.value, splits.value


def documents(n, tokens, heads, **changes):
    rows = n * tokens
    return dict(dict(q_offsets=4096, k_offsets=4096, seqs=n, q_len=rows, k_len=rows, hq=heads, hkv=heads, q_token=heads * 64, k_token=heads * 64,
                     v_token=heads * 64), **changes)


def test_plan_follows_the_checks():
    assert plan(d=60) == (SHAPE, 0, 0)
    assert plan(q=0) == (NULL, 0, 0)
    assert plan(q_len=0) == (0, 0, 0)
    st, rows, splits = plan()
    assert st == 0 and rows in (32, 128) and splits == 1
    assert plan(k_len=8000, q_len=4, k_seq=8000 * 64, v_seq=8000 * 64)[2] > 1
    rows = ctypes.c_int()
    assert _clib.load().g16_attention_plan(None, ctypes.byref(rows), ctypes.byref(rows)) == NULL
    assert _clib.load().g16_attention_plan(ctypes.create_string_buffer(head() + bytes(16)), None, ctypes.byref(rows)) == NULL


@pytest.mark.parametrize("n,tokens,heads", [(50000, 10, 12), (100000, 10, 12), (100000, 100, 12), (1000000, 3, 12)])
def test_many_documents_fit_a_launch_where_nothing_is_joined(n, tokens, heads):
    # one workgroup for every 128 (or 32) rows of a document and head, of which a launch takes 2^24 - 1
    st, rows, splits = plan(**documents(n, tokens, heads))
    assert st == 0 and splits == 1 and (n * tokens // rows + n) * heads < 1 << 24


def test_what_no_launch_takes_is_rejected():
    assert plan(**documents(1 << 24, 1, 2)) == (SHAPE, 0, 0)
    assert size("g16_attention", **documents(1 << 24, 1, 2)) == 0
    assert call("g16_attention", **documents(1 << 24, 1, 2)) == SHAPE
    # rows of all sequences past 32 bits
    equal = dict(seqs=1 << 22, q_len=1 << 22, k_len=8, hq=2, hkv=2)
    assert plan(**equal) == (SHAPE, 0, 0) and call("g16_attention", **equal) == SHAPE


@pytest.mark.parametrize("name", ["g16_attention", "g16_attention_decode"])
def test_an_infinite_cap_is_rejected(name):
    assert call(name, softcap=float("inf")) == SHAPE


def test_numbers_that_fp32_does_not_hold_are_refused():
    assert attn._numbers("attention", None, 0.0, 64) == (0.125, 0.0)
    assert attn._numbers("attention", -3.0, 1e-40, 64) == (-3.0, 1e-40)
    for scale, cap in ((1e39, 0.0), (-1e300, 0.0), (float("nan"), 0.0), (1.0, 1e39), (1.0, float("inf")), (1.0, float("nan")), (1.0, -1.0),
                       (1.0, 1e-60)):
        with pytest.raises(ValueError, match="attention: s"):
            attn._numbers("attention", scale, cap, 64)
