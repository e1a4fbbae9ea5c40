"""CPU tests of rotary, the caches in 8 bits and attention over them: argument structs, what the library rejects before a launch, and
what the Python functions refuse."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gtx16_fp16 as g
from gtx16_fp16 import _clib, attn, cache, positions

SHAPE, ALIGN, NULL, WORKSPACE, DTYPE = -1, -2, -3, -4, -6


def call(name, head):
    # (every call here is rejected or has nothing to do, so nothing is launched)
    return _clib.fast().struct_call(_clib.address(name), head, 0)


ROTARY = ["x", "out", "positions", "freqs", "x_seq", "x_token", "x_head", "seqs", "tokens", "heads", "d", "pairs", "axes", "s0", "s1", "s2", "s3",
          "interleaved", "is_f32"]


def rotary_head(**changes):
    v = dict(x=4096, out=4096, positions=4096, freqs=4096, x_seq=0, x_token=256, x_head=64, seqs=1, tokens=3, heads=4, d=64, pairs=32, axes=1, s0=32,
             s1=0, s2=0, s3=0, interleaved=0, is_f32=0) | changes
    return positions._ARGS.pack(*(v[n] for n in ROTARY))


@pytest.mark.parametrize("changes,status", [
    (dict(d=60), SHAPE), (dict(d=0), SHAPE), (dict(d=4104, pairs=0, s0=0), SHAPE), (dict(pairs=33, s0=33), SHAPE), (dict(pairs=-1, s0=-1), SHAPE),
    (dict(axes=0), SHAPE), (dict(axes=5), SHAPE), (dict(s0=31), SHAPE), (dict(axes=2, s0=33, s1=-1), SHAPE), (dict(heads=-1), SHAPE), (dict(tokens=-1), SHAPE),
    (dict(interleaved=2), SHAPE), (dict(seqs=1 << 16, tokens=1 << 16), SHAPE), (dict(is_f32=2), DTYPE), (dict(x=0), NULL), (dict(out=0), NULL),
    (dict(positions=0), NULL), (dict(freqs=0), NULL), (dict(x=4098), ALIGN), (dict(out=4104), ALIGN), (dict(x_token=3), ALIGN), (dict(x_head=4), ALIGN)])
def test_rotary_is_rejected_before_a_launch(changes, status):
    assert call("g16_rotary", rotary_head(**changes)) == status


def test_rotary_with_nothing_to_do():
    for n in ("seqs", "tokens", "heads"):
        assert call("g16_rotary", rotary_head(**{n: 0}, x=0)) == 0
    assert _clib.load().g16_rotary(None, None) == NULL


CACHE = ["k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "slots", "k_token", "k_head", "v_token", "v_head", "kc_page", "kc_token", "kc_head", "vc_page",
         "vc_token", "vc_head", "ks_page", "ks_token", "ks_head", "vs_page", "vs_token", "vs_head", "rows", "pages", "page", "hkv", "d", "code", "is_f32",
         "reserved"]


def cache_head(**changes):
    v = dict.fromkeys(CACHE, 0)
    v.update({n: 4096 for n in CACHE[:7]}, k_token=128, k_head=64, v_token=128, v_head=64, kc_page=2048, kc_token=128, kc_head=64, vc_page=2048, vc_token=128,
             vc_head=64, rows=3, pages=2, page=16, hkv=2, d=64, code=1)
    v.update(changes)
    return cache._ARGS.pack(*(v[n] for n in CACHE))


@pytest.mark.parametrize("name", ["g16_cache_write", "g16_cache_read"])
@pytest.mark.parametrize("changes,status", [
    (dict(d=60), SHAPE), (dict(d=136), SHAPE), (dict(d=0), SHAPE), (dict(rows=-1), SHAPE), (dict(pages=-1), SHAPE), (dict(page=-1), SHAPE), (dict(hkv=-1), SHAPE),
    (dict(pages=1 << 16, page=1 << 16), SHAPE), (dict(code=0), DTYPE), (dict(code=3), DTYPE), (dict(is_f32=2), DTYPE), (dict(k=0), NULL), (dict(v=0), NULL),
    (dict(slots=0), NULL), (dict(k_cache=0), NULL), (dict(v_scale=0), NULL), (dict(k=4104), ALIGN), (dict(k_cache=4100), ALIGN), (dict(kc_token=12), ALIGN),
    (dict(vc_page=4), ALIGN)])
def test_caches_are_rejected_before_a_launch(name, changes, status):
    assert call(name, cache_head(**changes)) == status


def test_caches_own_rules_and_nothing_to_do():
    assert call("g16_cache_write", cache_head(k_token=4)) == ALIGN
    for name in ("g16_cache_write", "g16_cache_read"):
        assert call(name, cache_head(rows=0, k=0)) == 0 and call(name, cache_head(hkv=0, k=0)) == 0
    assert _clib.load().g16_cache_write(None, None) == NULL and _clib.load().g16_cache_read(None, None) == NULL


BASE = (["q", "k", "v", "shared_k", "shared_v", "out", "q_offsets", "k_offsets", "visible", "lengths", "pages", "slopes"]
        + ["q_seq", "q_token", "q_head", "k_seq", "k_token", "k_head", "v_seq", "v_token", "v_head",
           "shared_k_token", "shared_k_head", "shared_v_token", "shared_v_head"]
        + ["seqs", "q_len", "k_len", "hq", "hkv", "d", "shared", "causal", "page", "max_pages", "num_pages", "is_f32", "num_cus"]
        + ["scale", "softcap", "reserved"])


def decode_head(**changes):
    v = dict.fromkeys(BASE, 0)
    v.update(q=4096, k=4096, v=4096, out=4096, lengths=4096, q_seq=128, q_head=64, k_seq=512, k_token=64, k_head=64, v_seq=512, v_token=64, v_head=64,
             seqs=2, q_len=1, k_len=8, page=8, hq=2, hkv=1, d=64, num_cus=256, scale=1.0, softcap=0.0)
    scales = dict(k_scale=4096, v_scale=4096, code=1) | {n: x for n, x in changes.items() if n in ("k_scale", "v_scale", "code")}
    v.update({n: x for n, x in changes.items() if n not in scales})
    return attn._ARGS8.pack(scales["k_scale"], scales["v_scale"], 8, 1, 1, 8, 1, 1, scales["code"], 0) + attn._ARGS.pack(*(v[n] for n in BASE))


def decode_call(**changes):
    return _clib.fast().args_call(_clib.address("g16_attention_decode8"), decode_head(**changes), None, 0, 0)


def decode_size(**changes):
    return _clib.fast().args_size(_clib.address("g16_attention_decode8_workspace_bytes"), decode_head(**changes))


@pytest.mark.parametrize("changes,status", [
    (dict(d=60), SHAPE), (dict(d=136), SHAPE), (dict(seqs=-1), SHAPE), (dict(hkv=0), SHAPE), (dict(hq=3, hkv=2), SHAPE), (dict(softcap=-1.0), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(is_f32=2), DTYPE), (dict(code=0), DTYPE), (dict(code=3), DTYPE), (dict(q=0), NULL), (dict(k=0), NULL),
    (dict(k_scale=0), NULL), (dict(v_scale=0), NULL), (dict(lengths=0), NULL), (dict(k=4100), ALIGN), (dict(k_token=12), ALIGN), (dict(v_seq=4), ALIGN),
    (dict(q=4104), ALIGN), (dict(q_head=3), ALIGN), (dict(pages=4096, page=4, max_pages=1), SHAPE), (dict(seqs=1 << 20, k_len=1 << 29), SHAPE),
    (dict(shared=3), NULL)])
def test_attention_is_rejected_before_a_launch(changes, status):
    assert decode_call(**changes) == status
    assert decode_size(**changes) == 0 or changes == dict(seqs=1 << 20, k_len=1 << 29)


def test_attentions_workspace():
    assert decode_size() == 0 and decode_size(k_len=512, page=512) == 0  # whole requests
    long = dict(k_len=8000, page=8000)
    assert decode_size(**long) > 0 and decode_call(**long) == WORKSPACE
    shared = dict(shared=64, shared_k=4096, shared_v=4096, shared_k_token=64, shared_v_token=64)
    assert decode_size(**shared) > 0 and decode_call(**shared) == WORKSPACE
    assert decode_call(seqs=0) == 0 and decode_call(hq=0) == 0
    # a cache's rows may be further apart than those of a cache that is not in 8 bits, and nearer (one key head for all tokens)
    assert decode_call(k_token=1 << 30, seqs=0) == 0


def test_tangents_are_refused():
    x, f = torch.zeros(3, 2, 64), torch.zeros(32)
    c, s, at = torch.zeros(2, 4, 2, 64, dtype=torch.int8), torch.zeros(2, 4, 2), torch.zeros(3, dtype=torch.int32)
    calls = [(lambda **a: g.rotary(a["x"], at, a["f"]), dict(x=x, f=f)),
             (lambda **a: g.cache_write(a["k"], a["v"], c, c, a["ks"], a["vs"], at), dict(k=x, v=x, ks=s, vs=s)),
             (lambda **a: g.cache_read(c, c, a["ks"], a["vs"], at), dict(ks=s, vs=s)),
             (lambda **a: g.attention_decode(a["q"], c, c, at, k_scale=a["ks"], v_scale=a["vs"]), dict(q=x, ks=s, vs=s))]
    for fn, operands in calls:
        for name in operands:
            with forward_ad.dual_level():
                given = dict(operands)
                given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
                with pytest.raises(RuntimeError, match="tangent"):
                    fn(**given)
                with pytest.raises(ValueError):  # (these tensors are on the CPU)
                    fn(**operands)


def test_structs_of_another_size_are_refused():
    with pytest.raises(ValueError):
        _clib.fast().struct_call(_clib.address("g16_rotary"), b"123", 0)
    with pytest.raises(ValueError):
        _clib.fast().struct_call(_clib.address("g16_rotary"), bytes(1024), 0)
