"""Single tokens over a cache of 8 bits: launches with a shared prefix by their query rows and heads, tokens far apart and on top of each
other, and what is near values that are not finite."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check
from _cache8 import random_cache
from test_gpu_attention8 import F16, F32, case, expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hkv,d,kw", [
    ([700, 0, 64, 1, 513], 4, 4, 64, dict(page=16)), ([600, 1300, 63], 8, 8, 128, {}), ([900, 33], 24, 8, 64, dict(page=24, softcap=20.0, biased=True)),
    ([640, 129, 31], 32, 4, 128, dict(page=64)), ([1000, 5], 28, 4, 128, dict(biased=True)), ([800, 65], 32, 4, 64, {}),
    ([1024], 4, 4, 128, {}), ([530] * 8, 32, 4, 128, dict(page=16)), ([20, 700], 16, 2, 128, {}), ([515, 70], 3, 3, 64, dict(by_head=True)),
    ([300, 0, 64], 4, 4, 128, {}), ([300, 12], 32, 4, 64, dict(page=16)),
], ids=str)
def test_shared_and_own_keys_in_one_launch(cuda, code, lengths, hq, hkv, d, kw):
    # one to eight query rows of a key head, heads by fours (past 512 keys) or by themselves, of 64 and 128 values
    args, more, ref = case(cuda, F16, code, lengths, hq, hkv, d, shared=200, seed=hq + d, **kw)
    y = g.attention_decode(*args, **more)
    check(y, ref)
    assert torch.equal(y, g.attention_decode(*args, **more))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("length", [70, 600])
def test_tokens_far_apart(cuda, dtype, length):
    # 2^24 bytes and more from a token to the next, which caches in the queries' type do not reach
    heads, d, step = 2, 64, (1 << 24) + 64
    gen = torch.Generator().manual_seed(9)
    cache, k, v = random_cache(1, length, heads, d, "int8", gen)
    room = torch.zeros(length * step, dtype=torch.int8, device=cuda)
    kc, vc = (room[at:].as_strided((1, length, heads, d), (0, step, d, 1)) for at in (0, 4096))
    kc.copy_(cache[0]), vc.copy_(cache[1])
    q = torch.randn(1, 4, d, generator=gen).to(dtype)
    y = g.attention_decode(q.to(cuda), kc, vc, torch.tensor([length], dtype=torch.int32, device=cuda), k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda))
    check(y, expected(q, [k[0]], [v[0]], [length]))


@pytest.mark.parametrize("length", [70, 600])
def test_tokens_of_one_place(cuda, length):
    # a stride of 0: all tokens are one key and value, whose mean is the value
    gen = torch.Generator().manual_seed(4)
    cache, k, v = random_cache(1, 1, 2, 64, "int8", gen)
    kc, vc, ks, vs = (t.to(cuda).expand(1, length, *t.shape[2:]) for t in cache)
    q = torch.randn(1, 4, 64, generator=gen).half()
    y = g.attention_decode(q.to(cuda), kc, vc, torch.tensor([length], dtype=torch.int32, device=cuda), k_scale=ks, v_scale=vs)
    check(y, expected(q, [k[0].expand(length, -1, -1)], [v[0].expand(length, -1, -1)], [length]))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv,d,length", [(4, 1, 128, 70), (8, 1, 64, 70), (16, 1, 64, 70), (32, 1, 64, 70), (16, 4, 64, 700)])
def test_rows_beside_infinite_queries(cuda, dtype, hq, hkv, d, length):
    (q, kc, vc, lengths), kw, (out, tol) = case(cuda, dtype, "e4m3", [length, 5], hq, hkv, d)
    q[0, 2, 5], q[1, 0, 0] = float("inf"), float("nan")
    y = g.attention_decode(q, kc, vc, lengths, **kw).cpu()
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 2] = bad[1, 0] = True
    assert torch.isnan(y[bad]).all()
    assert ((y.double() - out).abs() <= tol)[~bad].all()
