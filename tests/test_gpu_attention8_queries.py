"""Single tokens over a cache of 8 bits with fp32 queries of any size: their products with the codes, before the scales, stay in range."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check
from _cache8 import random_cache
from test_gpu_attention8 import expected

pytestmark = pytest.mark.gpu


def made(hq, hkv, d, length, seed):
    gen = torch.Generator().manual_seed(seed)
    cache, k, v = random_cache(1, length, hkv, d, "int8", gen)
    return cache, k, v, torch.randn(1, hq, d, generator=gen)


def call(cuda, q, cache, length, **kw):
    return g.attention_decode(q.to(cuda), cache[0].to(cuda), cache[1].to(cuda), torch.tensor([length], dtype=torch.int32, device=cuda),
                              k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda), **kw)


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (8, 2, 128), (8, 1, 72), (12, 1, 64), (40, 1, 128)])
@pytest.mark.parametrize("length", [100, 700])
@pytest.mark.parametrize("e", [63, 66, 112, 118])
def test_large_queries_of_small_keys(cuda, hq, hkv, d, length, e):
    cache, k, v, q = made(hq, hkv, d, length, e)
    q *= 2.0 ** e
    cache[2] *= 2.0 ** -e
    check(call(cuda, q, cache, length), expected(q, [k[0] * 2.0 ** -e], [v[0]], [length]))
    # some rows large, the others small, where all keys weigh alike
    q[:, ::2] *= 2.0 ** (-e - 40)
    check(call(cuda, q, cache, length, scale=-0.1), expected(q, [k[0] * 2.0 ** -e], [v[0]], [length], scale=-0.1))


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (12, 1, 128)])
def test_large_queries_take_one_key(cuda, hq, hkv, d):
    cache, k, v, q = made(hq, hkv, d, 100, 3)
    q *= 2.0 ** 117  # (scores below 2^124)
    y = call(cuda, q, cache, 100)
    for h in range(hq):
        want = v[0, (k[0, :, h // (hq // hkv)] @ q[0, h].double()).argmax(), h // (hq // hkv)]
        # a code times the three parts of the weight with its scale, whose sum is rounded twice, then the quotient and the product with it
        assert ((y[0, h].cpu().double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all(), h
