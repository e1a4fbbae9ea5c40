"""Single tokens over a cache of 8 bits with fp32 queries: values whose scales are far apart, of which the large ones get next to no weight."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check
from _cache8 import random_cache
from test_gpu_attention8 import expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (8, 1, 64), (16, 1, 128), (32, 1, 72)])
@pytest.mark.parametrize("length,at", [(40, 3), (130, 70), (130, 129), (900, 0), (900, 700), (900, 899)])
@pytest.mark.parametrize("low,high", [(-20, 20), (-60, 40), (-90, 60), (-40, 120)])
def test_a_large_value_without_weight(cuda, hq, hkv, d, length, at, low, high):
    # The key at `at` has values 2^(high - low) times the others' and scores that leave it exp(-300) or so: less than fp32 holds, so
    # the others alone make the result. Half of the heads see it with the weight of the rest instead.
    gen = torch.Generator().manual_seed(length + at)
    cache, k, v = random_cache(1, length, hkv, d, "int8", gen)
    q = torch.randn(1, hq, d, generator=gen)
    k[0, at] = 0.0
    cache[0][0, at] = 0
    k[0, at, :, 0], cache[0][0, at, :, 0], cache[2][0, at] = 127.0, 127, 1.0
    group = hq // hkv
    for h in range(hq):  # the score of that key: -300, or about the others'
        q[0, h, 0] = -300.0 * d ** 0.5 / 127.0 if (h % group) % 2 == 0 else 0.0
    k[0, :, :, 0] *= (torch.arange(length) == at)[:, None]  # (the others do not see the query's first value)
    cache[0][0, :, :, 0] *= (torch.arange(length) == at)[:, None]
    factor = torch.full((length, 1), 2.0 ** low)
    factor[at] = 2.0 ** high
    cache[3][0] *= factor
    v[0] *= factor.double()[..., None]
    y = g.attention_decode(q.to(cuda), cache[0].to(cuda), cache[1].to(cuda), torch.tensor([length], dtype=torch.int32, device=cuda),
                           k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda))
    check(y, expected(q, [k[0]], [v[0]], [length]))


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (8, 2, 128), (12, 1, 64), (20, 1, 128)])
@pytest.mark.parametrize("length", [60, 200, 1500])
@pytest.mark.parametrize("rise,fall", [(300.0, 120), (300.0, -120), (40.0, 60), (40.0, -60), (-200.0, 100), (-200.0, -100)])
def test_scores_and_scales_that_move_along_the_keys(cuda, hq, hkv, d, length, rise, fall):
    # scores rise (or fall) by `rise` from the first key to the last, values fall by 2^-fall: the sums are now those of the first
    # keys, now of the last
    gen = torch.Generator().manual_seed(length)
    cache, k, v = random_cache(1, length, hkv, d, "int8", gen)
    q = torch.randn(1, hq, d, generator=gen)
    q[:, :, 0] = d ** 0.5 / 127.0
    part = torch.linspace(0.0, 1.0, length).double()
    k *= 0.0
    cache[0].zero_()
    k[0, :, :, 0], cache[0][0, :, :, 0] = 127.0, 127
    cache[2][0] = (rise * part).float()[:, None]
    k[0] *= cache[2][0].double()[..., None]
    factor = 2.0 ** torch.round(fall * (0.5 - part))
    cache[3][0] *= factor.float()[:, None]
    v[0] *= factor[:, None, None]
    y = g.attention_decode(q.to(cuda), cache[0].to(cuda), cache[1].to(cuda), torch.tensor([length], dtype=torch.int32, device=cuda),
                           k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda))
    check(y, expected(q, [k[0]], [v[0]], [length]))
