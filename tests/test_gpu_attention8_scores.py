"""Single tokens over a cache of 8 bits whose scores are far larger than any softmax tells apart: the best key's value alone."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _cache8 import random_cache

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (8, 2, 128), (8, 1, 72), (12, 1, 64), (40, 1, 128)])
@pytest.mark.parametrize("length", [100, 700])
@pytest.mark.parametrize("dtype,eq,ek,kw", [(F32, 20, 0, {}), (F32, 30, 0, {}), (F32, 40, 5, {}), (F32, 60, 30, {}), (F32, 20, -60, dict(scale=2.0 ** 90)),
                                            (F16, 13, 14, {}), (F16, 13, 30, {}), (F32, 40, 0, dict(biased=True)), (F16, 10, 0, dict(scale=-1e6))], ids=str)
def test_one_key_alone(cuda, hq, hkv, d, length, dtype, eq, ek, kw):
    gen = torch.Generator().manual_seed(length)
    cache, k, v = random_cache(1, length, hkv, d, "int8", gen)
    q = (torch.randn(1, hq, d, generator=gen) * 2.0 ** eq).to(dtype)
    cache[2] *= 2.0 ** ek
    kw = dict(kw)
    if kw.pop("biased", False):
        kw["slopes"] = torch.full((hq,), 0.5, device=cuda)
    y = g.attention_decode(q.to(cuda), cache[0].to(cuda), cache[1].to(cuda), torch.tensor([length], dtype=torch.int32, device=cuda),
                           k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda), **kw).cpu()
    scale, u = kw.get("scale", d ** -0.5), 2.0 ** -11 if dtype == F16 else 2.0 ** -24
    for h in range(hq):
        s = (k[0, :, h // (hq // hkv)] * 2.0 ** ek @ q[0, h].double()) * scale
        first, second = s.topk(2).values.tolist()
        # the scores' own rounding leaves the order: 4 sqrt(d) 2^-24 of the products' sizes, and 100 more for the second key's weight
        size = ((k[0, :, h // (hq // hkv)].abs() * 2.0 ** ek) @ q[0, h].double().abs()).max().item() * abs(scale)
        if first - second < 100 + 0.5 * length * ("slopes" in kw) + 8 * d ** 0.5 * 2.0 ** -24 * size:
            continue
        want = v[0, s.argmax(), h // (hq // hkv)]
        # the weight's parts, the quotient and the result are rounded
        assert ((y[0, h].double() - want).abs() <= (u + 2.0 ** -16 * (dtype == F16) + 4 * 2.0 ** -24) * want.abs()).all(), h
