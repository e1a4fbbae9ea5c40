"""Attention whose scores are far larger than any softmax tells apart: the best key's value alone. Prompts, single tokens, and a shared
prefix before a cache in 8 bits."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _cache8 import random_cache

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def check(y, q, k, v, scale):
    """y, q [rows, hq, d], k, v [keys, hkv, d] on the CPU: rows whose best key stands out."""
    y, q, k, v = y.cpu(), q.cpu().double(), k.cpu().double(), v.cpu().double()
    group, seen = q.shape[1] // k.shape[1], 0
    u = 2.0 ** -11 if y.dtype == F16 else 2.0 ** -24
    for r in range(q.shape[0]):
        for h in range(q.shape[1]):
            kk = k[:, h // group]
            s = (kk @ q[r, h]) * scale
            first, second = s.topk(2).values.tolist()
            # the products' own rounding, 4 sqrt(d) 2^-24 of their sizes, leaves the order, and 100 more leave the second key nothing
            if first - second < 100 + 8 * q.shape[2] ** 0.5 * 2.0 ** -24 * (kk.abs() @ q[r, h].abs()).max().item() * abs(scale):
                continue
            want = v[s.argmax(), h // group]
            # the weight (fp16 queries': of a shared prefix and of 16 bits, too), the quotient and the result are rounded
            assert ((y[r, h].double() - want).abs() <= ((2 if y.dtype == F16 else 1) * u + 4 * 2.0 ** -24) * want.abs()).all(), (r, h)
            seen += 1
    assert seen


CASES = [(F32, 30, 0, {}), (F32, 40, 5, {}), (F32, 60, 30, {}), (F32, 20, -60, dict(scale=2.0 ** 90)), (F16, 12, 12, {}), (F16, 11, 5, dict(scale=-1e6)),
         (F16, 12, 12, dict(scale=3.0))]


def operands(cuda, rows, keys, hq, hkv, d, dtype, eq, ek, seed):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(*s, generator=gen) for s in ((rows, hq, d), (keys, hkv, d), (keys, hkv, d)))
    return (q * 2.0 ** eq).to(dtype).to(cuda), (k * 2.0 ** ek).to(dtype).to(cuda), v.to(dtype).to(cuda)


@pytest.mark.parametrize("dtype,eq,ek,kw", CASES, ids=str)
@pytest.mark.parametrize("rows,keys,hq,hkv,d", [(1, 100, 2, 2, 64), (40, 300, 4, 2, 128), (200, 257, 3, 3, 64), (17, 3000, 2, 1, 96), (3, 33, 8, 1, 32)])
def test_prompts(cuda, rows, keys, hq, hkv, d, dtype, eq, ek, kw):
    q, k, v = operands(cuda, rows, keys, hq, hkv, d, dtype, eq, ek, rows)
    check(g.attention(q[None], k[None], v[None], **kw)[0], q, k, v, kw.get("scale", d ** -0.5))


@pytest.mark.parametrize("dtype,eq,ek,kw", CASES, ids=str)
@pytest.mark.parametrize("keys,shared,hq,hkv,d", [(100, 0, 2, 2, 64), (3000, 0, 8, 2, 128), (200, 70, 8, 1, 72), (10, 900, 40, 1, 128), (600, 300, 4, 4, 64)])
def test_single_tokens(cuda, keys, shared, hq, hkv, d, dtype, eq, ek, kw):
    q, k, v = operands(cuda, 1, keys + shared, hq, hkv, d, dtype, eq, ek, keys)
    prefix = dict(shared_k=k[:shared], shared_v=v[:shared]) if shared else {}
    n = torch.tensor([keys], dtype=torch.int32, device=cuda)
    check(g.attention_decode(q, k[None, shared:], v[None, shared:], n, **prefix, **kw), q, k, v, kw.get("scale", d ** -0.5))


@pytest.mark.parametrize("dtype,eq,ek,kw", CASES, ids=str)
@pytest.mark.parametrize("keys,shared,hq,hkv,d", [(100, 70, 2, 2, 64), (700, 300, 8, 2, 128), (200, 70, 8, 1, 72), (10, 900, 40, 1, 128), (600, 300, 4, 4, 64)])
def test_a_prefix_before_a_cache_in_8_bits(cuda, keys, shared, hq, hkv, d, dtype, eq, ek, kw):
    q, k, v = operands(cuda, 1, shared, hq, hkv, d, dtype, eq, ek, keys)
    cache, k8, v8 = random_cache(1, keys, hkv, d, "int8", torch.Generator().manual_seed(1))
    cache[2] *= 2.0 ** ek
    n = torch.tensor([keys], dtype=torch.int32, device=cuda)
    y = g.attention_decode(q, cache[0].to(cuda), cache[1].to(cuda), n, shared_k=k, shared_v=v, k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda), **kw)
    both = torch.cat((k.cpu().double(), k8[0] * 2.0 ** ek)), torch.cat((v.cpu().double(), v8[0]))
    check(y, q, *both, kw.get("scale", d ** -0.5))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq", [2, 12])
def test_a_key_of_the_prefix_and_its_like_in_8_bits(cuda, dtype, hq):
    # the same key before and in the cache, exactly: half of the weight each, however large the score
    d, gen = 64, torch.Generator().manual_seed(0)
    cache, _, v8 = random_cache(1, 5, 1, d, "int8", gen)
    cache[0].zero_()
    cache[0][0, 2, 0, 0], cache[2][0] = 64, 2.0 ** -4
    k, v = torch.zeros(7, 1, d), torch.randn(7, 1, d, generator=gen).to(dtype)
    k[4, 0, 0] = 4.0
    q = torch.zeros(1, hq, d)
    q[:, :, 0] = 2.0 ** 10 * (1 + torch.arange(hq) / 16)
    want = (v[4].double() + v8[0, 2]) / 2
    n = torch.tensor([5], dtype=torch.int32, device=cuda)
    u = 2.0 ** -11 if dtype == F16 else 2.0 ** -24
    for step in range(50):  # scores from 2^23 on, which are rounded alike on both sides
        scale = 2.0 ** (step / 3 + 11) * 1.07
        y = g.attention_decode(q.to(dtype).to(cuda), cache[0].to(cuda), cache[1].to(cuda), n, shared_k=k.to(dtype).to(cuda), shared_v=v.to(cuda),
                               k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda), scale=scale).cpu()
        # (the other keys, of score 0, get nothing) the weights are 1 and exact; their sums' products and the result are rounded
        off = (y[0].double() - want).abs() - (u * want.abs() + (2.0 ** -16 if dtype == F16 else 2.0 ** -21) * (v[4].double().abs() + v8[0, 2].abs()))
        assert (off <= 0).all(), scale
