"""GPU tests of fp32 attention over fp32's range: values of unlike sizes beside each other, in both shapes of
workgroup of a prompt and for single tokens. The bounds are ``_attention``'s, which go by each row's scores
and each column's values, with nothing added for the sizes around them."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check, tokens
from _attention_batched import prompts
from _plans import prompt_plan

pytestmark = pytest.mark.gpu

F32 = torch.float32
# (sequences, rows and keys of each, query heads, key heads): a workgroup's rows
SHAPES = {32: (2, 45, 50, 2, 1), 128: (12, 140, 140, 24, 12)}


def data(shape, d=64, seed=0):
    n, rows, keys, hq, hkv = SHAPES[shape]
    assert prompt_plan(rows, keys, hq, hkv, d, True, n, packed=False)[0] == shape
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(n, m, h, d, generator=gen) for m, h in ((rows, hq), (keys, hkv), (keys, hkv))]


def compare(cuda, q, k, v, **rest):
    n, rows, keys = q.shape[0], q.shape[1], k.shape[1]
    y = g.attention(q.to(cuda), k.to(cuda), v.to(cuda), **rest)
    check(y.flatten(0, 1), prompts(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), [rows] * n, [keys] * n, **rest))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("f", [1e3, 1e6, 1e8, 1e12, 1e25])
@pytest.mark.parametrize("large", ["q", "k"])
def test_channels_of_unlike_size_in_queries_and_keys(cuda, shape, f, large):
    # the scores are those of unit normal queries and keys
    q, k, v = data(shape, seed=1)
    by = torch.ones(64)
    by[5:13] = f if large == "q" else 1 / f
    compare(cuda, q * by, k / by, v)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("small", [1e-4, 1e-8, 1e-15, 1e-30])
def test_channels_of_unlike_size_in_values(cuda, shape, small):
    q, k, v = data(shape, seed=2)
    v[..., 3:9] *= small
    v[..., 40:] /= small
    compare(cuda, q, k, v)


@pytest.mark.parametrize("shape", SHAPES)
def test_keys_and_values_of_unlike_size_in_one_tile(cuda, shape):
    q, k, v = data(shape, seed=3)
    k[:, ::3] *= 1e-7
    v[:, 1::4] *= 1e-9
    v[:, ::5] *= 1e9
    compare(cuda, q, k, v, causal=True)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e20, 1e30])
def test_small_queries_on_large_keys_and_the_other_way_round(cuda, shape, size):
    q, k, v = data(shape, seed=4)
    compare(cuda, q * size, k / size, v)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1e-35, 1e33, 2.5e38])
def test_values_near_the_ends_of_the_range(cuda, shape, size):
    q, k, v = data(shape, seed=5)
    compare(cuda, q, k, v.clamp(-1, 1) * size)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinite_and_nan_operands(cuda, shape, bad):
    # One row's query, one key and one value. The cap makes an infinite score as good as a large one, so every other
    # row, and where they are infinite those rows, too, have their values.
    q, k, v = data(shape, seed=6)
    n, rows, keys, hq, hkv = SHAPES[shape]
    size = max((q[i].abs().transpose(0, 1).unflatten(0, (hkv, -1)) @ k[i].abs().permute(1, 2, 0)[:, None]).max().item() for i in range(n)) / 8
    large = 3e38 if bad > 0 else -3e38
    args, same = [q.clone(), k.clone(), v.clone()], [q.clone(), k.clone(), v.clone()]
    for at, value in ((args, bad), (same, large)):
        at[0][0, 3, 0, 7] = at[1][1, 30, 0, 2] = value
    args[2][0, 11, 0, 9] = bad
    y = g.attention(*(t.to(cuda) for t in args), softcap=20.0).cpu()
    out = prompts(*(t.flatten(0, 1) for t in same), [rows] * n, [keys] * n, softcap=20.0)[0].unflatten(0, (n, rows))
    # (_attention's bound, with the largest score of the finite operands and the largest value)
    e = 2 * (4 * 8 * 2.0 ** -24 * size + 8 * 2.0 ** -24 * 40 + 2.0 ** -22) + 4 * keys ** 0.5 * 2.0 ** -24
    tol = 2.0 ** -24 * out.abs() + e * v.abs().max()
    assert not torch.isfinite(y[0, :, :hq // hkv, 9]).any()
    keep = torch.ones(y.shape, dtype=torch.bool)
    keep[0, :, :hq // hkv, 9] = False
    if bad != bad:
        assert y[0, 3, 0].isnan().all() and y[1, :, :hq // hkv].isnan().all()
        keep[0, 3, 0] = keep[1, :, :hq // hkv] = False
    over = ((y.double() - out).abs() / tol)[keep]
    assert torch.isfinite(over).all() and over.max() <= 1.0, f"{over.max():.3g} times the bound"


@pytest.mark.parametrize("shared", [0, 300])
@pytest.mark.parametrize("requests", [3, 70])
def test_tokens_with_channels_of_unlike_size(cuda, shared, requests):
    gen = torch.Generator().manual_seed(7)
    by = torch.ones(64)
    by[5:13], by[20:24] = 1e7, 1e-9
    lengths = [(37 * i) % 90 + 1 for i in range(requests)]
    q = torch.randn(requests, 4, 64, generator=gen) * by
    k, v = torch.randn(requests, 90, 2, 64, generator=gen) / by, torch.randn(requests, 90, 2, 64, generator=gen) * by
    sk, sv = (torch.randn(shared, 2, 64, generator=gen) / by, torch.randn(shared, 2, 64, generator=gen) * by) if shared else (None, None)
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    y = g.attention_decode(put(q), put(k), put(v), torch.tensor(lengths, dtype=torch.int32, device=cuda), shared_k=put(sk), shared_v=put(sv))
    check(y, tokens(q, list(k), list(v), lengths, sk, sv))
