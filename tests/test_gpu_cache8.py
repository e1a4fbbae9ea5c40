"""A cache of 8 bits on the GPU, bit for bit against the formats' definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _cache8 import CODES, coded, empty, numbers

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def rows_of(n, heads, d, dtype, seed=0):
    """k, v [n, heads, d] on the CPU: normal rows, and some of each kind that is written in its own way."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for _ in "kv":
        x = torch.randn(n, heads, d, generator=gen)
        x *= 2.0 ** torch.randint(-12, 5, (n, heads, 1), generator=gen)
        kinds = torch.randint(0, 12, (n, heads), generator=gen)
        x[kinds == 0] = 0.0
        x[kinds == 1] *= -0.0
        ties = torch.randint(-253, 254, (n, heads, d), generator=gen) * 0.5  # halves of a code where the scale is 1
        ties[..., 0] = 127.0
        x = torch.where((kinds == 2)[..., None], ties, x)
        fives = torch.randint(-14, 15, (n, heads, d), generator=gen) * 2.0 ** torch.randint(-6, 5, (n, heads, d), generator=gen)
        fives[..., -1] = 448.0  # an e4m3 scale's border, exactly
        x = torch.where((kinds == 3)[..., None], fives * 2.0 ** -3, x)
        if dtype == F32:
            x[kinds == 4] *= 2.0 ** -100  # about the least
            x[kinds == 5] *= 2.0 ** 120
            x[kinds == 6] *= 2.0 ** -140
        else:
            x[kinds == 4] *= 2.0 ** -22  # fp16's subnormals
            x[kinds == 5] *= 2.0 ** 9
        out.append(x.to(dtype))
    return out


def check(cache, before, k, v, slots, code):
    """`cache` after a write of k, v to `slots` (CPU) that it was `before`, every byte of it."""
    pages, page, heads, d = cache[0].shape
    last = {}
    for r, s in enumerate(slots.reshape(-1).tolist()):
        if 0 <= s < pages * page:
            last[s] = r
    at, rows = torch.tensor(list(last), dtype=torch.long), torch.tensor(list(last.values()), dtype=torch.long)
    for x, codes, scale, old_codes, old_scale in ((k, cache[0], cache[2], before[0], before[2]), (v, cache[1], cache[3], before[1], before[3])):
        y, s = coded(x.reshape(-1, heads, d)[rows], code)
        want, want_s = numbers(old_codes).reshape(-1, heads, d), old_scale.cpu().double().reshape(-1, heads)
        want[at], want_s[at] = y, s
        torch.testing.assert_close(numbers(codes).reshape(-1, heads, d), want, rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(scale.cpu().double().reshape(-1, heads), want_s, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,heads,d,pages,page,by_head", [(1, 1, 8, 1, 1, False), (1, 12, 64, 1, 300, False), (17, 3, 72, 5, 7, False), (40, 8, 128, 9, 16, True),
                                                          (40, 8, 128, 9, 16, False), (300, 2, 16, 30, 24, True), (33, 5, 24, 4, 16, False),
                                                          (70, 1, 32, 3, 64, True), (20, 9, 96, 2, 16, False), (2500, 2, 40, 200, 16, False)])
def test_written_codes(cuda, code, dtype, n, heads, d, pages, page, by_head):
    k, v = rows_of(n, heads, d, dtype, seed=n + d)
    gen = torch.Generator().manual_seed(1)
    slots = torch.randperm(max(n, pages * page), generator=gen)[:n].to(torch.int32)  # some past the end where it is small
    slots[n // 2] = -1 if n > 2 else slots[n // 2]
    cache = empty(pages, page, heads, d, code, cuda, by_head)
    before = [t.clone() for t in cache]
    g.cache_write(k.to(cuda), v.to(cuda), *cache, slots.to(cuda))
    check(cache, before, k, v, slots, code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_what_is_not_finite(cuda, code, dtype):
    k, v = (torch.randn(6, 2, 64).to(dtype) for _ in "kv")
    k[0, 0, 3], k[1, 1, 63], v[2, 0, 0], v[3, 1, 17] = float("inf"), float("nan"), float("-inf"), float("nan")
    cache = empty(1, 8, 2, 64, code, cuda)
    before = [t.clone() for t in cache]
    slots = torch.arange(6, dtype=torch.int32)
    g.cache_write(k.to(cuda), v.to(cuda), *cache, slots.to(cuda))
    check(cache, before, k, v, slots, code)
    kk, vv = g.cache_read(*cache, slots.to(cuda), out_dtype=dtype)
    assert torch.isnan(kk[0, 0]).all() and torch.isnan(kk[1, 1]).all() and torch.isnan(vv[2, 0]).all() and torch.isnan(vv[3, 1]).all()
    assert torch.isnan(kk).sum() == torch.isnan(vv).sum() == 128


@pytest.mark.parametrize("n,slots", [(2, 1), (64, 3), (700, 100), (5000, 4000), (5000, 1), (70000, 50000)])
def test_one_slot_several_times(cuda, n, slots):
    # the last row's codes and scale, whole, wherever the rows stand
    gen = torch.Generator().manual_seed(n)
    at = torch.randint(0, slots, (n,), generator=gen).to(torch.int32)
    k, v = (torch.randn(n, 1, 8, generator=gen).half() for _ in "kv")
    for _ in range(3):
        cache = empty(slots, 1, 1, 8, "int8", cuda)
        before = [t.clone() for t in cache]
        g.cache_write(k.to(cuda), v.to(cuda), *cache, at.to(cuda))
        check(cache, before, k, v, at, "int8")


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape,heads,d,pages,page,by_head", [((1,), 1, 8, 1, 1, False), ((3, 5), 3, 72, 5, 7, False), ((129,), 8, 128, 9, 16, True),
                                                              ((2, 2, 2), 2, 64, 3, 16, False), ((1000,), 1, 24, 3, 10, True), ((0,), 2, 64, 3, 16, False)])
def test_read(cuda, code, dtype, shape, heads, d, pages, page, by_head):
    k, v = rows_of(pages * page, heads, d, dtype, seed=d)
    cache = empty(pages, page, heads, d, code, cuda, by_head)
    g.cache_write(k.to(cuda), v.to(cuda), *cache, torch.arange(pages * page, dtype=torch.int32, device=cuda))
    gen = torch.Generator().manual_seed(2)
    slots = torch.randint(-3, pages * page + 3, shape, generator=gen).to(torch.int32)
    got = g.cache_read(*cache, slots.to(cuda), out_dtype=dtype)
    inside = ((slots >= 0) & (slots < pages * page))[..., None, None]
    for y, x in zip(got, (k, v)):
        c, s = coded(x, code)
        want = (c * s[..., None]).float().to(dtype)  # (a product of 8 and 24 bits, rounded to fp32 first)
        want = torch.where(inside, want[slots.long().clamp(0, pages * page - 1)], torch.zeros((), dtype=dtype))
        assert y.dtype == dtype and y.shape == (*shape, heads, d) and y.is_contiguous()
        torch.testing.assert_close(y.cpu(), want, rtol=0, atol=0, equal_nan=True)


def test_types_of_rows_and_of_what_is_read(cuda):
    k, v = rows_of(20, 2, 64, F16)
    cache = empty(2, 10, 2, 64, "int8", cuda)
    slots = torch.arange(20, dtype=torch.int32, device=cuda)
    g.cache_write(k.to(cuda), v.to(cuda), *cache, slots)
    a, b = (g.cache_read(*cache, slots, out_dtype=t)[0] for t in (F32, F16))
    assert a.dtype == F32 and torch.equal(a.half(), b)


def test_views(cuda):
    # slices of a fused projection, batches of tokens, rows that have to be copied, caches inside larger tensors
    fused = torch.randn(2, 5, 9, 64, device=cuda).half()
    k, v = fused[:, :, 3:6], fused[:, :, 6:]
    slots = torch.randperm(32, device=cuda)[:10].to(torch.int32).view(2, 5)
    both = torch.full((2, 16, 2, 3, 64), 7, dtype=torch.int8, device=cuda)
    scales = torch.full((2, 3, 16, 2), 0.25, device=cuda)
    cache = [both[:, :, 0], both[:, :, 1], scales[..., 0].transpose(1, 2), scales[..., 1].transpose(1, 2)]
    before = [t.clone() for t in cache]
    g.cache_write(k, v, *cache, slots)
    check(cache, before, k.cpu(), v.cpu(), slots.cpu(), "int8")
    odd = torch.randn(10, 3 * 64 + 1, device=cuda).half()[:, 1:].unflatten(1, (3, 64))
    before = [t.clone() for t in cache]
    g.cache_write(odd, odd.flip(0), *cache, slots.view(-1)[::2].repeat(2))
    check(cache, before, odd.cpu(), odd.flip(0).cpu(), slots.view(-1)[::2].repeat(2).cpu(), "int8")


def test_slots_past_32_bits_of_bytes(cuda):
    heads, d, page = 8, 128, 16
    pages = (1 << 32) // (heads * d * page) + 4  # over 4 GiB of codes
    k_cache = torch.empty(pages, page, heads, d, dtype=torch.int8, device=cuda)
    v_cache = torch.empty_like(k_cache)
    k_scale, v_scale = (torch.empty(pages, page, heads, device=cuda) for _ in "kv")
    slots = torch.tensor([pages * page - 1, 0, pages * page - 40, pages * page], dtype=torch.int32, device=cuda)
    k, v = (torch.randn(4, heads, d, device=cuda).half() for _ in "kv")
    g.cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots)
    for y, x in zip(g.cache_read(k_cache, v_cache, k_scale, v_scale, slots, out_dtype=F32), (k, v)):
        c, s = coded(x.cpu(), "int8")
        assert torch.equal(y.cpu()[:3], (c * s[..., None]).float()[:3]) and not y[3].any()


def test_many_rows(cuda):
    # more rows than a launch has, slots that come again in a later one, and rows that are not written
    n, pages, page = 70000, 9, 5000
    gen = torch.Generator().manual_seed(3)
    slots = torch.randint(-9000, pages * page, (n,), generator=gen, dtype=torch.int32)
    slots[[5, 40000, 69999]] = 17
    slots[[6, 32767, 32768]] = 18
    k, v = (torch.randn(n, 2, 8, generator=gen).half() for _ in "kv")
    cache = empty(pages, page, 2, 8, "int8", cuda)
    before = [t.clone() for t in cache]
    g.cache_write(k.to(cuda), v.to(cuda), *cache, slots.to(cuda))
    check(cache, before, k, v, slots, "int8")


def test_graphs(cuda):
    cache = empty(4, 16, 2, 64, "e4m3", cuda)
    k, v = (torch.randn(9, 2, 64, device=cuda).half() for _ in "kv")
    slots = torch.randperm(64, device=cuda)[:9].to(torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            g.cache_write(k, v, *cache, slots)
            got = g.cache_read(*cache, slots)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        k.mul_(1.5), v.neg_(), slots.copy_(torch.randperm(64, device=cuda)[:9])
        before = [t.clone() for t in cache]
        graph.replay()
        torch.cuda.synchronize()
        check(cache, before, k.cpu(), v.cpu(), slots.cpu(), "e4m3")
        again = g.cache_read(*cache, slots)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_nothing(cuda):
    cache = empty(2, 4, 2, 64, "int8", cuda)
    before = [t.clone() for t in cache]
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    g.cache_write(torch.empty(0, 2, 64, dtype=F16, device=cuda), torch.empty(0, 2, 64, dtype=F16, device=cuda), *cache, none)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    void = empty(0, 4, 2, 64, "int8", cuda)
    x = torch.ones(3, 2, 64, dtype=F16, device=cuda)
    slots = torch.arange(3, dtype=torch.int32, device=cuda)
    g.cache_write(x, x, *void, slots)
    assert not torch.stack(g.cache_read(*void, slots)).any()


def test_refusals(cuda):
    kc, vc, ks, vs = empty(2, 4, 2, 64, "int8", cuda)
    x, slots = torch.zeros(3, 2, 64, dtype=F16, device=cuda), torch.arange(3, dtype=torch.int32, device=cuda)
    e4 = empty(2, 4, 2, 64, "e4m3", cuda)[0]
    shifted = torch.zeros(2 * 4 * 2 * 64 + 4, dtype=torch.int8, device=cuda)[4:].view(2, 4, 2, 64)
    whole = dict(kc=kc, vc=vc, ks=ks, vs=vs)
    for bad in (dict(kc=e4), dict(vc=e4), dict(kc=kc.half()), dict(kc=kc[0]), dict(ks=ks.double()), dict(ks=ks[..., :1]), dict(vs=vs.cpu()), dict(kc=shifted),
                dict(vc=vc.transpose(2, 3)), dict(kc=kc.cpu()), dict(kc=kc[..., :60], vc=vc[..., :60])):
        with pytest.raises(ValueError):
            g.cache_write(x, x, *(whole | bad).values(), slots)
        with pytest.raises(ValueError):
            g.cache_read(*(whole | bad).values(), slots)
    for kk, vv, at in ((x, x[:2], slots), (x.bfloat16(), x.bfloat16(), slots), (x.float(), x, slots), (x[:, :1], x[:, :1], slots), (x, x, slots.long()),
                       (x, x, slots[:2]), (x, x, slots[:, None]), (x.cpu(), x.cpu(), slots), (x, x, slots.cpu())):
        with pytest.raises(ValueError):
            g.cache_write(kk, vv, kc, vc, ks, vs, at)
    with pytest.raises(ValueError, match="of their own"):
        g.cache_write(x, x, kc[:1].expand(2, -1, -1, -1), vc, ks, vs, slots)
    with pytest.raises(ValueError):
        g.cache_read(kc, vc, ks, vs, slots, out_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        g.cache_read(kc, vc, ks, vs, slots.long())
    with pytest.raises(RuntimeError, match="no gradient"):
        g.cache_write(x.clone().requires_grad_(), x, kc, vc, ks, vs, slots)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_read_where_written_is_near(cuda, code):
    # Half a step: max / 254 of a head, or 2^-4 of a value and half of the smallest one's step. int8's two quotients, the
    # product read and the difference taken here are rounded to fp32, 2^-24 each of at most 127 steps: 4 * 254 * 2^-24 < 2^-14
    # of half a step.
    k, v = (torch.randn(400, 4, 128, device=cuda) for _ in "kv")
    cache = empty(25, 16, 4, 128, code, cuda)
    slots = torch.randperm(400, device=cuda).to(torch.int32)
    g.cache_write(k, v, *cache, slots)
    for y, x in zip(g.cache_read(*cache, slots, out_dtype=F32), (k, v)):
        top = x.abs().amax(-1, keepdim=True)
        bound = top / 254 * (1 + 2.0 ** -14) if code == "int8" else x.abs() * 2.0 ** -4 + top / 224 * 2.0 ** -10
        assert ((y - x).abs() <= bound).all()
    assert cache[0].dtype == CODES[code]
