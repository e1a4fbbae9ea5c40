"""A cache of 8 bits on the GPU as autograd sees it, and what many rows of one slot cost."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _cache8 import empty

pytestmark = pytest.mark.gpu


def rows(n, heads, d, cuda):
    return [torch.randn(n, heads, d, device=cuda).half() for _ in "kv"]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("usual", [True, False])
def test_a_gradient_wanted_of_the_cache_is_refused(cuda, which, usual):
    # e4m3 codes are floating numbers, of which autograd takes a gradient; `usual`: what the extension looks at, else the Python functions
    cache = empty(3, 16, 2, 64, "e4m3", cuda)
    k, v = rows(3, 2, 64, cuda)
    slots, lengths = torch.arange(3, dtype=torch.int32, device=cuda), torch.ones(3, dtype=torch.int32, device=cuda)
    q = torch.randn(3, 4, 64, device=cuda).half()
    if not usual:
        k, v, slots, lengths = k[None], v[None], slots[None], lengths.repeat(2)[::2]
    calls = (lambda: g.cache_write(k, v, *cache, slots), lambda: g.cache_read(*cache, slots),
             lambda: g.attention_decode(q, cache[0], cache[1], lengths, k_scale=cache[2], v_scale=cache[3]))
    g.cache_write(k, v, *cache, slots)
    cache[which].requires_grad_()
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        for call in calls:
            call()


@pytest.mark.parametrize("usual", [True, False])
def test_a_write_is_seen_by_autograd(cuda, usual):
    # what torch's own operations in place do: a tensor that backward needs as it was is missed
    cache = empty(2, 16, 2, 64, "int8", cuda, fill=0)
    k, v = rows(3, 2, 64, cuda)
    slots = torch.arange(3, dtype=torch.int32, device=cuda)
    if not usual:
        k, v, slots = k[None], v[None], slots[None]
    before = [t._version for t in cache]
    w = torch.ones_like(cache[2], requires_grad=True)
    loss = (w * cache[2]).sum()
    view = cache[3][0]
    g.cache_write(k, v, *cache, slots)
    assert all(t._version > n for t, n in zip(cache, before)) and view._version == cache[3]._version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    g.cache_read(*cache, slots)
    after = [t._version for t in cache]
    g.attention_decode(torch.randn(2, 4, 64, device=cuda).half(), cache[0], cache[1], torch.ones(2, dtype=torch.int32, device=cuda), k_scale=cache[2],
                       v_scale=cache[3])
    assert [t._version for t in cache] == after  # (nobody else changes them)


def test_a_cache_made_in_inference_mode(cuda):
    with torch.inference_mode():
        cache = empty(2, 16, 2, 64, "int8", cuda, fill=0)
    k, v = rows(3, 2, 64, cuda)
    slots = torch.arange(3, dtype=torch.int32, device=cuda)
    g.cache_write(k, v, *cache, slots)
    with torch.inference_mode():
        g.cache_write(k, v, *cache, slots + 3)
    a, b = (g.cache_read(*cache, s)[0] for s in (slots, slots + 3))
    assert a.any() and torch.equal(a, b)


def test_many_rows_of_one_slot_cost_no_more(cuda):
    # Rows of a padded batch may all name one slot that nobody reads: they are passed over together. (Rows of slots of their own take
    # 46 us; twice that leaves room for a busy card. Where each was compared by itself, they took 400 to 750.)
    n = 32768
    k, v = rows(n, 8, 128, cuda)
    cache = empty(n // 16, 16, 8, 128, "int8", cuda)
    own = torch.randperm(n, device=cuda).to(torch.int32)
    one = torch.full_like(own, 5)
    half = torch.where(torch.arange(n, device=cuda) % 2 == 0, own, one).to(torch.int32)
    tail = own.clone()
    tail[n // 4:] = 5

    def least(slots):
        times = []
        for _ in range(7):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            for _ in range(4):
                g.cache_write(k, v, *cache, slots)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    apart = least(own)
    for slots in (one, half, tail):
        assert least(slots) <= 2 * apart
