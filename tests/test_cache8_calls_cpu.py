"""CPU tests of the caches in 8 bits: tangents of e4m3 codes, and what strides the library takes before a launch."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gtx16_fp16 as g
from test_cache8_cpu import ALIGN, SHAPE, WORKSPACE, decode_call, decode_size


def test_tangents_of_e4m3_codes_are_refused():
    x, at = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    c, s = torch.zeros(2, 4, 2, 64).to(torch.float8_e4m3fn), torch.zeros(2, 4, 2)
    calls = (lambda kc, vc: g.cache_write(x, x, kc, vc, s, s, at), lambda kc, vc: g.cache_read(kc, vc, s, s, at),
             lambda kc, vc: g.attention_decode(x, kc, vc, at, k_scale=s, v_scale=s))
    for call in calls:
        for which in range(2):
            with forward_ad.dual_level():
                given = [c, c]
                given[which] = forward_ad.make_dual(c, torch.zeros_like(c))
                with pytest.raises(RuntimeError, match="tangent"):
                    call(*given)
                with pytest.raises(ValueError):  # (these tensors are on the CPU)
                    call(c, c)


@pytest.mark.parametrize("step", [1 << 30, 1 << 24, 0, 8])
def test_tokens_far_apart_and_on_top_of_each_other_are_taken(step):
    # without a workspace the call ends where everything else has been looked at, before a launch
    long = dict(k_len=8000, page=8000, k_token=step, v_token=step)
    assert decode_size(**long) > 0 and decode_call(**long) == WORKSPACE


def test_a_workspace_does_not_lift_the_other_checks():
    long = dict(k_len=8000, page=8000)
    assert decode_call(**long, k_token=(1 << 30) + 4) == ALIGN and decode_call(**long, v_head=4) == ALIGN
    # keys are counted in 32 bits with room: up to 2^30 in all
    assert decode_call(k_len=(1 << 30) + 1, page=(1 << 30) + 1) == SHAPE and decode_size(k_len=(1 << 30) + 1, page=(1 << 30) + 1) == 0
