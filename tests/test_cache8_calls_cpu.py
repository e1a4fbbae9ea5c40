"""CPU tests of the caches in 8 bits: tangents of e4m3 codes, and what strides the library takes before a launch."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gtx16_fp16 as g


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
