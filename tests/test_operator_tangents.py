"""CPU test: operands with a forward-mode tangent are refused, whichever they are (before anything else is looked at)."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gtx16_fp16 as g


def calls():
    q, k = torch.zeros(2, 8, 4, 64), torch.zeros(2, 8, 2, 64)
    attn = dict(q=q, k=k, v=k, shared_k=k[0], shared_v=k[0], slopes=torch.zeros(4))
    n = torch.ones(2, dtype=torch.int32)
    lora = dict(x2d=torch.zeros(4, 8), w_t=torch.zeros(8, 8), down=torch.zeros(1, 8, 8), up=torch.zeros(1, 8, 8), scale=torch.zeros(1),
                bias=torch.zeros(8))
    index = torch.zeros(4, dtype=torch.int32)

    def decode(q, k, v, **rest):
        return g.attention_decode(q[:, 0], k, v, n, **rest)

    return [(g.attention, attn), (decode, attn), (lambda **a: g.lora_mm_t(index=index, **a), lora)]


def test_tangents_are_refused():
    for call, operands in calls():
        for name in operands:
            with forward_ad.dual_level():
                given = dict(operands)
                given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
                with pytest.raises(RuntimeError, match="tangent"):
                    call(**given)
                # without one, the other checks answer (these tensors are on the CPU)
                with pytest.raises(ValueError):
                    call(**operands)
