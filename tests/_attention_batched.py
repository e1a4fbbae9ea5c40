"""``_attention.prompts`` for larger inputs: the same formulas and bounds in 64 bits, a sequence and key head at a time."""
from __future__ import annotations

import math

import torch

from _attention import bound


def prompts(q, k, v, lens_q, lens_k, causal=False, visible=None, shared_k=None, shared_v=None, scale=None, softcap=0.0, slopes=None):
    """Packed q [sum lens_q, hq, d], k, v [sum lens_k, hkv, d] in their own type: (out, bound) of the same rows."""
    hq, d = q.shape[1:]
    hkv = k.shape[1]
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    mean, err = torch.zeros_like(out), torch.zeros(q.shape[0], hq, 1, dtype=torch.float64)
    front = 0 if shared_k is None else shared_k.shape[0]
    a = b = 0
    for n, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        pos_q, pos_k = front + lk - lq + torch.arange(lq), torch.arange(front + lk)
        seen = torch.ones(lq, front + lk, dtype=torch.bool)
        if causal:
            seen = pos_k[None] <= pos_q[:, None]
            if visible is not None:
                seen = seen | (pos_k < int(visible[n]))[None]
        rows = slice(a, a + lq)
        for h in range(hkv if lq else 0):
            kk, vv = k[b:b + lk, h].double(), v[b:b + lk, h].double()
            if front:
                kk, vv = torch.cat((shared_k[:, h].double(), kk)), torch.cat((shared_v[:, h].double(), vv))
            if not kk.shape[0]:
                continue
            heads = slice(h * group, (h + 1) * group)
            qq = q[rows, heads].double().transpose(0, 1).contiguous()  # [group, lq, d]
            s = (qq @ kk.T) * scale
            size = (qq.abs() @ kk.abs().T) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes[heads].double()[:, None, None] * (pos_q[:, None] - pos_k[None]).abs()
            some = seen.any(1)
            s = s.masked_fill(~seen, -math.inf)
            w = torch.exp(s - s.amax(-1, keepdim=True).masked_fill(~some[None, :, None], 0.0))
            w = w / w.sum(-1, keepdim=True).masked_fill(~some[None, :, None], 1.0)
            out[rows, heads] = (w @ vv).transpose(0, 1)
            mean[rows, heads] = (w @ vv.abs()).transpose(0, 1)
            top, high = size.masked_fill(~seen, 0.0).amax(-1), s.abs().masked_fill(~seen, 0.0).amax(-1)
            e = 4 * math.sqrt(d) * 2.0 ** -24 * top + 8 * 2.0 ** -24 * (high + softcap) + 2.0 ** -22
            e = 2 * e + 4 * seen.sum(1).double().clamp(min=1).sqrt() * 2.0 ** -24
            err[rows, heads] = (e * some).transpose(0, 1)[..., None]
        a, b = a + lq, b + lk
    return out, bound(out, mean, err, q.dtype)
