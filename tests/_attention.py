"""Plain attention in 64 bits, row by row of a sequence, and how far fp32 arithmetic may be from it.

``reference`` takes numpy-free CPU tensors and returns the output and a bound for each of its values; the
bound is what the formulas allow, not what a kernel happens to reach:

* the output is rounded once to its type (u = 2^-11 or 2^-24 of its magnitude);
* with fp16 inputs each weight is rounded to fp16, which moves the result by at most u times the
  weighted mean of |v|;
* an error e of a score (log units) changes its weight by a factor 1 + e, and so the result by at most 2 e
  times the weighted mean of |v|. e: the fp32 product q.k over d terms (random roundings: 4 sqrt(d) 2^-24 of
  the sum of |q k|, scaled), and the handful of fp32 steps from there to the exponential, each 2^-24 of
  the score's magnitude or of the softcap, eight of them, and 2^-22 for the exponential itself;
* the sums over n weights in fp32: 4 sqrt(n) 2^-24.
"""
from __future__ import annotations

import math

import torch

NEG = float("-inf")


def one_sequence(q, k, v, pos_q, pos_k, seen, scale, cap, slopes):
    """q [rows, hq, d], k, v [keys, hkv, d] (doubles), positions, seen [rows, keys]: (out, bound) [rows, hq, d]."""
    rows, hq, d = q.shape
    keys, hkv = k.shape[:2]
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    mean, err = torch.zeros_like(out), torch.zeros(rows, hq, 1, dtype=torch.float64)
    for h in range(hq):
        for i in range(rows):
            at = seen[i].nonzero().flatten()
            if not at.numel():
                continue
            kk, vv = k[at, h // (hq // hkv)], v[at, h // (hq // hkv)]
            s = (kk @ q[i, h]) * scale
            size = (kk.abs() @ q[i, h].abs()) * abs(scale)
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s - float(slopes[h]) * (pos_q[i] - pos_k[at]).abs()
            w = torch.exp(s - s.max())
            w = w / w.sum()
            out[i, h] = w @ vv
            mean[i, h] = w @ vv.abs()
            e = 4 * math.sqrt(d) * 2.0 ** -24 * size.max() + 8 * 2.0 ** -24 * (s.abs().max() + cap) + 2.0 ** -22
            err[i, h] = 2 * e + 4 * math.sqrt(at.numel()) * 2.0 ** -24
    return out, mean, err


def bound(out, mean, err, dtype):
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    # (fp16: the smallest step of a subnormal output, too)
    return u * out.abs() + (u * (dtype == torch.float16) + err) * mean + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


def prompts(q, k, v, lens_q, lens_k, causal=False, visible=None, shared_k=None, shared_v=None, scale=None, softcap=0.0,
            slopes=None):
    """Packed q [sum lens_q, hq, d], k, v [sum lens_k, hkv, d] in their own type: (out, bound) of the same rows."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    outs, bounds, a, b = [], [], 0, 0
    for n, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        kk, vv = k[b:b + lk].double(), v[b:b + lk].double()
        front = 0
        if shared_k is not None:
            front = shared_k.shape[0]
            kk, vv = torch.cat((shared_k.double(), kk)), torch.cat((shared_v.double(), vv))
        pos_q, pos_k = front + lk - lq + torch.arange(lq), torch.arange(front + lk)
        seen = torch.ones(lq, front + lk, dtype=torch.bool)
        if causal:
            seen = pos_k[None] <= pos_q[:, None]
            if visible is not None:
                seen = seen | (pos_k < int(visible[n]))[None]
        o, m, e = one_sequence(q[a:a + lq].double(), kk, vv, pos_q, pos_k, seen, scale, softcap, slopes)
        outs.append(o)
        bounds.append(bound(o, m, e, q.dtype))
        a, b = a + lq, b + lk
    return torch.cat(outs), torch.cat(bounds)


def tokens(q, k, v, lengths, shared_k=None, shared_v=None, scale=None, softcap=0.0, slopes=None):
    """q [requests, hq, d]; k, v: a list of each request's keys [n, hkv, d]."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    outs, bounds = [], []
    for b, n in enumerate(lengths):
        kk, vv, front = k[b][:n].double(), v[b][:n].double(), 0
        if shared_k is not None:
            front = shared_k.shape[0]
            kk, vv = torch.cat((shared_k.double(), kk)), torch.cat((shared_v.double(), vv))
        o, m, e = one_sequence(q[b:b + 1].double(), kk, vv, torch.tensor([front + n - 1]), torch.arange(front + n),
                               torch.ones(1, front + n, dtype=torch.bool), scale, softcap, slopes)
        outs.append(o)
        bounds.append(bound(o, m, e, q.dtype))
    return torch.cat(outs), torch.cat(bounds)


def check(y, ref, what=""):
    out, tol = ref
    y = y.detach().double().cpu().reshape(out.shape)
    assert torch.isfinite(y).all(), f"{what}: not finite"
    over = ((y - out).abs() / tol).max().item() if out.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.3g} times the bound"
