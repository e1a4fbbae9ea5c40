"""Codes of 8 bits in 64-bit arithmetic, on the CPU, from the formats' definitions."""
from __future__ import annotations

import torch

LEAST = 2.0 ** -96
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def coded(x, code):
    """x [.., d] -> (codes as the numbers they stand for before scaling, scales [..]), doubles, exact."""
    x = x.double()
    top = torch.where(torch.isfinite(x).all(-1), x.abs().amax(-1), torch.full(x.shape[:-1], float("inf"), dtype=torch.float64))
    lost, none = torch.isinf(top), top < LEAST
    safe = torch.where(lost | none, torch.ones_like(top), top)
    if code == "int8":  # (a quotient of two fp32 numbers rounded to 64 bits and then to 32 is the one rounded to 32)
        scale = (safe / 127.0).float().double()
        y = torch.round(x * (127.0 / safe).float().double()[..., None])
    else:
        scale = 2.0 ** torch.ceil(torch.log2(safe / 448.0) - 1e-9)
        scale = torch.where(safe > 448.0 * scale, 2 * scale, scale)
        y = x / scale[..., None]
        step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
        y = torch.round(y / step) * step
    y = torch.where((lost | none)[..., None], torch.zeros_like(y), y)
    return y, torch.where(lost, torch.full_like(scale, float("nan")), torch.where(none, torch.zeros_like(scale), scale))


def numbers(cache):
    """A cache's codes as doubles on the CPU."""
    return cache.contiguous().view(torch.uint8).cpu().view(cache.dtype).float().double()


def empty(pages, page, heads, d, code, device, by_head=False, fill=0x35):
    """(k_cache, v_cache, k_scale, v_scale) full of something."""
    def one(*shape, dtype):
        t = torch.full(shape, fill, dtype=torch.uint8, device=device)
        return t.view(dtype).squeeze(-1) if dtype == torch.float32 else t.view(dtype)

    order = (pages, heads, page) if by_head else (pages, page, heads)
    got = [one(*order, d, dtype=CODES[code]) for _ in "kv"] + [one(*order, 4, dtype=torch.float32) for _ in "kv"]
    return [t.transpose(1, 2) for t in got] if by_head else got


def random_cache(pages, page, heads, d, code, gen, device="cpu", by_head=False, loud=1.0):
    """A cache of normal values with its dequantised keys and values, [pages, page, heads, d] doubles."""
    out = []
    for factor in (loud, 1.0):
        y, scale = coded(factor * torch.randn(pages, page, heads, d, generator=gen), code)
        out.append((y.float().to(CODES[code]), scale.float(), y * scale[..., None]))
    (kc, ks, k), (vc, vs, v) = out
    move = (lambda t: t.transpose(1, 2).contiguous().to(device).transpose(1, 2)) if by_head else (lambda t: t.to(device))
    return [move(t) for t in (kc, vc, ks, vs)], k, v
