"""Low-rank adapters of many requests beside one linear layer's product (``lora_mm_t``).

No counterpart in the reference; arguments and checks follow ``mm_t``. The kernels are those of
``csrc/lora.hip``.
"""
from __future__ import annotations

import struct

import torch

from . import _clib
from .direct import direct
from .kernels import scratch_buffer, stream_handle
from .ops import _aligned, _sm_count, mm_t

MAX_RANK = 128  # G16_LORA_MAX_RANK

# g16_lora_args without its workspace
_ARGS = struct.Struct("@7P8i")
assert _ARGS.size == 7 * 8 + 8 * 4


def _check(x2d: torch.Tensor, w_t: torch.Tensor, down: torch.Tensor, up: torch.Tensor, index: torch.Tensor, scale) -> None:
    dev = x2d.device
    if x2d.dim() != 2 or w_t.dim() != 2:
        raise ValueError("lora_mm_t: x2d and w_t must be matrices")
    K, N = w_t.shape
    if not (down.dim() == 3 and up.dim() == 3 and down.dtype == up.dtype == torch.float16 and down.device == up.device == dev):
        raise ValueError(f"lora_mm_t: down and up must be fp16 tensors of three dimensions on {dev}")
    n, r = down.shape[:2]
    if down.shape[2] != K or up.shape != (n, N, r):
        raise ValueError(f"lora_mm_t: down {tuple(down.shape)} and up {tuple(up.shape)} must be [adapters, rank, {K}] and "
                         f"[adapters, {N}, rank]")
    if r % 8 or r > MAX_RANK:
        raise ValueError(f"lora_mm_t: the rank must be a multiple of 8 up to {MAX_RANK}, got {r}")
    if not (index.dtype == torch.int32 and index.shape == (x2d.shape[0],) and index.device == dev):
        raise ValueError(f"lora_mm_t: index must be an int32 tensor of shape ({x2d.shape[0]},) on {dev}")
    if scale is not None and not (scale.dtype == torch.float32 and scale.shape == (n,) and scale.device == dev):
        raise ValueError(f"lora_mm_t: scale must be an fp32 tensor of shape ({n},) on {dev}")
    if torch.is_grad_enabled() and (x2d.requires_grad or down.requires_grad or up.requires_grad):
        raise RuntimeError("lora_mm_t has no gradient: call it under torch.no_grad()")


def lora_mm_t(x2d: torch.Tensor, w_t: torch.Tensor, down: torch.Tensor, up: torch.Tensor, index: torch.Tensor, *,
              scale: torch.Tensor | None = None, bias: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``mm_t(x2d, w_t, bias)`` with a low-rank adapter beside it for each row:
    out[m] = x2d[m] @ w_t + bias + scale[a] * (x2d[m] @ down[a].T) @ up[a].T with a = index[m].

    down [adapters, rank, K] and up [adapters, N, rank] fp16 (the layouts of a pair of linear layers), rank a
    multiple of 8 up to 128 (pad smaller ones with zeros); index int32, one adapter a row in any order,
    negative (or past the last adapter) for none; scale fp32 [adapters] or None. x2d, w_t, bias and out_dtype
    are mm_t's, and so is the shared product, rounding of fp32 activations included; the adapters' part is
    computed from the activations as they are, in fp32, and added before the one rounding to out_dtype."""
    out = direct().lora_mm_t(x2d, w_t, down, up, index, scale, bias, out_dtype)
    if out is not None:
        return out
    if out_dtype not in (torch.float32, torch.float16):
        raise ValueError(f"out_dtype must be float32 or float16, got {out_dtype}")
    _check(x2d, w_t, down, up, index, scale)
    x2d = _aligned(x2d)
    y = mm_t(x2d, w_t, bias, torch.float32)
    M, K = x2d.shape
    N, (n, r) = w_t.shape[1], down.shape[:2]
    dev = x2d.device
    out = y if out_dtype == torch.float32 else torch.empty(M, N, device=dev, dtype=out_dtype)
    if out.numel() == 0:
        return out
    if n == 0 or r == 0 or K == 0:
        return out.copy_(y) if out is not y else y
    down, up, index = _aligned(down), _aligned(up), index.contiguous()
    scale = None if scale is None else scale.contiguous()
    head = _ARGS.pack(x2d.data_ptr(), down.data_ptr(), up.data_ptr(), index.data_ptr(), 0 if scale is None else scale.data_ptr(),
                      y.data_ptr(), out.data_ptr(), M, K, N, r, n, x2d.dtype == torch.float32, out_dtype == torch.float16,
                      _sm_count(dev))
    fast = _clib.fast()
    size, shrink, expand = _entry_points()
    stream = stream_handle(dev.index or 0)
    nbytes = fast.args_size(size, head)
    # (without a workspace, expand computes both products)
    ws = scratch_buffer(dev, stream, nbytes).data_ptr() if nbytes else None
    for fn in (shrink, expand) if nbytes else (expand,):
        status = fast.args_call(fn, head, ws, nbytes, stream)
        if status != 0:
            _clib.check(status, "adapters")
    return out


_entry: tuple[int, ...] = ()


def _entry_points() -> tuple[int, ...]:
    global _entry
    if not _entry:
        _entry = tuple(_clib.address(n) for n in ("g16_lora_workspace_bytes", "g16_lora_shrink", "g16_lora_expand"))
    return _entry
