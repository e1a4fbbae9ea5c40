"""Low-rank adapters of many requests beside one linear layer's product (``lora_mm_t``).

No counterpart in the reference; arguments and checks follow ``mm_t``. The kernels are those of
``csrc/lora.hip``; ``AdapterLinear`` is a ``FastLinear`` with adapters of its own.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

from . import _clib
from .direct import direct, refuse_gradients, refuse_tangents
from .kernels import scratch_buffer, stream_handle
from .linear import FastLinear
from .ops import _aligned, _sm_count, mm_t

MAX_RANK = 128  # G16_LORA_MAX_RANK
MAX_SIDE = 1 << 21  # G16_LORA_MAX_SIDE

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
    if K > MAX_SIDE or N > MAX_SIDE:
        raise ValueError(f"lora_mm_t: K and N may be up to {MAX_SIDE}, got {K} and {N}")
    if not (index.dtype == torch.int32 and index.shape == (x2d.shape[0],) and index.device == dev):
        raise ValueError(f"lora_mm_t: index must be an int32 tensor of shape ({x2d.shape[0]},) on {dev}")
    if scale is not None and not (scale.dtype == torch.float32 and scale.shape == (n,) and scale.device == dev):
        raise ValueError(f"lora_mm_t: scale must be an fp32 tensor of shape ({n},) on {dev}")


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
    if forward_ad._current_level >= 0:
        refuse_tangents("lora_mm_t", x2d, w_t, down, up, scale, bias)
    out = direct().lora_mm_t(x2d, w_t, down, up, index, scale, bias, out_dtype)
    if out is not None:
        return out
    if out_dtype not in (torch.float32, torch.float16):
        raise ValueError(f"out_dtype must be float32 or float16, got {out_dtype}")
    _check(x2d, w_t, down, up, index, scale)
    refuse_gradients("lora_mm_t", x2d, w_t, down, up, scale, bias)
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
    # (without a workspace, expand computes both products; the tensor is held until both are enqueued)
    ws = scratch_buffer(dev, stream, nbytes) if nbytes else None
    for fn in (shrink, expand) if nbytes else (expand,):
        status = fast.args_call(fn, head, None if ws is None else ws.data_ptr(), nbytes, stream)
        if status != 0:
            _clib.check(status, "adapters")
    return out


class AdapterLinear(FastLinear):
    """A ``FastLinear`` with ``adapters`` low-rank adapters beside its weight, one of them, or none, for each
    row: ``layer(x, index)`` with index as in ``lora_mm_t``, one value for each row of x (all leading
    dimensions flattened, in their order); ``layer(x)`` is the FastLinear.

    State: FastLinear's ``weight_t`` and ``bias``, and ``down`` [adapters, rank, in_features], ``up`` [adapters,
    out_features, rank] in fp16, ``scale`` [adapters] in fp32. A new layer's adapters change nothing (``up`` is
    zero)."""

    def __init__(self, in_features: int, out_features: int, adapters: int, rank: int, bias: bool = True, device=None):
        super().__init__(in_features, out_features, bias, device)
        if rank % 8 or not 0 < rank <= MAX_RANK:
            raise ValueError(f"AdapterLinear: the rank must be a multiple of 8 up to {MAX_RANK}, got {rank}")
        self.register_buffer("down", torch.zeros(adapters, rank, in_features, dtype=torch.float16, device=device))
        self.register_buffer("up", torch.zeros(adapters, out_features, rank, dtype=torch.float16, device=device))
        self.register_buffer("scale", torch.ones(adapters, dtype=torch.float32, device=device))

    @classmethod
    def from_fast(cls, layer: FastLinear, adapters: int, rank: int) -> "AdapterLinear":
        """``layer``'s own weight and bias (not copies) with ``adapters`` new adapters beside them."""
        m = cls(layer.in_features, layer.out_features, adapters, rank, layer.bias is not None, device="meta")
        dev = layer.weight_t.device
        m.weight_t, m.bias = layer.weight_t, layer.bias
        m.down = torch.zeros(m.down.shape, dtype=torch.float16, device=dev)
        m.up = torch.zeros(m.up.shape, dtype=torch.float16, device=dev)
        m.scale = torch.ones(adapters, dtype=torch.float32, device=dev)
        return m

    def forward(self, x: torch.Tensor, index: torch.Tensor | None = None) -> torch.Tensor:
        if index is None:
            return super().forward(x)
        dtype = x.dtype if x.dtype in (torch.float16, torch.float32) else torch.float32
        x2 = x.reshape(-1, self.in_features)
        y = lora_mm_t(x2 if x2.dtype == dtype else x2.float(), self.weight_t, self.down, self.up, index.reshape(-1), scale=self.scale,
                      bias=self.bias, out_dtype=dtype)
        return y.view(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, adapters={self.down.shape[0]}, rank={self.down.shape[1]}"


_entry: tuple[int, ...] = ()


def _entry_points() -> tuple[int, ...]:
    global _entry
    if not _entry:
        _entry = tuple(_clib.address(n) for n in ("g16_lora_workspace_bytes", "g16_lora_shrink", "g16_lora_expand"))
    return _entry
