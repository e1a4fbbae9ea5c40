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
from .kernels import SKINNY_MAX_M, scratch_buffer, stream_handle
from .linear import FastLinear
from .ops import _aligned, _gemm_route, _sm_count, mm_t, mm_t_prepacked

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
    return _add_adapters(x2d, mm_t(x2d, w_t, bias, torch.float32), down, up, index, scale, out_dtype)


def _add_adapters(x2d: torch.Tensor, y: torch.Tensor, down: torch.Tensor, up: torch.Tensor, index: torch.Tensor, scale,
                  out_dtype: torch.dtype) -> torch.Tensor:
    """The adapters' part beside the shared product ``y`` (fp32, written to where out_dtype is fp32); checked operands."""
    (M, K), N = x2d.shape, y.shape[1]
    n, r = down.shape[:2]
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

    Types, shapes and fallbacks are FastLinear's: with an index, too, large batches read the prepacked copy of the
    weight, and what the kernels cannot take (CPU tensors, other devices, sizes that are no multiples of 8, converted
    buffers) or have no gradient for is computed by torch operations, the adapters' part in fp32; gradients then reach
    x and, where they require them, ``down``, ``up`` and ``scale``. ``prepack_decode`` has no effect on calls with an
    index: token by token the host makes the shared product and the adapters' part in one go, which costs less than
    the decode layout saves.

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

    def _plain(self, x: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
        # FastLinear's result and the adapters, by torch operations
        y = super().forward(x)
        acc = torch.promote_types(y.dtype, torch.float32)
        x2, add = x.reshape(-1, self.in_features).to(acc), []
        for a in index.unique().tolist():
            if 0 <= a < self.down.shape[0]:
                at = (index == a).nonzero().flatten()
                add.append((at, self.scale[a].to(acc) * (x2[at] @ self.down[a].to(acc).t() @ self.up[a].to(acc).t())))
        if not add:
            return y
        part = torch.zeros(x2.shape[0], self.out_features, device=x2.device, dtype=acc).index_copy(
            0, torch.cat([at for at, _ in add]), torch.cat([z for _, z in add]))
        return (y.reshape(part.shape).to(acc) + part).to(y.dtype).view(y.shape)

    def _takes(self, x: torch.Tensor) -> bool:
        # what lora_mm_t computes with these buffers
        d, u = self.down, self.up
        return (x.is_cuda and self._operands_ok(self.weight_t, None, x.device) and d.dtype == u.dtype == torch.float16
                and d.device == u.device == self.scale.device == x.device
                and not (torch.is_grad_enabled() and any(t.requires_grad for t in (x, d, u, self.scale))))

    def _may_pack(self, M: int, dev: torch.device) -> bool:
        # whether a prepacked weight can serve M rows
        K, N = self.in_features, self.out_features
        return self.prepack_weight and M > SKINNY_MAX_M and not (K | N) % 8 and _gemm_route(_clib.load(), M, N, K, dev)[7] != 0

    def forward(self, x: torch.Tensor, index: torch.Tensor | None = None) -> torch.Tensor:
        if index is None:
            return super().forward(x)
        w, scale, bias = self.weight_t, self.scale, self.bias
        dtype = x.dtype if x.dtype in (torch.float16, torch.float32) else torch.float32
        x2, rows = x.reshape(-1, self.in_features), index.reshape(-1)
        M, y = x2.shape[0], None
        # (first what needs no look at the operands here: small calls are bound by the host)
        if M and x.is_cuda and forward_ad._current_level < 0 and not self._may_pack(M, x.device):
            y = direct().lora_mm_t(x2, w, self.down, self.up, rows, scale, bias, dtype)
        if y is None:
            if not (rows.dtype == torch.int32 and rows.shape[0] == M and rows.device == x.device):
                raise ValueError(f"AdapterLinear: index must hold {M} int32 values on {x.device}, one for each row of x")
            if M == 0 or not self._takes(x):
                return self._plain(x, rows)
            x2 = x2 if x2.dtype == dtype else x2.float()
            scale = scale if scale.dtype == torch.float32 else scale.float()
            wp = self._packed_for(x2) if self._may_pack(M, x.device) else None
            if wp is None:
                y = lora_mm_t(x2, w, self.down, self.up, rows, scale=scale, bias=bias, out_dtype=dtype)
            else:  # (lora_mm_t with the shared product from the prepacked weight, whose bits are mm_t's)
                _check(x2, w, self.down, self.up, rows, scale)
                refuse_tangents("AdapterLinear", x, self.down, self.up, scale)
                x2 = _aligned(x2)
                y = mm_t_prepacked(x2, w, wp, bias, torch.float32, _cast_source=x if self.share_cast else None)
                y = _add_adapters(x2, y, self.down, self.up, rows, scale, dtype)
        return y.view(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, adapters={self.down.shape[0]}, rank={self.down.shape[1]}"


_entry: tuple[int, ...] = ()


def _entry_points() -> tuple[int, ...]:
    global _entry
    if not _entry:
        _entry = tuple(_clib.address(n) for n in ("g16_lora_workspace_bytes", "g16_lora_shrink", "g16_lora_expand"))
    return _entry
