"""CPU tests of ``AdapterLinear``: where the kernels do not serve a call it falls back like ``FastLinear``, with the adapters."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def layer(K=96, N=72, n=3, r=8, device="cpu", bias=True):
    gen = torch.Generator().manual_seed(0)
    m = g.AdapterLinear(K, N, n, r, bias=bias)
    m.weight_t.copy_(0.05 * torch.randn(K, N, generator=gen))
    if bias:
        m.bias.copy_(torch.randn(N, generator=gen))
    m.down.copy_(torch.randn(n, r, K, generator=gen) * K ** -0.5)
    m.up.copy_(0.2 * torch.randn(n, N, r, generator=gen))
    m.scale.copy_(torch.tensor([1.0, 0.5, -2.0])[:n])
    x = torch.randn(5, 4, K, generator=gen)
    index = (torch.arange(20, dtype=torch.int32) % (n + 2) - 1).view(5, 4)  # -1 and n: none
    return m.to(device), x.to(device), index.to(device)


def formula(m, x, index):
    x, out = x.double(), x.double() @ m.weight_t.double()
    if m.bias is not None:
        out = out + m.bias.double()
    for a in range(m.down.shape[0]):
        rows = (index == a)[..., None]
        out = out + torch.where(rows, m.scale[a].double() * (x @ m.down[a].double().t() @ m.up[a].double().t()), 0.0)
    return out


def near(y, want, dtype):
    # 2^-11 of the output in fp16, 2^-8 in bfloat16; fp32 sums over at most 256 terms of magnitude up to 64 here; on the GPU
    # fp32 activations of more than 8 rows are rounded to fp16
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}.get(dtype, 2.0 ** -24)
    assert ((y.double() - want).abs() <= u * want.abs() + 2.0 ** -11 * 16).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K,N", [(96, 72), (100, 72), (96, 70), (256, 256)])
@pytest.mark.parametrize("bias", [True, False])
def test_sizes_the_kernels_do_not_take(device, K, N, bias):
    m, x, index = layer(K, N, device=device, bias=bias)
    with torch.no_grad():
        y = m(x, index)
        assert y.shape == (5, 4, N) and y.dtype == torch.float32
        near(y, formula(m, x, index), torch.float32)
        assert m(x[:0], index[:0]).shape == (0, 4, N)
        none = torch.full_like(index, -3)
        near(m(x, none), m(x).double(), torch.float32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("convert", ["half", "float", "bfloat16", "double"])
def test_converted_buffers(device, convert):
    m, x, index = layer(device=device)
    m = getattr(m, convert)()
    with torch.no_grad():
        near(m(x, index), formula(m, x, index), torch.float32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16, torch.float64])
def test_types(device, dtype):
    m, x, index = layer(device=device)
    x = x.to(dtype)
    with torch.no_grad():
        y = m(x, index)
    assert y.dtype == (dtype if dtype in (torch.float16, torch.float32) else torch.float32)
    near(y, formula(m, x, index), y.dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_reach_the_input_and_trained_adapters(device):
    m, x, index = layer(device=device)
    for wanted in (("x",), ("down", "up", "scale"), ("x", "down", "up", "scale")):
        ops = {"x": x, "down": m.down, "up": m.up, "scale": m.scale}
        plain = {k: v.detach().clone().double().requires_grad_(k in wanted) for k, v in ops.items()}
        for k, v in ops.items():
            v = v.detach().clone().requires_grad_(k in wanted)
            ops[k] = v
            if k != "x":
                setattr(m, k, v)
        w = torch.linspace(-1, 1, 20 * 72, device=device).view(5, 4, 72)
        (m(ops["x"], index) * w).sum().backward()
        twin = g.AdapterLinear(96, 72, 3, 8, device=device)
        for k in ("weight_t", "bias"):
            setattr(twin, k, getattr(m, k))
        for k in ("down", "up", "scale"):
            setattr(twin, k, plain[k])
        (formula(twin, plain["x"], index) * w).sum().backward()
        for k in wanted:
            # (a gradient has its operand's type: fp16 for down and up)
            got, want = ops[k].grad.double(), plain[k].grad
            assert ((got - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -12 * want.abs().max()).all(), (wanted, k)
        assert all(ops[k].grad is None for k in ops if k not in wanted)


def test_gradients_against_differences():
    m, x, index = layer(K=24, N=16)
    m, x = m.double(), x[:2].double()
    index = index[:2]
    given = [t.detach().clone().requires_grad_() for t in (x, m.down, m.up, m.scale)]

    def call(x, down, up, scale):
        m.down, m.up, m.scale = down, up, scale
        return m(x, index)

    assert torch.autograd.gradcheck(call, given)


@pytest.mark.parametrize("device", DEVICES)
def test_the_index_is_checked(device):
    m, x, index = layer(device=device)
    for bad in (index[:3], index.long(), index.float()):
        with pytest.raises(ValueError), torch.no_grad():
            m(x, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("x_type", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,N", [(4096, 512, 1024), (2304, 256, 4096), (600, 512, 512)])
def test_the_prepacked_weight_serves_calls_with_an_index(cuda, x_type, M, K, N):
    m, _, _ = layer(K, N, device=cuda)
    gen = torch.Generator().manual_seed(1)
    x, index = torch.randn(M, K, generator=gen).to(x_type).to(cuda), (torch.arange(M, dtype=torch.int32) % 5 - 1).to(cuda)
    with torch.no_grad():
        y = m(x, index)
        assert (m._wp is not None) == (g.ops._gemm_route(g._clib.load(), M, N, K, cuda)[7] == 256 or M >= N and bool(
            g.ops._gemm_route(g._clib.load(), M, N, K, cuda)[7]))
        assert torch.equal(y, g.lora_mm_t(x, m.weight_t, m.down, m.up, index, scale=m.scale, bias=m.bias, out_dtype=x_type))
        m.weight_t.mul_(2)  # (a stale copy would show)
        assert torch.equal(m(x, index), g.lora_mm_t(x, m.weight_t, m.down, m.up, index, scale=m.scale, bias=m.bias, out_dtype=x_type))
