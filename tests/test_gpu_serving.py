"""GPU tests of ``AdapterLinear`` and of the serving example, whole, against plain fp32 torch."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

import gtx16_fp16 as g

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "serve_adapters.py"
    spec = importlib.util.spec_from_file_location("serve_adapters", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def layer(dev, dtype=torch.float16):
    gen = torch.Generator().manual_seed(0)
    fast = g.FastLinear.from_linear(torch.nn.Linear(256, 128)).to(dev)
    m = g.AdapterLinear.from_fast(fast, 3, 16)
    m.down.copy_(torch.randn(m.down.shape, generator=gen) / 16)
    m.up.copy_(torch.randn(m.up.shape, generator=gen) / 4)
    m.scale.copy_(torch.tensor([1.0, 0.5, 2.0]))
    return fast, m, torch.randn(4, 7, 256, generator=gen).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16])
def test_adapter_linear(cuda, dtype):
    fast, m, x = layer(cuda, dtype)
    assert m.weight_t is fast.weight_t and m.bias is fast.bias
    index = torch.arange(-1, 27, device=cuda, dtype=torch.int32).view(4, 7) % 4 - 1
    with torch.no_grad():
        assert torch.equal(m(x), fast(x))
        y = m(x, index)
    assert y.shape == (4, 7, 128) and y.dtype == (torch.float32 if dtype == torch.bfloat16 else dtype)
    z = x.double().cpu()
    want = z @ m.weight_t.double().cpu() + m.bias.double().cpu()
    for a in range(3):
        rows = index.cpu() == a
        want[rows] += float(m.scale[a]) * (z[rows] @ m.down[a].double().cpu().T) @ m.up[a].double().cpu().T
    # activations and output rounded to fp16 at the worst: 2^-10 of sums of magnitude up to |x||w| < 64 here
    assert (y.double().cpu() - want).abs().max() < 2.0 ** -10 * 64
    none = torch.full((4, 7), -1, device=cuda, dtype=torch.int32)
    with torch.no_grad():
        assert torch.equal(m(x.float(), none), g.mm_t(x.float().reshape(-1, 256), m.weight_t, m.bias).view(4, 7, 128))


def test_adapter_linear_state_and_refusals(cuda):
    _, m, x = layer(cuda)
    assert set(m.state_dict()) == {"weight_t", "bias", "down", "up", "scale"}
    other = g.AdapterLinear(256, 128, 3, 16, device=cuda)
    other.load_state_dict(m.state_dict())
    index = torch.zeros(4, 7, device=cuda, dtype=torch.int32)
    with torch.no_grad():
        assert torch.equal(other(x, index), m(x, index))
    for rank in (0, 12, 136):
        with pytest.raises(ValueError):
            g.AdapterLinear(256, 128, 3, rank)
    with pytest.raises(ValueError), torch.no_grad():
        m(x, index[:3])


@pytest.mark.parametrize("argv", [["--layers", "2", "--requests", "5", "--tokens", "20", "--system", "70"],
                                  ["--layers", "1", "--requests", "1", "--tokens", "3", "--system", "1", "--prompt", "1"],
                                  ["--layers", "1", "--requests", "40", "--tokens", "4", "--system", "700", "--width", "1024", "--heads", "8"]])
def test_the_serving_example(cuda, argv):
    # fp16 activations through every layer: 2^-11 a rounding, some dozens of them in a row
    assert example().main([*argv, "--check"]) < 2e-2
