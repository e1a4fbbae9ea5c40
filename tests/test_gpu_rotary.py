"""Rotary positions on the GPU against the formula in 64 bits.

Bound of a value: its cosine and sine are off by at most 2^-23 each, and by 2^-51 of the angle, whose product and reduction are
made in 64 bits; the fp32 rotation rounds a product and the result (2^-24 of each); then comes the output's own rounding."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def reference(x, positions, freqs, sections=None, interleaved=False):
    """(out, bound) in doubles on the CPU; x [.., heads, d], positions as the call has them."""
    x, positions, freqs, dtype = x.cpu().double(), positions.cpu().double(), freqs.cpu().double(), x.dtype
    pairs = freqs.shape[0]
    if sections is None:
        angle = positions[..., None] * freqs
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
        angle = torch.stack([positions[a] * freqs[i] for i, a in enumerate(axis)], -1) if pairs else positions[0][..., None] * freqs
    z = torch.polar(torch.ones_like(angle), angle)[..., None, :]
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    y = z * torch.complex(a, b)
    off = (2.0 ** -23 + 2.0 ** -24 + 2.0 ** -51 * angle.abs()[..., None, :]) * (a.abs() + b.abs())
    out, tol = x.clone(), torch.zeros_like(x)
    if interleaved:
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = y.real, y.imag
        tol[..., 0:2 * pairs:2], tol[..., 1:2 * pairs:2] = off, off
    else:
        out[..., :pairs], out[..., pairs:2 * pairs] = y.real, y.imag
        tol[..., :pairs], tol[..., pairs:2 * pairs] = off, off
    u, least = (2.0 ** -11, 2.0 ** -25) if dtype == F16 else (2.0 ** -24, 1e-37)
    turned = tol > 0
    return out, torch.where(turned, tol * (1 + u) + u * out.abs() + least, torch.zeros_like(tol))


def close(got, x, positions, freqs, **kw):
    out, tol = reference(x, positions, freqs, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    off = (got.cpu().double() - out).abs()
    assert (off <= tol).all(), f"{(off - tol).max().item():.3g} over the bound"


def freqs_of(pairs, device):
    return torch.tensor([10000.0 ** (-i / max(1, pairs)) for i in range(pairs)], dtype=F32, device=device)


def normal(*shape, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,d,pairs", [(1, 1, 8, 4), (1, 24, 64, 32), (7, 5, 72, 36), (33, 40, 128, 64), (5, 3, 128, 20), (6, 2, 80, 10), (9, 4, 64, 5),
                                                (3, 2, 24, 0), (4, 3, 96, 48), (2, 2, 256, 128), (3, 1, 4096, 2048), (2, 3, 16, 1), (129, 41, 32, 16)])
def test_against_the_formula(cuda, dtype, interleaved, rows, heads, d, pairs):
    x = normal(rows, heads, d, dtype=dtype, device=cuda)
    positions = torch.arange(rows, dtype=torch.int32, device=cuda) * 37 + 5
    freqs = freqs_of(pairs, cuda)
    close(g.rotary(x, positions, freqs, interleaved=interleaved), x, positions, freqs, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("sections", [(16, 24, 24), (1, 62, 1), (64,), (0, 64), (10, 20, 30, 4), (0, 0, 64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(cuda, dtype, sections, interleaved):
    x = normal(2, 19, 6, 128, dtype=dtype, device=cuda)
    gen = torch.Generator().manual_seed(3)
    positions = torch.randint(-2000, 2000, (len(sections), 2, 19), generator=gen).to(torch.int32).to(cuda)
    freqs = freqs_of(64, cuda)
    kw = dict(sections=sections, interleaved=interleaved)
    close(g.rotary(x, positions, freqs, **kw), x, positions, freqs, **kw)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_far_positions(cuda, dtype):
    far = [0, 1, -1, 4095, 1 << 20, -(1 << 20), (1 << 24) + 1, (1 << 30) + 12345, (1 << 31) - 1, -(1 << 31)]
    positions = torch.tensor(far, dtype=torch.int32, device=cuda)
    x, freqs = normal(len(far), 3, 128, dtype=dtype, device=cuda), freqs_of(64, cuda)
    close(g.rotary(x, positions, freqs), x, positions, freqs)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_views(cuda, dtype):
    # slices of a fused projection, an equal batch, other orders, rows that cannot be read in place
    fused = normal(10, 12, 64, dtype=dtype, device=cuda)
    freqs = freqs_of(32, cuda)
    p10 = torch.arange(10, dtype=torch.int32, device=cuda)
    for x, p in ((fused[:, 2:9], p10), (fused.unflatten(0, (2, 5))[:, :, :4], p10.view(2, 5)), (fused.transpose(0, 1), p10.repeat(2)[:12]),
                 (fused.view(10, -1)[:, 3:3 + 64].unsqueeze(1), p10), (fused[:, :, :].expand(10, 12, 64)[::3], p10[::3]),
                 (fused[:1].expand(10, 12, 64), p10)):
        close(g.rotary(x, p, freqs), x, p, freqs)


def test_negative_positions_turn_back(cuda):
    x, freqs = normal(50, 4, 128, dtype=F32, device=cuda), freqs_of(64, cuda)
    p = torch.arange(50, dtype=torch.int32, device=cuda) * 1001
    back = g.rotary(g.rotary(x, p, freqs), -p, freqs)
    assert (back - x).abs().max() <= 8 * 2.0 ** -23 * x.abs().max()


def test_many_threads(cuda):
    # past the number of pieces from which a thread takes several heads, with heads left over
    x = normal(4099, 42, 64, dtype=F16, device=cuda)
    p = torch.arange(4099, dtype=torch.int32, device=cuda)
    freqs = freqs_of(32, cuda)
    close(g.rotary(x, p, freqs), x, p, freqs)


@pytest.mark.parametrize("shape", [(0, 4, 64), (3, 0, 64), (0, 5, 4, 64), (2, 0, 4, 64)])
def test_nothing(cuda, shape):
    x = torch.empty(shape, dtype=F16, device=cuda)
    assert g.rotary(x, torch.empty(shape[:-2], dtype=torch.int32, device=cuda), freqs_of(32, cuda)).shape == x.shape


def test_infinities_stay_with_their_pairs(cuda):
    x = normal(3, 2, 64, dtype=F16, device=cuda)
    x[1, 0, 5], x[1, 1, 63] = float("inf"), float("nan")
    p = torch.arange(3, dtype=torch.int32, device=cuda) + 1
    y = g.rotary(x, p, freqs_of(16, cuda))
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1, 0, 5] = bad[1, 0, 21] = bad[1, 1, 63] = True
    assert (torch.isfinite(y) == ~bad).all()


def test_streams_and_graphs(cuda):
    x, freqs = normal(64, 10, 128, dtype=F16, device=cuda), freqs_of(64, cuda)
    p = torch.arange(64, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g.rotary(x, p, freqs)
        with torch.cuda.graph(graph, stream=side):
            y = g.rotary(x, p, freqs)
    torch.cuda.current_stream().wait_stream(side)
    for shift in (0, 100, 7):
        p.add_(shift)
        graph.replay()
        eager = g.rotary(x, p, freqs)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        close(eager, x, p, freqs)


def test_refusals(cuda):
    x, p, f = torch.zeros(3, 2, 64, dtype=F16, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda), freqs_of(32, cuda)
    for bad in (dict(x=x.bfloat16()), dict(x=x[0]), dict(x=x[..., :60]), dict(positions=p.long()), dict(positions=p[:2]), dict(freqs=f.double()),
                dict(freqs=freqs_of(33, cuda)), dict(freqs=f[:, None]), dict(sections=(16, 17)), dict(sections=()), dict(sections=(8, 8, 8, 4, 4)),
                dict(sections=(-1, 33)), dict(sections=(16, 16)), dict(positions=p.cpu()), dict(freqs=f.cpu()), dict(x=x.cpu())):
        kw = dict(x=x, positions=p, freqs=f) | bad
        with pytest.raises(ValueError):
            g.rotary(kw.pop("x"), kw.pop("positions"), kw.pop("freqs"), **kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        g.rotary(x.requires_grad_(), p, f)
    with torch.no_grad():
        g.rotary(x, p, f)
