"""Serve requests with adapters of their own after a shared system prompt.

    python examples/serve_adapters.py [--layers 4 --requests 12 --tokens 32 --rotary --cache int8 --check]

A small half-precision decoder with random weights: its projections are ``AdapterLinear`` layers (one
fp16 weight for all requests, a low-rank adapter for each), its attention has grouped heads, a bias that
grows with the distance in place of positions (or, with ``--rotary``, rotary positions), and capped scores. The system
prompt's keys and values are computed once; every request's own prompt follows it (``attention`` with ``shared_k``),
and the tokens after that are generated for all requests together (``attention_decode`` over pages of 16 keys, in
fp16 or, with ``--cache int8`` or ``e4m3``, written by ``cache_write``). ``--check`` computes every request again by itself, in
fp32 and in plain torch, and compares the logits.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "gtx16-fp16_amd"))
import gtx16_fp16 as g  # noqa: E402

PAGE = 16
SOFTCAP = 30.0
CACHES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def layer(n_in: int, n_out: int, adapters: int, rank: int, gen: torch.Generator, device) -> g.AdapterLinear:
    m = g.AdapterLinear(n_in, n_out, adapters, rank, bias=False, device=device)
    for t, size in ((m.weight_t, n_in ** -0.5), (m.down, n_in ** -0.5), (m.up, 0.1)):
        t.copy_(size * torch.randn(t.shape, generator=gen))
    m.scale.copy_(0.5 + torch.rand(adapters, generator=gen))
    return m


class Block(nn.Module):
    def __init__(self, width, heads, key_heads, adapters, rank, gen, device):
        super().__init__()
        self.heads, self.key_heads, self.d = heads, key_heads, width // heads
        self.norm1, self.norm2 = (nn.RMSNorm(width, device=device, dtype=torch.float16) for _ in range(2))
        make = lambda a, b: layer(a, b, adapters, rank, gen, device)  # noqa: E731
        self.qkv = make(width, (heads + 2 * key_heads) * self.d)
        self.out, self.up, self.down = make(width, width), make(width, 4 * width), make(4 * width, width)

    def split(self, x, index, at, freqs):
        """q, k, v [rows, heads, d], views of the fused projection's output; rotated (freqs) where rows stand ``at``."""
        y = self.qkv(self.norm1(x), index).unflatten(-1, (-1, self.d))
        if freqs is None:
            return y.split((self.heads, self.key_heads, self.key_heads), dim=-2)
        qk = g.rotary(y[:, :self.heads + self.key_heads], at, freqs)
        return *qk.split((self.heads, self.key_heads), dim=-2), y[:, self.heads + self.key_heads:]

    def rest(self, x, attended, index):
        x = x + self.out(attended.flatten(-2), index)
        return x + self.down(torch.nn.functional.gelu(self.up(self.norm2(x), index)), index)


class Server(nn.Module):
    """``requests`` slots, each with an adapter and pages for its own keys in every layer."""

    def __init__(self, width=512, heads=8, key_heads=2, layers=4, vocab=1024, adapters=5, rank=16, seed=0, device="cuda",
                 rotary=False, cache="fp16"):
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        self.blocks = nn.ModuleList(Block(width, heads, key_heads, adapters, rank, gen, device) for _ in range(layers))
        self.embed = (0.7 * torch.randn(vocab, width, generator=gen)).half().to(device)
        self.head = g.FastLinear(width, vocab, bias=False, device=device)
        self.head.weight_t.copy_(self.embed.t())
        d = width // heads
        self.slopes = None if rotary else torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device=device)
        self.freqs = torch.tensor([10000.0 ** (-2 * i / d) for i in range(d // 2)], device=device) if rotary else None
        self.device, self.coded = device, CACHES[cache]
        self.shared: list = []

    def prefix(self, ids: torch.Tensor) -> None:
        """The system prompt, which has no adapter: its keys and values are kept for all requests."""
        x, index = self.embed[ids], torch.full((len(ids),), -1, dtype=torch.int32, device=self.device)
        whole = torch.tensor([0, len(ids)], dtype=torch.int32, device=self.device)
        at = torch.arange(len(ids), dtype=torch.int32, device=self.device)
        self.shared = []
        for b in self.blocks:
            q, k, v = b.split(x, index, at, self.freqs)
            self.shared.append((k.contiguous(), v.contiguous()))
            x = b.rest(x, g.attention(q, k, v, q_offsets=whole, causal=True, slopes=self.slopes, softcap=SOFTCAP), index)

    def start(self, prompts: list[torch.Tensor], adapter: torch.Tensor, most: int) -> torch.Tensor:
        """The requests' prompts, packed, of any lengths; the logits of each one's next token."""
        lens = torch.tensor([len(p) for p in prompts])
        n, per = len(prompts), -(-(int(lens.max()) + most) // PAGE)
        offsets = torch.cat((torch.zeros(1, dtype=torch.long), lens.cumsum(0))).to(torch.int32).to(self.device)
        self.adapter, self.lengths = adapter, lens.to(torch.int32).to(self.device)
        self.pages = torch.randperm(n * per).view(n, per).to(torch.int32).to(self.device)
        b0 = self.blocks[0]
        shape = (n * per, PAGE, b0.key_heads, b0.d)
        scaled = self.coded != torch.float16
        self.cache = [(*(torch.empty(shape, dtype=self.coded, device=self.device) for _ in "kv"),
                       *(torch.empty(shape[:3], device=self.device) if scaled else None for _ in "kv")) for _ in self.blocks]
        index = adapter.repeat_interleave(lens.to(self.device), output_size=int(lens.sum()))
        seq = torch.repeat_interleave(torch.arange(n, device=self.device), lens.to(self.device), output_size=int(lens.sum()))
        at = torch.arange(int(lens.sum()), device=self.device) - offsets[seq]
        slots = self.slots(seq, at)
        at = (at + len(self.shared[0][0])).to(torch.int32)
        x = self.embed[torch.cat(prompts).to(self.device)]
        for b, (sk, sv), cache in zip(self.blocks, self.shared, self.cache):
            q, k, v = b.split(x, index, at, self.freqs)
            self.keep(k, v, cache, slots)
            x = b.rest(x, g.attention(q, k, v, q_offsets=offsets, causal=True, shared_k=sk, shared_v=sv, slopes=self.slopes,
                                      softcap=SOFTCAP), index)
        return self.head(x[offsets[1:].long() - 1])

    def slots(self, seq: torch.Tensor, at: torch.Tensor) -> torch.Tensor:
        """Where the cache has token ``at`` of request ``seq``: tokens counted through all pages."""
        return (self.pages[seq, (at // PAGE).long()] * PAGE + at % PAGE).to(torch.int32)

    def keep(self, k, v, cache, slots) -> None:
        kc, vc, ks, vs = cache
        if ks is not None:
            g.cache_write(k, v, kc, vc, ks, vs, slots)
        else:
            kc.view(-1, *kc.shape[2:])[slots.long()], vc.view(-1, *vc.shape[2:])[slots.long()] = k, v

    def step(self, ids: torch.Tensor) -> torch.Tensor:
        """One more token of every request; the logits of the next."""
        slots = self.slots(torch.arange(len(ids), device=self.device), self.lengths)
        at = self.lengths + len(self.shared[0][0])
        self.lengths += 1
        x = self.embed[ids]
        for b, (sk, sv), cache in zip(self.blocks, self.shared, self.cache):
            q, k, v = b.split(x, self.adapter, at, self.freqs)
            self.keep(k, v, cache, slots)
            kc, vc, ks, vs = cache
            x = b.rest(x, g.attention_decode(q, kc, vc, self.lengths, pages=self.pages, shared_k=sk, shared_v=sv, slopes=self.slopes,
                                             softcap=SOFTCAP, k_scale=ks, v_scale=vs), self.adapter)
        return self.head(x)


def plain(server: Server, system: torch.Tensor, ids: torch.Tensor, adapter: int) -> torch.Tensor:
    """Logits after every token of one request, its system prompt before it, in fp32 torch."""
    n0, n = len(system), len(system) + len(ids)
    x = server.embed[torch.cat((system, ids))].float()
    pos = torch.arange(n, device=x.device)
    away = (pos[:, None] - pos[None]).float()

    def product(m, x):
        y = x @ m.weight_t.float()
        if adapter >= 0:  # the system prompt has none
            y[n0:] += m.scale[adapter] * ((x[n0:] @ m.down[adapter].float().T) @ m.up[adapter].float().T)
        return y

    for b in server.blocks:
        norm = lambda w, x: torch.nn.functional.rms_norm(x, x.shape[-1:], w.weight.float())  # noqa: E731
        q, k, v = (t.transpose(0, 1) for t in product(b.qkv, norm(b.norm1, x)).unflatten(-1, (-1, b.d)).split(
            (b.heads, b.key_heads, b.key_heads), dim=-2))
        if server.freqs is not None:
            angle = pos[:, None] * server.freqs.double()
            z = torch.polar(torch.ones_like(angle), angle).to(torch.complex64)
            q, k = (torch.cat(((y := z * torch.complex(*t.chunk(2, -1))).real, y.imag), -1) for t in (q, k))
        k, v = (t.repeat_interleave(b.heads // b.key_heads, 0) for t in (k, v))
        s = SOFTCAP * torch.tanh((q @ k.transpose(1, 2)) * b.d ** -0.5 / SOFTCAP)
        s = s if server.slopes is None else s - server.slopes[:, None, None] * away
        a = torch.softmax(s.masked_fill(away < 0, float("-inf")), -1) @ v
        x = x + product(b.out, a.transpose(0, 1).flatten(1))
        x = x + product(b.down, torch.nn.functional.gelu(product(b.up, norm(b.norm2, x))))
    return x[n0:] @ server.head.weight_t.float()


@torch.no_grad()
def main(argv: list[str] | None = None) -> float:
    """Returns the largest relative difference of logits from the plain ones (0.0 without ``--check``)."""
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("--width", 512), ("--heads", 8), ("--key-heads", 2), ("--layers", 4), ("--requests", 12), ("--system", 300),
                        ("--prompt", 60), ("--tokens", 32)):
        ap.add_argument(name, type=int, default=value)
    ap.add_argument("--rotary", action="store_true", help="rotary positions in place of the distance bias")
    ap.add_argument("--cache", choices=CACHES, default="fp16", help="what the requests' own keys and values are kept in")
    ap.add_argument("--check", action="store_true", help="compare with plain torch in fp32")
    a = ap.parse_args(argv)
    server = Server(a.width, a.heads, a.key_heads, a.layers, rotary=a.rotary, cache=a.cache)
    dev, gen = server.device, torch.Generator().manual_seed(1)
    vocab = server.embed.shape[0]
    system = torch.randint(0, vocab, (a.system,), generator=gen).to(dev)
    prompts = [torch.randint(0, vocab, (1 + int(torch.randint(0, a.prompt, (1,), generator=gen)),), generator=gen) for _ in range(a.requests)]
    adapter = torch.randint(-1, 5, (a.requests,), generator=gen).to(torch.int32).to(dev)
    server.prefix(system)
    logits = [server.start(prompts, adapter, a.tokens)]
    ids = []
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.tokens - 1):
        ids.append(logits[-1].argmax(-1))
        logits.append(server.step(ids[-1]))
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    print(f"{a.requests} requests, {a.layers} layers: {took / max(1, a.tokens - 1) * 1e3:.2f} ms a token step", flush=True)
    worst = 0.0
    if a.check:
        for r, p in enumerate(prompts):
            said = torch.stack([t[r] for t in ids]) if ids else torch.empty(0, dtype=torch.long, device=dev)
            ref = plain(server, system, torch.cat((p.to(dev), said)), int(adapter[r]))[len(p) - 1:]
            got = torch.stack([x[r] for x in logits]).float()
            worst = max(worst, float((got - ref).norm() / ref.norm()))
        print(f"largest relative difference of a request's logits from plain fp32: {worst:.2e}", flush=True)
    return worst


if __name__ == "__main__":
    main()
