"""Serving one attention layer with a paged q8_0 cache: a shared system prompt,
a batch of prompts behind it, then one token per request and step.

    python k-search_b200/examples/paged_serving.py [--requests 16] [--system 2048] [--prompt 300] [--steps 32]

The layer is a fused QKV projection and attention with random weights; the
hidden states are random too. What a step does with the cache is what a server
does: plan the pages, write the new rows, attend. The last step is compared
with attention over the cache's contents in fp32.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import kq  # noqa: E402


class Layer:
    """Fused QKV projection of hidden states [T, E] -> q, k, v views of one [T, Hq + 2 Hkv, D] tensor."""

    def __init__(self, E: int, Hq: int, Hkv: int, D: int, dtype: torch.dtype, device, seed: int = 0):
        g = torch.Generator(device).manual_seed(seed)
        self.Hq, self.Hkv, self.D = Hq, Hkv, D
        self.w = (torch.randn(E, (Hq + 2 * Hkv) * D, generator=g, device=device) * E ** -0.5).to(dtype)

    def qkv(self, x: torch.Tensor):
        y = (x @ self.w).view(x.shape[0], self.Hq + 2 * self.Hkv, self.D)
        return y.split_with_sizes((self.Hq, self.Hkv, self.Hkv), 1)


class Server:
    def __init__(self, layer: Layer, requests: int, pages: int, page_size: int, max_blocks: int, device):
        self.layer, self.page_size, self.device = layer, page_size, device
        shape = (pages, page_size, layer.Hkv, layer.D // 32, 34)
        self.k_cache = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.tables = torch.full((requests, max_blocks), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.prefix = 0

    def _place(self, k, v, cached, new, tables, total):
        plan = kq.page_plan(cached, new, tables, self.free, self.page_size, total)
        kq.page_write(k, v, plan.slots, self.k_cache, self.v_cache)
        return plan

    def _take(self, used: int):
        # a server keeps its free list on the host and knows what a step needs
        # from the lengths, as here; plan.counts says the same on the device
        self.free = self.free[used:]

    def system_prompt(self, x: torch.Tensor) -> torch.Tensor:
        """Caches the shared prompt (whole pages) and puts its pages in front of every request's table."""
        n = x.shape[0]
        assert n % self.page_size == 0, "a shared prefix is whole pages"
        q, k, v = self.layer.qkv(x)
        lens = torch.tensor([0, n], dtype=torch.int32, device=self.device)
        table = torch.full((1, self.tables.shape[1]), -1, dtype=torch.int32, device=self.device)
        plan = self._place(k, v, lens[:1], lens[1:], table, n)
        pages = n // self.page_size
        self._take(pages)
        self.tables[:, :pages] = table[:, :pages]
        self.lens += n
        self.prefix = n
        return kq.flash_prompt_ragged(q, k, v, plan.cu_new)

    def prompts(self, x: torch.Tensor, new_lens: list[int]) -> torch.Tensor:
        """Packed prompts [sum(new_lens), E] behind what is cached: their rows see the cache's contents."""
        q, k, v = self.layer.qkv(x)
        new = torch.tensor(new_lens, dtype=torch.int32, device=self.device)
        plan = self._place(k, v, self.lens, new, self.tables, x.shape[0])
        self._take(sum(-(-n // self.page_size) for n in new_lens))
        total = x.shape[0] + self.prefix * len(new_lens)
        keys, values = kq.page_read(self.k_cache, self.v_cache, self.tables, plan.cu_seqlens, total, q.dtype)
        self.lens = plan.seq_lens
        return kq.flash_prompt_ragged(q, keys, values, plan.cu_new, plan.cu_seqlens)

    def token(self, x: torch.Tensor, host_lens: list[int]) -> torch.Tensor:
        """One token per request [B, E]; host_lens are the lengths before it."""
        q, k, v = self.layer.qkv(x)
        plan = self._place(k, v, self.lens, torch.ones_like(self.lens), self.tables, x.shape[0])
        self._take(sum(n % self.page_size == 0 for n in host_lens))
        self.lens = plan.seq_lens
        return kq.flash_decode_paged(q.contiguous(), self.k_cache, self.v_cache, self.tables, plan.seq_lens,
                                     prefix_len=self.prefix, max_seqlen=max(host_lens) + 1)


def reference(server: Server, q: torch.Tensor, total: int) -> torch.Tensor:
    """The last step's attention in fp32 over the cache's contents."""
    cu = torch.nn.functional.pad(server.lens.cumsum(0), (1, 0)).to(torch.int32)
    k, v = kq.page_read(server.k_cache, server.v_cache, server.tables, cu, total)
    group, out = q.shape[1] // k.shape[1], []
    ends = cu.tolist()
    for b in range(q.shape[0]):
        kb, vb = (t[ends[b]:ends[b + 1]].float().repeat_interleave(group, 1) for t in (k, v))
        s = torch.einsum("hd,jhd->hj", q[b].float(), kb) * q.shape[2] ** -0.5
        out.append(torch.einsum("hj,jhd->hd", s.softmax(1), vb))
    return torch.stack(out)


def run(requests=16, system=2048, prompt=300, steps=32, Hq=32, Hkv=8, D=128, page_size=16, dtype=torch.float16,
        quiet=False) -> dict:
    device = torch.device("cuda")
    E = 512
    layer = Layer(E, Hq, Hkv, D, dtype, device)
    g = torch.Generator(device).manual_seed(1)
    hidden = lambda n: torch.randn(n, E, generator=g, device=device).to(dtype)  # noqa: E731
    new = [1 + (prompt * (b + 1)) // requests for b in range(requests)]
    blocks = -(-(system + max(new) + steps) // page_size)
    pages = system // page_size + sum(-(-(n + steps) // page_size) for n in new)
    server = Server(layer, requests, pages, page_size, blocks, device)

    server.system_prompt(hidden(system))
    server.prompts(hidden(sum(new)), new)
    lens = [system + n for n in new]
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for step in range(steps):
        x = hidden(requests)
        if step == 1:
            begin.record()
        out = server.token(x, lens)
        lens = [n + 1 for n in lens]
    end.record()
    torch.cuda.synchronize()
    q = layer.qkv(x)[0]
    want = reference(server, q, sum(lens))
    result = {
        "lens": server.lens.tolist() == lens,
        "error": ((out.float() - want).norm() / want.norm()).item(),
        "us_per_step": begin.elapsed_time(end) / (steps - 1) * 1e3 if steps > 1 else float("nan"),
        "device_error": kq.device_error(),
    }
    if not quiet:
        print(f"{requests} requests behind {system} tokens, {steps} steps: {result['us_per_step']:.0f} us per step, "
              f"relative error of the last {result['error']:.1e}")
    return result


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("requests", 16), ("system", 2048), ("prompt", 300), ("steps", 32), ("page-size", 16)):
        p.add_argument(f"--{name}", type=int, default=value)
    run(**vars(p.parse_args()))
