#!/usr/bin/env python3
"""An attention layer with 4-bit weights and a 4-bit key/value cache, the operators together as a server calls them.

x -> w4a16_gemm (the fused q, k, v projection) -> kv4_write (new tokens' keys and values join the cache) -> kv4_attention
(over everything the cache holds) -> w4a16_gemm (the output projection).  Run as a script it serves a few sequences of
ragged prompts: the first prompt is read back (kv4_read) and written for a second sequence as a shared prefix, the prompts
are answered whole, tokens follow one by one from a captured graph, and everything is compared with the same layer computed
in fp32 from the values that the cache holds.

    python w4a16-gemm_amd/kv4_layer.py [--hidden 1024] [--heads 8] [--kv-heads 2] [--group 128] [--page 64] [--steps 8]
"""
from __future__ import annotations

import argparse
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
if HERE not in sys.path:
    sys.path.insert(0, HERE)


class Pages:
    """Which pages of the cache each sequence has: a block table on the GPU, pages given out in order."""

    def __init__(self, torch, sequences, most_tokens, page_size, device):
        self.page_size, self.width = page_size, -(-most_tokens // page_size)
        order = torch.randperm(sequences * self.width, generator=torch.Generator().manual_seed(0))
        self.table = order.view(sequences, self.width).to(device=device, dtype=torch.int32)
        self.count = sequences * self.width

    def slots(self, sequence, position):
        """Slots of tokens, int64: sequence and position are int64 tensors of the same shape."""
        page = self.table[sequence, position // self.page_size].long()
        return page * self.page_size + position % self.page_size


class Layer:
    """Projections held as w4a16_gemm takes them and a cache for `pages` pages."""

    def __init__(self, torch, hidden, heads, kv_heads, head_dim, group, pages, page_size, seed=0, device="cuda"):
        import w4a16_kv
        import w4a16_opt
        self.torch, self.gemm, self.kv = torch, w4a16_opt.w4a16_gemm, w4a16_kv
        self.hidden, self.heads, self.kv_heads, self.head_dim, self.group = hidden, heads, kv_heads, head_dim, group
        gen = torch.Generator(device).manual_seed(seed)
        rows = (heads + 2 * kv_heads) * head_dim

        def packed(n, k):
            w = torch.randn(n, k, generator=gen, device=device, dtype=torch.float32) * k**-0.5
            return w4a16_opt.quantize_pack(w.half(), 128)

        self.qkv, self.out = packed(rows, hidden), packed(hidden, heads * head_dim)
        self.cache = w4a16_kv.kv4_cache(pages, page_size, kv_heads, head_dim, group, device=device)

    def project(self, x):
        """q, k, v of x [tokens, hidden]: views of one product, which the cache's operators take as they are."""
        h, g, d = self.heads, self.kv_heads, self.head_dim
        y = self.gemm(self.qkv[0], x, self.qkv[1]).view(x.size(0), h + 2 * g, d)
        return y[:, :h], y[:, h:h + g], y[:, h + g:]

    def __call__(self, x, slots, table, seq_lens, q_start=None, max_q=0, window=0):
        """x [tokens, hidden] fp16, the last tokens of each sequence; seq_lens counts them in."""
        q, k, v = self.project(x)
        self.kv.kv4_write(self.cache, k, v, slots, self.group)
        y = self.kv.kv4_attention(q, self.cache, table, seq_lens, self.group, q_start=q_start, max_q=max_q, window=window)
        return self.gemm(self.out[0], y.reshape(x.size(0), -1), self.out[1])

    def plain(self, x, slots_of, q_start, window=0):
        """The same in fp32 from what the cache holds: slots_of[b] are sequence b's slots in order."""
        torch, h, g, d = self.torch, self.heads, self.kv_heads, self.head_dim
        q = self.project(x)[0].float()
        out = torch.zeros(x.size(0), h, d, device=x.device)
        for b, slots in enumerate(slots_of):
            i0, i1 = int(q_start[b]), int(q_start[b + 1])
            if i0 == i1:
                continue
            k, v = (t.float().repeat_interleave(h // g, 1).transpose(0, 1).contiguous()
                    for t in self.kv.kv4_read(self.cache, slots, d, self.group))
            at = torch.arange(slots.numel(), device=x.device)
            pos = slots.numel() - (i1 - i0) + torch.arange(i1 - i0, device=x.device)
            see = at <= pos[:, None]
            if window:
                see &= at > pos[:, None] - window
            s = (q[i0:i1].transpose(0, 1) @ k.transpose(1, 2).contiguous()) * d**-0.5
            out[i0:i1] = (s.masked_fill(~see, float("-inf")).softmax(-1) @ v).transpose(0, 1)
        return self.gemm(self.out[0], out.half().reshape(x.size(0), -1), self.out[1])


def serve(torch, hidden=1024, heads=8, kv_heads=2, head_dim=128, group=128, page=64, steps=8, prompts=(200, 0, 333, 64), window=0):
    """Serves len(prompts) sequences; returns the largest errors, relative to the largest output, of prompts and of steps.
    Sequence 1 has sequence 0's prompt as a prefix, copied from the cache, and so none of its own."""
    dev = torch.device("cuda")
    lens = [n if i != 1 else prompts[0] for i, n in enumerate(prompts)]
    pages = Pages(torch, len(lens), max(lens) + steps, page, dev)
    layer = Layer(torch, hidden, heads, kv_heads, head_dim, group, pages.count, page)
    gen = torch.Generator(dev).manual_seed(1)

    def tokens(n):
        return torch.randn(n, hidden, generator=gen, device=dev, dtype=torch.float32).half()

    def of(b, first, last):
        return pages.slots(torch.full((last - first,), b, device=dev), torch.arange(first, last, device=dev))

    def error(got, want):
        return float((got - want).abs().max() / want.abs().max())

    # the prompts, ragged, in one call
    q_start = torch.tensor([0, *prompts], dtype=torch.int32).cumsum(0).to(device=dev, dtype=torch.int32)
    x = tokens(sum(prompts))
    slots = torch.cat([of(b, 0, n) for b, n in enumerate(prompts)])
    seen = torch.tensor(prompts, dtype=torch.int32, device=dev)
    y = layer(x, slots, pages.table, seen, q_start, max(prompts), window)
    prompt_error = error(y, layer.plain(x, [of(b, 0, n) for b, n in enumerate(prompts)], q_start.tolist(), window))

    # sequence 1 starts from sequence 0's prompt: values that the cache gave back are quantised to the same bytes or next to them
    k, v = layer.kv.kv4_read(layer.cache, of(0, 0, prompts[0]), head_dim, group)
    layer.kv.kv4_write(layer.cache, k, v, of(1, 0, prompts[0]), group)

    # one token of every sequence a step, from a graph: its inputs stay where they are
    at = torch.tensor(lens, dtype=torch.int64, device=dev)
    x, slots, seq_lens = tokens(len(lens)), torch.zeros_like(at), torch.zeros(len(lens), dtype=torch.int32, device=dev)
    rows = torch.arange(len(lens), device=dev)

    def ready(i):
        x.copy_(tokens(len(lens)))
        slots.copy_(pages.slots(rows, at + i))
        seq_lens.copy_(at + i + 1)

    ready(0)
    layer(x, slots, pages.table, seq_lens, window=window)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = layer(x, slots, pages.table, seq_lens, window=window)
    step_error = 0.0
    for i in range(steps):
        ready(i)
        graph.replay()
        want = layer.plain(x, [of(b, 0, n + i + 1) for b, n in enumerate(lens)], list(range(len(lens) + 1)), window)
        step_error = max(step_error, error(y, want))
    return prompt_error, step_error


def main() -> int:
    import torch
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("hidden", 1024), ("heads", 8), ("kv-heads", 2), ("head-dim", 128), ("group", 128), ("page", 64), ("steps", 8),
                          ("window", 0)):
        ap.add_argument(f"--{name}", type=int, default=default)
    args = ap.parse_args()
    prompt, step = serve(torch, **vars(args))
    per = args.head_dim + 8 * args.head_dim // args.group
    print(f"prompts: largest error {prompt:.2e} of the largest output; {args.steps} steps: {step:.2e}")
    print(f"cache: {per} bytes a token and KV head, {4 * args.head_dim / per:.2f} times less than fp16")
    return 0


if __name__ == "__main__":
    sys.exit(main())
