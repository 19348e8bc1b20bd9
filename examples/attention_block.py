"""An attention layer as a serving program runs it: INT8 projections around attention over a
paged 4-bit cache, prompts of several sequences in one call, then token by token in a HIP graph.

    python examples/attention_block.py [--tokens 64]

Weights and inputs are random; it prints the time of the prompt and of a decode step.
"""

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "consumer-int8-kernels_amd"))
from consumer_int8 import attention, ops  # noqa: E402


def int8_weight(n, k, device="cuda"):
    """Random INT8 [n, k] with a BF16 scale a row, of about unit gain."""
    codes = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=device)
    return codes, torch.full((n,), 1 / (73.3 * k**0.5), dtype=torch.bfloat16, device=device)


def project(x, weight, out):
    """out = x @ weight.T: W8A16 for a few rows, W8A8 with the rows quantized for more."""
    codes, scale = weight
    if x.shape[0] <= 16:
        ops.channel_gemv(x, codes, scale, out)
        return
    x_codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    x_scale = torch.empty(x.shape[0], device=x.device)
    ops.quantize_rows(x, x_codes, x_scale)
    ops.fused_channel_mm(x_codes, codes, x_scale, scale, out)


class Pages:
    """Which pages each sequence has. Page tables only grow, so a captured graph sees new pages
    in the same tensors."""

    def __init__(self, seqs, width, page_size, device="cuda"):
        self.page_size, self.width = page_size, width
        self.free = list(range(seqs * width))[::-1]
        self.host = [[] for _ in range(seqs)]
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.host_lens = [0] * seqs

    def extend(self, counts):
        """Room for counts[s] more tokens of each sequence: their positions and slots."""
        positions, slots = [], []
        for s, count in enumerate(counts):
            first = self.host_lens[s]
            if -(-(first + count) // self.page_size) > self.width:
                raise RuntimeError("Sequence longer than its page table")
            while len(self.host[s]) * self.page_size < first + count:
                self.host[s].append(self.free.pop())
            for t in range(first, first + count):
                positions.append(t)
                slots.append(self.host[s][t // self.page_size] * self.page_size + t % self.page_size)
            self.host_lens[s] = first + count
        rows = [pages + [-1] * (self.width - len(pages)) for pages in self.host]
        self.table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.lens.copy_(torch.tensor(self.host_lens, dtype=torch.int32))
        device = self.table.device
        return torch.tensor(positions, device=device), torch.tensor(slots, device=device)


class AttentionBlock:
    def __init__(self, hidden, q_heads, kv_heads, dim, pages, page_size, max_rows, window=0, device="cuda"):
        self.q_heads, self.kv_heads, self.dim, self.window = q_heads, kv_heads, dim, window
        self.qkv_weight = int8_weight((q_heads + 2 * kv_heads) * dim, hidden, device)
        self.out_weight = int8_weight(hidden, q_heads * dim, device)
        self.q_norm = torch.ones(dim, device=device)
        self.k_norm = torch.ones(dim, device=device)
        self.rope = attention.rope_table(max_rows, dim, device=device)
        self.cache = attention.new_cache(pages, kv_heads, page_size, dim, device)
        self.workspace = attention.new_workspace(dim, device)

    def __call__(self, x, positions, slots, page_table, context_lens, q_starts=None, max_q=1):
        """BF16 x [T, hidden]: rows q_starts[s] .. of each sequence, or one row each. Returns the
        layer's output and, for callers that look inside, the queries and what they attended to."""
        tokens, heads, kv, dim = x.shape[0], self.q_heads, self.kv_heads, self.dim
        qkv = torch.empty(tokens, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device=x.device)
        project(x, self.qkv_weight, qkv)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        # The normed queries replace the projected ones; keys and values go straight to the cache.
        attention.append_fp4(q, k, v, self.q_norm, self.k_norm, self.rope, positions, None, slots, q,
                             *self.cache)
        mixed = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=x.device)
        attention.attention_fp4(q, *self.cache, page_table, context_lens, q_starts, self.workspace, mixed,
                                None, dim**-0.5, max_q, self.window)
        out = torch.empty_like(x)
        project(mixed.flatten(1), self.out_weight, out)
        return out, q, mixed


def timed(call, steps=1):
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(steps):
        call()
    torch.cuda.synchronize()
    return (time.perf_counter() - start) / steps * 1e6


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--tokens", type=int, default=64, help="tokens to decode")
    args = parser.parse_args()
    torch.manual_seed(0)
    prompts, page_size, hidden = [700, 1, 2048, 33], 64, 5120
    width = -(-(max(prompts) + args.tokens) // page_size)
    pages = Pages(len(prompts), width, page_size)
    block = AttentionBlock(hidden, 40, 8, 128, len(prompts) * width, page_size, width * page_size)

    x = torch.randn(sum(prompts), hidden, device="cuda").bfloat16()
    starts = torch.tensor([0] + prompts, device="cuda").cumsum(0).int()
    positions, slots = pages.extend(prompts)
    prompt = lambda: block(x, positions, slots, pages.table, pages.lens, starts, max(prompts))
    prompt()
    print(f"prompts of {prompts} tokens: {timed(prompt):.0f} us")

    # One step in a graph: its inputs are refilled before each replay.
    token = torch.randn(len(prompts), hidden, device="cuda").bfloat16()
    positions, slots = pages.extend([1] * len(prompts))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(token, positions, slots, pages.table, pages.lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, *_ = block(token, positions, slots, pages.table, pages.lens)
    graph.replay()
    print(f"a step of {len(prompts)} sequences in a graph: {timed(graph.replay, 100):.1f} us")
    for _ in range(args.tokens - 1):
        new = pages.extend([1] * len(prompts))
        positions.copy_(new[0])
        slots.copy_(new[1])
        token.copy_(out)
        graph.replay()
    print(f"after {args.tokens} tokens: contexts {pages.lens.tolist()}, outputs of rms "
          f"{out.float().square().mean().sqrt().item():.3f}")


if __name__ == "__main__":
    main()
