"""An attention layer as a serving program runs it: INT8 projections around attention over a
paged 4-bit cache, prompts of several sequences in one call, then token by token in a HIP graph, then
by trees of drafted tokens, each verified in one step.

    python examples/attention_block.py [--tokens 64]

Weights and inputs are random; it prints the time of the prompt and of a decode step.
"""

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "consumer-int8-kernels_amd"))
from consumer_int8 import attention, ops, sampling  # noqa: E402


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

    def keep(self, lens):
        """The first lens[s] tokens of each sequence stay, the slots of the others are given anew."""
        self.host_lens = list(lens)
        self.lens.copy_(torch.tensor(self.host_lens, dtype=torch.int32))


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

    def __call__(self, x, positions, slots, page_table, context_lens, q_starts=None, max_q=1, parents=None):
        """BF16 x [T, hidden]: rows q_starts[s] .. of each sequence, or one row each; with `parents` they
        are trees. Returns the layer's output and, for callers that look inside, the queries and what
        they attended to."""
        tokens, heads, kv, dim = x.shape[0], self.q_heads, self.kv_heads, self.dim
        qkv = torch.empty(tokens, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device=x.device)
        project(x, self.qkv_weight, qkv)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        # The normed queries replace the projected ones; keys and values go straight to the cache.
        attention.append_fp4(q, k, v, self.q_norm, self.k_norm, self.rope, positions, None, slots, q,
                             *self.cache)
        mixed = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=x.device)
        if parents is None:
            attention.attention_fp4(q, *self.cache, page_table, context_lens, q_starts, self.workspace, mixed,
                                    None, dim**-0.5, max_q, self.window)
        else:
            attention.attention_fp4_tree(q, *self.cache, page_table, context_lens, q_starts, parents,
                                         self.workspace, mixed, None, dim**-0.5, max_q, self.window)
        out = torch.empty_like(x)
        project(mixed.flatten(1), self.out_weight, out)
        return out, q, mixed


class DraftedSteps:
    """Decoding with drafts: a drafter (here the layer's head on the embeddings alone) grows the same tree
    for each of `seqs` sequences from its last token, and one pass over all rows decides which stand.
    Everything stays on the device; the buffers are the same in every step, so that both halves can be
    captured into graphs."""

    def __init__(self, block, hidden, vocab, seqs, tree, device="cuda"):
        self.block, self.tree, self.seqs, rows = block, tree, seqs, seqs * len(tree)
        self.embed = torch.randn(vocab, hidden, device=device).bfloat16()
        self.head = int8_weight(vocab, hidden, device)
        self.parents = torch.tensor(tree * seqs, dtype=torch.int32, device=device)
        self.q_starts = torch.arange(0, rows + 1, len(tree), dtype=torch.int32, device=device)
        depth = []
        for parent in tree:
            depth.append(0 if parent < 0 else depth[parent] + 1)
        self.depth = torch.tensor(depth * seqs, device=device)
        self.levels = [[i for i, d in enumerate(depth) if d == level] for level in range(max(depth) + 1)]
        self.tokens = torch.zeros(rows, dtype=torch.int64, device=device)
        self.draft = torch.zeros(rows, vocab, device=device)
        self.target = torch.empty(rows, vocab, device=device)
        self.temperature = torch.ones(rows, device=device)
        self.uniforms = torch.empty(rows, device=device)
        self.positions, self.slots = (torch.zeros(rows, dtype=torch.int64, device=device) for _ in "ps")
        self.path = torch.empty(rows, dtype=torch.int32, device=device)
        self.accepted = torch.empty(seqs, dtype=torch.int32, device=device)
        self.next = torch.zeros(seqs, dtype=torch.int64, device=device)
        self.workspace = sampling.new_workspace(device)

    def probs(self, x, temperature, out):
        logits = torch.empty(x.shape[0], self.embed.shape[0], dtype=torch.bfloat16, device=x.device)
        project(x, self.head, logits)
        sampling.token_probs(logits, temperature, self.workspace, out)

    def propose(self):
        """Tokens of the trees from self.next on, a level at a time, each child drawn from its parent's
        probabilities."""
        n = len(self.tree)
        tokens, draft = self.tokens.view(self.seqs, n), self.draft.view(self.seqs, n, -1)
        tokens[:, 0] = self.next
        for level in self.levels[:-1]:
            rows = self.embed[tokens[:, level].flatten()]
            found = torch.empty(rows.shape[0], draft.shape[2], device=rows.device)
            self.probs(rows, self.temperature[:rows.shape[0]], found)
            draft[:, level] = found.view(self.seqs, len(level), -1)
            for i in level:
                children = [c for c, parent in enumerate(self.tree) if parent == i]
                if children:
                    tokens[:, children] = torch.multinomial(draft[:, i], len(children), replacement=True)

    def verify(self, page_table, context_lens):
        """The target's pass over all trees: path, accepted and next say what stands, and the accepted
        rows' keys and values are in each sequence's first slots."""
        x = self.embed[self.tokens]
        out, q, mixed = self.block(x, self.positions, self.slots, page_table, context_lens, self.q_starts,
                                   len(self.tree), self.parents)
        self.probs(x + out, self.temperature, self.target)
        sampling.verify_drafts(self.target, self.draft, self.tokens, self.parents, self.q_starts, self.uniforms,
                               self.workspace, self.path, self.accepted, self.next)
        attention.move_fp4(*self.block.cache, self.path, self.slots, self.q_starts)
        return q, mixed

    def extend(self, pages):
        """Room for the trees; a row's position is its depth's."""
        first = torch.tensor(pages.host_lens, device=self.depth.device).repeat_interleave(len(self.tree))
        self.positions.copy_(first + self.depth)
        self.slots.copy_(pages.extend([len(self.tree)] * self.seqs)[1])

    def keep(self, pages):
        """What was accepted stays: the host learns how many."""
        n = len(self.tree)
        pages.keep([context - n + a for context, a in zip(pages.host_lens, self.accepted.tolist())])


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
    tree = [-1, 0, 0, 1, 1, 2, 3]  # two children, two more of the first, one each of the next two
    width = -(-(max(prompts) + args.tokens * (2 + len(tree))) // page_size)
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

    steps = DraftedSteps(block, hidden, 32000, len(prompts), tree)
    verify = lambda: steps.verify(pages.table, pages.lens)
    steps.extend(pages)
    steps.propose()
    steps.uniforms.uniform_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify()
    torch.cuda.current_stream().wait_stream(side)
    steps.keep(pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        verify()
    total = 0
    for _ in range(args.tokens):
        steps.extend(pages)
        steps.propose()
        steps.uniforms.uniform_()
        graph.replay()
        steps.keep(pages)
        total += sum(steps.accepted.tolist())
    print(f"trees of {len(tree)} rows: {total / args.tokens / len(prompts):.2f} tokens a step and sequence")
    steps.extend(pages)
    print(f"a step of {len(prompts)} trees in a graph: {timed(graph.replay, 100):.1f} us")


if __name__ == "__main__":
    main()
