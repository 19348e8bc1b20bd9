"""Decoding with drafts in examples/attention_block.py: trees appended, attended to, turned into
probabilities, verified and moved, several steps in a HIP graph, each against the same step run eagerly
bit for bit and against the 64-bit forms over what the cache holds."""

import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import drafts as OD
from tests.test_gpu_attention_block import example  # noqa: F401

pytestmark = pytest.mark.gpu

TREE = [-1, 0, 0, 1, 1, 2, 3, 0, 6]


def slots_of(pages, s, tokens):
    return torch.tensor([pages.host[s][t // pages.page_size] * pages.page_size + t % pages.page_size for t in tokens],
                        device="cuda")


def unpacked(block, slots):
    from consumer_int8 import attention

    k, v = (torch.empty(len(slots), block.kv_heads, block.dim, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    attention.unpack_fp4(*block.cache, slots, k, v)
    return k.double().cpu().numpy(), v.double().cpu().numpy()


def check_mixed(block, pages, q, mixed, before, window):
    """mixed against the formula; `before`: keys and values of all contexts as the step saw them."""
    heads, kv, dim, n = q.shape[1], block.kv_heads, block.dim, len(TREE)
    for s, context in enumerate(pages.host_lens):
        k, v = before[s]
        rows = slice(s * n, s * n + n)
        queries, got = (t[rows].double().cpu().numpy() for t in (q, mixed))
        seen = OD.tree_seen(TREE, context, window).repeat(heads // kv, 0)
        for h in range(kv):
            mine = slice(h * (heads // kv), (h + 1) * (heads // kv))
            out, lse, mean, off = OD.attention64(queries[:, mine].reshape(-1, dim), k[:, h], v[:, h], seen, dim**-0.5)
            bound, _ = OA.attention_bounds(out, lse, mean, off)
            assert np.all(np.abs(got[:, mine].reshape(-1, dim) - out) <= bound), (s, h)


@pytest.mark.parametrize("heads,kv,dim,window,seqs", [(8, 2, 128, 0, 3), (6, 3, 64, 24, 2), (16, 1, 256, 0, 2),
                                                      (32, 2, 128, 7, 5)])
def test_drafted_steps(example, heads, kv, dim, window, seqs):  # noqa: F811
    print("drafted steps", heads, kv, dim, window, seqs, flush=True)
    torch.manual_seed(dim + heads)
    page_size, hidden, vocab, n = 16, 512, 1024, len(TREE)
    prompts = [70, 1, 129, 16, 250][:seqs]
    width = -(-(max(prompts) + 8 * n) // page_size)
    pages = example.Pages(seqs, width, page_size)
    block = example.AttentionBlock(hidden, heads, kv, dim, seqs * width, page_size, width * page_size, window)
    x = torch.randn(sum(prompts), hidden, device="cuda").bfloat16()
    starts = torch.tensor([0] + prompts, device="cuda").cumsum(0).int()
    positions, slots = pages.extend(prompts)
    block(x, positions, slots, pages.table, pages.lens, starts, max(prompts))

    steps = example.DraftedSteps(block, hidden, vocab, seqs, TREE)
    steps.temperature[:] = torch.tensor([1.0, 0.6] * (seqs * n))[:seqs * n]
    run = lambda: steps.verify(pages.table, pages.lens)  # noqa: E731
    steps.extend(pages)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    steps.propose()
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    steps.keep(pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, mixed = run()
    taken = 0
    for step in range(5):
        steps.extend(pages)
        steps.propose()
        steps.uniforms.copy_(torch.rand(seqs * n))
        contexts = list(pages.host_lens)
        cache = [t.clone() for t in block.cache]
        graph.replay()
        torch.cuda.synchronize()
        found = [t.clone() for t in (q, mixed, steps.target, steps.path, steps.accepted, steps.next, *block.cache)]
        for t, old in zip(block.cache, cache):
            t.copy_(old)
        again = run()
        for a, b in zip(found, (*again, steps.target, steps.path, steps.accepted, steps.next, *block.cache)):
            assert torch.equal(a, b), step
        # What attention saw: without the moves.
        for t, old in zip(block.cache, cache):
            t.copy_(old)
        block(steps.embed[steps.tokens], steps.positions, steps.slots, pages.table, pages.lens, steps.q_starts, n,
              steps.parents)
        before = [unpacked(block, slots_of(pages, s, range(c))) for s, c in enumerate(contexts)]
        check_mixed(block, pages, q, mixed, before, window)
        for t, new in zip(block.cache, found[6:]):
            t.copy_(new)
        # The accepted rows by the 64-bit form of what was verified, and their keys and values in place.
        target, draft = (t.double().cpu().numpy() for t in (steps.target, steps.draft))
        assert np.abs(target.sum(1) - 1).max() < 1e-5
        tokens, uniforms = steps.tokens.cpu().numpy(), steps.uniforms.cpu().numpy()
        for s, context in enumerate(contexts):
            rows = slice(s * n, s * n + n)
            path, following, margin = OD.verify(target[rows], draft[rows], tokens[rows], TREE, uniforms[rows])
            assert margin > 1e-11
            assert steps.path[rows].tolist() == path + [-1] * (n - len(path))
            assert steps.accepted[s] == len(path) and steps.next[s] == following
            now = unpacked(block, slots_of(pages, s, range(context)))
            order = list(range(context - n)) + [context - n + r for r in path]
            for a, b in zip(now, before[s]):
                assert np.array_equal(a[:len(order)], b[order])
            taken += len(path)
        steps.keep(pages)
        assert pages.host_lens == [c - n + a for c, a in zip(contexts, steps.accepted.tolist())]
    assert taken >= 5 * seqs
