"""examples/attention_block.py on the GPU: prompts of several sequences, then steps in a HIP graph,
against eager steps bit for bit and against attention in 64 bits over what the cache holds."""

import sys

import numpy as np
import pytest
import torch

from oracle import attention as OA
from tests.conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(ops):
    sys.path.insert(0, str(REPO / "examples"))
    import attention_block

    return attention_block


def check(block, pages, q, mixed, starts, window):
    """mixed against the formula, over every context as the cache holds it."""
    from consumer_int8 import attention

    heads, kv, dim = q.shape[1], block.kv_heads, block.dim
    for s, context in enumerate(pages.host_lens):
        slots = torch.tensor([pages.host[s][t // pages.page_size] * pages.page_size + t % pages.page_size
                              for t in range(context)], device="cuda")
        k, v = (torch.empty(context, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in "kv")
        attention.unpack_fp4(*block.cache, slots, k, v)
        rows = slice(starts[s], starts[s + 1])
        queries = q[rows].double().cpu().numpy()
        high = np.arange(context - len(queries), context) + 1
        low = np.maximum(high - window, 0) if window else np.zeros_like(high)
        k, v = (t.double().cpu().numpy() for t in (k, v))
        high, low = (np.repeat(t, heads // kv) for t in (high, low))
        got = mixed[rows].double().cpu().numpy()
        for h in range(kv):
            group = slice(h * (heads // kv), (h + 1) * (heads // kv))
            out, lse, mean, off = OA.attention64(queries[:, group].reshape(-1, dim), k[:, h], v[:, h], high, low,
                                                 dim**-0.5)
            bound, _ = OA.attention_bounds(out, lse, mean, off)
            assert np.all(np.abs(got[:, group].reshape(-1, dim) - out) <= bound), (s, h)


@pytest.mark.parametrize("heads,kv,dim,window", [(8, 2, 128, 0), (6, 3, 64, 24), (4, 1, 256, 0)])
def test_prompt_then_steps(example, heads, kv, dim, window):
    print("attention_block", heads, kv, dim, window, flush=True)
    torch.manual_seed(dim)
    prompts, page_size, hidden, steps = [70, 1, 129, 16], 16, 512, 5
    width = -(-(max(prompts) + steps) // page_size)
    pages = example.Pages(len(prompts), width, page_size)
    block = example.AttentionBlock(hidden, heads, kv, dim, len(prompts) * width, page_size, width * page_size,
                                   window)
    x = torch.randn(sum(prompts), hidden, device="cuda").bfloat16()
    starts = np.concatenate([[0], np.cumsum(prompts)])
    positions, slots = pages.extend(prompts)
    out, q, mixed = block(x, positions, slots, pages.table, pages.lens, torch.tensor(starts).int().cuda(),
                          max(prompts))
    check(block, pages, q, mixed, starts, window)
    assert torch.isfinite(out.float()).all()

    n = len(prompts)
    token = torch.randn(n, hidden, device="cuda").bfloat16()
    positions, slots = pages.extend([1] * n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(token, positions, slots, pages.table, pages.lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, q, mixed = block(token, positions, slots, pages.table, pages.lens)
    for step in range(steps):
        if step:
            new = pages.extend([1] * n)
            positions.copy_(new[0])
            slots.copy_(new[1])
            token.copy_(out)
        graph.replay()
        check(block, pages, q, mixed, np.arange(n + 1), window)
        replayed = [t.clone() for t in (out, q, mixed)]
        eager = block(token, positions, slots, pages.table, pages.lens)
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))
