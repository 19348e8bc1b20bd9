"""GPU checks of speculative decoding's operators at the ends of their ranges; forms and bounds are those of
tests/test_gpu_drafts.py."""

import math

import numpy as np
import pytest
import torch

from tests.helpers import guard_intact, with_guard
from tests.test_gpu_attention import bf16_randn, random_cache, say
from tests.test_gpu_drafts import attention, check_probs, check_tree, random_tree, run_tree, sampling  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(7, 1000), (7, 40003), (200, 40003)])
def test_probs_of_far_logits(sampling, rows, vocab, dtype):  # noqa: F811
    """Logits further apart than the largest number, at temperatures that bring them together again."""
    say("far logits", rows, vocab, dtype)
    rng = np.random.default_rng(rows + vocab)
    x = rng.uniform(-3.3e38, 3.3e38, (rows, vocab))
    x[:, 7], x[:, vocab - 3] = 3.3e38, -3.3e38
    x[0, :vocab // 2] = -math.inf
    t = np.float32([1.5e38, 3e38, 4e37, math.inf, 1.0, 0.5, 1e37] + [2e38] * (rows - 7))
    x = torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()
    check_probs(sampling, x, t, torch.empty(rows, vocab, device="cuda"))


def test_trees_of_many_sequences_and_heads(attention):  # noqa: F811
    """65535 sequences of 128 key heads: more than the prompt kernel's launch holds, which trees do not
    take. The first and the last have rows."""
    say("trees of many sequences and heads")
    rng = np.random.default_rng(8)
    dim, page, hk, group, seqs = 64, 16, 128, 3, 65535
    lens, counts = np.zeros(seqs, np.int64), np.zeros(seqs, np.int64)
    lens[[0, -1]], counts[[0, -1]] = [100, 37], [30, 34]
    starts = np.concatenate([[0], np.cumsum(counts)])
    cache = random_cache(attention, rng, 12, hk, page, dim)
    table = np.zeros((seqs, 7), np.int32)
    table[0], table[-1] = rng.permutation(12)[:7], rng.permutation(12)[:7]
    parents = np.concatenate([random_tree(rng, n, 0.5) for n in (30, 34)])
    q = bf16_randn(rng, 64, hk * group, dim).cuda()
    out, lse = run_tree(attention, q, cache, table, lens, starts, parents, 0.1, 64, 0)
    check_tree(q, cache, table, lens, starts, parents, 0.1, 0, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [262209, 1000003, 1 << 21, (1 << 21) + 5])
def test_probs_of_one_long_row(sampling, vocab, dtype):  # noqa: F811
    say("one long row", vocab, dtype)
    rng = np.random.default_rng(vocab)
    x = torch.from_numpy((3 * rng.standard_normal((1, vocab))).astype(np.float32)).to(dtype).cuda()
    for t in (None, [0.0], [0.7]):
        out, guard = with_guard((1, vocab), torch.float32, 5.0)
        check_probs(sampling, x, t, out)
        assert guard_intact(guard, 5.0)
