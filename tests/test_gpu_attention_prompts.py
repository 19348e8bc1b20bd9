"""Prompts through many tiles a workgroup, so that every LDS buffer is used over and over by waves
that have drifted apart: against the 64-bit form, and for the same bits on a second call."""

import numpy as np
import pytest
import torch

from tests.helpers import host
from tests.test_gpu_attention import (bf16_randn, check_attention, f64, random_cache,  # noqa: F401
                                      attention, run_attention, say, tables)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,hq,hk,lens,counts,window", [
    (64, 14, 2, [8000], [300], 0),               # 63 tiles of 128 tokens
    (64, 14, 2, [8000, 700], [300, 700], 1500),
    (64, 16, 16, [2000], [2000], 0),
    (64, 4, 2, [2000], [2000], 700),
    (64, 3, 1, [9001, 3003], [203, 1501], 0),
    (128, 10, 2, [2111], [2111], 0),
    (256, 6, 1, [1500], [1500], 900),
])
def test_many_tiles(attention, dim, hq, hk, lens, counts, window):  # noqa: F811
    say("prompts", dim, hq, hk, lens, counts, window)
    rng = np.random.default_rng(sum(lens) + dim + hq)
    page = 32
    pages = sum(-(-n // page) for n in lens) + 3
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = [0] + list(np.cumsum(counts))
    q = bf16_randn(rng, starts[-1], hq, dim).cuda()
    out, lse = run_attention(attention, q, cache, table, lens, starts, dim**-0.5, max(counts), window)
    check_attention(q, cache, table, lens, starts, dim**-0.5, max(counts), window, out, lse)
    for _ in range(3):
        again, lse2 = run_attention(attention, q, cache, table, lens, starts, dim**-0.5, max(counts), window)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_values_in_many_tiles(attention, dim):  # noqa: F811
    """Blocks of values that are NaN, in tiles that some rows see in part and others whole: they
    reach the rows that see their token, in their own channels, and no others."""
    rng = np.random.default_rng(dim)
    page, n, heads = 16, 900, 2
    cache = random_cache(attention, rng, 60, 1, page, dim)
    table = tables(rng, [n], 60, page)
    q = bf16_randn(rng, n, heads, dim).cuda()
    clean, clean_lse = run_attention(attention, q, cache, table, [n], [0, n], 0.1, n, 0)
    want = host(torch.zeros(n, dim, dtype=torch.bool))
    blocks = dim // 32
    for token, block in [(899, 0), (700, 1), (511, 0), (512, 1), (400, 0)]:
        block = block * (blocks - 1)
        cache.v_scales[int(table[0, token // page]), 0, token % page, block] = 255
        want[token:, 32 * block:32 * block + 32] = True
    out, lse = run_attention(attention, q, cache, table, [n], [0, n], 0.1, n, 0)
    nan = np.isnan(f64(out))
    assert np.array_equal(nan, np.repeat(want[:, None], heads, 1))
    assert np.array_equal(f64(out)[~nan], f64(clean)[~nan]) and torch.equal(lse, clean_lse)
