"""attention_fp4 and append_fp4 at the ends of what their arguments may be."""

import numpy as np
import pytest
import torch

from tests.test_gpu_attention import (attention, bf16_randn, check_attention, random_cache,  # noqa: F401
                                      run_attention, say, tables)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,hq,hk,lens,counts", [
    (128, 8, 2, [3, 90, 0], [8, 8, 5]),        # some queries are before the first token
    (64, 2, 1, [2100, 4], [20, 20]),
    (256, 6, 1, [40, 700], [100, 100]),        # prompts
    (64, 4, 4, [100, 300], [200, 150]),
])
def test_windows_past_the_page_table_hide_nothing(attention, dim, hq, hk, lens, counts):  # noqa: F811
    say("windows", dim, hq, hk, lens, counts)
    rng = np.random.default_rng(dim + sum(lens))
    page = 16
    pages = sum(-(-n // page) for n in lens) + 1
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    holds = table.shape[1] * page
    starts = [0] + list(np.cumsum(counts))
    q = bf16_randn(rng, starts[-1], hq, dim).cuda()
    want, want_lse = run_attention(attention, q, cache, table, lens, starts, 0.09, max(counts), 0)
    check_attention(q, cache, table, lens, starts, 0.09, max(counts), 0, want, want_lse)
    for window in (holds, holds + 1, 2**31 - 9, 2**31 - 2, 2**31 - 1, 2**31, 2**32 + 1, 2**63 - 1):
        out, lse = run_attention(attention, q, cache, table, lens, starts, 0.09, max(counts), window)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), window
    for window in (holds - 1, max(lens) - 1):
        out, lse = run_attention(attention, q, cache, table, lens, starts, 0.09, max(counts), window)
        check_attention(q, cache, table, lens, starts, 0.09, max(counts), window, out, lse)
