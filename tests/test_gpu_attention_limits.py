"""attention_fp4 and append_fp4 at the ends of what their arguments may be."""

import numpy as np
import pytest
import torch

from oracle import attention as OA
from tests.helpers import host
from tests.test_gpu_attention import (attention, bf16_randn, check_attention, dev, f64, random_cache,  # noqa: F401
                                      rope_inputs, run_attention, say, tables)

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


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [3, 9000])
def test_pairs_of_an_axis_that_there_is_not_are_nan(attention, tokens, interleaved):  # noqa: F811
    """One axis, whose positions may be [T] or [1, T], and pairs that name axes 0, 1 and -1."""
    rng = np.random.default_rng(tokens)
    dim, rot, hq, hk = 64, 48, 2, 2
    table, at, _ = rope_inputs(rng, 50, rot, tokens, 1)
    of = np.zeros(rot // 2, dtype=np.int32)
    q, k = bf16_randn(rng, tokens, hq, dim).cuda(), bf16_randn(rng, tokens, hk, dim).cuda()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    attention.qk_norm_rope(q, k, None, None, dev(table), dev(at), None, q_out, k_out, 1e-6, interleaved)
    plain = q_out.clone(), k_out.clone()
    attention.qk_norm_rope(q, k, None, None, dev(table), dev(at[0]), dev(of), q_out, k_out, 1e-6, interleaved)
    assert torch.equal(q_out, plain[0]) and torch.equal(k_out, plain[1])
    of[3], of[10], of[23] = 1, -1, 2**31 - 1
    attention.qk_norm_rope(q, k, None, None, dev(table), dev(at), dev(of), q_out, k_out, 1e-6, interleaved)
    for x, got in ((q, q_out), (k, k_out)):
        y, size = OA.norm_rope64(f64(x), None, 0, table, rot, at, of, interleaved)
        nan = np.isnan(y)
        assert nan.sum() == tokens * 2 * 6 and np.array_equal(np.isnan(f64(got)), nan)
        assert np.all((np.abs(f64(got) - y) <= OA.norm_rope_bound(y, size, dim))[~nan])
    # appended, such a pair makes its blocks NaN
    cache = attention.new_cache(tokens // 16 + 1, hk, 16, dim)
    slots = torch.arange(tokens, device="cuda")
    attention.append_fp4(None, k, k, None, None, dev(table), dev(at), dev(of), slots, None, *cache, 1e-6, interleaved)
    with np.errstate(invalid="ignore"):
        codes, scales = OA.fp4_quantize(OA.norm_rope32(host(k.float()), None, 0, table, rot, at, of, interleaved))
    k_back, v_back = torch.empty_like(k), torch.empty_like(k)
    attention.unpack_fp4(*cache, slots, k_back, v_back)
    assert np.array_equal(f64(k_back), OA.fp4_values(codes, scales), equal_nan=True) and (scales == 255).any()


@pytest.mark.parametrize("tokens,heads", [(1, 4), (5, 6), (600, 4)])
def test_heads_that_take_turns_in_a_row(attention, tokens, heads):  # noqa: F811
    """Projections laid out [tokens, heads, 3, dim]: views of one buffer that share no element, in place."""
    rng = np.random.default_rng(tokens)
    dim, rot = 64, 64
    qkv = bf16_randn(rng, tokens, heads, 3, dim).cuda()
    apart = [qkv[:, :, i].contiguous() for i in range(3)]
    table, at, _ = rope_inputs(rng, 700, rot, tokens, 1)
    w = dev(np.exp(0.5 * rng.standard_normal(dim)).astype(np.float32))
    args = w, w, dev(table), dev(at[0]), None
    want = [torch.empty_like(t) for t in apart[:2]]
    attention.qk_norm_rope(*apart[:2], *args, *want)
    cache, cache2 = (attention.new_cache(tokens // 16 + 1, heads, 16, dim) for _ in range(2))
    slots = torch.arange(tokens, device="cuda")
    attention.append_fp4(*apart, *args, slots, torch.empty_like(apart[0]), *cache)
    q, k, v = qkv.unbind(2)
    mixed = qkv.clone().unbind(2)
    attention.append_fp4(*mixed, *args, slots, mixed[0], *cache2)
    assert torch.equal(mixed[0], want[0]) and torch.equal(mixed[1], apart[1]) and torch.equal(mixed[2], apart[2])
    assert all(torch.equal(a, b) for a, b in zip(cache, cache2))
    attention.qk_norm_rope(q, k, *args, q, k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, apart[2])


def test_more_contexts_than_a_launch_holds(attention):  # noqa: F811
    """65535 sequences of 129 key heads, of no token or of one: 2^23 + 65407 contexts, which 512 threads
    each would not fit. One token's output is its value, exactly."""
    rng = np.random.default_rng(1)
    seqs, heads, dim, page, pages, scale = 65535, 129, 64, 16, 40, 0.125
    cache = random_cache(attention, rng, pages, heads, page, dim)
    gen = torch.Generator("cuda").manual_seed(1)
    q = torch.randn(seqs, heads, dim, device="cuda", generator=gen, dtype=torch.float32).bfloat16()
    table = torch.randint(0, pages, (seqs, 1), device="cuda", generator=gen, dtype=torch.int32)
    lens = torch.randint(0, 2, (seqs,), device="cuda", generator=gen, dtype=torch.int32)
    out, lse = torch.full_like(q, 5.0), torch.full((seqs, heads), 5.0, device="cuda")
    attention.attention_fp4(q, *cache, table, lens, None, attention.new_workspace(dim), out, lse, scale)
    torch.cuda.synchronize()
    k, v = (torch.empty(pages, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    attention.unpack_fp4(*cache, torch.arange(pages, device="cuda") * page, k, v)
    for first in range(0, seqs, 4096):
        part = slice(first, min(first + 4096, seqs))
        at, one = table[part, 0].long(), lens[part].bool()
        assert torch.equal(out[part], torch.where(one[:, None, None], v[at], 0))
        assert (lse[part][~one] == -torch.inf).all()
        terms = q[part].double() * k[at].double() * scale
        score, off = terms.sum(-1), terms.abs().sum(-1) * (dim + 2) * 2.0**-24
        assert ((lse[part].double() - score).abs() <= off + 2.0**-15 + score.abs() * 2.0**-21)[one].all()
