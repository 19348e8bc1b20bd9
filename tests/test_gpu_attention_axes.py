"""append_fp4 with several position axes, code for code against the FP32 form; head counts and sizes
that give a wave four groups of heads; prompts in a HIP graph."""

import numpy as np
import pytest
import torch

from oracle import attention as OA
from tests.helpers import host
from tests.test_gpu_attention import (attention, bf16_randn, dev, f64, layer, rope_inputs, say)  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,rot,hq,hk,tokens,axes,normed,interleaved", [
    (64, 64, 16, 16, 27, 3, True, True),
    (64, 48, 0, 3, 41, 2, False, False),
    (128, 128, 32, 8, 1, 3, True, False),
    (128, 64, 28, 4, 130, 4, True, True),
    (256, 256, 6, 2, 19, 3, True, False),
    (128, 96, 5, 1, 33, 5, True, False),          # more than four axes
    (64, 32, 14, 2, 50, 16, False, True),
    (256, 64, 24, 4, 4100, 3, True, False),       # four groups of heads a wave
    (64, 64, 16, 16, 4200, 3, True, True),
    (128, 128, 40, 8, 3000, 7, True, False),
])
def test_append_with_several_axes(attention, dim, rot, hq, hk, tokens, axes, normed, interleaved):  # noqa: F811
    say("append_fp4, axes", dim, rot, hq, hk, tokens, axes, interleaved)
    rng = np.random.default_rng(dim + rot + tokens + axes)
    page = 32
    pages = tokens // page + 2
    width = (hq + 2 * hk) * dim
    qkv = (bf16_randn(rng, tokens, width) * torch.exp(bf16_randn(rng, 1, width))).cuda()
    q, k, v = (t.unflatten(1, (-1, dim)) if t.shape[1] else None
               for t in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    qw, kw = ([np.exp(0.5 * rng.standard_normal(dim)).astype(np.float32) for _ in "qk"] if normed else (None, None))
    table, at, of = rope_inputs(rng, 300, rot, tokens, axes)
    if tokens > 20:
        at[axes - 1, 7], of[1] = 300, axes  # a position past the table, and an axis that there is not
    cache = attention.new_cache(pages, hk, page, dim)
    slots = rng.permutation(pages * page)[:tokens]
    q_out = torch.empty(tokens, hq, dim, dtype=torch.bfloat16, device="cuda") if hq else None
    attention.append_fp4(q, k, v, dev(qw) if hq else None, dev(kw), dev(table), dev(at), dev(of), dev(slots), q_out,
                         *cache, 1e-6, interleaved)
    if hq:
        y, size = OA.norm_rope64(f64(q), qw, 1e-6, table, rot, at, of, interleaved)
        nan = np.isnan(y)
        assert np.array_equal(np.isnan(f64(q_out)), nan)
        assert np.all((np.abs(f64(q_out) - y) <= OA.norm_rope_bound(y, size, dim))[~nan])
    where = slots // page, slice(None), slots % page
    k32 = OA.norm_rope32(host(k.float()), kw, 1e-6, table, rot, at, of, interleaved)
    for x, c, s in ((k32, cache.k_codes, cache.k_scales), (host(v.float()), cache.v_codes, cache.v_scales)):
        with np.errstate(invalid="ignore"):
            codes, scales = OA.fp4_quantize(x)
        assert np.array_equal(host(s)[where], scales)
        assert np.array_equal(OA.fp4_values(host(c)[where], scales), OA.fp4_values(codes, scales), equal_nan=True)


@pytest.mark.parametrize("dim,hq,hk,tokens,interleaved", [(64, 16, 16, 9000, False), (256, 24, 4, 4500, True),
                                                          (128, 40, 8, 3500, False)])
def test_four_groups_a_wave(attention, dim, hq, hk, tokens, interleaved):  # noqa: F811
    """Norm and rotation without a cache, one axis."""
    say("qk_norm_rope", dim, hq, hk, tokens)
    rng = np.random.default_rng(tokens)
    rot = dim // 2
    q, k = bf16_randn(rng, tokens, hq, dim).cuda(), bf16_randn(rng, tokens, hk, dim).cuda()
    qw, kw = (np.exp(0.5 * rng.standard_normal(dim)).astype(np.float32) for _ in "qk")
    table, at, _ = rope_inputs(rng, 9000, rot, tokens, 1)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    attention.qk_norm_rope(q, k, dev(qw), dev(kw), dev(table), dev(at[0]), None, q_out, k_out, 1e-6, interleaved)
    for x, w, got in ((q, qw, q_out), (k, kw, k_out)):
        y, size = OA.norm_rope64(f64(x), w, 1e-6, table, rot, at, None, interleaved)
        assert np.all(np.abs(f64(got) - y) <= OA.norm_rope_bound(y, size, dim))


@pytest.mark.parametrize("dim,hq,hk", [(64, 14, 2), (128, 8, 2), (256, 6, 1)])
def test_prompts_in_a_graph(attention, dim, hq, hk):  # noqa: F811
    """Chunks of prompts, decodes and drafted tokens in one captured call, replayed with other lengths
    and starts, against eager calls."""
    rng = np.random.default_rng(dim)
    page, seqs, width, tokens, max_q = 16, 4, 60, 420, 300
    pages = dev(rng.permutation(seqs * width).astype(np.int32).reshape(seqs, width))
    table = attention.rope_table(1024, dim)
    cache = attention.new_cache(seqs * width, hk, page, dim)
    eager_cache = attention.new_cache(seqs * width, hk, page, dim)
    ws, ws2 = attention.new_workspace(dim), attention.new_workspace(dim)
    qkv = bf16_randn(rng, tokens, (hq + 2 * hk) * dim).cuda()
    lens, starts = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (seqs, seqs + 1))
    at, slots = (torch.zeros(tokens, dtype=torch.int64, device="cuda") for _ in range(2))

    def load(lengths, counts):
        place, slot = np.zeros(tokens, dtype=np.int64), np.full(tokens, -1, dtype=np.int64)
        begin, host_pages = np.concatenate([[0], np.cumsum(counts)]), pages.cpu().numpy()
        for s, (n, c) in enumerate(zip(lengths, counts)):
            t = np.arange(n - c, n)
            place[begin[s]:begin[s + 1]] = t
            slot[begin[s]:begin[s + 1]] = host_pages[s, t // page].astype(np.int64) * page + t % page
        for to, x in ((lens, np.int32(lengths)), (starts, np.int32(begin)), (at, place), (slots, slot)):
            to.copy_(dev(x))
        qkv.copy_(bf16_randn(rng, *qkv.shape).cuda())
        return int(begin[-1])

    def call(c, w):
        return layer(attention, qkv, hq, hk, dim, (None, None), table, at, slots, c, pages, lens, starts, max_q, w)

    load([300, 1, 60, 9], [300, 1, 60, 9])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(cache, ws)
    torch.cuda.current_stream().wait_stream(side)
    for t, e in zip(cache, eager_cache):
        e.copy_(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(cache, ws)
    for lengths, counts in [([310, 301, 61, 14], [10, 300, 1, 5]), ([610, 302, 161, 15], [300, 1, 100, 1]),
                            ([611, 303, 162, 16], [1, 1, 1, 1]), ([960, 500, 163, 20], [220, 197, 1, 2])]:
        used = load(lengths, counts)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = call(eager_cache, ws2)
        assert torch.equal(out[:used], want[:used])
        assert all(torch.equal(a, b) for a, b in zip(cache, eager_cache))
