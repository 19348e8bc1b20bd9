"""GPU checks of the attention operators against their 64-bit forms (oracle/attention.py), with
bounds derived there; codes and scales bit for bit against the FP32 form."""

import math

import numpy as np
import pytest
import torch

from oracle import attention as OA
from tests.helpers import guard_intact, host, to_dev, with_guard

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attention(ops):
    from consumer_int8 import attention as module

    return module


def bf16_randn(rng, *shape, scale=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).bfloat16()


def f64(t):
    return t.detach().double().cpu().numpy()


def say(*a):
    print(*a, flush=True)


# ---- norm and rotation ------------------------------------------------------------------


def rope_inputs(rng, rows, rot, tokens, axes):
    angle = rng.uniform(-math.pi, math.pi, (rows, rot // 2))
    table = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)
    at = rng.integers(0, rows, (axes, tokens))
    of = rng.integers(0, axes, rot // 2).astype(np.int32) if axes > 1 else None
    return table, at, of


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("dim,rot,hq,hk,tokens,axes,normed,interleaved,layout", [
    (64, 64, 1, 1, 1, 1, True, False, "rows"),
    (64, 16, 14, 2, 37, 3, True, True, "rows"),
    (64, 48, 16, 16, 5, 2, False, False, "apart"),
    (128, 128, 32, 8, 1, 1, True, False, "rows"),
    (128, 32, 28, 4, 129, 1, True, True, "heads"),
    (128, 0, 7, 1, 33, 1, True, False, "apart"),
    (128, 112, 5, 5, 300, 4, True, False, "inplace"),
    (256, 64, 24, 4, 66, 1, True, False, "inplace"),
    (256, 256, 3, 1, 2, 3, False, True, "rows"),
    (256, 80, 16, 2, 517, 1, True, False, "rows"),
    (128, 128, 40, 8, 2050, 1, True, False, "rows"),
    (128, 128, 8, 8, 9000, 1, False, True, "inplace"),
])
def test_qk_norm_rope(attention, dim, rot, hq, hk, tokens, axes, normed, interleaved, layout):
    rng = np.random.default_rng(dim + rot + hq + tokens)
    say("qk_norm_rope", dim, rot, hq, hk, tokens, axes, layout)
    width = (hq + 2 * hk) * dim + 16
    qkv = (bf16_randn(rng, tokens, width) * torch.exp(bf16_randn(rng, tokens, 1, scale=2))).cuda()
    q, k = qkv[:, :hq * dim].unflatten(1, (hq, dim)), qkv[:, hq * dim:(hq + hk) * dim].unflatten(1, (hk, dim))
    if layout == "heads":  # heads outside
        q, k = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    qw, kw = ([np.exp(0.5 * rng.standard_normal(dim)).astype(np.float32) for _ in "qk"] if normed else (None, None))
    table, at, of = rope_inputs(rng, 700, rot, tokens, axes) if rot else (None, None, None)
    want = [OA.norm_rope64(f64(x), w, 1e-6, table, rot, at, of, interleaved) for x, w in ((q, qw), (k, kw))]
    rest = host(qkv[:, (hq + hk) * dim:].view(torch.int16)).copy()
    if layout == "inplace":
        q_out, k_out, guards = q, k, []
    else:
        (q_out, qb), (k_out, kb) = (with_guard((tokens, h, dim), torch.bfloat16, 3.0) for h in (hq, hk))
        guards = [qb, kb]
    positions = None if at is None else dev(at[0] if axes == 1 else at)
    attention.qk_norm_rope(q, k, dev(qw), dev(kw), dev(table), positions, dev(of), q_out, k_out, 1e-6, interleaved)
    torch.cuda.synchronize()
    for got, (y, size) in zip((q_out, k_out), want):
        assert np.all(np.abs(f64(got) - y) <= OA.norm_rope_bound(y, size, dim))
    assert all(guard_intact(b, 3.0) for b in guards)
    assert np.array_equal(host(qkv[:, (hq + hk) * dim:].view(torch.int16)), rest)


def test_rotation_outside_the_table_is_nan_and_inside_is_untouched(attention):
    q = torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.ones(4, 1, 64, dtype=torch.bfloat16, device="cuda")
    table = attention.rope_table(10, 32)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    at = torch.tensor([0, 9, 10, -1], device="cuda")
    attention.qk_norm_rope(q, k, None, None, table, at, None, q_out, k_out)
    bad = host(torch.isnan(q_out.float()).any(-1))
    assert bad.tolist() == [[False] * 2] * 2 + [[True] * 2] * 2
    assert torch.isnan(q_out[2:, :, :32].float()).all() and (q_out[2:, :, 32:] == 1).all()
    axes = torch.zeros(16, dtype=torch.int32, device="cuda")
    axes[3], axes[5] = 2, -1
    attention.qk_norm_rope(q, k, None, None, table, at.clamp(0, 9).repeat(2, 1), axes, q_out, k_out)
    nan = torch.isnan(q_out.float())
    assert nan[:, :, [3, 5, 19, 21]].all() and int(nan.sum()) == 4 * 2 * 4


def test_norm_of_zeros_infinities_and_nan(attention):
    q = torch.zeros(3, 1, 128, dtype=torch.bfloat16, device="cuda")
    q[1, 0, 5], q[2, 0, 7] = math.inf, math.nan
    k = torch.zeros_like(q)
    w = torch.ones(128, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    attention.qk_norm_rope(q, k, w, w, None, None, None, q_out, k_out, 1e-6)
    assert (q_out[0] == 0).all() and (k_out == 0).all()
    assert torch.isnan(q_out[1, 0, 5]) and (q_out[1, 0, 6:] == 0).all()
    assert torch.isnan(q_out[2].float()).all()


# ---- the cache --------------------------------------------------------------------------


@pytest.mark.parametrize("dim,rot,hq,hk,tokens,page,normed,interleaved,pool", [
    (64, 64, 0, 2, 1, 16, True, False, "plain"),
    (64, 32, 14, 2, 77, 32, True, True, "pool"),
    (128, 128, 32, 8, 64, 16, True, False, "plain"),
    (128, 0, 0, 5, 33, 64, False, False, "pool"),
    (128, 64, 7, 7, 1000, 128, True, False, "plain"),
    (256, 64, 24, 4, 259, 1024, True, False, "pool"),
    (256, 256, 3, 1, 3, 16, False, True, "plain"),
    (128, 128, 40, 8, 4100, 64, True, False, "pool"),
])
def test_append_and_unpack(attention, dim, rot, hq, hk, tokens, page, normed, interleaved, pool):
    rng = np.random.default_rng(dim + rot + hk + tokens)
    say("append_fp4", dim, rot, hq, hk, tokens, page, pool)
    pages = tokens // page + 7
    width = (hq + 2 * hk) * dim
    qkv = (bf16_randn(rng, tokens, width) * torch.exp(bf16_randn(rng, 1, width))).cuda()
    qkv[0, -32:] = 0
    q, k, v = qkv.split([hq * dim, hk * dim, hk * dim], 1)
    q, k, v = (t.unflatten(1, (-1, dim)) if t.shape[1] else None for t in (q, k, v))
    qw, kw = ([np.exp(0.5 * rng.standard_normal(dim)).astype(np.float32) for _ in "qk"] if normed else (None, None))
    table, at, _ = rope_inputs(rng, 500, rot, tokens, 1) if rot else (None, None, None)
    if pool == "plain":
        cache = attention.new_cache(pages, hk, page, dim)
        for t in cache:
            t.fill_(0xA5)
    else:  # all four parts of a page in one record, as one pool
        sizes = [hk * page * dim // n for n in (2, 32, 2, 32)]
        flat = torch.full((pages, sum(sizes) + 64), 0xA5, dtype=torch.uint8, device="cuda")
        parts = flat.split(sizes + [64], 1)[:4]
        cache = attention.Fp4Cache(*(t.unflatten(1, (hk, page, -1)) for t in parts))
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 2:
        slots[1], slots[-1] = -1, pages * page  # padding, and outside
    q_out = torch.empty(tokens, hq, dim, dtype=torch.bfloat16, device="cuda") if hq else None
    attention.append_fp4(q, k, v, dev(qw) if hq else None, dev(kw), dev(table), None if at is None else dev(at[0]),
                         None, dev(slots), q_out, *cache, 1e-6, interleaved)
    torch.cuda.synchronize()
    if hq:
        y, size = OA.norm_rope64(f64(q), qw, 1e-6, table, rot, at, None, interleaved)
        assert np.all(np.abs(f64(q_out) - y) <= OA.norm_rope_bound(y, size, dim))
    kept = [i for i, s in enumerate(slots) if 0 <= s < pages * page]
    where = slots[kept] // page, slice(None), slots[kept] % page
    k32 = OA.norm_rope32(host(k.float()), kw, 1e-6, table, rot, at, None, interleaved)
    for x, c, s in ((k32, cache.k_codes, cache.k_scales), (host(v.float()), cache.v_codes, cache.v_scales)):
        codes, scales = OA.fp4_quantize(x[kept])
        got_codes, got_scales = host(c), host(s)
        # -0 and 0 are the same value: compare values where codes are zeros
        assert np.array_equal(got_scales[where], scales)
        assert np.array_equal(OA.fp4_values(got_codes[where], scales), OA.fp4_values(codes, scales))
        written = np.zeros(got_codes.shape[:3], dtype=bool)
        written[where] = True
        assert (got_codes[~written] == 0xA5).all() and (got_scales[~written] == 0xA5).all()
    if pool == "pool":
        assert (flat[:, -64:] == 0xA5).all()
    # the quantized keys lie by the formula's: half a step, and what FP32 moves
    y, size = OA.norm_rope64(f64(k), kw, 1e-6, table, rot, at, None, interleaved)
    codes, scales = OA.fp4_quantize(k32)
    unit = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, -1)
    assert np.all(np.abs(OA.fp4_values(codes, scales) - y) <= unit * np.where(np.abs(y) > 4 * unit, 1, np.where(
        np.abs(y) > 2 * unit, 0.5, 0.25)) + size * 20 * 2.0**-24)

    k_back, v_back = (torch.full((tokens, hk, dim), 9.0, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    attention.unpack_fp4(*cache, dev(slots), k_back, v_back)
    for back, c, s in ((k_back, cache.k_codes, cache.k_scales), (v_back, cache.v_codes, cache.v_scales)):
        want = np.zeros((tokens, hk, dim))
        want[kept] = OA.fp4_values(host(c)[where], host(s)[where])
        assert np.array_equal(f64(back), want)


def test_every_rounding_of_a_block(attention):
    """Values around each threshold and scale boundary, tiny and huge blocks, infinities."""
    edges = np.float32([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7])
    block = np.concatenate([edges, np.nextafter(edges, np.float32(9)), np.nextafter(edges, np.float32(-9)),
                            np.float32([7, -7])])
    rows = []
    for e in [-140, -133, -126, -125, -124, -60, 0, 1, 60, 120, 124, 125]:
        with np.errstate(over="ignore"):
            rows += [np.ldexp(block, e), np.ldexp(-block * np.float32(0.93), e)]
    rows += [np.float32([3.3e38] + [1] * 31), np.float32([math.inf] + [1] * 31), np.float32([math.nan] * 32)]
    v = torch.from_numpy(np.stack(rows)).bfloat16()  # what BF16 keeps of them
    v = torch.cat([v, v], 1).unsqueeze(1).contiguous().cuda()
    t = v.shape[0]
    cache = attention.new_cache(4, 1, 16, 64)
    slots = torch.arange(t, device="cuda")
    attention.append_fp4(None, v, v, None, None, None, None, None, slots, None, *cache)
    codes, scales = OA.fp4_quantize(host(v.float())[:, 0])
    got = host(cache.v_codes)[:, 0].reshape(-1, 32)[:t], host(cache.v_scales)[:, 0].reshape(-1, 2)[:t]
    assert np.array_equal(got[1], scales)
    assert np.array_equal(got[0], codes)
    k, v2 = torch.empty_like(v), torch.empty_like(v)
    attention.unpack_fp4(*cache, slots, k, v2)
    assert np.array_equal(f64(v2)[:, 0], OA.fp4_values(codes, scales), equal_nan=True)


def test_keys_are_quantized_from_fp32(attention):
    """A rotated key is not rounded to BF16 first: thresholds between BF16 neighbours."""
    rng = np.random.default_rng(8)
    k = bf16_randn(rng, 500, 2, 128).cuda()
    table, at, _ = rope_inputs(rng, 64, 128, 500, 1)
    cache = attention.new_cache(32, 2, 16, 128)
    slots = torch.arange(500, device="cuda")
    attention.append_fp4(None, k, k, None, None, dev(table), dev(at[0]), None, slots, None, *cache)
    codes, scales = OA.fp4_quantize(OA.norm_rope32(host(k.float()), None, 0, table, 128, at, None, False))
    got = host(cache.k_codes).transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:500]
    assert np.array_equal(OA.fp4_values(got, scales), OA.fp4_values(codes, scales))


# ---- attention --------------------------------------------------------------------------


def random_cache(attention, rng, pages, heads, page, dim, spread=1.0):
    cache = attention.new_cache(pages, heads, page, dim)
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.copy_(to_dev(rng.integers(0, 256, codes.shape).astype(np.uint8)))
        scales.copy_(to_dev((126 + np.rint(spread * rng.standard_normal(scales.shape))).astype(np.uint8)))
    return cache


def tables(rng, lens, pages, page, width=None):
    used = [-(-n // page) for n in lens]
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), max([1] + used) if width is None else width), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def run_attention(attention, q, cache, table, lens, starts, scale, max_q, window, workspace=None):
    out, buf = with_guard(tuple(q.shape), torch.bfloat16, 5.0)
    out.fill_(5.0)
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    if workspace is None:
        workspace = attention.new_workspace(q.shape[2]).fill_(math.nan)
    attention.attention_fp4(q, *cache, dev(table), dev(np.int32(lens)), None if starts is None else dev(np.int32(starts)),
                            workspace, out, lse, scale, max_q, window)
    torch.cuda.synchronize()
    assert guard_intact(buf, 5.0)
    return out, lse


def check_attention(q, cache, table, lens, starts, scale, max_q, window, out, lse):
    """Every sequence and head against the 64-bit form."""
    hq, hk, page = q.shape[1], cache.k_codes.shape[1], cache.k_codes.shape[2]
    group, qh, oh, lh = hq // hk, f64(q), f64(out), f64(lse)
    kc, ks, vc, vs = (host(t) for t in cache)
    if starts is None:
        starts = list(range(len(lens) + 1))
    for i, n in enumerate(lens):
        count = starts[i + 1] - starts[i]
        shown = min(count, max_q)
        if not shown:
            continue
        at = table[i, :-(-n // page)]
        for h in range(hk):
            k, v = (OA.fp4_values(c[at, h], s[at, h]).reshape(-1, q.shape[2])[:n] for c, s in ((kc, ks), (vc, vs)))
            rows = slice(starts[i], starts[i] + shown)
            heads = slice(h * group, (h + 1) * group)
            high = np.repeat(np.arange(n - count, n - count + shown) + 1, group)
            low = np.maximum(high - window, 0) if window else np.zeros_like(high)
            o, l, mean, off = OA.attention64(qh[rows, heads].reshape(-1, q.shape[2]), k, v, high, low, scale)
            do, dl = OA.attention_bounds(o, l, mean, off)
            got_o, got_l = oh[rows, heads].reshape(o.shape), lh[rows, heads].reshape(l.shape)
            empty = np.isneginf(l)
            assert np.array_equal(np.isneginf(got_l), empty) and (got_o[empty] == 0).all()
            bad = np.abs(got_o - o) > do
            assert not bad.any(), (i, h, np.argwhere(bad)[:4], np.abs(got_o - o)[bad][:4], do[bad][:4])
            assert np.all(np.abs(got_l - l)[~empty] <= dl[~empty]), (i, h, np.abs(got_l - l).max(), dl.max())


CASES = [
    # dim, query heads, key heads, page, context lengths, query counts (None: one each), window
    (64, 1, 1, 16, [1], None, 0),
    (64, 14, 2, 16, [0, 1, 2, 15, 16, 17, 31, 32, 33, 500], None, 0),
    (64, 16, 16, 128, [129, 1000], None, 100),
    (128, 32, 8, 16, [517], None, 0),
    (128, 32, 8, 64, [63, 64, 65, 2049, 127, 1, 0, 4095], None, 0),
    (128, 5, 1, 32, [100, 3000], None, 1),
    (128, 40, 8, 32, [700, 20, 0, 333], None, 33),
    (128, 64, 2, 16, [300, 45], None, 0),          # 32 heads share a key head
    (128, 96, 2, 16, [300, 45], None, 0),          # 48 do
    (256, 24, 4, 64, [1, 64, 1300], None, 0),
    (256, 6, 1, 16, [5000], None, 700),
    (256, 3, 3, 1024, [1025, 2], None, 0),
    (128, 8, 2, 16, [90, 7, 300], [2, 3, 5], 0),   # drafted tokens
    (256, 24, 4, 32, [1600, 33, 4], [4, 4, 4], 0),
    (64, 14, 2, 16, [50, 300], [8, 7], 20),
    (128, 4, 2, 16, [3, 40, 10], [8, 40, 0], 0),   # more queries than tokens: rows that see nothing
    (128, 28, 4, 32, [200, 1000], [130, 77], 64),
    (64, 2, 2, 16, [333], [333], 0),
    (128, 40, 8, 64, [517, 1], [517, 1], 0),
    (256, 6, 1, 16, [300, 290], [100, 290], 0),
    (128, 16, 1, 128, [2000, 5, 700], [1, 5, 300], 0),  # decode, a short prompt and a chunk together
    (64, 8, 8, 64, [1500, 1400], [600, 1], 256),
    (128, 12, 4, 16, [4100], [65], 0),
    (256, 2, 2, 64, [900], [450], 100),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_attention(attention, case):
    dim, hq, hk, page, lens, counts, window = case
    say("attention_fp4", case)
    rng = np.random.default_rng(sum(lens) + dim + hq)
    pages = sum(-(-n // page) for n in lens) + 3
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = None if counts is None else [0] + list(np.cumsum(counts))
    tokens = len(lens) if counts is None else starts[-1] + 2  # two rows of padding
    wide = bf16_randn(rng, tokens, (hq + 2 * hk) * dim).cuda()
    q = wide[:, :hq * dim].unflatten(1, (hq, dim))
    max_q = 1 if counts is None else max(counts)
    scale = dim ** -0.5
    out, lse = run_attention(attention, q, cache, table, lens, starts, scale, max_q, window)
    check_attention(q, cache, table, lens, starts, scale, max_q, window, out, lse)
    if counts is not None:
        assert (out[starts[-1]:] == 5).all() and (lse[starts[-1]:] == 5).all()
    again, lse2 = run_attention(attention, q, cache, table, lens, starts, scale, max_q, window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_attention_of_peaked_scores(attention):
    """Weights that span everything: the running maximum climbs, falls and jumps."""
    rng = np.random.default_rng(5)
    lens, page, dim = [900, 1200], 16, 128
    cache = random_cache(attention, rng, 140, 2, page, dim, spread=3.0)
    table = tables(rng, lens, 140, page)
    q = bf16_randn(rng, 2, 8, dim, scale=4).cuda()
    for scale in (1.0, -0.5, 0.0, 30.0):
        out, lse = run_attention(attention, q, cache, table, lens, None, scale, 1, 0)
        check_attention(q, cache, table, lens, None, scale, 1, 0, out, lse)


@pytest.mark.parametrize("counts", [None, [3, 1], [150, 40]])
def test_what_lies_beyond_a_sequence_does_not_matter(attention, counts):
    """NaN scales in every row past the lengths, in unused pages and in masked tokens' pages."""
    rng = np.random.default_rng(6)
    lens, page, dim = [181, 47], 32, 128
    cache = random_cache(attention, rng, 16, 2, page, dim)
    table = tables(rng, lens, 16, page, width=9)
    starts = None if counts is None else [0] + list(np.cumsum(counts))
    q = bf16_randn(rng, 2 if counts is None else starts[-1], 8, dim).cuda()
    max_q = max(counts or [1])
    want, want_lse = run_attention(attention, q, cache, table, lens, starts, 0.1, max_q, 0)
    for i, n in enumerate(lens):
        last = table[i, n // page] if n % page else None
        if last is not None:
            for s in (cache.k_scales, cache.v_scales):
                s[int(last), :, n % page:] = 255
    unused = sorted(set(range(16)) - set(table[table >= 0].tolist()))
    for s in (cache.k_scales, cache.v_scales):
        s[unused] = 255
    table[0, 7:], table[1, 5:] = unused[0], 10**6  # entries past the lengths
    out, lse = run_attention(attention, q, cache, table, lens, starts, 0.1, max_q, 0)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("counts", [None, [64]])
def test_pages_outside_the_cache_are_not_attended_to(attention, counts):
    rng = np.random.default_rng(7)
    page, dim, n = 16, 64, 160
    cache = random_cache(attention, rng, 12, 1, page, dim)
    table = tables(rng, [n], 12, page)
    starts = None if counts is None else [0, counts[0]]
    q = bf16_randn(rng, 1 if counts is None else counts[0], 4, dim).cuda()
    kept = [p for j, p in enumerate(table[0]) if j not in (0, 4)]
    table[0, 0], table[0, 4] = -1, 12
    out, lse = run_attention(attention, q, cache, table, [n], starts, 0.2, (counts or [1])[0], 0)
    k, v = (OA.fp4_values(host(c)[kept, 0], host(s)[kept, 0]).reshape(-1, dim)
            for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    at = np.concatenate([np.arange(16) + 16 * j for j in range(10) if j not in (0, 4)])
    count = q.shape[0]
    high = np.array([(at <= n - count + i).sum() for i in range(count)]).repeat(4)
    o, l, mean, off = OA.attention64(f64(q).reshape(-1, dim), k, v, high, np.zeros_like(high), 0.2)
    do, dl = OA.attention_bounds(o, l, mean, off)
    assert np.all(np.abs(f64(out).reshape(-1, dim) - o) <= do) and np.all(np.abs(f64(lse).reshape(-1) - l) <= dl)


@pytest.mark.parametrize("counts", [None, [40]])
def test_nan_and_infinite_values_reach_their_rows_alone(attention, counts):
    rng = np.random.default_rng(9)
    page, dim, n = 16, 128, 100
    cache = random_cache(attention, rng, 8, 2, page, dim)
    table = tables(rng, [n], 8, page)
    starts = None if counts is None else [0, counts[0]]
    q = bf16_randn(rng, 1 if counts is None else counts[0], 4, dim).cuda()
    clean, _ = run_attention(attention, q, cache, table, [n], starts, 0.1, (counts or [1])[0], 0)
    q2 = q.clone()
    q2[-1, 1, 3] = math.nan
    cache.v_scales[int(table[0, 99 // page]), 1, 99 % page, 2] = 255  # the last token's values
    out, lse = run_attention(attention, q2, cache, table, [n], starts, 0.1, (counts or [1])[0], 0)
    nan = torch.isnan(out.float())
    assert nan[-1, 1].all() and torch.isnan(lse[-1, 1])
    assert torch.equal(out[-1, 0], clean[-1, 0])
    for h in (2, 3):
        assert nan[-1, h, 64:96].all() and torch.equal(out[-1, h, :64], clean[-1, h, :64])
        assert torch.equal(out[-1, h, 96:], clean[-1, h, 96:])
    assert torch.equal(out[:-1], clean[:-1])


def test_lengths_and_starts_outside_their_ranges(attention):
    """Lengths past the page table and starts past the queries are clamped; max_q bounds."""
    rng = np.random.default_rng(10)
    page, dim = 16, 64
    cache = random_cache(attention, rng, 8, 2, page, dim)
    table = rng.permutation(8).astype(np.int32).reshape(2, 4)
    q = bf16_randn(rng, 6, 4, dim).cuda()
    out, lse = run_attention(attention, q, cache, table, [1000, -5], [-3, 4, 99], 0.1, 6, 0)
    check_attention(q, cache, table, [64, 0], [0, 4, 6], 0.1, 6, 0, out, lse)
    out, lse = run_attention(attention, q, cache, table, [64, 30], [0, 4, 6], 0.1, 3, 0)
    check_attention(q, cache, table, [64, 30], [0, 4, 6], 0.1, 3, 0, out, lse)
    assert (out[3] == 5).all()


@pytest.mark.parametrize("counts", [None, [70]])
def test_offsets_past_32_bits(attention, counts):
    """Pages and slots past 4 GiB of codes."""
    page, dim, heads = 64, 256, 8
    pages = (5 << 30) // (heads * page * dim // 2)
    rng = np.random.default_rng(11)
    cache = attention.Fp4Cache(*(torch.empty(pages, heads, page, dim // n, dtype=torch.uint8, device="cuda")
                                 for n in (2, 32, 2, 32)))
    table = np.int32([[pages - 1, 3, pages - 2]])
    n = 150
    slots = np.int64(table[0, np.arange(n) // page]) * page + np.arange(n) % page
    k, v = bf16_randn(rng, n, heads, dim).cuda(), bf16_randn(rng, n, heads, dim).cuda()
    attention.append_fp4(None, k, v, None, None, None, None, None, dev(slots), None, *cache)
    k_back, v_back = torch.empty_like(k), torch.empty_like(v)
    attention.unpack_fp4(*cache, dev(slots), k_back, v_back)
    for x, back in ((k, k_back), (v, v_back)):
        assert np.array_equal(f64(back), OA.fp4_values(*OA.fp4_quantize(host(x.float()))))
    count = 1 if counts is None else counts[0]
    q = bf16_randn(rng, count, heads, dim).cuda()
    out, lse = run_attention(attention, q, cache, table, [n], None if counts is None else [0, count], 0.0625, count, 0)
    small = attention.Fp4Cache(*(t[[pages - 1, 3, pages - 2]].contiguous() for t in cache))
    del cache
    check_attention(q, small, np.int32([[0, 1, 2]]), [n], [0, count], 0.0625, count, 0, out, lse)


def test_long_context_and_many_sequences(attention):
    """One sequence whose context is split over the whole GPU among many short ones."""
    rng = np.random.default_rng(12)
    page, dim, hk = 16, 128, 2
    lens = [40000] + [int(x) for x in rng.integers(0, 300, 99)]
    pages = sum(-(-n // page) for n in lens) + 1
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    q = bf16_randn(rng, 100, 8, dim).cuda()
    out, lse = run_attention(attention, q, cache, table, lens, None, 0.09, 1, 0)
    check_attention(q, cache, table, lens, None, 0.09, 1, 0, out, lse)


@pytest.mark.parametrize("dim,hq,hk,seqs,count", [(256, 16, 4, 80, 5), (64, 8, 4, 300, 1), (128, 30, 2, 130, 3)])
def test_more_contexts_than_workgroups(attention, dim, hq, hk, seqs, count):
    rng = np.random.default_rng(seqs)
    page = 32
    lens = [int(x) for x in rng.integers(0, 130, seqs)]
    lens[seqs // 2], lens[-1] = 3001, 2500
    pages = sum(-(-n // page) for n in lens) + 1
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    q = bf16_randn(rng, seqs * count, hq, dim).cuda()
    starts = [i * count for i in range(seqs + 1)]
    out, lse = run_attention(attention, q, cache, table, lens, starts, 0.09, count, 0)
    check_attention(q, cache, table, lens, starts, 0.09, count, 0, out, lse)


@pytest.mark.parametrize("dim,hq,hk,lens,counts,window", [
    (128, 16, 2, [3000, 10, 2500, 7], [5, 0, 16, 1], 0),
    (128, 16, 2, [700, 10, 1000, 7], [5, 0, 16, 1], 0),
    (256, 24, 4, [2600, 21], [9, 21], 0),
    (64, 14, 2, [5000, 3, 18], [18, 3, 18], 300),
    (64, 2, 2, [2200, 33, 60], [128, 33, 65], 0),
    (128, 66, 2, [4200, 1], [3, 1], 0),              # blocks of rows end inside a token
    (128, 66, 2, [400, 30], [3, 1], 50),
    (256, 2, 1, [2100] + [66] * 69, [64] * 70, 0),   # more contexts than workgroups
    (128, 5, 1, [3000, 2100], [26, 25], 0),          # 130 and 125 rows
    (64, 4, 4, [20, 3000, 2], [30, 100, 40], 0),     # rows that see nothing
])
def test_blocks_of_rows(attention, dim, hq, hk, lens, counts, window):
    rng = np.random.default_rng(sum(lens) + dim)
    page = 16
    pages = sum(-(-n // page) for n in lens) + 1
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = [0] + list(np.cumsum(counts))
    q = bf16_randn(rng, starts[-1], hq, dim).cuda()
    out, lse = run_attention(attention, q, cache, table, lens, starts, 0.09, max(counts), window)
    check_attention(q, cache, table, lens, starts, 0.09, max(counts), window, out, lse)
    # as many as max_q shows, whatever the blocks
    out, lse = run_attention(attention, q, cache, table, lens, starts, 0.09, 2, window)
    check_attention(q, cache, table, lens, starts, 0.09, 2, window, out, lse)


def test_long_chunk_behind_a_long_context(attention):
    rng = np.random.default_rng(13)
    page, dim, hk = 64, 128, 1
    lens, starts = [20000, 900], [0, 160, 200]
    cache = random_cache(attention, rng, 340, hk, page, dim)
    table = tables(rng, lens, 340, page)
    q = bf16_randn(rng, 200, 4, dim).cuda()
    out, lse = run_attention(attention, q, cache, table, lens, starts, 0.09, 160, 0)
    check_attention(q, cache, table, lens, starts, 0.09, 160, 0, out, lse)


def test_refusals(attention):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    cache = attention.new_cache(4, 2, 16, 64)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    ws = attention.new_workspace(64)
    out, slots = torch.empty_like(q), torch.zeros(2, dtype=torch.int64, device="cuda")

    def attend(**kw):
        a = dict(q=q, cache=cache, table=table, lens=lens, starts=None, ws=ws, out=out, lse=None)
        a.update(kw)
        attention.attention_fp4(a["q"], *a["cache"], a["table"], a["lens"], a["starts"], a["ws"], a["out"], a["lse"], 0.1)

    for text, kw in [("Unexpected dtype", dict(q=q.half())), ("Unexpected dtype", dict(table=table.long())),
                     ("same CUDA device", dict(lens=lens.cpu())), ("contiguous channels", dict(q=q.transpose(1, 2))),
                     ("Expected heads", dict(q=q[0])), ("inputs' shapes", dict(out=out[:1])),
                     ("noncontiguous", dict(out=torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1))),
                     ("workspace", dict(ws=ws[:-1])), ("page_table", dict(lens=lens[:1])),
                     ("q_starts [seqs + 1]", dict(starts=lens)), ("FP32 lse", dict(lse=torch.empty(2, 3, device="cuda"))),
                     ("cache codes", dict(cache=cache._replace(v_scales=cache.k_codes))),
                     ("pages must be contiguous", dict(cache=cache._replace(
                         k_codes=torch.zeros(4, 16, 2, 32, dtype=torch.uint8, device="cuda").transpose(1, 2)))),
                     ("must not overlap", dict(out=q))]:
        with pytest.raises(RuntimeError, match=text.replace("[", r"\[").replace("+", r"\+")):
            attend(**kw)
    with pytest.raises(RuntimeError, match="table and positions together"):
        attention.qk_norm_rope(q, q, None, None, attention.rope_table(8, 64), None, None, out, out)
    with pytest.raises(RuntimeError, match="Several axes"):
        attention.qk_norm_rope(q, q, None, None, attention.rope_table(8, 64), torch.stack([slots, slots]), None, out, out)
    with pytest.raises(RuntimeError, match="overlap"):
        attention.qk_norm_rope(q, q, None, None, None, None, None, out, out)
    with pytest.raises(RuntimeError, match="Queries need an output"):
        attention.append_fp4(q, q[:, :2], q[:, :2], None, None, None, None, None, slots, None, *cache)
    with pytest.raises(RuntimeError, match="slots"):
        attention.append_fp4(None, q[:, :2], q[:, :2], None, None, None, None, None, slots[:1], None, *cache)
    attend()


def test_empty_calls(attention):
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    cache = attention.new_cache(4, 2, 16, 64)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    attention.qk_norm_rope(q, q[:, :2], None, None, attention.rope_table(8, 64), none, None, q.clone(), q[:, :2].clone())
    attention.append_fp4(None, q[:, :2], q[:, :2], None, None, None, None, None, none, None, *cache)
    attention.unpack_fp4(*cache, none, q[:, :2].clone(), q[:, :2].clone())
    i32 = torch.zeros(3, dtype=torch.int32, device="cuda")
    ws = attention.new_workspace(64)
    attention.attention_fp4(q, *cache, i32[:0].view(0, 2), i32[:0], None, ws, q.clone(), None, 0.1)
    attention.attention_fp4(q, *cache, i32[:2].view(2, 1), i32[:2], i32, ws, q.clone(), None, 0.1)
    one = torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.ones_like(one)
    attention.attention_fp4(one, *cache, i32[:0].view(2, 0), i32[:2] + 9, None, ws, out, None, 0.1)
    torch.cuda.synchronize()
    assert (out == 0).all()  # a page table without columns


# ---- streams, graphs and the operators together --------------------------------------------


def layer(attention, qkv, hq, hk, dim, weights, table, positions, slots, cache, pages, lens, starts, max_q, ws):
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    rotated = torch.empty(qkv.shape[0], hq, dim, dtype=torch.bfloat16, device="cuda")
    attention.append_fp4(q, k, v, *weights, table, positions, None, slots, rotated, *cache)
    out = torch.empty_like(rotated)
    attention.attention_fp4(rotated, *cache, pages, lens, starts, ws, out, None, dim ** -0.5, max_q)
    return out


def test_a_prompt_at_once_and_token_by_token(attention):
    """The same tokens in one chunk, in chunks and one by one: the same cache bit for bit, and
    outputs within the rounding of either."""
    rng = np.random.default_rng(14)
    hq, hk, dim, page, n = 8, 2, 128, 16, 75
    qkv = bf16_randn(rng, n, (hq + 2 * hk) * dim).cuda()
    weights = [dev(np.exp(0.3 * rng.standard_normal(dim)).astype(np.float32)) for _ in "qk"]
    table, pages = attention.rope_table(128, dim), dev(rng.permutation(8).astype(np.int32).reshape(1, 8))
    at = torch.arange(n, device="cuda")
    slots = pages[0, at // page].long() * page + at % page
    ws = attention.new_workspace(dim)
    results, caches = [], []
    for chunks in ([n], [1] * n, [40, 3, 17, 15]):
        cache = attention.new_cache(8, hk, page, dim)
        got, first = [], 0
        for c in chunks:
            part = slice(first, first + c)
            got.append(layer(attention, qkv[part], hq, hk, dim, weights, table, at[part], slots[part], cache, pages,
                             dev(np.int32([first + c])), dev(np.int32([0, c])), c, ws))
            first += c
        results.append(torch.cat(got).float())
        caches.append(cache)
    for c in caches[1:]:
        assert all(torch.equal(a, b) for a, b in zip(c, caches[0]))
    for r in results[1:]:
        assert float((r - results[0]).norm() / results[0].norm()) < 2.0**-7


def test_side_stream_and_graph(attention):
    """On a side stream behind a long producer, and captured once and replayed on growing
    contexts, against eager calls."""
    rng = np.random.default_rng(15)
    hq, hk, dim, page, s = 8, 2, 128, 16, 5
    weights, table = (None, None), attention.rope_table(4096, dim)
    pages = dev(rng.permutation(s * 40).astype(np.int32).reshape(s, 40))
    cache = random_cache(attention, rng, s * 40, hk, page, dim)
    eager_cache = attention.Fp4Cache(*(t.clone() for t in cache))
    ws, ws2 = attention.new_workspace(dim), attention.new_workspace(dim)
    qkv = bf16_randn(rng, s, (hq + 2 * hk) * dim).cuda()
    lens, at = (torch.zeros(s, dtype=t, device="cuda") for t in (torch.int32, torch.int64))
    slots = torch.zeros(s, dtype=torch.int64, device="cuda")

    def load(lengths, x):
        lens.copy_(dev(np.int32(lengths)))
        at.copy_(lens.long() - 1)
        slots.copy_(pages[torch.arange(s, device="cuda"), at // page].long() * page + at % page)
        qkv.copy_(x)

    load([1, 2, 30, 200, 600], qkv.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(attention, qkv, hq, hk, dim, weights, table, at, slots, cache, pages, lens, None, 1, ws)
    torch.cuda.current_stream().wait_stream(side)
    for t, e in zip(cache, eager_cache):
        e.copy_(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(attention, qkv, hq, hk, dim, weights, table, at, slots, cache, pages, lens, None, 1, ws)
    for lengths in ([2, 3, 31, 201, 601], [1, 640, 5, 17, 33], [300, 301, 302, 303, 304], [640, 1, 1, 1, 1]):
        load(lengths, bf16_randn(rng, *qkv.shape).cuda())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = layer(attention, qkv, hq, hk, dim, weights, table, at, slots, eager_cache, pages, lens, None, 1, ws2)
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(cache, eager_cache))
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big.T / 4096
        x = qkv.clone()
        got = layer(attention, x, hq, hk, dim, weights, table, at, slots, cache, pages, lens, None, 1, ws)
    side.synchronize()
    assert torch.equal(got, want)
