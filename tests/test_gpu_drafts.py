"""GPU checks of the operators of speculative decoding against their 64-bit forms (oracle/drafts.py),
with bounds derived there and in oracle/attention.py."""

import math

import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import drafts as OD
from tests.helpers import guard_intact, host, with_guard
from tests.test_gpu_attention import bf16_randn, dev, f64, random_cache, say, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attention(ops):
    from consumer_int8 import attention as module

    return module


@pytest.fixture(scope="module")
def sampling(ops):
    from consumer_int8 import sampling as module

    return module


# ---- trees ------------------------------------------------------------------------------


def run_tree(attention, q, cache, table, lens, starts, parents, scale, max_q, window, workspace=None):
    out, buf = with_guard(tuple(q.shape), torch.bfloat16, 5.0)
    out.fill_(5.0)
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    if workspace is None:
        workspace = attention.new_workspace(q.shape[2]).fill_(math.nan)
    attention.attention_fp4_tree(q, *cache, dev(table), dev(np.int32(lens)), dev(np.int32(starts)),
                                 dev(np.int32(parents)), workspace, out, lse, scale, max_q, window)
    torch.cuda.synchronize()
    assert guard_intact(buf, 5.0)
    return out, lse


def check_tree(q, cache, table, lens, starts, parents, scale, window, out, lse):
    hq, hk, page, dim = q.shape[1], cache.k_codes.shape[1], cache.k_codes.shape[2], q.shape[2]
    group, qh, oh, lh = hq // hk, f64(q), f64(out), f64(lse)
    kc, ks, vc, vs = (host(t) for t in cache)
    for i, n in enumerate(lens):
        rows = slice(starts[i], starts[i + 1])
        if rows.start == rows.stop:
            continue
        seen = np.repeat(OD.tree_seen(parents[rows], n, window), group, axis=0)
        at = table[i, :-(-n // page)]
        for h in range(hk):
            k, v = (OA.fp4_values(c[at, h], s[at, h]).reshape(-1, dim)[:n] for c, s in ((kc, ks), (vc, vs)))
            mine = slice(h * group, (h + 1) * group)
            o, l, mean, off = OD.attention64(qh[rows, mine].reshape(-1, dim), k, v, seen, scale)
            do, dl = OA.attention_bounds(o, l, mean, off)
            # Numbers below 2^-126 are 0 to the exponential, the products and the roundings: for each token a
            # weight (its largest is 1 or more, which the sum of weights divides by), its product, the sum it
            # is added to and the sum's factor where parts join, and the output.
            do = do + (n * (np.abs(v).max(initial=0) + 3) + 1) * 2.0**-126
            got_o, got_l = oh[rows, mine].reshape(o.shape), lh[rows, mine].reshape(l.shape)
            empty = np.isneginf(l)
            assert np.array_equal(np.isneginf(got_l), empty) and (got_o[empty] == 0).all()
            bad = np.abs(got_o - o) > do
            assert not bad.any(), (i, h, np.argwhere(bad)[:4], np.abs(got_o - o)[bad][:4], do[bad][:4])
            assert np.all(np.abs(got_l - l)[~empty] <= dl[~empty])


def random_tree(rng, n, wide=1.0):
    """Parents of n rows; some rows hang on the context, with numbers that name no row before them."""
    at = np.arange(n)
    parents = np.floor(at * rng.random(n) ** wide).astype(np.int64)
    stray = rng.random(n) < 0.1
    parents[stray] = rng.choice([-1, -2**31, 2**31 - 1, n + 3], stray.sum())
    parents[:1] = rng.choice([-1, 0, 5])
    return parents


TREES = [
    # dim, query heads, key heads, page, context lengths (rows counted), rows, window
    (64, 1, 1, 16, [1], [1], 0),
    (64, 14, 2, 16, [20, 2, 15, 16, 17, 33, 500], [4, 2, 0, 7, 1, 3, 11], 0),
    (64, 16, 16, 128, [129, 1000], [64, 33], 100),
    (64, 8, 8, 64, [1500, 1400], [60, 1], 17),
    (128, 32, 8, 16, [600], [8], 0),
    (128, 32, 8, 64, [63, 64, 65, 2049, 127, 10, 4095], [9, 1, 64, 33, 32, 10, 17], 0),
    (128, 40, 8, 32, [700, 64, 333], [64, 64, 26], 0),
    (128, 5, 1, 32, [100, 3000], [13, 40], 1),
    (128, 40, 8, 32, [700, 20, 5, 333], [26, 20, 5, 7], 3),
    (128, 64, 2, 16, [300, 45], [6, 9], 0),          # 32 heads share a key head
    (128, 96, 2, 16, [300, 45], [3, 2], 20),         # 48 do
    (128, 28, 4, 32, [9000, 300, 2000], [11, 11, 11], 1024),
    (128, 4, 2, 16, [3, 40, 10], [8, 40, 0], 0),     # more rows than tokens
    (128, 4, 2, 16, [3, 20], [8, 40], 2),
    (256, 24, 4, 64, [1, 64, 1300], [1, 26, 26], 0),
    (256, 6, 1, 16, [5000], [64], 700),
    (256, 3, 3, 1024, [1025, 2], [50, 2], 0),
    (256, 24, 4, 64, [20000], [26], 0),
    (256, 2, 2, 64, [900, 61], [64, 61], 5),
    (256, 16, 1, 32, [640], [64], 0),
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_tree_attention(attention, case):
    dim, hq, hk, page, lens, counts, window = case
    say("attention_fp4_tree", case)
    rng = np.random.default_rng(sum(lens) + dim + hq)
    pages = sum(-(-n // page) for n in lens) + 3
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = [0] + list(np.cumsum(counts))
    parents = np.concatenate([random_tree(rng, n, 0.5) for n in counts] + [[9, 9]])
    wide = bf16_randn(rng, starts[-1] + 2, (hq + 2 * hk) * dim).cuda()  # two rows of padding
    q = wide[:, :hq * dim].unflatten(1, (hq, dim))
    out, lse = run_tree(attention, q, cache, table, lens, starts, parents, dim ** -0.5, max(counts), window)
    check_tree(q, cache, table, lens, starts, parents, dim ** -0.5, window, out, lse)
    assert (out[starts[-1]:] == 5).all() and (lse[starts[-1]:] == 5).all()
    again, lse2 = run_tree(attention, q, cache, table, lens, starts, parents, dim ** -0.5, max(counts), window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dim,group,count,window", [(64, 2, 9, 0), (128, 4, 5, 0), (128, 8, 64, 0), (256, 6, 30, 12),
                                                    (128, 5, 40, 70)])
def test_a_chain_is_what_attention_gives(attention, dim, group, count, window):
    say("chain", dim, group, count, window)
    rng = np.random.default_rng(dim + count)
    lens, page, hk = [700, count, 3000], 32, 2
    pages = sum(-(-n // page) for n in lens) + 1
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = np.int32([0, count, 2 * count, 3 * count])
    q = bf16_randn(rng, 3 * count, hk * group, dim).cuda()
    out, lse = run_tree(attention, q, cache, table, lens, starts, np.tile(np.arange(-1, count - 1), 3), 0.1, count, window)
    want, want_lse = torch.empty_like(out), torch.empty_like(lse)
    attention.attention_fp4(q, *cache, dev(table), dev(np.int32(lens)), dev(starts), attention.new_workspace(dim), want,
                            want_lse, 0.1, count, window)
    if group * count <= 128:  # the same parts, joined in the same order
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    parents = np.tile(np.arange(-1, count - 1), 3)
    for o, l in ((out, lse), (want, want_lse)):
        check_tree(q, cache, table, lens, starts, parents, 0.1, window, o, l)


@pytest.mark.parametrize("hq,count", [(4, 12), (16, 50)])
def test_what_a_row_does_not_see_does_not_reach_it(attention, hq, count):
    """Keys and values of a branch, of rows past the context and of unused pages become NaN: only rows
    of the branch change."""
    say("unseen", hq, count)
    rng = np.random.default_rng(hq)
    page, dim, hk, n = 16, 128, 1, 203
    cache = random_cache(attention, rng, 20, hk, page, dim)
    table = tables(rng, [n], 20, page, width=15)
    parents = random_tree(rng, count, 0.6)
    parents[0], parents[1:4] = -1, 0
    q = bf16_randn(rng, count, hq, dim).cuda()
    clean, clean_lse = run_tree(attention, q, cache, table, [n], [0, count], parents, 0.1, count, 0)
    spoilt = 2  # of the tree
    token = n - count + spoilt
    cache.v_scales[int(table[0, token // page]), 0, token % page, 1] = 255
    cache.k_scales[int(table[0, token // page]), 0, token % page, 3] = 255
    for s in (cache.k_scales, cache.v_scales):
        s[int(table[0, n // page]), :, n % page:] = 255
        s[sorted(set(range(20)) - set(table[0, :13].tolist()))] = 255
    table[0, 13:] = [10**6, -7]
    out, lse = run_tree(attention, q, cache, table, [n], [0, count], parents, 0.1, count, 0)
    below = np.array([spoilt in chain for chain in OD.ancestors(parents)])
    assert below.any() and not below.all()
    assert torch.isnan(out[dev(below)].float()).all() and torch.isnan(lse[dev(below)]).all()
    assert torch.equal(out[dev(~below)], clean[dev(~below)]) and torch.equal(lse[dev(~below)], clean_lse[dev(~below)])


def test_tree_pages_outside_the_cache_and_bad_starts(attention):
    """Tokens of no page are seen by nobody; starts and lengths are clamped; rows past max_q are left."""
    say("tree pages")
    rng = np.random.default_rng(3)
    page, dim = 16, 64
    cache = random_cache(attention, rng, 12, 1, page, dim)
    table = tables(rng, [150], 12, page)
    q = bf16_randn(rng, 20, 4, dim).cuda()
    parents = random_tree(rng, 20, 0.5)
    seen = OD.tree_seen(parents, 150)
    hole = table.copy()
    hole[0, 2], hole[0, 9] = -1, 12  # the second holds rows of the tree
    out, lse = run_tree(attention, q, cache, hole, [150], [0, 20], parents, 0.2, 20, 0)
    seen[:, 32:48], seen[:, 144:] = False, False
    k, v = (OA.fp4_values(host(c)[table[0], 0], host(s)[table[0], 0]).reshape(-1, dim)[:150]
            for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    o, l, mean, off = OD.attention64(f64(q).reshape(-1, dim), k, v, seen.repeat(4, 0), 0.2)
    do, dl = OA.attention_bounds(o, l, mean, off)
    assert np.all(np.abs(f64(out).reshape(-1, dim) - o) <= do) and np.all(np.abs(f64(lse).reshape(-1) - l) <= dl)
    # two sequences of a clamped table
    table = rng.permutation(8).astype(np.int32).reshape(2, 4)
    parents[12:] = random_tree(rng, 8)
    out, lse = run_tree(attention, q, cache, table, [1000, -5], [-3, 12, 99], parents, 0.1, 20, 0)
    check_tree(q, cache, table, [64, 0], [0, 12, 20], parents, 0.1, 0, out, lse)
    out, lse = run_tree(attention, q, cache, table, [64, 30], [0, 12, 20], parents, 0.1, 9, 0)
    whole, whole_lse = run_tree(attention, q, cache, table, [64, 30], [0, 12, 20], parents, 0.1, 12, 0)
    assert torch.equal(out[:9], whole[:9]) and torch.equal(out[12:], whole[12:]) and (out[9:12] == 5).all()


# ---- probabilities ----------------------------------------------------------------------


def check_probs(sampling, x, t, out, workspace=None):
    """x a tensor of logits, maybe a view of wider rows; against the 64-bit form."""
    sampling.token_probs(x, None if t is None else dev(np.float32(t)), workspace or sampling.new_workspace().fill_(math.nan),
                         out)
    torch.cuda.synchronize()
    want, bound = OD.token_probs64(f64(x), 1.0 if t is None else np.float32(t))
    got = f64(out)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bad = ~(np.abs(got - want) <= bound) & ~nan
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], bound[bad][:4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 7, 0), (1, 32000, 0), (5, 2049, 3), (2, 50001, 0),
                                            (52, 4097, 7), (1, 300001, 0), (511, 130, 0), (513, 1000, 1), (600, 8193, 0)])
def test_token_probs(sampling, rows, vocab, pad, dtype):
    say("token_probs", rows, vocab, pad, dtype)
    rng = np.random.default_rng(rows + vocab)
    x = torch.from_numpy((3 * rng.standard_normal((rows, vocab + pad))).astype(np.float32)).to(dtype).cuda()[:, :vocab]
    t = np.where(rng.random(rows) < 0.2, 0, rng.uniform(0.3, 2, rows))
    buf = torch.full((rows, vocab + 2 * pad), 5.0, device="cuda")
    check_probs(sampling, x, t, buf[:, :vocab])
    assert (buf[:, vocab:] == 5).all()
    out, guard = with_guard((rows, vocab), torch.float32, 5.0)
    check_probs(sampling, x, None, out)
    assert guard_intact(guard, 5.0)
    if dtype == torch.float32:  # in place
        want = torch.empty(rows, vocab, device="cuda")
        sampling.token_probs(x, None, sampling.new_workspace(), want)
        sampling.token_probs(x, None, sampling.new_workspace(), x)
        assert torch.equal(x, want)


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_probs_of_unusual_rows(sampling, rows):
    """Masked logits, infinities, NaN, ties, far below zero, temperatures of all kinds; alone and among
    ordinary rows."""
    say("unusual rows", rows)
    rng = np.random.default_rng(rows)
    vocab = 5000
    inf, nan = math.inf, math.nan
    special = []  # (row, temperature)
    base = 2 * rng.standard_normal(vocab)
    masked = np.where(rng.random(vocab) < 0.999, -inf, base)
    lowest = np.where(rng.random(vocab) < 0.99, -3.3895e38, base)
    first_masked = base.copy()
    first_masked[:4100] = -inf  # whole chunks of nothing
    for row in (masked, lowest, first_masked, base - 5000, base - 1e30, np.full(vocab, -inf), np.zeros(vocab),
                np.full(vocab, -3.3895e38)):
        special += [(row, t) for t in (1.0, 0.0, 1e-30, 1e-45, 0.01, 3e38, inf)]
    one = np.full(vocab, -inf)
    one[4999] = -7
    special += [(one, 0.0), (one, 2.0)]
    for row in (base, masked):
        for value in (nan, inf):
            at = row.copy()
            at[[4500, 77]] = value
            special += [(at, 0.0), (at, 1.0)]
    special += [(base, -1.0), (base, nan), (base, -0.0), (np.full(vocab, -inf), -1.0)]
    for first in range(0, len(special), rows):
        part = special[first:first + rows]
        part += [(base, 1.0)] * (rows - len(part))
        x = torch.from_numpy(np.stack([r for r, _ in part]).astype(np.float32)).bfloat16().cuda()
        check_probs(sampling, x, [t for _, t in part], torch.empty(rows, vocab, device="cuda"))


# ---- verification -----------------------------------------------------------------------


def run_verify(sampling, target, draft, tokens, parents, starts, uniforms, workspace=None):
    rows, seqs = len(tokens), len(starts) - 1
    path, a = with_guard((rows,), torch.int32, -77)
    accepted, b = with_guard((seqs,), torch.int32, -77)
    following, c = with_guard((seqs,), torch.int64, -77)
    path.fill_(-77)
    if workspace is None:
        workspace = sampling.new_workspace().fill_(math.nan)
    sampling.verify_drafts(target, draft, dev(np.int64(tokens)), None if parents is None else dev(np.int32(parents)),
                           dev(np.int32(starts)), dev(np.float32(uniforms)), workspace, path, accepted, following)
    torch.cuda.synchronize()
    assert all(guard_intact(g, -77) for g in (a, b, c))
    return host(path), host(accepted), host(following)


def check_verify(sampling, target, draft, tokens, parents, starts, uniforms, least=1e-11):
    """Against the 64-bit form; no comparison in it may be nearer than `least`, past all roundings of
    sums of up to 2^20 values (2^20 * 2^-53 = 1.2e-10 at worst, 2^-43 as they grow in trees)."""
    got = run_verify(sampling, target, draft, tokens, parents, starts, uniforms)
    p, q = f64(target), None if draft is None else f64(draft)
    lengths = []
    for s, (begin, end) in enumerate(zip(starts[:-1], starts[1:])):
        rows = slice(begin, end)
        path, following, margin = OD.verify(p[rows], None if q is None else q[rows], tokens[rows],
                                            None if parents is None else parents[rows], uniforms[rows])
        assert margin > least, margin
        want = np.full(end - begin, -1)
        want[:len(path)] = path
        assert np.array_equal(got[0][rows], want), (s, got[0][rows], want)
        assert got[1][s] == len(path) and got[2][s] == following, (s, got[1][s], len(path), got[2][s], following)
        lengths.append(len(path))
    assert (got[0][starts[-1]:] == -77).all()
    return lengths


def random_probs(rng, rows, vocab, grain=None):
    p = rng.random((rows, vocab)) ** 6
    p /= p.sum(1, keepdims=True)
    if grain:  # whole multiples of 1 / grain, so that sums of them are exact
        p = np.floor(p * grain) / grain
    return p.astype(np.float32)


def drafts_of(rng, target, draft, starts, tree):
    """Tokens that the drafter would give, and their parents."""
    tokens, parents = np.zeros(len(target), np.int64), np.zeros(len(target), np.int64)
    for begin, end in zip(starts[:-1], starts[1:]):
        n = end - begin
        parents[begin:end] = random_tree(rng, n, 0.7) if tree else np.arange(-1, n - 1)
        for i in range(1, n):
            parent = parents[begin + i]
            source = (draft if draft is not None else target)[begin + (parent if 0 <= parent < i else 0)].astype(float)
            tokens[begin + i] = rng.choice(target.shape[1], p=source / source.sum()) if source.sum() else 0
    return tokens, parents


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("counts,vocab", [([1], 1), ([1], 5), ([4], 7), ([3, 0, 1, 9, 64, 2], 50), ([8] * 33, 1001),
                                          ([26, 5], 32000), ([17], 70001), ([6] * 300, 300), ([70, 64, 65], 40)])
def test_verify(sampling, counts, vocab, drawn, tree):
    say("verify_drafts", counts[:8], len(counts), vocab, drawn, tree)
    rng = np.random.default_rng(vocab + len(counts))
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = starts[-1] + 2
    target = random_probs(rng, rows, vocab)
    draft = None
    if drawn:  # near the target, so that drafts stand now and then
        draft = target * rng.random((rows, vocab)).astype(np.float32) ** 0.5
        draft = (draft / draft.sum(1, keepdims=True)).astype(np.float32)
    tokens, parents = drafts_of(rng, target, draft, starts, tree)
    lengths = check_verify(sampling, dev(target), None if draft is None else dev(draft), tokens,
                           parents if tree else None, starts, rng.random(rows, dtype=np.float32))
    if len(counts) == 300 and drawn:
        assert len(set(lengths)) >= 4, "ways of all lengths"


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("drawn", [False, True])
def test_verify_of_exact_sums(sampling, drawn, tree):
    """Probabilities in whole 1/256: all sums and products are exact in 64 bits for as many rejections as
    happen here, so even results on a border are equal: numbers are whole 1/16 too."""
    say("exact sums", drawn, tree)
    rng = np.random.default_rng(2)
    counts = [5] * 400
    starts = np.concatenate([[0], np.cumsum(counts)])
    target, draft = (random_probs(rng, 2000, 12, 256) for _ in "pq")
    tokens, parents = drafts_of(rng, target, draft if drawn else None, starts, tree)
    uniforms = (rng.integers(0, 16, 2000) / 16).astype(np.float32)
    if tree:  # two rejections at most are followed by another child: 2^-8, 2^-16, 2^-24, 2^-32, 2^-40
        parents[:] = np.tile([-1, 0, 0, 0, 2], 400)
    check_verify(sampling, dev(target), dev(draft) if drawn else None, tokens, parents if tree else None, starts, uniforms,
                 least=-1)


def test_verify_of_unusual_rows(sampling):
    """Values that are no probabilities, tokens that are none, numbers outside [0, 1), rows without
    weight, parents that name nothing, strided rows, targets that are certain."""
    say("unusual verification")
    rng = np.random.default_rng(4)
    counts, vocab = [7] * 60, 90
    starts = np.concatenate([[0], np.cumsum(counts)])
    for trial in range(4):
        rows = starts[-1]
        wide_p, wide_q = (dev(random_probs(rng, rows, vocab + 11)) for _ in "pq")
        p, q = wide_p[:, 3:3 + vocab], wide_q[:, 5:5 + vocab]
        for x in (p, q):
            for value in (math.nan, math.inf, -math.inf, -1.0, 0.0):
                x[dev(rng.random((rows, vocab)) < 0.05)] = value
        p[dev(rng.random(rows) < 0.1)] = 0
        q[dev(rng.random(rows) < 0.1)] = 0
        sure = rng.random(rows) < 0.2
        p[dev(sure)] = 0
        p[dev(sure), 40] = 1
        tokens = rng.integers(-3, vocab + 3, rows)
        tokens[rng.random(rows) < 0.3] = 40
        tokens[:3] = [-2**62, 2**40 + 40, 2**32]
        uniforms = rng.random(rows, dtype=np.float32)
        odd = rng.random(rows) < 0.2
        uniforms[odd] = rng.choice(np.float32([math.nan, math.inf, -math.inf, -0.5, 1.0, 7.0, 0.0]), odd.sum())
        parents = np.concatenate([random_tree(rng, n, 0.7) for n in counts]) if trial % 2 else None
        check_verify(sampling, p, q if trial >= 2 else None, tokens, parents, starts, uniforms)


def test_verify_all_but_one_token_rejected(sampling):
    """63 certain choices that fail leave the token that has the rest, in another chunk than theirs."""
    say("one token left")
    vocab = 9000
    p = np.zeros((64, vocab), np.float32)
    p[0, :4032:64] = 2.0**-7
    p[0, 8999] = 1 - 63 * 2.0**-7
    tokens = np.concatenate([[0], np.arange(0, 4032, 64)])
    uniforms = np.full(64, 0.999, np.float32)
    got = run_verify(sampling, dev(p), None, tokens, [-1] + [0] * 63, [0, 64], uniforms)
    assert got[1].tolist() == [1] and got[2].tolist() == [8999]
    # and where all fail that have weight, the target's row is drawn from
    p[0, 8999] = 0
    p *= 2
    got = run_verify(sampling, dev(p), None, tokens, [-1] + [0] * 63, [0, 64], np.full(64, 0.9999, np.float32))
    assert got[1].tolist() in ([1], [2]) and (got[1][0] == 2 or got[2][0] in tokens)


@pytest.mark.parametrize("drawn,tree", [(True, False), (True, True), (False, True)])
def test_verified_tokens_follow_the_target(sampling, drawn, tree):
    """16384 sequences at once: each frequency of the first new token within 5 standard deviations of
    the target's, though the drafter is far from it."""
    say("law", drawn, tree)
    rng = np.random.default_rng(5)
    seqs, vocab, n = 16384, 9, 4
    p, q = (random_probs(rng, 1, vocab)[0].astype(float) for _ in "pq")
    p, q = p / p.sum(), q / q.sum()
    starts = np.arange(0, (seqs + 1) * n, n)
    tokens = rng.choice(vocab, seqs * n, p=q)
    target, draft = (torch.tensor(x, dtype=torch.float32, device="cuda").expand(seqs * n, vocab).contiguous() for x in (p, q))
    parents = np.tile([-1, 0, 0, 1], seqs) if tree else None
    path, accepted, following = run_verify(sampling, target, draft if drawn else None, tokens, parents, starts,
                                           rng.random(seqs * n, dtype=np.float32))
    first = np.where(accepted > 1, tokens[starts[:-1] + np.maximum(path[starts[:-1] + 1], 0)], following)
    got = np.bincount(first, minlength=vocab) / seqs
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / seqs)), (got, p)
    assert (accepted > 1).any() and (accepted == 1).any()


@pytest.mark.parametrize("probe", [False, True])
def test_verify_of_shared_sums(sampling, probe):
    """Trees whose sums several workgroups share: each from the others', and (the measurement library's
    build) each adding up all of them itself, as after a wait in vain. Replayed in a graph, where the
    workspace holds the sums of the replay before."""
    say("shared sums", probe)
    rng = np.random.default_rng(7)
    counts, vocab = [12, 1, 0, 30, 7], 20011
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = starts[-1]
    target = random_probs(rng, rows, vocab)
    draft = (target * rng.random((rows, vocab)) ** 0.5).astype(np.float32)
    draft = (draft / draft.sum(1, keepdims=True)).astype(np.float32)
    if not probe:
        tokens, parents = drafts_of(rng, target, draft, starts, True)
        ws, t, q = sampling.new_workspace().fill_(0), dev(target), dev(draft)
        ids, par, at = dev(np.int64(tokens)), dev(np.int32(parents)), dev(np.int32(starts))
        u = torch.zeros(rows, device="cuda")
        path, accepted, following = (torch.empty(n, dtype=d, device="cuda") for n, d in
                                     ((rows, torch.int32), (5, torch.int32), (5, torch.int64)))
        call = lambda: sampling.verify_drafts(t, q, ids, par, at, u, ws, path, accepted, following)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for trial in range(6):
            uniforms = rng.random(rows, dtype=np.float32)
            u.copy_(dev(uniforms))
            graph.replay()
            got = [host(x).copy() for x in (path, accepted, following)]
            check_verify(sampling, t, q, tokens, parents, starts, uniforms)
            eager = run_verify(sampling, t, q, tokens, parents, starts, uniforms)
            assert all(np.array_equal(a, b) for a, b in zip(got, eager))
        return
    import ctypes

    from consumer_int8 import _abi

    _abi.load()
    lib = ctypes.CDLL(str(_abi.LIB_PATH.with_name("libci8_probe.so")))
    lib.probe_verify_drafts.argtypes = [ctypes.c_void_p] * 6 + [ctypes.c_int64] * 3 + [ctypes.c_void_p] * 5
    for trial in range(3):
        tokens, parents = drafts_of(rng, target, draft, starts, True)
        uniforms = rng.random(rows, dtype=np.float32)
        want = run_verify(sampling, dev(target), dev(draft), tokens, parents, starts, uniforms)
        held = [dev(x) for x in (target, draft, np.int64(tokens), np.int32(parents), np.int32(starts), uniforms)]
        out = [torch.empty(n, dtype=d, device="cuda") for n, d in
               ((rows, torch.int32), (5, torch.int32), (5, torch.int64))]
        ws = sampling.new_workspace().fill_(math.nan)
        status = lib.probe_verify_drafts(*(x.data_ptr() for x in held), 5, rows, vocab, ws.data_ptr(),
                                         *(x.data_ptr() for x in out), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert status == 0 and all(np.array_equal(host(a), b) for a, b in zip(out, want))


def test_verify_offsets_past_32_bits(sampling):
    """Rows past 2^32 values."""
    say("verify past 32 bits")
    stride = 1 << 31
    buf = torch.empty(2 * stride + 1000, device="cuda")
    rows = buf.as_strided((3, 1000), (stride, 1))
    rows[:] = dev(random_probs(np.random.default_rng(6), 3, 1000))
    tokens = [0, 5, 9]
    for uniforms in ([0.3, 0, 0], [0.3, 0.9999, 0]):
        check_verify(sampling, rows, None, np.int64(tokens), None, [0, 3], np.float32(uniforms))
    out = torch.empty(3, 1000, device="cuda")
    check_probs(sampling, rows, [1.0, 0.0, 0.5], out)


# ---- moving rows ------------------------------------------------------------------------


@pytest.mark.parametrize("dim,heads,page,counts,pool", [(64, 1, 16, [5], False), (64, 16, 32, [20, 0, 64, 3], True),
                                                        (128, 8, 64, [26] * 9, False), (128, 40, 16, [9, 200], True),
                                                        (256, 4, 128, [33, 1, 65], True), (256, 5, 1024, [300], False)])
def test_move(attention, dim, heads, page, counts, pool):
    say("move_fp4", dim, heads, page, counts, pool)
    rng = np.random.default_rng(dim + heads)
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows_all = starts[-1] + 2
    pages = rows_all // page + 5
    if pool:
        sizes = [heads * page * dim // n for n in (2, 32, 2, 32)]
        buf = torch.zeros(pages, sum(sizes), dtype=torch.uint8, device="cuda")
        parts = buf.split(sizes, 1)
        cache = attention.Fp4Cache(*(t.unflatten(1, (heads, page, dim // n)) for t, n in zip(parts, (2, 32, 2, 32))))
    else:
        cache = attention.new_cache(pages, heads, page, dim)
    for t in cache:
        t.copy_(dev(rng.integers(0, 256, tuple(t.shape)).astype(np.uint8)))
    slots = rng.permutation(pages * page)[:rows_all]
    slots[rng.random(rows_all) < 0.05] = rng.choice([-1, pages * page, -2**60, 2**60])
    rows = np.full(rows_all, -1, np.int64)
    for begin, end in zip(starts[:-1], starts[1:]):
        n = end - begin
        rows[begin:end] = np.where(rng.random(n) < 0.5, rng.integers(-2, n + 3, n), np.arange(n) + rng.integers(0, 3, n))
    rows[starts[-1]:] = [1, 1]  # of no sequence
    def flat(t):  # [slots, heads, bytes]
        return host(t).transpose(0, 2, 1, 3).reshape(pages * page, heads, -1)
    want = [OD.move(flat(t), rows, slots, starts) for t in cache]
    attention.move_fp4(*cache, dev(np.int32(rows)), dev(slots), dev(np.int32(starts)))
    torch.cuda.synchronize()
    for t, w in zip(cache, want):
        assert np.array_equal(flat(t), w)


# ---- all of it together -----------------------------------------------------------------


def test_refusals_of_tensors(attention, sampling):
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda")
    cache = attention.new_cache(4, 2, 16, 64)
    table, lens = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.full((1,), 9, dtype=torch.int32, device="cuda")
    starts, parents = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    ws, out = attention.new_workspace(64), torch.empty_like(q)

    def tree(starts=starts, parents=parents, max_q=4, ws=ws):
        attention.attention_fp4_tree(q, *cache, table, lens, starts, parents, ws, out, None, 0.1, max_q)

    tree()
    for bad in [dict(parents=parents.long()), dict(parents=parents[:3]), dict(parents=parents.cpu()), dict(max_q=65),
                dict(max_q=0), dict(starts=starts.repeat(2)), dict(ws=ws[:100])]:
        with pytest.raises(RuntimeError):
            tree(**bad)
    slots = torch.arange(4, device="cuda")
    attention.move_fp4(*cache, parents, slots, starts)
    for bad in [(parents.long(), slots, starts), (parents, slots.int(), starts), (parents, slots[:3], starts),
                (parents, slots, starts[:0]), (parents, slots.cpu(), starts)]:
        with pytest.raises(RuntimeError):
            attention.move_fp4(*cache, *bad)
    x, ws, p = torch.zeros(4, 10, device="cuda"), sampling.new_workspace(), torch.zeros(4, 10, device="cuda")
    t = torch.ones(4, device="cuda")
    sampling.token_probs(x, t, ws, p)
    for bad in [(x.half(), t, ws, p), (x.t(), t, ws, p.t()), (x, t[:3], ws, p), (x, t.double(), ws, p), (x, t, ws[:100], p),
                (x, t, ws, p[:, :9]), (x, t, ws, p.bfloat16()), (x[0], t, ws, p), (x, t, ws, x[:, :0]),
                (x[:, :0], t, ws, p[:, :0]), (x, t.cpu(), ws, p)]:
        with pytest.raises(RuntimeError):
            sampling.token_probs(*bad)
    ids, i32, one, one64 = torch.zeros(4, dtype=torch.int64, device="cuda"), parents.clone(), lens.clone(), slots[:1].clone()
    good = [p, p, ids, parents, starts, t, ws, i32, one, one64]
    sampling.verify_drafts(*good)
    for i, bad in [(0, p.double()), (1, p[:, :9]), (1, p[:3]), (2, ids.int()), (3, ids), (4, ids), (5, t[:3]), (6, ws[:9]),
                   (7, i32[:3]), (8, i32), (9, one), (7, parents), (5, t.cpu()), (8, i32[:1])]:
        with pytest.raises(RuntimeError):
            sampling.verify_drafts(*good[:i], bad, *good[i + 1:])


# ---- more sequences, other streams, graphs -----------------------------------------------

MANY = [
    # dim, query heads, key heads, page, context lengths, rows, window: trees of more than 32 rows that are cut
    # into runs, with as many contexts as workgroups and with more, and more than 64 sequences
    (128, 40, 40, 64, [3000, 2400, 9], [64, 40, 9], 0),
    (64, 40, 40, 32, [2500, 33, 2400, 2400, 700, 64, 2330], [64, 33, 64, 33, 50, 64, 1], 0),
    (128, 10, 2, 16, [40] * 40 + [2600] + [17] * 39, [7] * 80, 0),
    (256, 4, 1, 16, [40] * 65 + [2600, 1], [9] * 66 + [1], 0),
    (128, 128, 1, 128, [700], [64], 0),   # 128 blocks of rows
    (64, 100, 1, 16, [2600, 30], [64, 30], 33),
    (64, 2, 2, 16, [50] * 70 + [4000], [3] * 71, 0),  # at most 32 rows, likewise
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(str(x)[:20].replace(" ", "") for x in c))
def test_tree_attention_of_many(attention, case):
    test_tree_attention(attention, case)


def step_of_all(attention, sampling, seed):
    """Tensors of one call of each operator, and the calls."""
    rng = np.random.default_rng(seed)
    dim, hq, hk, page, counts, lens = 128, 16, 2, 16, [9, 1, 20], [500, 40, 2500]
    n, vocab = sum(counts), 33000
    pages = sum(-(-x // page) for x in lens) + 2
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = np.int32(np.concatenate([[0], np.cumsum(counts)]))
    t = dict(q=bf16_randn(rng, n, hq, dim).cuda(), table=dev(table), lens=dev(np.int32(lens)), starts=dev(starts),
             parents=dev(np.int32(np.concatenate([random_tree(rng, c, 0.5) for c in counts]))),
             logits=torch.from_numpy(3 * rng.standard_normal((n, vocab)).astype(np.float32)).cuda(),
             draft=torch.from_numpy(random_probs(rng, n, vocab)).cuda(),
             tokens=dev(rng.integers(0, vocab, n)), uniforms=dev(rng.random(n).astype(np.float32)),
             slots=dev(rng.permutation(pages * page)[:n].astype(np.int64)),
             out=torch.empty(n, hq, dim, dtype=torch.bfloat16, device="cuda"), lse=torch.empty(n, hq, device="cuda"),
             probs=torch.empty(n, vocab, device="cuda"), path=torch.empty(n, dtype=torch.int32, device="cuda"),
             accepted=torch.empty(3, dtype=torch.int32, device="cuda"),
             next=torch.empty(3, dtype=torch.int64, device="cuda"), **cache._asdict())
    spaces = attention.new_workspace(dim), sampling.new_workspace()

    def run():
        attention.attention_fp4_tree(t["q"], *cache, t["table"], t["lens"], t["starts"], t["parents"], spaces[0], t["out"],
                                     t["lse"], dim ** -0.5, 20, 0)
        sampling.token_probs(t["logits"], None, spaces[1], t["probs"])
        sampling.verify_drafts(t["probs"], t["draft"], t["tokens"], t["parents"], t["starts"], t["uniforms"], spaces[1],
                               t["path"], t["accepted"], t["next"])
        attention.move_fp4(*cache, t["path"], t["slots"], t["starts"])

    def results():
        return [t[name].clone() for name in ("out", "lse", "probs", "path", "accepted", "next", *cache._fields)]

    return t, run, results


def refill(t, other):
    for name in ("q", "parents", "logits", "draft", "tokens", "uniforms", "k_codes", "k_scales", "v_codes", "v_scales"):
        t[name].copy_(other[name])


def test_graphs_of_all_replay_with_other_inputs(attention, sampling):
    t, run, results = step_of_all(attention, sampling, 1)
    others = [step_of_all(attention, sampling, seed)[0] for seed in (2, 3)]
    original = {name: x.clone() for name, x in t.items()}
    wants = []
    for inputs in (original, *others):
        refill(t, inputs)
        run()
        wants.append(results())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    torch.cuda.synchronize()
    for turn in range(2):
        for inputs, want in zip((original, *others), wants):
            refill(t, inputs)
            for name in ("out", "lse", "probs", "path", "accepted", "next"):
                t[name].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(results(), want)), turn


def test_streams_side_by_side(attention, sampling):
    """Two streams at once, each with its own workspaces, against the calls one after the other."""
    calls = [step_of_all(attention, sampling, seed) for seed in (4, 5)]
    saved = [{name: x.clone() for name, x in t.items()} for t, _, _ in calls]
    wants = []
    for t, run, results in calls:
        run()
        wants.append(results())
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for (t, _, _), old in zip(calls, saved):
            refill(t, old)
        torch.cuda.synchronize()
        for stream, (_, run, _) in zip(streams, calls):
            with torch.cuda.stream(stream):
                run()
        torch.cuda.synchronize()
        for (_, _, results), want in zip(calls, wants):
            assert all(torch.equal(a, b) for a, b in zip(results(), want))


def test_tree_and_move_past_32_bits(attention):
    """Pages whose bytes start past 2^32: 1.1 million of 4 KiB."""
    rng = np.random.default_rng(32)
    dim, hq, hk, page, pages = 128, 4, 1, 64, 1_100_000
    cache = attention.new_cache(pages, hk, page, dim)
    used = [pages - 1, 3, pages - 20, pages - 7]
    small = random_cache(attention, rng, 4, hk, page, dim)
    for big, part in zip(cache, small):
        big[used] = part
    lens, counts = [200], [12]
    parents = random_tree(rng, 12, 0.5)
    q = bf16_randn(rng, 12, hq, dim).cuda()
    out, lse = run_tree(attention, q, cache, np.int32([used]), lens, [0, 12], parents, 0.1, 12, 0)
    want, want_lse = run_tree(attention, q, small, np.int32([[0, 1, 2, 3]]), lens, [0, 12], parents, 0.1, 12, 0)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    rows, starts = np.int32([0, 3, 2, 3]), np.int32([0, 4])
    here = np.int64([used[0] * page + 1, used[1] * page + 2, used[2] * page, used[3] * page + 63])
    there = np.int64([1, page + 2, 2 * page, 3 * page + 63])
    attention.move_fp4(*cache, dev(rows), dev(here), dev(starts))
    attention.move_fp4(*small, dev(rows), dev(there), dev(starts))
    for big, part in zip(cache, small):
        assert torch.equal(big[used], part)
