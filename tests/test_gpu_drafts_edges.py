"""GPU checks of speculative decoding's operators at the ends of their ranges, and where several workgroups
share a row: probabilities that are none, rows without weight and logits of all kinds at vocabularies
that are cut into chunks, and chains of more rows than the split kernel takes. Forms and bounds are those
of tests/test_gpu_drafts.py; tests/test_drafts_plan_edges.py checks which kernels these sizes go to."""

import ctypes
import math

import numpy as np
import pytest
import torch

from tests.helpers import guard_intact, host, with_guard
from tests.test_gpu_attention import bf16_randn, dev, random_cache, say, tables
from tests.test_gpu_drafts import (attention, check_probs, check_tree, check_verify, drafts_of,  # noqa: F401
                                   random_probs, random_tree, run_tree, run_verify, sampling)

pytestmark = pytest.mark.gpu

VOCAB = 20011  # verify_drafts: more than one chunk with all numbers of sequences used here
LONG = 40003  # token_probs: chunks where rows are few

# ---- logits far apart, many sequences, one long row --------------------------------------


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


# ---- verification over several chunks ---------------------------------------------------


def unusual(rng, counts, trial):
    """Rows of p and q that are strided and hold values that are no probabilities, tokens that are none."""
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows, vocab = starts[-1], VOCAB
    p, q = (random_probs(rng, rows, vocab) for _ in "pq")
    tokens, _ = drafts_of(rng, p, q if trial >= 2 else None, starts, False)
    parents = np.concatenate([random_tree(rng, n, 0.7) for n in counts]) if trial % 2 else None
    for x in (p, q):
        for value in (math.nan, math.inf, -math.inf, -1.0, 0.0):
            x[rng.random((rows, vocab)) < 0.05] = value
        for row in np.flatnonzero(rng.random(rows) < 0.15):  # a chunk of nothing
            x[row, rng.integers(0, 10) * 2000:][:2100] = 0
    p[rng.random(rows) < 0.1] = 0
    q[rng.random(rows) < 0.1] = 0
    sure = rng.random(rows) < 0.2
    p[sure] = 0
    p[sure, 15040] = 1
    tokens[rng.random(rows) < 0.2] = 15040
    strange = rng.random(rows) < 0.1
    tokens[strange] = rng.choice([-1, -2**62, vocab, 2**40 + 40, 2**32], strange.sum())
    uniforms = rng.random(rows, dtype=np.float32)
    odd = rng.random(rows) < 0.2
    uniforms[odd] = rng.choice(np.float32([math.nan, math.inf, -math.inf, -0.5, 1.0, 7.0, 0.0]), odd.sum())
    return starts, p, q, tokens, parents, uniforms


def strided(x, before, behind):
    wide = torch.full((x.shape[0], before + x.shape[1] + behind), math.nan, device="cuda")
    view = wide[:, before:before + x.shape[1]]
    view.copy_(dev(x))
    return view


@pytest.mark.parametrize("trial", range(4))
def test_verify_of_unusual_rows_in_chunks(sampling, trial):  # noqa: F811
    say("unusual verification in chunks", trial)
    starts, p, q, tokens, parents, uniforms = unusual(np.random.default_rng(40 + trial), [7] * 20 + [0, 1, 64], trial)
    check_verify(sampling, strided(p, 3, 8), strided(q, 5, 4) if trial >= 2 else None, tokens, parents, starts, uniforms)


def probe_verify(target, draft, tokens, parents, starts, uniforms):
    """The measurement library's build, whose workgroups add up all chunks themselves."""
    from consumer_int8 import _abi

    _abi.load()
    lib = ctypes.CDLL(str(_abi.LIB_PATH.with_name("libci8_probe.so")))
    lib.probe_verify_drafts.argtypes = [ctypes.c_void_p] * 6 + [ctypes.c_int64] * 3 + [ctypes.c_void_p] * 5
    seqs, (rows, vocab) = len(starts) - 1, target.shape
    held = [dev(x) for x in (target, draft, np.int64(tokens), np.int32(parents), np.int32(starts), np.float32(uniforms))]
    out = [torch.full((n,), -77, dtype=d, device="cuda") for n, d in
           ((rows, torch.int32), (seqs, torch.int32), (seqs, torch.int64))]
    ws = torch.full((1 << 18,), math.nan, device="cuda")
    status = lib.probe_verify_drafts(*(x.data_ptr() for x in held), seqs, rows, vocab, ws.data_ptr(),
                                     *(x.data_ptr() for x in out), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0
    return [host(x) for x in out]


def test_verify_of_unusual_rows_without_waits(sampling):  # noqa: F811
    say("unusual verification without waits")
    starts, p, q, tokens, parents, uniforms = unusual(np.random.default_rng(50), [7] * 20 + [0, 1, 64], 3)
    want = run_verify(sampling, dev(p), dev(q), tokens, parents, starts, uniforms)
    got = probe_verify(p, q, tokens, parents, starts, uniforms)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_verify_all_but_one_token_rejected_in_chunks(sampling):  # noqa: F811
    """63 certain choices that fail, of all chunks, leave the token that has the rest; where nothing has, the
    target's row is drawn from."""
    say("one token left, in chunks")
    p = np.zeros((64, VOCAB), np.float32)
    at = np.arange(63) * 317
    p[0, at] = 2.0**-7
    p[0, VOCAB - 1] = 1 - 63 * 2.0**-7
    tokens, parents = np.concatenate([[0], at]), np.array([-1] + [0] * 63)
    uniforms = np.full(64, 0.999, np.float32)
    assert check_verify(sampling, dev(p), None, tokens, parents, [0, 64], uniforms) == [1]
    p[0, VOCAB - 1] = 0
    p *= 2
    uniforms[1:] = 1 - 2.0**-24
    for first in (0.0, 0.3, 0.9999):
        uniforms[0] = first
        assert check_verify(sampling, dev(p), None, tokens, parents, [0, 64], uniforms) == [1]


@pytest.mark.parametrize("tree", [False, True])
def test_verify_of_nothing_left_in_chunks(sampling, tree):  # noqa: F811
    """A drafter's row that is larger than the target's everywhere leaves nothing: the target's row is drawn
    from; a row without weight gives -1. Among sequences of which something is left."""
    say("nothing left, in chunks", tree)
    rng = np.random.default_rng(60)
    counts = [5, 4, 1, 3, 6, 1, 2]
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = starts[-1]
    p, q = (random_probs(rng, rows, VOCAB) for _ in "pq")
    larger = [0, 3, 4]
    for s in larger:
        q[starts[s]:starts[s + 1]] = 2 * p[starts[s]:starts[s + 1]]
    p[starts[5]] = 0
    p[starts[6]:starts[7]] = 0
    tokens, parents = drafts_of(rng, p, q, starts, False)
    if tree:  # children of row 0, all but the last
        parents = np.concatenate([np.r_[-1, [0] * max(n - 2, 0), 1][:n] for n in counts])
    uniforms = rng.random(rows, dtype=np.float32)
    for s in larger:
        uniforms[starts[s] + 1:starts[s + 1]] = 0.75
    inputs = (tokens, parents if tree else None, starts, uniforms)
    lengths = check_verify(sampling, dev(p), dev(q), *inputs)
    assert [lengths[s] for s in larger + [5, 6]] == [1] * 5
    following = run_verify(sampling, dev(p), dev(q), *inputs)[2]
    assert following[5] == -1 and following[6] == -1 and (following[larger] >= 0).all()
    if tree:
        got = probe_verify(p, q, tokens, parents, starts, uniforms)
        assert all(np.array_equal(a, b) for a, b in zip(got, run_verify(sampling, dev(p), dev(q), *inputs)))


# ---- probabilities of unusual rows, in chunks and in whole rows of all registers ---------


def unusual_logits(rng, vocab):
    inf, nan = math.inf, math.nan
    base = 2 * rng.standard_normal(vocab)
    masked = np.where(rng.random(vocab) < 0.999, -inf, base)
    lowest = np.where(rng.random(vocab) < 0.99, -3.3895e38, base)
    first_masked, last_masked, one, ties = base.copy(), base.copy(), np.full(vocab, -inf), base.copy()
    first_masked[:30000] = -inf  # whole chunks of nothing
    last_masked[9000:] = -inf
    one[vocab - 2] = -7
    ties[[1500, 30000, vocab - 1]] = 64.0
    special = []  # (row, temperature)
    for row in (masked, lowest, first_masked, last_masked, ties, base - 5000, base - 1e30, np.full(vocab, -inf),
                np.zeros(vocab), np.full(vocab, -3.3895e38)):
        special += [(row, t) for t in (1.0, 0.0, 1e-30, 1e-45, 0.01, 3e38, inf)]
    special += [(one, 0.0), (one, 2.0)]
    for row in (base, masked, ties):
        for value in (nan, inf):
            for places in ([4500, 77], [vocab - 1], [20000, 39000]):
                at = row.copy()
                at[places] = value
                special += [(at, 0.0), (at, 1.0)]
    return special + [(base, -1.0), (base, nan), (base, -0.0), (np.full(vocab, -inf), -1.0), (base, 1.0)]


@pytest.mark.parametrize("rows,dtype", [(1, torch.float32), (5, torch.bfloat16), (5, torch.float32),
                                        (200, torch.bfloat16), (200, torch.float32), (300, torch.bfloat16)])
def test_probs_of_unusual_long_rows(sampling, rows, dtype):  # noqa: F811
    say("unusual long rows", rows, dtype)
    rng = np.random.default_rng(rows)
    special = unusual_logits(rng, LONG)
    if rows == 1:
        special = special[::4]
    for first in range(0, len(special), rows):
        part = special[first:first + rows]
        part += [special[-1]] * (rows - len(part))
        x = torch.from_numpy(np.stack([r for r, _ in part]).astype(np.float32)).to(dtype).cuda()
        check_probs(sampling, x, [t for _, t in part], torch.empty(rows, LONG, device="cuda"))


# ---- chains of more rows ----------------------------------------------------------------


@pytest.mark.parametrize("dim,group,count,window", [
    (64, 1, 33, 0), (64, 2, 50, 40), (64, 8, 16, 0), (128, 4, 9, 0), (128, 8, 8, 9), (128, 2, 64, 0), (256, 1, 17, 0),
    (256, 6, 5, 0), (256, 4, 32, 20),                               # the tree kernel, blocks in attention_fp4
    (64, 1, 32, 3), (128, 8, 4, 0), (128, 1, 1, 0), (256, 4, 4, 0)])  # the split kernel, both
def test_a_chain_of_any_length(attention, dim, group, count, window):  # noqa: F811
    """A chain as a tree and as attention_fp4 takes it: both by the formula, and bit for bit where both are
    the split kernel's, of at most 32 rows a key head (16 at 256 channels)."""
    say("chain of any length", dim, group, count, window)
    rng = np.random.default_rng(dim + count)
    lens, page, hk = [700, count, 3000, 64], 32, 2
    pages = sum(-(-n // page) for n in lens) + 1
    cache = random_cache(attention, rng, pages, hk, page, dim)
    table = tables(rng, lens, pages, page)
    starts = np.int32(np.arange(5) * count)
    parents = np.tile(np.arange(-1, count - 1), 4)
    q = bf16_randn(rng, 4 * count, hk * group, dim).cuda()
    out, lse = run_tree(attention, q, cache, table, lens, starts, parents, 0.1, count, window)
    want, want_lse = torch.empty_like(out), torch.empty_like(lse)
    attention.attention_fp4(q, *cache, dev(table), dev(np.int32(lens)), dev(starts), attention.new_workspace(dim), want,
                            want_lse, 0.1, count, window)
    if group * count <= (16 if dim == 256 else 32):
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    for o, l in ((out, lse), (want, want_lse)):
        check_tree(q, cache, table, lens, starts, parents, 0.1, window, o, l)
