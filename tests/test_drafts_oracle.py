"""CPU checks of the operators of speculative decoding: their plain forms (oracle/drafts.py), the
C boundary's refusals, the torch surface. No kernel is launched here."""

import ctypes
import re

import numpy as np
import pytest

from oracle import attention as OA
from oracle import drafts as OD
from tests.conftest import HEADER_PATH, LIB_PATH
from tests.test_attention_oracle import FAKE, cache, codes, heads, refused

HEADER = HEADER_PATH.parent / "consumer_int8_drafts.h"


def test_header_library_and_binding_agree(lib):
    from consumer_int8 import _abi

    declared = sorted(set(re.findall(r"^int (ci8_\w+)\s*\(", HEADER.read_text(), re.M)))
    assert declared == ["ci8_attention_fp4_tree", "ci8_move_fp4", "ci8_token_probs", "ci8_verify_drafts"]
    assert sorted(_abi.DRAFTS_SIGNATURES) == declared
    raw = ctypes.CDLL(str(LIB_PATH))
    assert all(hasattr(raw, name) for name in declared)


# ---- the plain forms --------------------------------------------------------------------


def test_tree_seen():
    # 0 - 1 - 3, 0 - 2 - 4 - 5, behind a context of 4
    seen = OD.tree_seen([-1, 0, 0, 1, 2, 4], 10)
    assert seen[:, :4].all()
    assert [np.flatnonzero(r[4:]).tolist() for r in seen] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 4, 5]]
    seen = OD.tree_seen([-1, 0, 0, 1, 2, 4], 10, window=2)
    assert [np.flatnonzero(r).tolist() for r in seen] == [[3, 4], [4, 5], [4, 6], [5, 7], [6, 8], [8, 9]]
    # a chain is what a causal mask says; parents that are none hang on the context
    for window in (0, 1, 3, 50):
        at = np.arange(9) + 11
        chain = OD.tree_seen(range(-1, 8), 20, window)
        t = np.arange(20)
        assert np.array_equal(chain, (t <= at[:, None]) & (t > at[:, None] - (window or 99)))
    assert OD.tree_seen([3, 7, 2, -9], 4).tolist() == np.eye(4, dtype=bool).tolist()
    # more rows than tokens
    assert [np.flatnonzero(r).tolist() for r in OD.tree_seen([-1, 0, 0, 2], 2)] == [[], [], [0], [0, 1]]


def test_attention64_is_that_of_a_chain():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((5, 8)), rng.standard_normal((12, 8)), rng.standard_normal((12, 8))
    high = np.arange(8, 13)
    want = OA.attention64(q, k, v, high, np.zeros(5, int), 0.3)
    got = OD.attention64(q, k, v, OD.tree_seen(range(-1, 4), 12), 0.3)
    for a, b in zip(want, got):
        assert np.allclose(a, b, rtol=1e-14, atol=0)


def test_token_probs64():
    x = np.array([[0.0, 1, 1, -np.inf], [-np.inf] * 4, [0, np.nan, 0, 0], [0, np.inf, np.inf, 0], [3, 1, 2, 0]])
    p, bound = OD.token_probs64(x, [0.5, 1, 0, 0, np.inf])
    e = np.exp([-2.0, 0, 0])
    assert np.allclose(p[0], [*(e / e.sum()), 0]) and (p[1] == 0).all() and np.isnan(p[2]).all()
    assert p[3].tolist() == [0, 1, 0, 0] and (p[4] == 0.25).all() and bound[0, 1] < 1e-5
    assert np.isnan(OD.token_probs64(x[4:], -1.0)[0]).all() and np.isnan(OD.token_probs64(x[3:4], 1.0)[0]).all()


def law(target, draft, parents, drafter, trials, rng):
    """Frequencies of a sequence's first new token."""
    counts = np.zeros(target.shape[1])
    for _ in range(trials):
        tokens = drafter(rng)
        path, following, _ = OD.verify(target, draft, tokens, parents, rng.random(len(tokens), dtype=np.float32))
        counts[tokens[path[1]] if len(path) > 1 else following] += 1
    return counts / trials


@pytest.mark.parametrize("drawn", [True, False])
def test_verified_tokens_follow_the_target(drawn):
    """Three children of one row: whichever stands, the first new token is distributed as p. 8000
    trials: each frequency within 5 of its standard deviations."""
    rng = np.random.default_rng(1)
    p, q = rng.random(6) ** 3, rng.random(6)
    p, q = p / p.sum(), q / q.sum()
    parents = [-1, 0, 0, 0]
    target, draft = np.tile(p, (4, 1)), np.tile(q, (4, 1))
    if drawn:
        got = law(target, draft, parents, lambda r: np.concatenate([[0], r.choice(6, 3, p=q)]), 8000, rng)
    else:
        got = law(target, None, parents, lambda r: np.array([0, 4, 1, 4]), 8000, rng)
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / 8000))


def test_verify_by_hand():
    p = np.array([[0.5, 0.25, 0.25, 0], [0, 0, 1, 0], [0.25, 0.25, 0.25, 0.25], [1, 0, 0, 0]])
    # certain choices: token 1 fails, then 0 has 0.5 of what is left, 0.75
    assert OD.verify(p, None, [9, 1, 0, 2], [-1, 0, 0, 2], [0.9, 0.5, 0.6, 0.2])[:2] == ([0, 2, 3], 0)
    assert OD.verify(p, None, [9, 1, 0, 2], [-1, 0, 0, 2], [0.9, 0.5, 0.7, 0.2])[:2] == ([0], 2)
    # all that has weight fails: drawn from p itself
    assert OD.verify(p, None, [9, 2], [-1, 0], [0.2, 0.5])[:2] == ([0], 0)
    assert OD.verify(p[1:], None, [9, 2], None, [0.2, 0.5])[:2] == ([0, 1], 0)
    # drawn: q(x) = 1 on token 0 stands with number < 0.5; else the rest is drawn
    q = np.tile([1.0, 0, 0, 0], (4, 1))
    assert OD.verify(p, q, [9, 0], None, [0.6, 0.49])[:2] == ([0, 1], 2)
    assert OD.verify(p, q, [9, 0], None, [0.6, 0.5])[:2] == ([0], 2)
    # numbers and tokens that are none
    assert OD.verify(p, None, [9, -1, 7], [-1, 0, 0], [float("nan"), 0, 0])[:2] == ([0], 0)
    assert OD.verify(p * np.nan, None, [9], None, [0.5])[:2] == ([0], -1)


def test_move_in_order():
    v = np.arange(10)
    assert OD.move(v, [0, 2, 4, -1, 9], [3, 5, 1, 0, 8], [0, 5]).tolist() == [0, 8, 2, 3, 4, 1, 6, 7, 8, 9]
    assert OD.move(v, [1, 1, 0, 1], [3, 5, 1, 99], [0, 2, 4]).tolist() == [0, 1, 2, 5, 4, 5, 6, 7, 8, 9]


# ---- refusals ---------------------------------------------------------------------------


def test_tree_refusals(lib):
    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref

    def call(q=None, c=None, table=FAKE << 10, width=4, lens=FAKE << 11, starts=FAKE << 14, parents=FAKE << 15, seqs=8,
             tokens=8, dim=128, ws=FAKE << 12, out=FAKE + (1 << 26), lse=FAKE << 13, scale=0.1, max_q=4, window=0):
        return lib.ci8_attention_fp4_tree(ref(q or heads(n=8)), ref(c or cache()), table, width, lens, starts, parents,
                                          seqs, tokens, dim, ws, out, lse, scale, max_q, window, None)

    refused(lib, call(starts=None), geometry, "A tree needs q_starts and parents")
    refused(lib, call(parents=None), geometry, "A tree needs q_starts and parents")
    refused(lib, call(max_q=65), large, "A tree has at most 64 queries")
    refused(lib, call(dim=80), geometry, "Unsupported head size")
    refused(lib, call(q=heads(n=6)), geometry, "a multiple of the cache's heads")
    for bad in [dict(seqs=-1), dict(seqs=1 << 17), dict(width=-1), dict(max_q=0), dict(window=-1),
                dict(scale=float("nan"))]:
        refused(lib, call(**bad), geometry, "Invalid attention")
    refused(lib, call(width=1 << 28), large, "Page table too large")
    wide = dict(q=heads(n=64), c=cache(n=1, page=1024), max_q=9, width=65532)
    refused(lib, call(**wide), large, "Page table too large for a tree of that many rows")  # 9 blocks
    refused(lib, call(**{**wide, "max_q": 8, "out": FAKE << 15}), overlap, "must not overlap anything else")
    refused(lib, call(parents=(FAKE << 15) + 2), alignment, "attention_fp4 requires aligned")
    refused(lib, call(out=FAKE << 15), overlap, "must not overlap anything else")
    refused(lib, call(lse=FAKE << 15), overlap, "must not overlap anything else")
    assert call(seqs=0, tokens=0) == 0 and call(seqs=3, tokens=0, parents=None) == 0


def test_move_refusals(lib):
    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref

    def call(c=None, rows=FAKE << 10, slots=FAKE << 11, starts=FAKE << 12, seqs=2, tokens=8, dim=128):
        return lib.ci8_move_fp4(ref(c or cache()), rows, slots, starts, seqs, tokens, dim, None)

    refused(lib, call(dim=96), geometry, "Unsupported head size")
    refused(lib, call(tokens=-1), geometry, "Invalid token count")
    refused(lib, call(tokens=1 << 25), large, "Too many tokens")
    refused(lib, call(c=cache(pages=0)), geometry, "Invalid cache")
    for seqs in (-1, 1 << 16):
        refused(lib, call(seqs=seqs), geometry, "Invalid move")
    for bad in [dict(rows=(FAKE << 10) + 2), dict(slots=(FAKE << 11) + 4), dict(starts=(FAKE << 12) + 1)]:
        refused(lib, call(**bad), alignment, "move_fp4 requires aligned")
    refused(lib, call(c=cache(v_codes=FAKE << 8)), overlap, "Cache buffers must not overlap")
    refused(lib, call(slots=FAKE << 8), overlap, "The cache must not overlap an input")
    many = cache(n=65535, k_codes=1 << 50, k_scales=1 << 51, v_codes=1 << 52, v_scales=1 << 53, pages=1,
                 **{k + "_page_stride": 0 for k in ("k_code", "k_scale", "v_code", "v_scale")})
    refused(lib, call(c=many, seqs=65535), large, "Too many sequences")
    assert call(seqs=0, tokens=0) == 0 and call(seqs=2, tokens=0) == 0


def test_token_probs_refusals(lib):
    geometry, alignment, overlap, large = codes()

    def call(x=FAKE, bits=16, xs=100, t=FAKE << 6, out=FAKE << 8, os=100, tokens=8, vocab=100, ws=FAKE << 10):
        return lib.ci8_token_probs(x, bits, xs, t, out, os, tokens, vocab, ws, None)

    for bad in [dict(tokens=-1), dict(vocab=0), dict(vocab=-5)]:
        refused(lib, call(**bad), geometry, "Invalid rows")
    refused(lib, call(bits=8), geometry, "Logits are BF16")
    for bad in [dict(tokens=(1 << 24) + 1), dict(vocab=(1 << 24) + 1)]:
        refused(lib, call(**bad), large, "Too many tokens")
    refused(lib, call(tokens=1 << 23, vocab=4, xs=4, os=4, x=1 << 50, out=1 << 51), large, "Too many tokens")
    for bad in [dict(xs=99), dict(os=99), dict(xs=-100)]:
        refused(lib, call(**bad), geometry, "must not overlap")
    for bad in [dict(x=None), dict(out=None)]:
        refused(lib, call(**bad), geometry, "Missing rows")
    refused(lib, call(xs=1 << 60), large, "Rows too large")
    for bad in [dict(x=FAKE + 1), dict(out=(FAKE << 8) + 2), dict(bits=32, x=FAKE + 2)]:
        refused(lib, call(**bad), alignment, "aligned")
    for bad in [dict(t=(FAKE << 6) + 2), dict(ws=(FAKE << 10) + 8), dict(ws=None)]:
        refused(lib, call(**bad), alignment, "token_probs requires aligned")
    for bad in [dict(out=FAKE), dict(out=FAKE + 400, bits=32), dict(out=FAKE, bits=32, os=104), dict(t=FAKE << 8),
                dict(ws=FAKE), dict(ws=FAKE << 8), dict(t=(FAKE << 10) + 64)]:
        refused(lib, call(**bad), overlap, "must not overlap anything else")
    assert call(tokens=0) == 0 and call(tokens=0, x=None, out=None, t=None) == 0


def test_verify_refusals(lib):
    geometry, alignment, overlap, large = codes()
    names = ["p", "ps", "q", "qs", "ids", "parents", "starts", "u", "seqs", "tokens", "vocab", "ws", "path", "accepted",
             "next"]
    usual = dict(p=FAKE << 4, ps=100, q=FAKE << 5, qs=100, ids=FAKE << 6, parents=FAKE << 7, starts=FAKE << 8,
                 u=FAKE << 9, seqs=2, tokens=8, vocab=100, ws=FAKE << 10, path=FAKE << 11, accepted=FAKE << 12,
                 next=FAKE << 13)

    def call(**more):
        return lib.ci8_verify_drafts(*({**usual, **more}[n] for n in names), None)

    for bad in [dict(tokens=-1), dict(vocab=0)]:
        refused(lib, call(**bad), geometry, "Invalid rows")
    for bad in [dict(seqs=-1), dict(seqs=16385)]:
        refused(lib, call(**bad), geometry, "at most 16384 sequences")
    refused(lib, call(vocab=(1 << 24) + 1), large, "Too many tokens")
    for bad in [dict(ps=99), dict(qs=99)]:
        refused(lib, call(**bad), geometry, "must not overlap")
    refused(lib, call(p=None), geometry, "Missing rows")
    for name in ("ids", "starts", "u", "path", "accepted", "next"):
        refused(lib, call(**{name: None}), geometry, "a buffer is missing")
    for name in ("ids", "parents", "starts", "u", "ws", "path", "accepted", "next"):
        refused(lib, call(**{name: usual[name] + 2}), alignment, "verify_drafts requires aligned")
    refused(lib, call(ws=None), alignment, "verify_drafts requires aligned")
    for out in ("path", "accepted", "next", "ws"):
        for other in ("p", "q", "ids", "parents", "starts", "u"):
            refused(lib, call(**{out: usual[other]}), overlap, "must not overlap anything else")
    refused(lib, call(accepted=usual["path"]), overlap, "must not overlap anything else")
    assert call(seqs=0, tokens=0, p=None, q=None) == 0


def test_schemas_and_fakes():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    from consumer_int8 import attention, sampling

    assert "Tensor(d!) next_tokens" in str(sampling.verify_drafts.default._schema)
    with FakeTensorMode():
        q = torch.empty(2, 4, 64, dtype=torch.bfloat16)
        c = attention.new_cache(4, 2, 16, 64, device="cpu")
        i32, i64, f32 = (torch.empty(2, dtype=t) for t in (torch.int32, torch.int64, torch.float32))
        assert attention.attention_fp4_tree(q, *c, torch.empty(2, 3, dtype=torch.int32), i32, i32, i32,
                                            torch.empty(66, 4), torch.empty_like(q), None, 0.1, 2) is None
        assert attention.move_fp4(*c, i32, i64, i32) is None
        ws, probs = sampling.new_workspace("cpu"), torch.empty(2, 9)
        assert sampling.token_probs(probs, f32, ws, probs) is None
        assert sampling.verify_drafts(probs, None, i64, None, i32, f32, ws, i32, i32, i64) is None


def test_no_cpu_implementation():
    import torch

    from consumer_int8 import sampling

    with pytest.raises(NotImplementedError):
        sampling.token_probs(torch.zeros(1, 4), None, sampling.new_workspace("cpu"), torch.zeros(1, 4))
