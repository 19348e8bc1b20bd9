"""CPU checks of the C boundary of speculative decoding's operators beside tests/test_drafts_oracle.py. No
kernel is launched here."""

import ctypes

import pytest

from tests.test_attention_oracle import FAKE, cache, codes, heads, refused

PARTS = ["k_codes", "k_scales", "v_codes", "v_scales"]


@pytest.mark.parametrize("name", ["rows", "slots", "starts", *PARTS])
def test_move_without_a_buffer(lib, name):
    usual = dict(rows=FAKE << 10, slots=FAKE << 11, starts=FAKE << 12)
    view = cache(**{name: None} if name in PARTS else {})

    def call(seqs, tokens):
        given = {**usual, **({} if name in PARTS else {name: None})}
        return lib.ci8_move_fp4(ctypes.byref(view), given["rows"], given["slots"], given["starts"], seqs, tokens, 128, None)

    refused(lib, call(2, 8), codes()[0], "Invalid move: a buffer is missing")
    assert call(0, 0) == 0 and call(2, 0) == 0 and call(0, 8) == 0


@pytest.mark.parametrize("name", ["q", "table", "lens", "ws", "out", *PARTS])
def test_tree_without_a_buffer(lib, name):
    usual = dict(table=FAKE << 10, lens=FAKE << 11, ws=FAKE << 12, out=FAKE + (1 << 26))
    view, q = cache(**{name: None} if name in PARTS else {}), heads(n=8)
    if name == "q":
        q.data = None

    def call(seqs, tokens, width=4):
        given = {**usual, **({name: None} if name in usual else {})}
        return lib.ci8_attention_fp4_tree(ctypes.byref(q), ctypes.byref(view), given["table"], width, given["lens"],
                                          FAKE << 14, FAKE << 15, seqs, tokens, 128, given["ws"], given["out"], None, 0.1,
                                          4, 0, None)

    refused(lib, call(2, 8), codes()[0], "Invalid attention: a buffer is missing")
    assert call(0, 0) == 0 and call(2, 0) == 0 and call(0, 8) == 0


def test_tree_without_pages_needs_no_table(lib):
    """An empty page table has no bytes: what refuses this call is the overlap behind it."""
    status = lib.ci8_attention_fp4_tree(ctypes.byref(heads(n=8)), ctypes.byref(cache()), None, 0, FAKE << 11, FAKE << 14,
                                        FAKE << 15, 2, 8, 128, FAKE << 12, FAKE << 15, None, 0.1, 4, 0, None)
    refused(lib, status, codes()[2], "must not overlap anything else")
