"""CPU checks of the C boundary of speculative decoding's operators beside tests/test_drafts_oracle.py. No
kernel is launched here."""

import ctypes

import pytest

from tests.test_attention_oracle import FAKE, cache, codes, refused

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
