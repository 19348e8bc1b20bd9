"""Launches of speculative decoding's operators: constants that bound what a call may cost, and which kernels
the sizes of tests/test_gpu_drafts_edges.py go to."""

import shutil
import subprocess

import pytest

from tests.conftest import PKG
from tests.test_drafts_plan import plan  # noqa: F401


def test_a_wait_in_vain_costs_no_more_than_the_sums(tmp_path):
    """A workgroup of verify_drafts that looks for others' sums in vain adds them up itself, in 94 us of 62
    chunks of 2048 tokens; a look takes it 0.16 us."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    (tmp_path / "p.cpp").write_text('#include <cstdio>\n#include "sampling_plan.h"\n'
                                    'int main() { std::printf("%d\\n", ci8::kMostPolls); }\n')
    subprocess.run([gxx, "-std=c++17", f"-I{PKG / 'csrc'}", str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    polls = int(subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout)
    assert 100 <= polls and polls * 0.16 <= 94


def test_one_long_row_is_cut_into_chunks(plan):  # noqa: F811
    """Up to 256 chunks of 8192 values, whatever their number would be in smaller ones."""
    sizes = [36864, 262144, 262145, 262208, 300001, 524287, 524289, 10**6, 2000003, 1 << 21]
    for vocab, (*_, length, chunks, bf16, fp32) in zip(sizes, plan("probs", [(1, v) for v in sizes])):
        assert bf16 and fp32 and chunks <= 256 and length * chunks >= vocab, (vocab, length, chunks)
    for *_, bf16, fp32 in plan("probs", [(1, (1 << 21) + 1), (1, 36863)]):
        assert not bf16 and not fp32


def test_sizes_of_edge_cases_have_chunks(plan):  # noqa: F811
    for length, count, each, rounds in plan("verify", [(seqs, 20011) for seqs in (1, 7, 23)]):
        assert count > 1 and rounds > 1 and count * length > 20011 - length
    few = plan("probs", [(rows, 40003) for rows in (1, 5, 200, 300)])
    assert [(bool(bf16), bool(fp32)) for *_, bf16, fp32 in few] == [(True, True)] * 2 + [(False, False), (True, False)]
    assert all(parts > 4 for _, _, _, parts, _, _ in few)
