"""Sizes of the launches of speculative decoding's operators (csrc/sampling_plan.h and
csrc/attention_plan.h, compiled with g++) over their whole ranges."""

import itertools
import shutil
import subprocess

import pytest

from tests.conftest import PKG

WORKSPACE = 1 << 20  # bytes

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "attention_plan.h"
#include "sampling_plan.h"
using namespace ci8;
int main(int argc, char** argv) {
  char what[16];
  long long a, b, c, d;
  while (std::scanf("%15s %lld %lld %lld %lld", what, &a, &b, &c, &d) == 5) {
    if (!std::strcmp(what, "probs")) {
      const Chunks whole = probs_parts(a, b), part = probs_chunks(a, b);
      std::printf("%d %d %d %d %d %d\n", whole.length, whole.count, part.length, part.count,
                  int(probs_in_chunks(a, b, part, true)), int(probs_in_chunks(a, b, part, false)));
    } else if (!std::strcmp(what, "verify")) {
      const Chunks plain = verify_chunks(a, b, false), rounds = verify_chunks(a, b, true);
      std::printf("%d %d %d %d\n", plain.length, plain.count, rounds.length, rounds.count);
    } else {
      std::printf("%d %lld\n", int(tree_fits(a, b, c, int(d))), (long long)move_blocks(c, int(d)));
    }
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    folder = tmp_path_factory.mktemp("drafts_plan")
    (folder / "p.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", f"-I{PKG / 'csrc'}", str(folder / "p.cpp"), "-o", str(folder / "p")],
                   check=True)

    def run(what, cases):
        lines = "".join(" ".join(map(str, [what, *c, *[0] * (4 - len(c))])) + "\n" for c in cases)
        out = subprocess.run([str(folder / "p")], input=lines, check=True, capture_output=True, text=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


SIZES = [1, 2, 3, 7, 511, 1000, 4095, 4096, 4097, 9999, 10000, 10001, 32000, 36863, 36864, 50001, 151936, 300001,
         (1 << 20) + 1, (1 << 24) - 1, 1 << 24]


def covers(length, count, size):
    return count >= 1 and length * count >= size and length * (count - 1) < size


def test_rows_of_probabilities_are_covered(plan):
    cases = list(itertools.product([1, 2, 52, 128, 191, 192, 255, 256, 257, 300, 511, 512, 4000, 1 << 23], SIZES))
    for (tokens, vocab), (length, count, part, parts, bf16, fp32) in zip(cases, plan("probs", cases)):
        assert covers(length, count, vocab) and length % 4096 == 0
        assert count == 1 or tokens * count <= 256 * 2
        assert covers(part, parts, vocab) and part % 1024 == 0 and part <= 8192
        for chosen in (bf16, fp32):  # a thread a chunk, and the sums fit
            assert not chosen or (parts <= 256 and tokens * parts * 8 <= WORKSPACE)


def test_verified_rows_are_covered(plan):
    cases = list(itertools.product([1, 2, 3, 16, 63, 64, 65, 300, 1024, 4097, 1 << 14], SIZES))
    for (seqs, vocab), (length, count, each, rounds) in zip(cases, plan("verify", cases)):
        for n, c in ((length, count), (each, rounds)):
            assert covers(n, c, vocab) and c <= 256
            assert c == 1 or (n % 4 == 0 and vocab > 10000)  # chunks start on 16 bytes
        assert seqs * count * 8 <= WORKSPACE or count == 1
        assert rounds == 1 or seqs * rounds * 66 * 8 <= WORKSPACE


def test_sums_of_trees_fit_32_bits(plan):
    cases = list(itertools.product([1, 1 << 12, 1 << 20, (1 << 26) - 4096], [1, 8, 64], [1, 4, 48, 1000], [64, 128, 256]))
    seen = set()
    for (tokens, max_q, group, dim), (fits, blocks) in zip(cases, plan("tree", cases)):
        rows = 32 if dim == 256 else 64
        most = 64 * -(-max_q * group // rows) * (tokens // 32 + 1 + 40)  # of 64 sequences
        assert bool(fits) == (2 * most < 2**31)
        seen.add(fits)
        assert (blocks - 1) * 256 < group * 2 * (dim // 32 + 1) <= blocks * 256
    assert seen == {0, 1}
