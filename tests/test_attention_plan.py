"""Sizes of the attention operators' launches (csrc/attention_plan.h, compiled with g++) against
counts by hand, and what the C boundary refuses because a launch cannot hold it."""

import ctypes
import shutil
import subprocess

import pytest

from tests.conftest import PKG
from tests.test_attention_oracle import codes, norm, refused, rotation

MOST_ITEMS = 2**32 - 1  # of a HIP launch, along x

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "attention_plan.h"
using namespace ci8;
int main(int argc, char** argv) {
  long long v[8] = {};
  for (int i = 1; i < argc;) {
    const char* what = argv[i++];
    const int n = !std::strcmp(what, "norm") ? 5 : 3;
    for (int j = 0; j < n; ++j) v[j] = std::atoll(argv[i++]);
    if (n == 5) {
      const NormRopeGrid g = norm_rope_grid(v[0], int(v[1]), int(v[2]), int(v[3]), v[4] != 0);
      std::printf("%lld %d %d\n", (long long)g.workgroups, g.per_wave, int(launch_fits(g.workgroups, kNormThreads)));
    } else {
      const int64_t n = unpack_workgroups(v[0], int(v[1]), int(v[2]));
      std::printf("%lld 0 %d\n", (long long)n, int(launch_fits(n, kUnpackThreads)));
    }
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    folder = tmp_path_factory.mktemp("attention_plan")
    (folder / "p.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", f"-I{PKG / 'csrc'}", str(folder / "p.cpp"), "-o", str(folder / "p")],
                   check=True)

    def run(*cases):
        args = [str(v) for case in cases for v in case]
        out = subprocess.run([str(folder / "p"), *args], check=True, capture_output=True, text=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


def test_norm_and_unpack_grids(plan):
    cases = [
        ("norm", 1, 32, 8, 128, 0),              # 10 groups, a wave each
        ("norm", 4096, 24, 4, 256, 0),           # 14 groups, 4 chunks
        ("norm", 1 << 24, 4, 4, 128, 0),         # 2 groups in a chunk: 2^22 workgroups
        ("norm", 1 << 24, 56, 8, 128, 0),        # 16 groups in 4 chunks: 2^24 workgroups of 256
        ("norm", (1 << 24) - 4, 56, 8, 128, 0),  # one less
        ("norm", 1 << 24, 40, 8, 128, 1),        # 14 groups
        ("norm", 1 << 24, 40, 12, 128, 1),       # 16 groups, 4 chunks
        ("norm", 1 << 24, 0, 48, 256, 1),        # 48 groups, 12 chunks
        ("unpack", 1, 1, 64), ("unpack", 33, 1, 64),
        ("unpack", 1 << 24, 16, 128),            # 2^32 threads
        ("unpack", (1 << 24) - 1, 16, 128),
    ]
    want = [(3, 1), (4096, 4), (1 << 22, 4), (1 << 24, 4), ((1 << 24) - 4, 4), (1 << 24, 4), (1 << 24, 4),
            (3 << 24, 4), (1, 0), (2, 0), (1 << 24, 0), ((1 << 24) - 1, 0)]
    got = plan(*cases)
    assert [g[:2] for g in got] == want
    assert [g[2] for g in got] == [int(n * 256 <= MOST_ITEMS) for n, _ in want]


def test_calls_that_no_launch_holds_are_refused(lib):
    """Each is past the limit by a little; nothing is launched."""
    from consumer_int8 import _abi as A

    *_, large = codes()
    ref, tokens = ctypes.byref, 1 << 24

    def heads(at, n, token_stride=None):
        return A.Heads(at << 42, n, n * 128 if token_stride is None else token_stride, 128)

    q, k = heads(1, 56), heads(2, 8)
    r = rotation(table=9 << 42, positions=10 << 42)
    refused(lib, lib.ci8_qk_norm_rope(ref(q), ref(k), ref(q), ref(k), ref(norm()), ref(r), tokens, 128, None),
            large, "Too many tokens")
    cache = A.Fp4CacheView(3 << 42, 4 << 42, 5 << 42, 6 << 42, 12 * 16 * 64, 12 * 16 * 4, 12 * 16 * 64, 12 * 16 * 4,
                           8, 12, 16)
    q, k, v = heads(1, 40), heads(2, 12), heads(7, 12, 0)
    refused(lib, lib.ci8_append_fp4(ref(q), ref(k), ref(v), ref(q), ref(norm()), ref(r), 11 << 42, ref(cache), tokens,
                                    128, None), large, "Too many tokens")
    cache.heads = 16
    for name in ("k", "v"):
        setattr(cache, name + "_code_page_stride", 16 * 16 * 64)
        setattr(cache, name + "_scale_page_stride", 16 * 16 * 4)
    refused(lib, lib.ci8_unpack_fp4(ref(cache), 11 << 42, 12 << 42, 13 << 42, tokens, 128, None),
            large, "Too many tokens")
