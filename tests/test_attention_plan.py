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
    const bool attend = !std::strcmp(what, "attend");
    const int n = attend || !std::strcmp(what, "norm") ? 5 : 3;
    for (int j = 0; j < n; ++j) v[j] = std::atoll(argv[i++]);
    if (attend) {
      const RowSplit r = row_split(v[0], v[1], int(v[2]), v[3]);
      const int64_t units = prompt_units(v[0], v[1], int(v[2]), v[3], int(v[4]));
      std::printf("%d %d %d %lld\n", r.few, int(r.split), int(r.prompt), (long long)units);
    } else if (n == 5) {
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


def test_kernels_and_units_of_attention(plan):
    """Tokens, sequences, query heads of a key head, longest, key heads."""
    cases = [
        ("attend", 64, 64, 4, 1, 8),          # decodes: up to 4 rows, one kernel
        ("attend", 64, 2, 4, 32, 8),          # 128 rows: still that one
        ("attend", 4096, 1, 5, 4096, 8),      # a prompt alone: the other, 80 full row tiles
        ("attend", 4100, 5, 5, 4096, 8),      # beside decodes: both
        ("attend", 300, 1, 48, 300, 2),       # 57 row tiles, the last of 64 rows
        ("attend", 301, 2, 48, 300, 2),       # 48 rows at least: too many for the first kernel
        ("attend", 65535, 65535, 1, 1, 65535),
        ("attend", 65535 * 33, 65535, 4, 33, 128),   # a row tile a sequence and head: 2^23 - 128 units
    ]
    want = [(4, 1, 0, 64 * 8), (128, 1, 0, 2 * 8), (0, 0, 1, 640), (16, 1, 1, 8 * 85), (0, 0, 1, 114), (0, 0, 1, 116),
            (1, 1, 0, (65535 * 65535 // 256 + 65535) * 65535), (0, 0, 1, 65535 * 128)]
    got = plan(*cases)
    assert [g[:3] for g in got] == [w[:3] for w in want]
    # units: never fewer than a count of the tiles
    assert [g[3] for g in got[:6]] == [w[3] for w in want[:6]] and got[7][3] == want[7][3]


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


def test_attention_that_no_launch_holds_is_refused(lib):
    """Prompts of 65535 sequences and 128 key heads: 2^23 - 128 workgroups of 512, and one a CU."""
    from consumer_int8 import _abi as A

    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref
    page = 128 * 16 * 64
    cache = A.Fp4CacheView(3 << 42, 4 << 42, 5 << 42, 6 << 42, page, page // 16, page, page // 16, 8, 128, 16)
    for seqs, count, group, status, text in [(65535, 33, 4, large, "Too many sequences"),
                                             (65535, 33, 5, geometry, "a multiple")]:
        q = A.Heads(1 << 42, 512, 512 * 128, 128)
        if group == 5:
            q.heads = 513
        refused(lib, lib.ci8_attention_fp4(ref(q), ref(cache), 7 << 42, 4, 8 << 42, 9 << 42, seqs, 1 << 21, 128,
                                           10 << 42, 11 << 42, None, 0.1, count, 0, None), status, text)


def test_heads_that_take_turns_and_touch_are_refused(lib):
    """Heads of [tokens, heads, 3, dim] half a head on, a token and half a head on, or of other strides."""
    from consumer_int8 import _abi as A

    *_, overlap, _large = codes()
    ref, base, dim = ctypes.byref, 1 << 40, 128

    def view(at, n=4, step=3 * dim, row=None):
        return A.Heads(base + 2 * at, n, n * step if row is None else row, step)

    q = view(0)
    for k in [view(dim // 2), view(3 * dim - 64), view(12 * dim + 64), view(15 * dim), view(dim, 4, 2 * dim, 12 * dim),
              view(dim, 3, 3 * dim, 12 * dim + 8)]:
        r = rotation(table=9 << 42, positions=10 << 42)
        refused(lib, lib.ci8_qk_norm_rope(ref(q), ref(k), ref(q), ref(k), ref(norm()), ref(r), 8, dim, None), overlap,
                "An output must be its input")
