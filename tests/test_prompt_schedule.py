"""The order of LDS stores, reads and barriers in csrc/attention_prompt.hip (csrc/prompt_schedule.h,
compiled with g++), against an enumeration of what waves between the same two barriers touch."""

import re
import shutil
import subprocess

import pytest

from tests.conftest import PKG

HALVES = (1, 2, 4)  # of a tile, at 256, 128 and 64 channels

PROGRAM = r"""
#include <cstdio>
#include "prompt_schedule.h"
using namespace ci8;
int main() {
  std::printf("%d %d %d %d %d\n", kKeyBuffers, kValueBuffers, kPoisonBuffers, kKeysStaged, kValuesStaged);
  for (int halves = 1; halves <= 8; ++halves) {
    std::printf("%d %d %d", barrier_half(halves), keys_ahead(halves), values_ahead(halves));
    for (int b = 0; b < halves; ++b) std::printf(" %d", int(schedule_holds(halves, b)));
    std::puts("");
  }
}
"""


@pytest.fixture(scope="module")
def schedule(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    folder = tmp_path_factory.mktemp("schedule")
    (folder / "s.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", f"-I{PKG / 'csrc'}", str(folder / "s.cpp"), "-o", str(folder / "s")],
                   check=True)
    lines = subprocess.run([str(folder / "s")], check=True, capture_output=True, text=True).stdout.split("\n")
    counts = [int(v) for v in lines[0].split()]
    rows = {n + 1: [int(v) for v in line.split()] for n, line in enumerate(lines[1:9])}
    return counts, rows


def conflicts(halves, barrier, counts, ahead, steps=12):
    """Pairs of a store and a read of one buffer between the same two barriers: waves may do them in
    either order."""
    keys, values, poison, keys_staged, values_staged = counts
    kinds = [("keys", keys, keys_staged, ahead[0]), ("values", values, values_staged, ahead[1]),
             ("poison", poison, values_staged, 0)]
    found, interval = set(), 0
    touched = {}  # (kind, buffer, interval) -> {(what, tile)}
    for step in range(steps):
        for b in range(halves):
            for kind, buffers, staged, early in kinds:
                if b == 0:
                    touched.setdefault((kind, (step + staged) % buffers, interval), set()).add(
                        ("store", step + staged))
                tile, half = divmod(step * halves + b + early, halves)
                if kind != "poison" or half == halves - 1:
                    touched.setdefault((kind, tile % buffers, interval), set()).add(("read", tile))
            if b == barrier:
                interval += 1
    for (kind, buffer, _), what in touched.items():
        if len({w for w, _ in what}) == 2:
            found.add(kind)
    return found


@pytest.mark.parametrize("halves", HALVES)
def test_no_store_meets_a_read(schedule, halves):
    counts, rows = schedule
    barrier, *ahead = rows[halves][:3]
    assert conflicts(halves, barrier, counts, ahead) == set()
    assert rows[halves][3 + barrier] == 1


def test_a_barrier_after_the_first_of_four_halves_parts_nothing(schedule):
    """Both the header's check and the enumeration see what such a barrier leaves open."""
    counts, rows = schedule
    assert conflicts(4, 0, counts, rows[4][1:3]) == {"keys", "values"}
    assert rows[4][3] == 0


@pytest.mark.parametrize("halves", [2, 3, 4, 5, 8])
def test_the_headers_check_is_the_enumeration(schedule, halves):
    counts, rows = schedule
    for barrier in range(halves):
        assert rows[halves][3 + barrier] == (not conflicts(halves, barrier, counts, rows[halves][1:3])), barrier


def test_the_kernel_goes_by_the_header():
    """The kernel's one barrier in a step, what it reads ahead, and its buffers are the header's."""
    text = (PKG / "csrc" / "attention_prompt.hip").read_text()
    loop = text[text.index("for (int t = t_begin; t < t_end; ++t)"):text.index("// A row's two lanes hold")]
    assert loop.count("__syncthreads") == 1
    assert re.search(r"if \(b == barrier_half\(kHalves\)\) \{\s*__builtin_amdgcn_sched_barrier\(0\);\s*__syncthreads", loop)
    assert "read_keys(buffer[(b + kKeysAhead) / kHalves], (b + kKeysAhead) % kHalves)" in loop
    assert "read_values(t + (b + kValuesAhead) / kHalves, (b + kValuesAhead) % kHalves)" in loop
    assert "schedule_holds(kHalves, barrier_half(kHalves))" in text
