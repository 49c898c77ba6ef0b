"""CPU simulation of the 4-bit kernels' record rings.

The kernels of blackwell_gemm_b200/csrc/moe_w4.cuh hand ring stages from one
producing thread to sets of warps through mbarriers waited on by phase parity.
These tests replay the steps under random schedules, copies landing in any
order, and check what the sums rest on:

* a warp reads a stage only while it holds the record that the warp came for;
* a stage is written again only after everything in it has been read;
* a place in TMEM is written only after its last MMA, read only when whole;
* no schedule deadlocks.

Planted mistakes (the second set releasing a stage that it has not waited for)
must make the simulation fail.
"""
from __future__ import annotations

import random

import pytest

from test_pipeline_protocol import Barrier

WARPS = 4  # to a set


class Ring:
    """Stages, their barriers, and copies under way."""

    def __init__(self, stages, releases, rng):
        self.rng = rng
        self.full = [Barrier(1) for _ in range(stages)]
        self.empty = [Barrier(releases) for _ in range(stages)]
        self.holds = [None] * stages    # what has landed there
        self.unread = [0] * stages      # readings of it that are still to come
        self.flying = []

    def produce(self, items):
        """items: readings that each stage item will get."""
        for i, readings in enumerate(items):
            s, lap = i % len(self.full), i // len(self.full)
            while not self.empty[s].try_wait((lap & 1) ^ 1):
                yield
            assert self.unread[s] == 0 and s not in [f[0] for f in self.flying], \
                f"stage {s} written before it was read"
            self.full[s].arrive(expect_tx=1)
            self.flying.append((s, i, readings))
            yield

    def land(self):
        """Copies land in any order, some of them late."""
        while True:
            if self.flying and self.rng.random() < 0.5:
                s, i, readings = self.flying.pop(self.rng.randrange(len(self.flying)))
                self.holds[s], self.unread[s] = i, readings
                self.full[s].complete_tx(1)
            yield

    def wait(self, i):
        s, lap = i % len(self.full), i // len(self.full)
        while not self.full[s].try_wait(lap & 1):
            yield

    def read(self, i):
        s = i % len(self.full)
        assert self.holds[s] == i, f"stage {s} holds {self.holds[s]}, not {i}"
        self.unread[s] -= 1

    def release(self, i):
        self.empty[i % len(self.empty)].arrive()


def run(tasks, background, rng, limit=400_000):
    """Steps tasks at random, some of them much slower than others."""
    weight = {id(t): rng.choice([1, 1, 8, 40]) for t in tasks + background}
    alive = list(tasks)
    for _ in range(limit):
        if not alive:
            return
        pool = alive + background
        t = rng.choices(pool, [weight[id(p)] for p in pool])[0]
        try:
            next(t)
        except StopIteration:
            alive.remove(t)
    raise AssertionError("no end: deadlock")


# --------------------------------------------- 64-row tiles (w4_stream_kernel)
def stream_kernel(segments, stages, rng, plant=None, places=4):
    """segments: records of each of a CTA's segments.  Set 0 unpacks the first
    record of a stage, set 1 the second; a single one is set 0's."""
    items, first = [], []     # per stage item: records in it; its first record's number
    n = 0
    for length in segments:
        for kb in range(0, length, 2):
            items.append(min(2, length - kb))
            first.append(n)
            n += items[-1]
    ring = Ring(stages, 2 * WARPS, rng)
    unpacked = [Barrier(WARPS) for _ in range(places)]
    used = [Barrier(1) for _ in range(places)]
    place = [None] * places   # [record, warps that wrote it]
    pipe = []                 # MMAs under way, in order

    def unpack(which):
        for i, records in enumerate(items):
            if which == 1 and records == 1:
                if plant != "release without waiting":
                    yield from ring.wait(i)
                ring.release(i)
                yield
                continue
            yield from ring.wait(i)
            record = first[i] + which
            w, lap = record % places, record // places
            while not used[w].try_wait((lap & 1) ^ 1):
                yield
            ring.read(i)
            if place[w] is None or place[w][0] != record:
                assert place[w] is None or place[w][1] == "done", "a place written before its MMA"
                place[w] = [record, 0]
            place[w][1] += 1
            yield
            ring.release(i)
            yield
            unpacked[w].arrive()
            yield

    def mma():
        for record in range(n):
            w = record % places
            while not unpacked[w].try_wait((record // places) & 1):
                yield
            assert place[w] == [record, WARPS], f"place {w} holds {place[w]}, not {record}"
            pipe.append(w)
            yield
        while pipe:
            yield

    def finish():
        while True:
            if pipe:
                w = pipe.pop(0)
                place[w][1] = "done"
                used[w].arrive()
            yield

    tasks = [ring.produce([WARPS * r for r in items]), mma()]
    tasks += [unpack(which) for which in (0, 1) for _ in range(WARPS)]
    run(tasks, [ring.land(), finish()], rng)
    assert all(u == 0 for u in ring.unread)


SEGMENTS = {
    "one record to a segment": [1] * 40,
    "two": [2] * 20,
    "three": [3] * 14,
    "a divided one at both ends": [1, 4, 4, 4, 3],
    "odd, divided at both ends": [2, 5, 5, 5, 5, 1],
    "long": [31, 31],
}


@pytest.mark.parametrize("segments", list(SEGMENTS))
@pytest.mark.parametrize("stages", [5, 6])
def test_unpacking_sets_hold(stages, segments):
    for seed in range(20):
        stream_kernel(SEGMENTS[segments], stages, random.Random(seed))


@pytest.mark.parametrize("stages", [5, 6])
def test_release_without_waiting_is_caught(stages):
    def fails(seed):
        try:
            stream_kernel([1] * 40, stages, random.Random(seed), "release without waiting")
        except AssertionError:
            return True
        return False
    assert any(fails(seed) for seed in range(40))


# ---------------------------------------- up to 32 rows (w4_rows_kernel)
def rows_kernel(segments, groups, stages, rng):
    """Groups of warps take stages in turn; a barrier of them all ends a segment."""
    items = [min(2, length - kb) for length in segments for kb in range(0, length, 2)]
    ends, at = [], 0
    for length in segments:
        at += (length + 1) // 2
        ends.append(at)
    ring = Ring(stages, WARPS, rng)
    arrived = [0] * len(ends)

    def take(group):
        begin = 0
        for segment, end in enumerate(ends):
            for i in range(begin, end):
                if i % groups != group:
                    continue
                yield from ring.wait(i)
                for _ in range(items[i]):
                    ring.read(i)
                    yield
                ring.release(i)
                yield
            arrived[segment] += 1
            while arrived[segment] < groups * WARPS:
                yield
            begin = end

    tasks = [ring.produce([WARPS * r for r in items])]
    tasks += [take(g) for g in range(groups) for _ in range(WARPS)]
    run(tasks, [ring.land()], rng)
    assert all(u == 0 for u in ring.unread)


def _fails(*args):
    for seed in range(30):
        try:
            rows_kernel(*args, random.Random(seed))
        except AssertionError:
            return True
    return False


@pytest.mark.parametrize("groups,stages", [(4, 8), (3, 6), (2, 4)])
def test_groups_of_warps_hold(groups, stages):
    for segments in ([64], [1, 32, 32, 9], [3, 3, 3, 3, 3, 3, 3], [1] * 30):
        for seed in range(10):
            rows_kernel(segments, groups, stages, random.Random(seed))


@pytest.mark.parametrize("groups,stages", [(3, 7), (2, 5)])
def test_stages_that_change_groups_are_caught(groups, stages):
    # a group that comes to a stage must have seen its last lap's copy land
    assert _fails([64], groups, stages)


def test_ring_depths_of_the_kernels(tmp_path):
    """What is compiled has a whole number of turns to a ring."""
    import shutil
    import subprocess
    from pathlib import Path
    from blackwell_gemm_b200 import build
    if shutil.which("nvcc") is None and not Path("/usr/local/cuda/bin/nvcc").exists():
        pytest.skip("no nvcc")
    source = tmp_path / "rings.cu"
    source.write_text("""
#include <cstdio>
#include "moe_w4.cuh"
using namespace b200;
template <int kTok, int kGroup> void show() {
  using C = W4RowsCfg<kTok, kGroup>;
  std::printf("%d %d %d %d\\n", kTok, kGroup, C::kGroups, C::kStages);
}
int main() {
  show<8, 32>(), show<8, 64>(), show<8, 128>(), show<16, 32>(), show<16, 64>(), show<16, 128>();
  show<32, 32>(), show<32, 64>();
}
""")
    exe = tmp_path / "rings"
    subprocess.run([build._nvcc(), "-std=c++17", *build.ARCH_FLAGS, "-I", str(build.INCLUDE), "-I",
                    str(build.CSRC), "-o", str(exe), str(source)], check=True)
    rows = [tuple(map(int, line.split())) for line in
            subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
            if line]
    assert len(rows) == 8
    for tok, group, groups, stages in rows:
        assert stages % groups == 0, (tok, group, groups, stages)
        assert not _fails([64], groups, stages)
