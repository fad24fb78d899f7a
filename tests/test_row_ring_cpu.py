"""The ring through which the one-launch block-scaled linear hands its quantised rows to the tensor cores, as a model: the schedule of
csrc/gb_row_ring.cuh, which the kernel is compiled with, under random legal orders of everything that the hardware may delay (copies that
land in any order, two issuers, warps that stand still).  No lane may take a stage for free before the slab that was in it has been
multiplied, and everything ends."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gridbook_b200", "csrc")
ACCUMULATORS, WARPS = 8, 4


@pytest.fixture(scope="module")
def ring(tmp_path_factory):
    at = tmp_path_factory.mktemp("ring")
    (at / "ring.cpp").write_text('#include "gb_row_ring.cuh"\nusing namespace gb_row_ring;\nextern "C" {\nint stages() { return kStages; }\n'
                                 'int step() { return kSlabsAStep; }\nint works_(int g, int r) { return works(g, r); }\n'
                                 'int first_(int g, int r) { return first_slab(g, r); }\nint row_(int g, int r) { return row(g, r); }\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(at / "ring.so"), str(at / "ring.cpp")], check=True)
    return ctypes.CDLL(str(at / "ring.so"))


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def over(self, parity):
        """What a wait for a phase of that parity is told."""
        return (self.phase & 1) != parity


def _steps(stages, step, works, first, row, rows, slabs, warp):
    """The (slab, row) of each step of a warp."""
    groups = [g for g in range(4 * warp, 4 * warp + 4) if works(g, rows)]
    for n0 in range(0, slabs, step):
        yield [(n0 + first(g, rows), row(g, rows)) for g in groups if n0 + first(g, rows) < slabs]


def _run(stages, schedule, rows, slabs, rng):
    """"early", "stuck" or "ok"."""
    full, empty = [Barrier(1 + rows) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    acc_full, acc_empty = [Barrier(1) for _ in range(ACCUMULATORS)], [Barrier(1) for _ in range(ACCUMULATORS)]
    multiplied, landing, early, written = [False] * slabs, [], [], []

    def producer():
        for n in range(slabs):
            while not empty[n % stages].over((n // stages & 1) ^ 1):
                yield
            landing.append(n)
            yield

    def memory():
        left = slabs
        while left:
            if landing and rng.random() < 0.5:
                full[landing.pop(rng.randrange(len(landing))) % stages].arrive()
                left -= 1
            yield

    def quantiser(warp):
        for step in schedule(rows, slabs, warp):
            for n, _ in step:
                while not empty[n % stages].over((n // stages & 1) ^ 1):
                    yield
            yield
            for n, r in step:
                if n >= stages and not multiplied[n - stages]:
                    early.append(n)
                written.append((n, r))
                full[n % stages].arrive()
            yield

    def issuer(i):
        for n in range(i, slabs, 2):
            while not acc_empty[n % ACCUMULATORS].over((n // ACCUMULATORS & 1) ^ 1):
                yield
            while not full[n % stages].over(n // stages & 1):
                yield
            yield
            multiplied[n] = True
            acc_full[n % ACCUMULATORS].arrive()
            empty[n % stages].arrive()
            yield

    def read_out():
        for n in range(slabs):
            while not acc_full[n % ACCUMULATORS].over(n // ACCUMULATORS & 1):
                yield
            yield
            acc_empty[n % ACCUMULATORS].arrive()

    actors = [producer(), memory(), issuer(0), issuer(1), read_out()] + [quantiser(w) for w in range(WARPS)]
    live = list(range(len(actors)))
    speed = [1.0] * len(actors)
    for turn in range(100000):
        if early:
            return "early"
        if not live:
            assert sorted(written) == [(n, r) for n in range(slabs) for r in range(rows)]
            return "ok"
        if turn % 100 == 0:
            speed = [rng.choice([0.02, 0.2, 1.0, 1.0]) for _ in actors]
        k = rng.choices(live, [speed[i] for i in live])[0]
        try:
            next(actors[k])
        except StopIteration:
            live.remove(k)
    return "stuck"


@pytest.mark.parametrize("rows", [1, 2, 3, 4])
@pytest.mark.parametrize("kb,tiles", [(1, 40), (2, 17), (7, 6), (9, 5), (11, 4), (13, 3), (23, 2), (32, 2), (45, 1)])
def test_no_stage_is_taken_early(ring, rows, kb, tiles):
    stages, step = ring.stages(), ring.step()

    def schedule(rows, slabs, warp):
        return _steps(stages, step, ring.works_, ring.first_, ring.row_, rows, slabs, warp)

    rng = random.Random(100 * kb + rows)
    assert {_run(stages, schedule, rows, kb * tiles, rng) for _ in range(25)} == {"ok"}


def test_the_model_sees_a_stage_taken_early():
    """Slabs dealt out from each tile's own start, as they once were: with an odd number of blocks a warp misses phases of its stages."""
    kb, tiles = 9, 5

    def schedule(rows, slabs, warp):
        for tile in range(tiles):
            for n in range(warp, kb, WARPS):
                yield [(tile * kb + n, r) for r in range(rows)]

    rng = random.Random(1)
    assert "early" in {_run(10, schedule, 4, kb * tiles, rng) for _ in range(40)}
