"""The ring of stages of the 4-bit linear layer, without a GPU: every division
that its planner makes (q4_plan.h, compiled here with g++), and a model of the
kernel's barriers on the rings that come of them, under random schedules.

A wait on a barrier tells its rounds apart by one bit, so it lets a warp through
that comes two rounds early.  The model knows which round each wait means."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMEM_LIMIT = 227 * 1024 - 512  # of a block, less what the kernel declares statically
CODES, SUMS = 8, 8             # warps


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("q4") / "q4_plan.so")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "rokoko_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "q4_plan_lib.cpp"), "-o", so], check=True, capture_output=True)
    fn = ctypes.CDLL(so).q4_plan_of

    def of(rows, n, k, group, type_bytes, sms=148):
        out = (ctypes.c_longlong * 9)()
        assert fn(rows, n, k, group, type_bytes, sms, out), (rows, n, k, group, type_bytes)
        return dict(zip(("stages", "accs", "sub", "steps", "smem", "pass_bytes", "grid", "tmem", "workspace"), out))
    return of


@pytest.fixture(scope="module")
def plans(plan):
    found = []
    for type_bytes in (2, 4):
        for group in (32, 64, 128, 384):
            for rows in list(range(1, 33)) + [70, 3000]:
                for n in [1, 31, 148, 149, 148 * 32, 148 * 32 + 1, 148 * 64, 148 * 64 + 1, 148 * 128, 148 * 128 + 1, 100003]:
                    for k in (1, 128, 129, 300, 512, 1111, 16384):
                        found.append(plan(rows, n, k, group, type_bytes))
    return found


class Late(Exception):
    """A wait let a warp through before the round that it means."""


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.round = count, count, 0

    def arrive(self):
        assert self.left > 0
        self.left -= 1
        if self.left == 0:
            self.round, self.left = self.round + 1, self.count


def run_ring(stages, accs, sub, steps, rng):
    """One run of the kernel's warps, each a generator that yields the (barrier, round) it waits for; a round r is over
    when the barrier has come to r + 1, and the hardware's parity test sees `round` and `r` modulo 2 only."""
    full = [Barrier(3) for _ in range(stages)]
    empty = [Barrier(5 if sub == 1 else 9) for _ in range(stages)]
    d_full, d_empty = [Barrier(1) for _ in range(accs)], [Barrier(4) for _ in range(accs)]
    filled, in_use = {}, {}

    def copies():
        for i in range(steps):
            yield empty[i % stages], i // stages - 1
            full[i % stages].arrive()

    def products():
        for i in range(steps):
            yield full[i % stages], i // stages
            assert filled[i % stages] == [i, i]  # both halves of this step, nothing else's
            for b in range(sub):
                d = i * sub + b
                yield d_empty[d % accs], d // accs - 1
                d_full[d % accs].arrive()
            empty[i % stages].arrive()

    def codes(first, half):
        for i in range(first, steps, CODES // 2):
            yield empty[i % stages], i // stages - 1
            assert in_use.get(i % stages, 0) == 0
            filled.setdefault(i % stages, [None, None])[half] = i
            full[i % stages].arrive()

    def sums(which):
        for i in range(which if sub == 1 else 0, steps, 2 if sub == 1 else 1):
            yield full[i % stages], i // stages
            in_use[i % stages] = in_use.get(i % stages, 0) + 1
            for b in range(0 if sub == 1 else which, sub, 2):
                d = i * sub + b
                yield d_full[d % accs], d // accs
                assert filled[i % stages] == [i, i]
                d_empty[d % accs].arrive()
            in_use[i % stages] -= 1
            empty[i % stages].arrive()

    warps = [copies(), products()] + [codes(w // 2, w % 2) for w in range(CODES)]
    warps += [sums(w // (SUMS // 2)) for w in range(SUMS)]
    wants = [next(w, None) for w in warps]
    # some warps are held up for long
    speed = [rng.choice((1.0, 1.0, 0.3, 0.02)) for _ in warps]
    while any(w is not None for w in wants):
        ready = [j for j, w in enumerate(wants) if w and (w[0].round + w[1]) % 2 == 1]
        assert ready, "no warp can go on"
        j = rng.choices(ready, [speed[j] for j in ready])[0]
        bar, r = wants[j]
        if bar.round <= r:
            raise Late(f"{stages} stages, {accs} accumulators, {sub} groups a block")
        wants[j] = next(warps[j], None)


def test_no_wait_of_any_planned_ring_is_early(plans):
    rings = sorted({(p["stages"], p["accs"], p["sub"]) for p in plans})
    assert len(rings) > 4
    for ring in rings:
        for seed in range(40):
            run_ring(*ring, steps=44, rng=random.Random(seed))


def test_the_model_finds_the_early_wait_of_an_odd_ring():
    """What the planner rules out: with one group a block the two sets of sums take turns, and nothing orders them."""
    for ring in ((5, 2, 1), (5, 4, 1), (7, 4, 1)):
        with pytest.raises(Late):
            for seed in range(2000):
                run_ring(*ring, steps=44, rng=random.Random(seed))


def test_planned_sizes_fit(plans):
    for p in plans:
        assert 4 <= p["stages"] <= 8 and p["accs"] in (2, 4) and p["smem"] <= SMEM_LIMIT and p["tmem"] <= 512
        assert p["pass_bytes"] <= p["workspace"] and p["grid"] >= 1 and p["steps"] >= 1
        assert p["sub"] > 1 or p["stages"] % 2 == 0
