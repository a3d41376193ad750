"""The planning of the expert layer's streamed products, compiled from the library's own header: the layers of tests/moe_runs.py reach the parts of
the loop that they are there for, and a split covers every unit with the warps that there are."""
import os
import shutil
import subprocess

import pytest

from tests.moe_runs import RUNS, SMS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "w4_plan_check")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "vela_b200", "csrc"),
                        os.path.join(ROOT, "tests", "host", "w4_plan_check.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def call(*args):
        r = subprocess.run([exe] + [str(int(a)) for a in args], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0
        return [int(v) for v in r.stdout.split()]
    return call


def cdiv(a, b):
    return -(-a // b)


def shows(plan, T, I_rows, K, E, k, group, what):
    """a product of E experts' [I_rows, K] for T tokens, every expert chosen by T k / E of them"""
    rt, nu = cdiv(I_rows, 16), cdiv(cdiv(K, 64), 2)
    ks, slots, chunks, room = plan(rt, nu, group, E, k, T, SMS)
    assert E == k                                   # every token takes every expert
    share = E * cdiv(T, 8) * rt // SMS              # row tiles of a block at least, over the slots of 8 tokens
    rounds = cdiv(min(share, rt), slots)
    assert chunks >= what.get("chunks", 1) and slots >= what.get("slots", 1) and rounds >= what.get("rounds", 0), (ks, slots, chunks, rounds)
    if what.get("past_room"):
        assert rounds > room // 8


@pytest.mark.parametrize("case,up,down", RUNS)
def test_runs_reach_what_they_are_for(plan, case, up, down):
    T, D, I, E, k, _, group, _ = case
    shows(plan, T, 2 * I, D, E, k, group, up)
    shows(plan, T, D, I, E, k, 0, down)


def test_splits_cover_the_units(plan):
    for nu in (1, 2, 3, 7, 12, 16, 17, 33, 61, 500):
        for uw_group in (0, 32, 64, 128):
            for rt, E, T in ((1, 1, 9), (96, 8, 32), (900, 64, 20)):
                ks, slots, chunks, _ = plan(rt, nu, uw_group, E, 1, T, SMS)
                uw = 2 if uw_group >= 64 else 1
                assert 1 <= ks <= 16 and slots == 16 // ks and ks * uw * chunks >= nu > ks * uw * (chunks - 1)
