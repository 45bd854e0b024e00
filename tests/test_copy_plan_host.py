"""Order of the copies between sequences of a cache (csrc/copy_plan.cuh), compiled for the host and carried out on numbers: every row
is what it would be if all rows were read before any is written."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "mdlarc_scale_b200" / "csrc"
SOURCE = r"""
#include "copy_plan.cuh"
#include <algorithm>
// steps: [most_steps][4] slot, begin, end, op; programs: [most_programs][4] first step, steps, lo, hi; serial
extern "C" int plan(const int* copies, int n, int n_seqs, int t_max, int most, int* steps, int* programs, char* serial, int* n_programs) {
  std::vector<CopyProgram> out;
  std::vector<char> ser;
  const int r = copy_plan(copies, n, n_seqs, t_max, most, out, ser);
  int s = 0;
  for (size_t p = 0; p < out.size(); ++p) {
    programs[4 * p] = s; programs[4 * p + 1] = (int)out[p].steps.size(); programs[4 * p + 2] = out[p].lo; programs[4 * p + 3] = out[p].hi;
    serial[p] = ser[p];
    for (const CopyStep& c : out[p].steps) { steps[4 * s] = c.slot; steps[4 * s + 1] = c.begin; steps[4 * s + 2] = c.end; steps[4 * s + 3] = c.op; ++s; }
  }
  *n_programs = (int)out.size();
  return r;
}
"""
STORE = 8        # op: number of the value, this much more for a store


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("copy_plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    return C.CDLL(str(d / "plan.so"))


def plan(lib, copies, seqs, rows, most=1900):
    c = np.ascontiguousarray(copies, np.int32).reshape(-1, 4)
    steps, progs = np.zeros((4 * len(c) + 8, 4), np.int32), np.zeros((4 * len(c) + 8, 4), np.int32)
    serial, n = np.zeros(4 * len(c) + 8, np.int8), C.c_int()
    r = lib.plan(c.ctypes.data_as(C.c_void_p), len(c), seqs, rows, most, steps.ctypes.data_as(C.c_void_p), progs.ctypes.data_as(C.c_void_p),
                 serial.ctypes.data_as(C.c_void_p), C.byref(n))
    out = [(steps[a:a + k], lo, hi, bool(s)) for (a, k, lo, hi), s in zip(progs[:n.value].tolist(), serial[:n.value])]
    return r, out


def wanted(copies, state):
    out = state.copy()
    for s, d, b, e in copies:
        out[d, b:e] = state[s, b:e]
    return out


def carry_out(programs, state, order):
    """Programs of one launch in any order (`order` shuffles them); serial ones begin another launch."""
    launches = [[]]
    for p in programs:
        if p[3]:
            launches.append([])
        launches[-1].append(p)
    for launch in launches:
        for i in order(len(launch)):
            steps, lo, hi, _ = launch[i]
            assert steps[0][3] < STORE               # the kernel keeps the program's rows in the first step
            for r in range(lo, hi):
                v = [None] * 5
                for slot, b, e, op in steps.tolist():
                    if op < STORE:
                        v[op] = state[slot, r]
                    elif b <= r < e:
                        state[slot, r] = v[op - STORE]
    return state


def check(lib, copies, seqs, rows, most=1900):
    state = np.arange(seqs * rows).reshape(seqs, rows)
    r, programs = plan(lib, copies, seqs, rows, most)
    assert r == 0
    for order in (range, lambda n: range(n - 1, -1, -1)):
        assert np.array_equal(carry_out(programs, state.copy(), order), wanted(copies, state))
    assert all(len(p[0]) <= most for p in programs)
    return programs


def test_fork_reads_once(lib):
    programs = check(lib, [(2, d, 0, 3 + d) for d in (0, 1, 3, 4)], 5, 9)
    assert len(programs) == 1 and sum(s[3] < STORE for s in programs[0][0].tolist()) == 1


def test_independent_copies_are_programs_of_their_own(lib):
    assert len(check(lib, [(0, 1, 0, 4), (2, 3, 1, 2), (4, 5, 0, 1)], 6, 4)) == 3


@pytest.mark.parametrize("copies", [
    [(0, 1, 0, 4), (1, 0, 0, 4)], [(0, 1, 0, 4), (1, 2, 0, 4), (2, 0, 0, 4)], [(0, 1, 0, 3), (1, 0, 2, 5)],
    [(0, 1, 0, 4), (1, 2, 1, 3), (2, 3, 0, 4)], [(3, 2, 0, 4), (2, 1, 0, 4), (1, 0, 0, 4), (3, 4, 0, 1)],
    [(0, 1, 0, 4), (1, 0, 0, 4), (0, 2, 0, 4), (1, 3, 2, 4), (2, 4, 0, 4)], [(1, 1, 0, 4), (1, 0, 0, 4)], [(0, 1, 2, 2), (1, 0, 0, 0)], []])
def test_chains_and_cycles(lib, copies):
    check(lib, copies, 5, 6)


@pytest.mark.parametrize("most", [1900, 24, 12])
@pytest.mark.parametrize("seed", range(60))
def test_random(lib, seed, most):
    g = np.random.default_rng(seed)
    seqs, rows = int(g.integers(1, 12)), int(g.integers(1, 9))
    copies = []
    for d in g.permutation(seqs)[:int(g.integers(0, seqs + 1))]:
        b = int(g.integers(0, rows + 1))
        copies.append((int(g.integers(0, seqs)), int(d), b, int(g.integers(b, rows + 1))))
    r, programs = plan(lib, copies, seqs, rows, most)
    if r == 3:
        assert most < 24
        return
    check(lib, copies, seqs, rows, most)


def test_long_forks_and_chains_are_cut(lib):
    assert len(check(lib, [(0, d, 0, 2) for d in range(1, 40)], 40, 2, 8)) > 1
    assert len(check(lib, [(d + 1, d, 0, 2) for d in range(39)], 40, 2, 8)) > 1


def test_refusals(lib):
    for bad in ([(0, 5, 0, 1)], [(-1, 0, 0, 1)], [(5, 0, 0, 1)], [(0, -1, 0, 1)], [(0, 1, -1, 1)], [(0, 1, 0, 7)], [(0, 1, 3, 2)]):
        assert plan(lib, bad, 5, 6)[0] == 1
    assert plan(lib, [(0, 1, 0, 1), (2, 1, 3, 4)], 5, 6)[0] == 2
    assert plan(lib, [(1, 1, 0, 1), (2, 1, 0, 4)], 5, 6)[0] == 2
    assert plan(lib, [(d, (d + 1) % 10, 0, 1) for d in range(10)], 10, 6, 19)[0] == 3
    assert plan(lib, [(d, (d + 1) % 10, 0, 1) for d in range(10)], 10, 6, 20)[0] == 0
