"""How attention over shared cached rows is cut into units of work (csrc/prefix_rules.cuh), compiled for the host: the lines that were
measured on 148 SMs stay, and every plan covers the work it is made for."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mdlarc_scale_b200" / "csrc"
SOURCE = r"""
#include "prefix_rules.cuh"
extern "C" void plan(const long long* in, long long* out) {
  const PrefixPlan p = prefix_plan(in[0], in[1], in[2], in[3], in[4], (int)in[5], (int)in[6], (int)in[7], in[8] != 0, in[9] != 0, (int)in[10]);
  const long long v[] = {p.shared.kernel, p.shared.tile, p.shared.tiles, p.shared.splits, p.shared.units,
                         p.own.kernel, p.own.tile, p.own.tiles, p.own.splits, p.own.units, p.together, p.grouped, p.parts};
  for (int i = 0; i < 13; ++i) out[i] = v[i];
}
"""
ROWS, TILES, TC, F32_FEW, F32 = range(5)


class Plan:
    pass


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), str(d / "rules.cpp"), "-o", str(d / "rules.so")], check=True)
    lib = C.CDLL(str(d / "rules.so"))

    def of(groups, items, prefix, own, kv, rep, dim=128, wide=False, tc=False, sms=148, total=None):
        total = max(1, groups) * items if total is None else total
        a, b = (C.c_longlong * 11)(groups, items, prefix, total, own, kv, rep, dim, wide, tc, sms), (C.c_longlong * 13)()
        lib.plan(a, b)
        p = Plan()
        p.shared, p.own = Plan(), Plan()
        for part, at in ((p.shared, 0), (p.own, 5)):
            part.kernel, part.tile, part.tiles, part.splits, part.units = b[at:at + 5]
        p.together, p.grouped, p.parts = b[10:]
        return p

    return of


def test_kernels_by_query_rows(plan):
    for rows, want in ((1, (ROWS, 8)), (8, (ROWS, 8)), (9, (TILES, 16)), (16, (TILES, 16)), (17, (TILES, 32)), (33, (TILES, 64)), (64, (TILES, 64)),
                       (65, (TC, 256)), (257, (TC, 256))):
        p = plan(3, rows, 5000, 0, 2, 1, tc=True)
        assert (p.shared.kernel, p.shared.tile) == want and p.shared.tiles == -(-rows // want[1]) and p.own.units == 0
    assert plan(3, 65, 5000, 0, 2, 1, tc=False).shared.kernel == TILES
    for rows, want in ((1, (F32_FEW, 1)), (2, (F32_FEW, 2)), (3, (F32_FEW, 4)), (4, (F32_FEW, 4)), (5, (F32, 16)), (17, (F32, 32)), (33, (F32, 64)), (300, (F32, 64))):
        p = plan(3, rows, 5000, 10, 2, 1, wide=True)
        assert (p.shared.kernel, p.shared.tile) == want
        assert p.together == (want == (F32_FEW, 1))          # units of one launch have one size
    assert plan(3, 4, 500, 100, 2, 2).together and not plan(3, 5, 500, 100, 2, 2).together


def test_few_samples_take_one_launch(plan):
    p = plan(1, 2, 190, 17, 4, 1, 64)
    assert p.grouped and p.shared.splits == 6 and p.own.splits == 1 and p.parts == 7
    assert plan(1, 2, 64 * 6, 64, 4, 1).grouped and not plan(1, 2, 64 * 6 + 1, 64, 4, 1).grouped and not plan(1, 2, 190, 65, 4, 1).grouped
    assert plan(1, 7, 64, 9, 4, 1).grouped and not plan(1, 8, 64, 9, 4, 1).grouped
    assert plan(37, 2, 190, 17, 4, 1).grouped and not plan(38, 2, 190, 17, 4, 1).grouped          # a CTA an SM
    assert plan(33, 2, 190, 17, 4, 1, sms=132).grouped and not plan(34, 2, 190, 17, 4, 1, sms=132).grouped
    assert not plan(1, 2, 190, 0, 4, 1).grouped and not plan(1, 2, 190, 17, 4, 1, wide=True).grouped


def test_lines_on_148_sms(plan):
    """One range for what runs at once; a wave of 256-row tiles against steps and joins."""
    p = plan(1, 64, 8191, 500, 8, 4, tc=True)
    assert p.own.splits == 3 and p.own.units == 1536 and p.shared.kernel == TC and p.shared.units <= 148
    p = plan(1, 256, 32768, 250, 8, 4, tc=True)
    assert p.shared.splits == 4 and p.shared.units == 128 and p.own.splits == 1
    p = plan(24, 5, 4096, 5, 8, 4)
    assert p.shared.kernel == TILES and p.shared.splits == 4 and p.own.splits == 1
    p = plan(64, 8, 1193, 300, 20, 1, 64)
    assert p.together and p.shared.splits == 2 and p.own.splits == 1


def test_any_sizes(plan):
    r = random.Random(5)
    for _ in range(4000):
        size = lambda most: int(round(most ** r.random()))      # noqa: E731
        groups, items, prefix, own, kv, rep = size(200) * r.randint(0, 3), size(300), size(200000), size(5000) * r.randint(0, 1), size(32), size(40)
        if groups == 0 and own == 0:
            continue
        dim, wide, tc, sms = r.choice((64, 128)), r.random() < 0.3, r.random() < 0.5, r.choice((20, 132, 148, 160))
        total = r.randint(1, items) if groups == 0 else groups * items
        p = plan(groups, items, prefix, own, kv, rep, dim, wide, tc, sms, total)
        for part, heads, rows, have, most in ((p.shared, groups, items * rep, groups > 0, 128), (p.own, total, rep, own > 0, 32)):
            if not have:
                assert part.units == 0 and part.splits == 0
                continue
            assert part.tile * part.tiles >= rows > part.tile * (part.tiles - 1)
            assert 1 <= part.splits <= most and part.units == heads * kv * part.tiles * part.splits
            assert part.kernel != TC or (tc and not wide)
            assert (part.kernel in (F32_FEW, F32)) == wide
        assert p.parts == p.shared.splits + p.own.splits >= 1
        assert p.own.kernel != TC
        if p.together:
            assert p.shared.kernel == p.own.kernel and (not wide or p.shared.tile == p.own.tile)
        if p.grouped:
            assert p.together and p.shared.kernel == ROWS and p.shared.tiles == 1 and p.shared.splits + items <= 8 and items * rep <= 8
