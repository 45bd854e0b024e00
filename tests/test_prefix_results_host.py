"""Every plan of attention over shared cached rows ends in results: kernels that write parts alone are followed by a join, and have memory
for their parts.  No GPU needed."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest
import torch

from mdlarc_scale_b200 import _lib

CSRC = Path(__file__).resolve().parent.parent / "mdlarc_scale_b200" / "csrc"
SOURCE = r"""
#include "prefix_rules.cuh"
extern "C" void plan(const long long* in, int* out) {
  const PrefixPlan p = prefix_plan(in[0], in[1], in[2], in[3], in[4], (int)in[5], (int)in[6], (int)in[7], in[8] != 0, in[9] != 0, (int)in[10]);
  out[0] = p.shared.kernel == AP_TC; out[1] = p.parts; out[2] = p.grouped; out[3] = p.joined;
}
extern "C" int rows(int begin, int end, int seq, int n_seqs, int t_max) { return ap_row_count(begin, end, seq, n_seqs, t_max); }
"""
LEAST, MOST = -2 ** 31, 2 ** 31 - 1
# groups, items of each, key heads, heads of a key head, dim, shared rows: units enough for one range each, no rows of the items' own
ONE_RANGE = [(64, 32, 8, 4, 128, 2048), (8, 64, 8, 4, 128, 1024), (20, 66, 20, 1, 64, 640), (1, 256, 32, 4, 128, 700)]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), str(d / "rules.cpp"), "-o", str(d / "rules.so")], check=True)
    lib = C.CDLL(str(d / "rules.so"))

    def of(groups, items, prefix, own, kv, rep, dim, wide=False, tc=True, sms=148):
        out = (C.c_int * 4)()
        lib.plan((C.c_longlong * 11)(groups, items, prefix, max(1, groups) * items, own, kv, rep, dim, wide, tc, sms), out)
        return tuple(out)
    of.rows = lib.rows
    return of


def test_rows_of_any_ends(plan):
    """Ends of any 32 bits: a range is counted, empty, or outside the cache, and never a difference that has wrapped around."""
    ends = [LEAST, LEAST + 1, -100, -2, -1, 0, 1, 2, 99, 100, 101, 10 ** 9, MOST - 1, MOST]
    for begin in ends:
        for end in ends:
            for seq in (LEAST, -1, 0, 4, 5, MOST):
                inside = begin >= 0 and end <= 100 and 0 <= seq < 5
                assert plan.rows(begin, end, seq, 5, 100) == (0 if end <= begin else end - begin if inside else -1), (begin, end, seq)


@pytest.mark.parametrize("groups,items,kv,rep,dim,prefix", ONE_RANGE)
def test_tensor_memory_results_of_one_range_are_joined(plan, groups, items, kv, rep, dim, prefix):
    tc, parts, grouped, joined = plan(groups, items, prefix, 0, kv, rep, dim)
    assert tc and parts == 1 and not grouped and joined


@pytest.mark.parametrize("groups,items,kv,rep,dim,prefix", ONE_RANGE)
def test_results_of_one_range_have_memory(groups, items, kv, rep, dim, prefix):
    from mdlarc_scale_b200 import build
    build.build()
    a = _lib.PrefixAttentionArgs(n_groups=groups, n_items=groups * items, n_heads=kv * rep, n_kv=kv, dim=dim, n_seqs=groups, t_max=prefix, scale=0.125,
                                 act_format=_lib.ACT_BF16, kv_format=_lib.ACT_BF16, max_group=items)
    need = _lib.load().arcb_prefix_attention_scratch_bytes(C.byref(a))
    assert need >= groups * items * kv * rep * (dim + 4) * 4
    # and a call without it is refused ahead of any launch
    for field in ("d_q", "d_k", "d_v", "d_out", "d_group_first", "d_group_seq", "d_group_len"):
        setattr(a, field, 4096)
    assert _lib.load().arcb_op_prefix_attention(C.byref(a), None) == _lib.E_ARG


def test_results_are_written_once(plan):
    """By the kernels themselves where there is one part of a result that they can finish, by the CTA of a group, or by a join."""
    r = random.Random(6)
    seen = set()
    for _ in range(6000):
        size = lambda most: int(round(most ** r.random()))      # noqa: E731
        groups, items, prefix, own, kv, rep = size(200) * r.randint(0, 3), size(300), size(40000), size(3000) * r.randint(0, 1), size(32), size(40)
        if groups == 0 and own == 0:
            continue
        tc, parts, grouped, joined = plan(groups, items, prefix, own, kv, rep, r.choice((64, 128)), r.random() < 0.3, r.random() < 0.7, r.choice((20, 148)))
        assert joined == (not grouped and (parts > 1 or tc))
        seen.add((tc, parts > 1, grouped))
    assert len(seen) == 5


def test_gradients_are_refused():
    """Neither operator has one: an output without it would end a backward pass in silence."""
    from mdlarc_scale_b200 import copy_cache_rows, prefix_attention
    q, k = torch.zeros((2, 2, 64)), torch.zeros((1, 2, 5, 64))
    first, seq, length = (torch.zeros(n, dtype=torch.int32) for n in (2, 1, 1))
    for at in range(3):
        args = [t.clone().requires_grad_(i == at) for i, t in enumerate((q, k, k))]
        with pytest.raises(ValueError, match="no gradient"):
            prefix_attention(*args, first, seq, length)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            prefix_attention(*args, first, seq, length)
    with pytest.raises(ValueError, match="no gradient"):
        prefix_attention(q, k, k, first, seq, length, out=torch.zeros_like(q, requires_grad=True))
    with pytest.raises(ValueError, match="no gradient"):
        copy_cache_rows(k.clone().requires_grad_(), [(0, 0, 0, 1)])
    with pytest.raises(ValueError, match="CUDA"):
        copy_cache_rows(k, [(0, 0, 0, 1)])
