"""Every item of every call has a result: one range without a part to join it with, items that bad groups leave out, indices at the ends of
32 bits.  Tolerances are those of test_gpu_prefix_attention.py."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from gpu_util import have_b200
from mdlarc_scale_b200 import _lib, prefix, prefix_attention
from test_gpu_prefix_attention import BF16, F16, F32, FORM_IDS, FORMS, Case

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not have_b200(), reason="needs a B200")]
CODES = {F16: _lib.ACT_F16, BF16: _lib.ACT_BF16, F32: _lib.ACT_F32}


def scratch_of(c, **hints):
    n, heads, dim = c.q.shape
    a = _lib.PrefixAttentionArgs(n_groups=len(c.sizes), n_items=n, n_heads=heads, n_kv=c.k.shape[1], dim=dim, n_seqs=c.k.shape[0], t_max=c.k.shape[2],
                                 scale=0.125, act_format=CODES[c.q.dtype], kv_format=CODES[c.k.dtype], **hints)
    return _lib.load().arcb_prefix_attention_scratch_bytes(C.byref(a))


@pytest.mark.parametrize("form", [(BF16, BF16), (F16, F16)], ids=["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv,most,prefix,groups", [(64, 8, 8, 100, 1024, 16), (128, 16, 4, 40, 700, 35), (64, 4, 2, 70, 641, 74)])
def test_shared_rows_alone_in_one_range(form, dim, heads, kv, most, prefix, groups):
    """Enough groups for one range each, more than 64 query rows, no rows of the items' own: parts of tensor memory's results, joined alone."""
    sizes = [most, 0, 1] + [(g * 37) % (most + 1) for g in range(groups - 3)]
    lens = [prefix, prefix, 0] + [prefix - (g * 131) % prefix for g in range(groups - 3)]
    c = Case(sizes, lens, [0] * sum(sizes), heads, kv, dim, form, seed=groups, own_in_group=True, rows=prefix + 9)
    hints = dict(max_group=most, max_prefix=prefix)
    assert scratch_of(c, **hints) == c.q.numel() // dim * (dim + 4) * 4          # one part of every result
    out = torch.full_like(c.q, math.nan)
    prefix_attention(c.q, c.k, c.v, *c.groups, out=out, **hints)
    c.check(out, mine=False)
    skip = torch.zeros(sum(sizes), dtype=torch.uint8, device="cuda")
    skip[0] = skip[-1] = 1
    c.check(prefix_attention(c.q, c.k, c.v, *c.groups, skip=skip, **hints), mine=False, skip=(0, sum(sizes) - 1))
    c.check(prefix_attention(c.q, c.k, c.v, *c.groups, scale=-0.2, **hints), scale=-0.2, mine=False)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("sizes,heads,kv", [([3, 2], 2, 2), ([5, 2], 16, 2), ([40, 3], 4, 2)])
def test_ends_of_32_bits(form, sizes, heads, kv):
    """Ends whose difference does not fit 32 bits: rows outside the cache count as not there and are reported, an end before the begin is no
    row and no error."""
    c = Case(sizes, [140, 130], [1 + i % 9 for i in range(sum(sizes))], heads, kv, 64, form, 31)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    item = 1
    for hints in (dict(max_group=max(sizes), max_prefix=140, max_own=9), {}):
        for begin, end, code in ((-2 ** 31, 0, 4), (-2 ** 31, 2 ** 31 - 1, 4), (-2, 2 ** 31 - 1, 4), (-1, 2 ** 31 - 1, 4), (-2 ** 31, -1, 4), (1, -2 ** 31, 0),
                                 (2 ** 31 - 1, -2 ** 31, 0), (2 ** 31 - 1, 2 ** 31 - 1, 0), (-2 ** 31, -2 ** 31, 0), (0, 2 ** 31 - 1, 4), (5, -3, 0)):
            keep, old = [t[item].clone() for t in c.items], c.own[item]
            c.items[1][item], c.items[2][item], c.own[item] = begin, end, 0
            status.zero_()
            out = c(status=status, **hints)
            assert status.item() == code, (begin, end)
            was, c.begin[item] = c.begin[item], 0
            c.check(out)
            c.begin[item], c.own[item] = was, old
            for t, v in zip(c.items, keep):
                t[item] = v


def dirty(c, **hints):
    """The next call's scratch has held other parts."""
    need = max(scratch_of(c, d_item_end=4096, **hints), scratch_of(c, **hints))
    torch.full((max(4, need) // 4,), 3.0, device="cuda")
    return torch.full_like(c.q, math.nan)


# items of three groups, heads, key heads, rows of the longest group, what the plan is told: one CTA a group, warps, CTAs of 16 to 64 query
# rows, tensor memory; results of one part where no item has rows of its own
@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("sizes,heads,kv,prefix,plan", [([3, 2, 4], 4, 4, 60, 60), ([3, 2, 4], 2, 2, 200, 200), ([3, 2, 4], 2, 1, 190, 4000), ([3, 2, 4], 16, 4, 60, 60),
                                                        ([9, 5, 16], 2, 1, 300, 300), ([30, 7, 50], 1, 1, 200, 200), ([80, 70, 100], 2, 2, 700, 4000)])
@pytest.mark.parametrize("dim", [64, 128])
def test_items_that_bad_groups_leave_out(form, sizes, heads, kv, prefix, plan, dim):
    """Items of groups that are wrong, and items between or behind groups, see their own rows alone, and nothing that scratch or output have held."""
    n, ends = sum(sizes), np.cumsum([0] + sizes).tolist()
    c = Case(sizes, [prefix, prefix - 7, prefix // 2], [i % 9 for i in range(n)], heads, kv, dim, form, seed=n)
    hints = dict(max_group=max(sizes), max_prefix=plan, max_own=9)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = [("first", 0, 2, [0]), ("first", 0, -2 ** 31, [0]), ("first", 0, n + 1, [0]), ("first", 3, n - 2, [2]), ("first", 3, 2 ** 31 - 1, [2]), ("first", 3, 0, [2]),
           ("first", 1, -5, [0, 1]), ("first", 1, 10 ** 6, [0, 1]), ("first", 2, n + 1, [1, 2]), ("seq", 1, 99999, [1]), ("len", 2, -1, [2]),
           ("group", 0, max(sizes) - 1, [2])]
    tensors, lengths, own = dict(zip(("first", "seq", "len"), c.groups)), list(c.prefix), list(c.own)
    assert tensors["first"].tolist() == ends
    for what, at, value, gone in bad:
        kw = dict(hints)
        if what == "group":
            kw["max_group"] = value
        else:
            old = tensors[what][at].clone()
            tensors[what][at] = value
        c.prefix = [0 if g in gone else p for g, p in enumerate(lengths)]
        for mine in (True, False):
            status.zero_()
            out = dirty(c, **kw)
            prefix_attention(c.q, c.k, c.v, *c.groups, *(c.items if mine else ()), out=out, status=status, **kw)
            assert status.item() == 4, (what, at, value)
            c.check(out, mine=mine)
        if what != "group":
            tensors[what][at] = old
    # no group but the last one, which ends where it begins
    tensors["first"].zero_()
    c.prefix = [0, 0, 0]
    for mine in (True, False):
        status.zero_()
        out = dirty(c, **hints)
        prefix_attention(c.q, c.k, c.v, *c.groups, *(c.items if mine else ()), out=out, status=status, **hints)
        assert status.item() == 4
        c.check(out, mine=mine)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_bounds_of_no_rows(form, monkeypatch):
    """0 rows is a bound, not an unknown one: the work is planned for as few as there can be, and what the tensors hold counts all the same."""
    planned, attend = [], prefix._attend

    def look(a, out, dev):
        packed = _lib.PrefixAttentionArgs.from_buffer_copy(a)
        planned.append((packed.max_group, packed.max_prefix, packed.max_own))
        attend(a, out, dev)

    monkeypatch.setattr(prefix, "_attend", look)
    c = Case([3, 20], [300, 101], [i * 13 % 90 for i in range(23)], 4, 2, 64, form, 15)
    for kw, want in ((dict(max_prefix=0, max_own=0), (0, 1, 1)), (dict(max_group=20, max_prefix=0), (20, 1, 0)), (dict(max_own=0), (0, 0, 1)), ({}, (0, 0, 0)),
                     (dict(max_prefix=300, max_own=90), (0, 300, 90))):
        c.check(c(**kw))
        assert planned.pop() == want
    for kw in (dict(max_prefix=-1), dict(max_own=-1), dict(max_group=-1)):
        with pytest.raises(ValueError):
            c(**kw)


@pytest.mark.parametrize("form", [(F16, BF16), (F32, F32)], ids=["f16-bf16", "f32"])
@pytest.mark.parametrize("value", [-7, 2 ** 31 - 1, -2 ** 31, 0, 201])
@pytest.mark.parametrize("kept", [0, 100])
def test_ends_that_are_all_wrong(form, value, kept):
    """Two thousand groups whose ends, but the first ones, are no items': the groups ahead of them have theirs, all other items their own rows."""
    groups, n = 2000, 200
    sizes = [1] * n + [0] * (groups - n)
    c = Case(sizes, [20] * n + [0] * (groups - n), [i % 5 for i in range(n)], 2, 1, 64, form, seed=kept)
    c.groups[0][kept + 1:] = value
    c.prefix = [20 if i < kept else 0 for i in range(groups)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    hints = dict(max_group=1, max_prefix=20, max_own=5)
    for mine in (True, False):
        status.zero_()
        out = dirty(c, **hints)
        prefix_attention(c.q, c.k, c.v, *c.groups, *(c.items if mine else ()), out=out, status=status, **hints)
        assert status.item() == 4
        c.check(out, mine=mine)
