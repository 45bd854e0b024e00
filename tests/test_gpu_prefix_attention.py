"""Attention of queries that share cached rows against softmax(scale q K^T) V in 64 bits.

Tolerance of a value o = sum_t p_t v_t, from the arithmetic alone: the output's rounding, u |o| with u half a step of its type, and
errors of the weights, each relative to p_t, so that their sum is bounded by a factor of A = sum_t p_t |v_t|.  The factor: a weight
rounded to the products' operand type in two pieces is 2^-16 off, in one half a step of the type (half: 2^-11; bfloat16, where
max_group, by default the number of items, allows more than 16 query rows a key head, 2^-8); a score is a sum of dim products in 32
bits whose every addition is off by 2^-23 of the partial sums, at most (dim + 4) 2^-23 S with S = scale sum_d |q_d k_d|, and the
exponential turns an absolute error of a score into a relative one of the weight, twice (numerator and denominator); sums over the
rows and joins of parts in 32 bits: 2^-23 for each of the chain's additions, at most (rows + 128) of them.
"""
import math

import numpy as np
import pytest
import torch

from gpu_util import have_b200
from mdlarc_scale_b200 import _lib, prefix_attention

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not have_b200(), reason="needs a B200")]
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
FORMS = [(F16, BF16), (BF16, BF16), (F16, F16), (F32, F32)]
FORM_IDS = ["f16-bf16", "bf16", "f16", "f32"]


class Case:
    """Ragged groups over one cache; every row that no item may see holds NaN."""

    def __init__(self, sizes, prefix, own, heads, kv, dim, form, seed=0, own_in_group=False, sharp=1.0, spread=1.0, rows=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = np.random.default_rng(seed)
        n = sum(sizes)
        self.sizes, self.prefix, self.own = list(sizes), list(prefix), list(own)
        first = np.concatenate([[0], np.cumsum(sizes)]).astype(int)
        group_of = np.repeat(np.arange(len(sizes)), sizes)
        self.begin = [prefix[x] if own_in_group else int(r.integers(0, 20)) for x in group_of]
        seqs = len(sizes) if rows else len(sizes) + n
        places = r.permutation(seqs)
        self.group_seq = places[:len(sizes)].tolist()
        self.item_seq = [self.group_seq[x] for x in group_of] if own_in_group else places[len(sizes):].tolist()
        rows = rows or max([*prefix, *[b + o for b, o in zip(self.begin, own)], 1]) + int(r.integers(0, 3))
        q_type, kv_type = form
        self.q = (torch.randn((n, heads, dim), device="cuda", generator=g) * sharp).to(q_type)
        k = torch.randn((seqs, kv, rows, dim), device="cuda", generator=g) * spread
        v = torch.randn((seqs, kv, rows, dim), device="cuda", generator=g) + 0.3
        seen = torch.zeros((seqs, rows), dtype=torch.bool, device="cuda")
        for s, p in zip(self.group_seq, prefix):
            seen[s, :p] = True
        for s, b, o in zip(self.item_seq, self.begin, own):
            seen[s, b:b + o] = True
        k[~seen[:, None].expand(-1, kv, -1)] = math.nan
        v[~seen[:, None].expand(-1, kv, -1)] = math.nan
        self.k, self.v = k.to(kv_type), v.to(kv_type)
        self.group_of = group_of
        ints = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")      # noqa: E731
        self.groups = (ints(first), ints(self.group_seq), ints(prefix))
        self.items = (ints(self.item_seq), ints(self.begin), ints(np.array(self.begin) + np.array(own)))
        self.scale = dim ** -0.5

    def __call__(self, **kw):
        return prefix_attention(self.q, self.k, self.v, *self.groups, *self.items, **kw)

    def check(self, out, scale=None, shared=True, mine=True, skip=()):
        scale = self.scale if scale is None else scale
        n, heads, dim = self.q.shape
        rep = heads // self.k.shape[1]
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        for i in range(n):
            g = self.group_of[i]
            p, b, o = self.prefix[g] if shared else 0, self.begin[i], self.own[i] if mine else 0
            if p + o == 0 or i in skip:
                assert not out[i].any(), f"item {i} sees nothing"
                continue
            keys, values = (torch.cat([x[self.group_seq[g], :, :p], x[self.item_seq[i], :, b:b + o]], 1).double() for x in (self.k, self.v))
            q = self.q[i].double().view(-1, rep, dim)
            weights = torch.softmax(torch.matmul(q, keys.transpose(1, 2)) * scale, -1)
            want = torch.matmul(weights, values).view(heads, dim)
            spread = torch.matmul(weights, values.abs()).view(heads, dim)
            size = (torch.matmul(q.abs(), keys.abs().transpose(1, 2)) * abs(scale)).amax(-1).view(heads, 1)
            u = torch.finfo(out.dtype).eps / 2
            many = n * rep > 16 and self.q.dtype == BF16
            pieces = {F32: 0.0, BF16: 2.0 ** -8 if many else 2.0 ** -16, F16: 2.0 ** -11}[self.k.dtype]
            tol = u * want.abs() + (pieces + 2 * (dim + 4) * 2.0 ** -23 * size + (p + o + 128) * 2.0 ** -23) * spread + 2.0 ** -24
            err = (out[i].double() - want).abs()
            assert bool((err <= tol).all()), f"item {i}: {float((err / tol).max()):.2f} of the tolerance, error {float(err.max()):.3g}"


def small(form, heads, kv, dim, seed, **kw):
    r = np.random.default_rng(seed)
    sizes = [int(x) for x in r.integers(1, 9, 4)]
    prefix = [int(x) for x in r.integers(0, 150, 4)]
    own = [int(x) for x in r.integers(0, 90, sum(sizes))]
    return Case(sizes, prefix, own, heads, kv, dim, form, seed, **kw)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (4, 4, 64), (20, 5, 64), (12, 2, 128), (32, 1, 128), (7, 7, 128), (40, 2, 64)])
def test_ragged_groups(form, heads, kv, dim):
    c = small(form, heads, kv, dim, heads * dim + kv)
    c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("prefix,own", [(0, 0), (0, 1), (1, 0), (1, 1), (15, 16), (16, 15), (63, 65), (64, 64), (65, 63), (128, 0), (0, 129), (257, 31)])
def test_lengths(form, prefix, own):
    for dim in (64, 128):
        c = Case([3], [prefix], [own, max(own - 1, 0), own], 4, 2, dim, form, prefix * 7 + own)
        c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("items,heads,kv", [(1, 2, 2), (15, 1, 1), (16, 1, 1), (17, 2, 2), (33, 1, 1), (9, 8, 1), (16, 4, 1), (65, 2, 2), (127, 1, 1), (43, 3, 1),
                                            (129, 1, 1), (70, 8, 2), (300, 2, 1)])
def test_query_tiles(form, items, heads, kv):
    """Numbers of query rows about the tiles' edges."""
    for dim in (64, 128):
        c = Case([items, 2], [201, 33], [i % 5 for i in range(items + 2)], heads, kv, dim, form, items)
        c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("items,heads,kv", [(17, 4, 1), (65, 2, 2), (43, 3, 1), (128, 1, 1), (129, 1, 1), (70, 8, 2), (257, 1, 1), (300, 2, 1)])
def test_query_tiles_of_a_long_cache(form, items, heads, kv):
    """Without hints the plan is made for groups as long as a cache: most ranges of these are short or empty."""
    for dim in (64, 128):
        for prefix in (3, 1153):
            c = Case([items, 2], [prefix, 130], [i % 5 for i in range(items + 2)], heads, kv, dim, form, items, own_in_group=True, rows=4144)
            c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("prefix", [0, 1, 127, 128, 129, 255, 257, 1025, 4097, 4140])
def test_lengths_in_a_long_cache(form, prefix):
    for dim in (64, 128):
        for items in (33, 70):
            c = Case([items], [prefix], [i % 3 for i in range(items)], 4, 2, dim, form, prefix, own_in_group=True, rows=4144)
            c.check(c())
            c.check(prefix_attention(c.q, c.k, c.v, *c.groups), mine=False)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_long_rows_in_many_ranges(form, dim):
    """Rows cut into as many ranges as the plan makes; all kinds of lengths in one call, some empty."""
    c = Case([2, 1, 3], [9001, 0, 517], [3000, 0, 1, 2, 4097, 64], 4, 2, dim, form, dim)
    c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_many_queries_over_a_long_prefix(form):
    c = Case([90, 70], [2900, 1031], [i * 7 % 40 for i in range(160)], 8, 2, 128, form, 5)
    c.check(c())
    c = Case([150, 3], [1500, 2100], [i * 7 % 40 for i in range(153)], 3, 3, 64, form, 6)
    c.check(c())
    c = Case([100, 71], [4600, 9003], [i % 4 for i in range(171)], 2, 1, 64, form, 7, own_in_group=True, rows=9008, sharp=3.0)
    c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("sizes,prefix,own", [([2], [190], 17), ([1, 2, 1], [0, 31, 33], 64), ([7, 6], [64, 1], 3), ([4, 1, 3, 2], [256, 200, 0, 97], 40), ([2, 2], [0, 0], 5)])
def test_few_items_over_a_short_prefix(form, sizes, prefix, own):
    """As few samples of a short prompt are: groups of one CTA."""
    for heads, kv, dim in ((4, 4, 64), (8, 8, 128), (2, 1, 128)):
        c = Case(sizes, prefix, [(own - 3 * i) % (own + 1) for i in range(sum(sizes))], heads, kv, dim, form, own)
        hints = dict(max_group=max(sizes), max_prefix=max(1, max(prefix)), max_own=own)
        c.check(c(**hints))
        assert torch.equal(c(**hints), c(**hints))
        c.check(c(**dict(hints, max_prefix=1, max_own=1)))          # bounds that are too small: longer ranges
        skip = torch.zeros(sum(sizes), dtype=torch.uint8, device="cuda")
        skip[-1] = 1
        c.check(c(skip=skip, **hints), skip=(sum(sizes) - 1,))


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("items", [2, 5, 33, 140])
def test_scores_that_grow_along_the_rows(form, items):
    """Maxima that have to be raised again and again, and ones that never are."""
    for dim in (64, 128):
        for ramp in ((0.05, 8.0), (8.0, 0.05)):
            c = Case([items], [1600], [i % 3 for i in range(items)], 4, 2, dim, form, items, own_in_group=True, rows=4144)
            c.k *= torch.linspace(*ramp, 4144, device="cuda").to(c.k.dtype)[None, None, :, None]
            c.check(c())


@pytest.mark.parametrize("form", FORMS[1:], ids=FORM_IDS[1:])
@pytest.mark.parametrize("items", [2, 33, 140])
def test_rows_whose_scores_are_infinite(form, items):
    """Keys of minus infinity under queries that are not negative: scores of minus infinity, weights of 0, as if the rows were not there.
    Half queries over bfloat16 keys are no case of it: a query is hi + lo there, lo is 0 or of either sign, and 0 times an infinity, like
    the sum of two that differ in sign, is no number."""
    gone = 260
    for dim in (64, 128):
        c = Case([items], [900], [0] * items, 4, 2, dim, form, items, own_in_group=True, rows=4144)
        c.q = c.q.abs() + 0.01
        seq = c.group_seq[0]
        c.k[seq, :, :gone] = -math.inf
        out = c()
        assert bool(torch.isfinite(out).all())
        c.k = c.k[:, :, gone:].contiguous()
        c.v = c.v[:, :, gone:].contiguous()
        c.prefix = [900 - gone]
        c.check(out)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_draft_tokens_of_a_sequence(form):
    """Item j of a group sees the shared rows and j + 1 rows behind them, of the same sequence."""
    sizes, prefix = [5, 1, 4], [130, 64, 1]
    c = Case(sizes, prefix, [j + 1 for s in sizes for j in range(s)], 8, 2, 128, form, 3, own_in_group=True)
    c.check(c())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_sharp_and_flat_softmax(form):
    for sharp, spread in ((40.0, 1.0), (0.0, 1.0), (1.0, 1e-3)):
        c = small(form, 4, 2, 64, 11, sharp=sharp, spread=spread)
        c.check(c())


def test_scales():
    for scale in (0.0, -0.3, 2.0):
        c = small((BF16, BF16), 4, 2, 64, 12)
        c.check(c(scale=scale), scale)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_one_part_alone(form):
    """Only shared rows, or only own ones: no join."""
    c = small(form, 8, 4, 64, 13)
    c.check(prefix_attention(c.q, c.k, c.v, *c.groups), mine=False)
    c.check(prefix_attention(c.q, c.k, c.v, item_seq=c.items[0], item_begin=c.items[1], item_end=c.items[2]), shared=False)
    c.check(prefix_attention(c.q, c.k, c.v, item_seq=c.items[0], item_begin=c.items[1], item_end=c.items[2], max_own=64), shared=False)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_own_rows_by_default(form):
    """Without item_seq and item_begin: sequence i from row 0."""
    n, rows = 5, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((n, 4, 64), device="cuda", generator=g).to(form[0])
    k, v = (torch.randn((n, 2, rows, 64), device="cuda", generator=g).to(form[1]) for _ in range(2))
    end = torch.tensor([0, 1, 70, 33, 64], dtype=torch.int32, device="cuda")
    same = prefix_attention(q, k, v, item_seq=torch.arange(n, dtype=torch.int32, device="cuda"), item_begin=torch.zeros(n, dtype=torch.int32, device="cuda"), item_end=end)
    assert torch.equal(prefix_attention(q, k, v, item_end=end), same)
    assert not same[0].any() and bool(torch.isfinite(same).all())


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_skipped_items(form):
    c = small(form, 4, 2, 128, 14)
    n = c.q.shape[0]
    skip = torch.zeros(n, dtype=torch.uint8, device="cuda")
    skip[1] = skip[n - 1] = 1
    c.check(c(skip=skip), skip=(1, n - 1))
    skip[:] = 1
    assert not c(skip=skip).any()
    skip[:] = 0
    skip[0] = 255
    c.check(prefix_attention(c.q, c.k, c.v, *c.groups, skip=skip), mine=False, skip=(0,))


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_hints_plan_and_do_not_cut(form):
    """Bounds that are too small, or far too large, change the ranges, not the rows."""
    c = Case([3, 20], [900, 301], [i * 13 % 300 for i in range(23)], 4, 2, 64, form, 15)
    for kw in (dict(max_prefix=1, max_own=1), dict(max_prefix=900, max_own=300), dict(max_group=20), dict(max_group=23, max_prefix=10 ** 6, max_own=10 ** 6)):
        c.check(c(**kw))


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_queries_in_a_wider_matrix(form):
    c = small(form, 4, 2, 64, 16)
    wide = torch.full((c.q.shape[0], 3 * 256 + 16), math.nan, device="cuda", dtype=form[0])
    wide[:, 256:512] = c.q.flatten(1)
    q = wide[:, 256:512].view(-1, 4, 64)
    want = c()
    got = prefix_attention(q, c.k, c.v, *c.groups, *c.items)
    assert torch.equal(got, want)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_runs_are_equal_and_outputs_are_all_written(form):
    c = Case([40, 3], [1201, 77], [i * 31 % 200 for i in range(43)], 8, 2, 128, form, 17)
    out = torch.full_like(c.q, math.nan)
    first = c(out=out).clone()
    assert c(out=out) is out and torch.equal(out, first) and bool(torch.isfinite(out).all())


def test_nothing_beyond_the_output_is_written():
    c = small((F16, BF16), 5, 5, 64, 18)
    n = c.q.shape[0]
    room = torch.full((n + 2, 5, 64), 7.0, device="cuda", dtype=F16)
    c.check(c(out=room[1:n + 1]))
    assert bool((room[0] == 7).all()) and bool((room[n + 1] == 7).all())


def test_streams_and_graphs():
    """Calls on two streams at once, and two captured ones that are replayed with other lengths and inputs."""
    cases = [Case([6, 2], [700, 90], [i * 9 % 60 for i in range(8)], 8, 2, 128, (BF16, BF16), s) for s in (20, 21)]
    want = [c() for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [None, None]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i] = c()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs, graphs = [torch.empty_like(w) for w in want], []
    for c, o in zip(cases, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c(out=o)
        graphs.append(graph)
    for c in cases:
        c.prefix[0] -= 333
        c.groups[2][0] -= 333
        c.own = [max(o - 1, 0) for o in c.own]
        c.items[2].copy_(torch.tensor(np.array(c.begin) + np.array(c.own), dtype=torch.int32))
        c.q.mul_(-0.5)
    for g in (graphs[1], graphs[0], graphs[1]):
        g.replay()
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        c.check(o)


def test_offsets_beyond_32_bits():
    """The last sequences of a 10 GB cache of keys and one of values."""
    rows, seqs = 40_016, 1024
    k = torch.zeros((seqs, 1, rows, 64), device="cuda", dtype=F16)
    v = torch.zeros((seqs, 1, rows, 64), device="cuda", dtype=F16)
    g = torch.Generator(device="cuda").manual_seed(2)
    for t in (k, v):
        t[seqs - 2:].copy_(torch.randn((2, 1, rows, 64), device="cuda", generator=g))
    c = Case.__new__(Case)
    c.q = torch.randn((20, 2, 64), device="cuda", generator=g).half()
    c.k, c.v, c.scale = k, v, 0.125
    c.sizes, c.prefix, c.own, c.group_of = [20], [rows], [i * 17 for i in range(20)], [0] * 20
    c.begin, c.group_seq, c.item_seq = [rows - o for o in c.own], [seqs - 1], [seqs - 2] * 20
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")      # noqa: E731
    c.groups, c.items = (ints([0, 20]), ints(c.group_seq), ints(c.prefix)), (ints(c.item_seq), ints(c.begin), ints([rows] * 20))
    c.check(c(max_group=20))


@pytest.mark.parametrize("form,items", [(F32, 20), (F32, 2), (BF16, 80), (F16, 3)])
def test_offsets_beyond_32_bits_of_other_kernels(form, items):
    rows, seqs = 40_016, 900
    k, v = (torch.zeros((seqs, 1, rows, 64), device="cuda", dtype=form) for _ in range(2))
    c = Case([items], [rows], [i % 7 for i in range(items)], 2, 1, 64, (form, form), 3, own_in_group=True, rows=rows + 8)
    for big, small_one in ((k, c.k), (v, c.v)):
        big[seqs - 1].copy_(small_one[0, :, :rows])
    own = [min(o, rows) for o in c.own]
    c.begin = [rows - o for o in own]
    c.own, c.k, c.v, c.group_seq, c.item_seq = own, k, v, [seqs - 1], [seqs - 1] * items
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")      # noqa: E731
    c.groups, c.items = (ints([0, items]), ints(c.group_seq), ints([rows])), (ints(c.item_seq), ints(c.begin), ints([rows] * items))
    c.check(c(max_own=7))


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("items,heads,kv", [(2, 2, 2), (5, 4, 2), (33, 2, 1), (140, 2, 1)])
def test_nan_in_a_query_of_any_size_of_group(form, items, heads, kv):
    for dim in (64, 128):
        c = Case([items], [700], [i % 9 for i in range(items)], heads, kv, dim, form, items, own_in_group=True, rows=4144)
        for hints in ({}, dict(max_group=items, max_prefix=300, max_own=9)):
            want = c(**hints)
            q = c.q.clone()
            q[items - 1, 1] = math.nan
            out = prefix_attention(q, c.k, c.v, *c.groups, *c.items, **hints)
            assert bool(torch.isnan(out[items - 1, 1]).all())
            out[items - 1, 1] = want[items - 1, 1]
            assert torch.equal(out, want)


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("sizes,heads,kv", [([3, 2], 2, 2), ([5, 2], 16, 2), ([40, 3], 4, 2)])
def test_bad_indices_in_any_size_of_group(form, sizes, heads, kv):
    c = Case(sizes, [140, 130], [1 + i % 9 for i in range(sum(sizes))], heads, kv, 64, form, 29)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    hints = dict(max_group=max(sizes), max_prefix=140, max_own=9)
    want, first = c(status=status, **hints), sizes[0]
    assert status.item() == 0
    for what, i, value in (("groups", 1, 99), ("groups", 1, -1), ("groups", 2, 10 ** 6), ("groups", 2, -3), ("groups", 0, 2), ("groups", 0, -2 ** 31), ("items", 0, 500),
                           ("items", 0, -2 ** 31), ("items", 1, -2), ("items", 2, 2 ** 31 - 1)):
        t = getattr(c, what)[i]
        old = t[0].clone()
        t[0] = value
        status.zero_()
        out = c(status=status, **hints)
        assert status.item() == 4, (what, i, value)
        t[0] = old
        assert torch.equal(out[first:], want[first:])
    status.zero_()
    assert torch.equal(c(status=status, **hints), want) and status.item() == 0


def test_nan_in_a_query_stays_in_its_item():
    c = small((F16, F16), 4, 2, 64, 22)
    c.q[2, 1] = math.nan
    out = c()
    assert bool(torch.isnan(out[2, 1]).all())
    out[2, 1] = 0
    assert bool(torch.isfinite(out).all())


def test_bad_indices_set_the_status():
    c = Case([3, 2], [40, 30], [9, 8, 7, 6, 5], 4, 2, 64, (F16, BF16), 23)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = c(status=status)
    assert status.item() == 0
    for what, i, value in (("groups", 1, 99), ("groups", 1, -1), ("groups", 2, 10 ** 6), ("groups", 2, -3), ("groups", 0, 2), ("items", 0, 50), ("items", 1, -2),
                           ("items", 2, 10 ** 6)):
        t = getattr(c, what)[i]
        old = t[0].clone()
        t[0] = value
        status.zero_()
        out = c(status=status)
        assert status.item() == 4, (what, i, value)
        t[0] = old
        assert torch.equal(out[3:], want[3:])        # the other group's items have theirs
    status.zero_()
    assert torch.equal(c(status=status), want) and status.item() == 0
    c(max_group=2, status=status)                    # a group of three
    assert status.item() == 4


def test_refusals():
    c = small((F16, BF16), 4, 2, 64, 24)
    n = c.q.shape[0]
    g, it = c.groups, c.items
    bad = [
        lambda: prefix_attention(c.q, c.k, c.v),                                             # nothing to attend
        lambda: prefix_attention(c.q[0], c.k, c.v, *g, *it),
        lambda: prefix_attention(c.q[:1].expand(n, -1, -1), c.k, c.v, *g, *it),              # one item's queries for all
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, max_own=2 ** 31),
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, scale=1e39),
        lambda: prefix_attention(c.q, c.k, c.v[:, :, :-1], *g, *it),
        lambda: prefix_attention(c.q, c.k.transpose(0, 1), c.v.transpose(0, 1), *g, *it),
        lambda: prefix_attention(c.q, c.k.cpu(), c.v, *g, *it),
        lambda: prefix_attention(c.q.double(), c.k, c.v, *g, *it),
        lambda: prefix_attention(c.q.bfloat16(), c.k.half(), c.v.half(), *g, *it),           # formats that do not go together
        lambda: prefix_attention(c.q.float(), c.k, c.v, *g, *it),
        lambda: prefix_attention(c.q, c.k, c.v.half(), *g, *it),
        lambda: prefix_attention(c.q[:, :3], c.k, c.v, *g, *it),                             # heads
        lambda: prefix_attention(c.q.transpose(1, 2).contiguous().transpose(1, 2), c.k, c.v, *g, *it),
        lambda: prefix_attention(c.q[..., :32].contiguous(), c.k[..., :32].contiguous(), c.v[..., :32].contiguous(), *g, *it),
        lambda: prefix_attention(c.q, c.k, c.v, g[0].long(), g[1], g[2], *it),
        lambda: prefix_attention(c.q, c.k, c.v, g[0], g[1][:-1], g[2], *it),
        lambda: prefix_attention(c.q, c.k, c.v, g[0], None, g[2], *it),
        lambda: prefix_attention(c.q, c.k, c.v, g[0][:1], g[1], g[2], *it),
        lambda: prefix_attention(c.q, c.k, c.v, *g, it[0], it[1], it[2][:-1]),
        lambda: prefix_attention(c.q, c.k, c.v, *g, it[0].cpu(), it[1], it[2]),
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, skip=torch.zeros(n, device="cuda")),
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, out=torch.empty((n, 4, 64), device="cuda")),
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, scale=math.inf),
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, scale=math.nan),
        lambda: prefix_attention(c.q, c.k, c.v, *g, *it, max_own=-1),
        lambda: prefix_attention(torch.empty(n * 256 + 4, device="cuda", dtype=F16)[4:].view(n, 4, 64), c.k, c.v, *g, *it),      # 8 bytes off
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, _lib.ArcbError)):
            call()
            pytest.fail(f"call {i} was accepted")
    empty = prefix_attention(c.q[:0], c.k, c.v, *g, it[0][:0], it[1][:0], it[2][:0])
    assert empty.shape == (0, 4, 64)
