"""Weights of attention over shared cached rows keep both of their 16-bit pieces, in every kernel.

Half of the rows have the largest score, the others one whose weight lies between two values of the cache's type; values are +1 and -1/2
times a column's factor, so that the two halves cancel but for what one piece alone would lose: an output of 0.27 half steps, where a
kernel that rounds weights to one piece gives 0.  Every key stands in three values of decreasing size, so that scores are exact to 2^-20.

Tolerance: u |o| for the output, and in parts of A = sum_t p_t |v_t|: half a step of the type squared for a weight in two pieces (bfloat16
2^-16, half 2^-22), twice (dim + 4) 2^-23 S for scores of size S (numerator and denominator), (rows + 128) 2^-23 for the sums and joins.  Half
pieces end at 2^-24, so that each is off by 2^-25 of the reference at most, which is never above the largest weight: 2^-25 max_t p_t
sum_t |v_t|.
"""
import math

import numpy as np
import pytest
import torch

from gpu_util import have_b200
from mdlarc_scale_b200 import prefix_attention

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not have_b200(), reason="needs a B200")]
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
FORMS = [(F16, BF16), (BF16, BF16), (F16, F16), (F32, F32)]
FORM_IDS = ["f16-bf16", "bf16", "f16", "f32"]
# items, heads, key heads, shared rows that the work is laid out for
SHAPES = [(2, 2, 2, 64), (3, 4, 4, 600), (8, 1, 1, 600), (4, 4, 1, 600), (16, 2, 2, 600), (5, 6, 2, 600), (20, 3, 3, 600), (8, 8, 2, 600), (33, 1, 1, 600),
          (64, 2, 2, 600), (70, 1, 1, 4000), (128, 2, 2, 4000), (40, 8, 2, 4000), (300, 1, 1, 4000)]


def ints(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def keys(scores, dim, kind):
    """Rows whose products with a query of ones are `scores`, to three pieces of the type."""
    k = torch.zeros((len(scores), dim), dtype=torch.float64)
    left = torch.as_tensor(scores, dtype=torch.float64)
    for d in (1, dim // 2, dim - 2):
        k[:, d] = left.to(kind).double()
        left = left - k[:, d]
    return k.to(kind).cuda()


def reference(q, k, v, scale):
    """Of queries [heads, dim] over rows [rows, dim] in 64 bits: result, sum of p |v|, size of the scores, max p sum |v|."""
    q, k, v = q.double(), k.double(), v.double()
    p = torch.softmax(q @ k.T * scale, -1)
    return p @ v, p @ v.abs(), (q.abs() @ k.abs().T).amax(-1, keepdim=True) * scale, p.amax(-1, keepdim=True) * v.abs().sum(0)


def tolerance(form, rows, dim, want, spread, size, floor, least=0):
    u = torch.finfo(form[0]).eps / 2
    two = {BF16: 2.0 ** -16, F16: 2.0 ** -22, F32: 0.0}[form[1]]
    small = 2.0 ** (-25 - least) if form[1] == F16 else 0.0
    return u * want.abs() + (two + 2 * (dim + 4) * 2.0 ** -23 * size + (rows + 128) * 2.0 ** -23) * spread + small * floor + 2.0 ** -30


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("items,heads,kv,plan", SHAPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_no_weight_loses_its_second_piece(form, items, heads, kv, plan, dim):
    half_step = torch.finfo(form[1] if form[1] != F32 else F16).eps / 2
    shared, own, pitch = 70, 6, 4112
    scale = dim ** -0.5
    score = math.log(0.5 * (1 + 0.9 * half_step)) / scale
    pattern = np.where(np.arange(pitch) % 2, 0.0, score)
    k = keys(pattern, dim, form[1])[None, None].expand(2, kv, -1, -1).contiguous()
    factor = torch.tensor([(-1.0) ** j * 2.0 ** (j % 3) for j in range(dim)])
    v = torch.from_numpy(np.where(np.arange(pitch) % 2, -0.5, 1.0))[:, None] * factor
    v = v.to(form[1]).cuda()[None, None].expand(2, kv, -1, -1).contiguous()
    q = torch.ones((items, heads, dim), device="cuda", dtype=form[0])
    hints = dict(max_group=items, max_prefix=plan, max_own=own)
    got = prefix_attention(q, k, v, ints([0, items]), ints([1]), ints([shared]), ints([0] * items), ints([2] * items), ints([2 + own] * items), **hints)
    rows = torch.cat([torch.arange(shared), torch.arange(2, 2 + own)]).cuda()
    want, spread, size, floor = reference(q[0], k[0, 0, rows], v[0, 0, rows], scale)
    tol = tolerance(form, shared + own, dim, want, spread, size, floor)
    assert bool((want.abs() > 2 * tol).all())          # one piece alone is told from two
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("items,heads,kv,plan", SHAPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_many_small_weights_beside_large_ones(form, items, heads, kv, plan, dim):
    """Every 50th row has the largest score and a value of 0, all others 2^-25.5 of its weight: the result is theirs alone.  A half cache's
    weights are kept down to 2^-28 of a range's largest one."""
    shared, own, pitch = 3011, 9, 4112
    scale = dim ** -0.5
    large = np.arange(pitch) % 50 == 7
    k = keys(np.where(large, 0.0, -25.5 * math.log(2) / scale), dim, form[1])[None, None].expand(1, kv, -1, -1).contiguous()
    v = torch.from_numpy(np.where(large, 0.0, 256.0))[:, None] * torch.tensor([2.0 ** (j % 3) for j in range(dim)])
    v = v.to(form[1]).cuda()[None, None].expand(1, kv, -1, -1).contiguous()
    q = torch.ones((items, heads, dim), device="cuda", dtype=form[0])
    hints = dict(max_group=items, max_prefix=plan, max_own=own)
    got = prefix_attention(q, k, v, ints([0, items]), ints([0]), ints([shared]), ints([0] * items), ints([0] * items), ints([own] * items), **hints)
    rows = torch.cat([torch.arange(shared), torch.arange(own)]).cuda()
    want, spread, size, floor = reference(q[0], k[0, 0, rows], v[0, 0, rows], scale)
    tol = tolerance(form, shared + own, dim, want, spread, size, floor, least=3)
    assert bool((want > 3 * tol).all())
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance"
