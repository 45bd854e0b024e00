"""Copies of rows between the sequences of a cache, to the bit, against indexing on the host."""
import numpy as np
import pytest
import torch

from gpu_util import have_b200
from mdlarc_scale_b200 import _lib, copy_cache_rows

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not have_b200(), reason="needs a B200")]


def bits(shape, dtype, seed):
    """Any bit pattern, NaN among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    raw = torch.randint(-2 ** 15, 2 ** 15, shape, device="cuda", dtype=torch.int16, generator=g)
    return raw.view(dtype) if dtype != torch.float32 else torch.stack([raw, raw.flip(0)], -1).view(torch.float32).squeeze(-1)


def as_int(t):
    return t.view({2: torch.int16, 4: torch.int32, 1: torch.int8}[t.element_size()])


def wanted(cache, copies):
    old = as_int(cache).cpu().numpy()
    new = old.copy()
    for s, d, b, e in np.asarray(copies).reshape(-1, 4).tolist():
        new[..., d, :, b:e, :] = old[..., s, :, b:e, :]
    return new


def check(cache, copies):
    want = wanted(cache, copies)
    copy_cache_rows(cache, copies)
    assert np.array_equal(as_int(cache).cpu().numpy(), want)


SHAPES = [((2, 3, 1, 16, 64), torch.bfloat16), ((3, 7, 5, 33, 128), torch.float16), ((2, 4, 2, 40, 64), torch.float32),
          ((5, 2, 9, 6), torch.bfloat16), ((1, 3, 3, 7, 2), torch.float16), ((4, 6, 1, 19, 5), torch.float32), ((1, 1, 1, 1, 8), torch.float16)]


@pytest.mark.parametrize("shape,dtype", SHAPES)
def test_single_rows_and_whole_sequences(shape, dtype):
    seqs, rows = shape[-4], shape[-2]
    for i, (b, e) in enumerate([(0, rows), (0, 1), (rows - 1, rows), (rows // 2, rows // 2), (rows // 3, rows)]):
        check(bits(shape, dtype, i), [(seqs - 1, 0, b, e)])


@pytest.mark.parametrize("shape,dtype", SHAPES[:3])
def test_fork(shape, dtype):
    seqs, rows = shape[-4], shape[-2]
    check(bits(shape, dtype, 1), [(1, d, d % rows, rows) for d in range(seqs) if d != 1])


def test_swap_rotation_and_chain():
    check(bits((2, 4, 2, 21, 64), torch.bfloat16, 1), [(0, 1, 0, 21), (1, 0, 0, 21)])
    check(bits((2, 4, 2, 21, 64), torch.bfloat16, 2), [(0, 1, 3, 17), (1, 2, 0, 9), (2, 0, 5, 21), (1, 3, 20, 21)])
    check(bits((2, 4, 2, 21, 64), torch.bfloat16, 3), [(0, 1, 0, 21), (1, 2, 0, 21), (2, 3, 0, 21)])


@pytest.mark.parametrize("seed", range(12))
def test_random(seed):
    g = np.random.default_rng(seed)
    seqs, rows = int(g.integers(2, 60)), int(g.integers(1, 90))
    copies = []
    for d in g.permutation(seqs)[:int(g.integers(1, seqs + 1))]:
        b = int(g.integers(0, rows + 1))
        copies.append((int(g.integers(0, seqs)), int(d), b, int(g.integers(b, rows + 1))))
    check(bits((2, seqs, 3, rows, 64), torch.bfloat16, seed), np.array(copies))


def test_many_sequences():
    """More steps than one launch's parameters hold, forks, chains and a long cycle."""
    seqs = 1300
    check(bits((1, seqs, 1, 2, 8), torch.float16, 0), [(0, d, 0, 2) for d in range(1, seqs)])
    check(bits((2, seqs, 1, 2, 8), torch.float16, 1), [(d + 1, d, 0, 2) for d in range(seqs - 1)])
    check(bits((2, seqs, 1, 2, 8), torch.float16, 2), [(d, (d + 1) % 700, 0, 2) for d in range(700)] + [(d, d + 900, 0, 1) for d in range(300)])


def test_offsets_beyond_32_bits():
    """A cache of 9 GB: rows of its last sequence go to the first, and back."""
    cache = torch.zeros((1, 3, 1, 1536 * 1024 - 16, 1024), device="cuda", dtype=torch.int16)
    rows = cache.shape[3]
    tail = torch.randint(-2 ** 15, 2 ** 15, (40, 1024), device="cuda", dtype=torch.int16)
    cache[0, 2, 0, rows - 40:] = tail
    copy_cache_rows(cache, [(2, 0, rows - 40, rows)])
    copy_cache_rows(cache, [(0, 1, rows - 41, rows)])
    assert torch.equal(cache[0, 0, 0, rows - 40:], tail) and torch.equal(cache[0, 1, 0, rows - 40:], tail)
    assert not cache[0, 0, 0, :rows - 40].any() and not cache[0, 1, 0, :rows - 40].any()


def test_streams_graphs_and_changed_lists():
    cache = bits((2, 5, 2, 30, 64), torch.bfloat16, 5)
    copies = np.array([[0, 1, 0, 30], [1, 2, 0, 30]], np.int32)
    want = wanted(cache, copies)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        copy_cache_rows(cache, copies)
        copies[:] = 0                                   # read before the call returns
    side.synchronize()
    assert np.array_equal(as_int(cache).cpu().numpy(), want)
    # two captured calls, replayed in the other order, an eager one between
    graphs, lists = [], [[(0, 1, 0, 30), (1, 0, 0, 30)], [(3, 4, 0, 10)]]
    for c in lists:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            copy_cache_rows(cache, c)
        graphs.append(graph)
    for step in ([(3, 4, 0, 10)], [(2, 3, 0, 30)], [(0, 1, 0, 30), (1, 0, 0, 30)], [(3, 4, 0, 10)]):
        want = wanted(cache, step)
        graphs[lists.index(step)].replay() if step in lists else copy_cache_rows(cache, step)
        torch.cuda.synchronize()
        assert np.array_equal(as_int(cache).cpu().numpy(), want)


def test_nothing_to_do():
    cache = bits((2, 5, 2, 30, 64), torch.bfloat16, 5)
    before = as_int(cache).clone()
    for copies in ([], np.zeros((0, 4), np.int64), [(1, 1, 0, 30)], [(0, 1, 4, 4)]):
        copy_cache_rows(cache, copies)
    assert torch.equal(as_int(cache), before)


def test_refusals_leave_the_cache():
    cache = bits((2, 5, 2, 30, 64), torch.bfloat16, 5)
    before = as_int(cache).clone()
    for bad in ([(0, 5, 0, 1)], [(-1, 0, 0, 1)], [(0, 1, 0, 31)], [(0, 1, 3, 2)], [(0, 1, 0, 1), (2, 1, 0, 1)], [(0, 1, -2, 3)],
                [(d, (d + 1) % 5, 0, 2) for d in range(5)] + [(0, 2, 0, 1)]):
        with pytest.raises((ValueError, _lib.ArcbError)):
            copy_cache_rows(cache, bad)
    for bad in ([(0, 1, 0)], [(0.0, 1.0, 0.0, 2.0)], [0, 1, 0, 2], np.array([[2 ** 40, 0, 0, 1]])):
        with pytest.raises(ValueError):
            copy_cache_rows(cache, bad)
    with pytest.raises(ValueError):
        copy_cache_rows(cache.transpose(0, 1), [(0, 1, 0, 1)])
    with pytest.raises(ValueError):
        copy_cache_rows(cache[0, 0], [(0, 1, 0, 1)])
    with pytest.raises(_lib.ArcbError):       # rows that are no multiple of 4 bytes
        copy_cache_rows(torch.zeros((1, 2, 1, 4, 3), device="cuda", dtype=torch.float16), [(0, 1, 0, 1)])
    torch.cuda.synchronize()
    assert torch.equal(as_int(cache), before)
