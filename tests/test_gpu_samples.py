"""Several continuations of one prompt: rows of the grid model that share a prompt's keys and values, and forked sequences of layered
models.

Logits of rows that share a prompt against rows that each hold it: the same numbers but for the order of the attention's additions
and, in the cache's bfloat16 beside half queries, weights of 16 bits instead of 24.  Both paths round their results at the same places,
so that a difference turns such a rounding over here and there (half: 2^-11 of a value, bfloat16: 2^-8); the rms of the logits'
difference stays within four of those of the rms of the logits."""
import numpy as np
import pytest
import torch

from gpu_util import have_b200
from mdlarc_scale_b200 import _lib, generate, predict_with_augmentations
from mdlarc_scale_b200.inference import generate_tokens
from mdlarc_scale_b200.layered import Segment
from mdlarc_scale_b200.registry import build_engine
from test_gpu_step_cluster import batch, engine

import logesun_util
import vodavik_util
from oracle import logesun as lo
from oracle import vodavik as vo

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not have_b200(), reason="needs a B200")]


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("prompts,samples", [(1, 2), (3, 4), (2, 9), (1, 17), (2, 33), (1, 70), (5, 8)])
def test_rows_that_share_a_prompt(prompts, samples, act):
    eng = engine(256, 192, 2, act, seed=samples)
    ids, pos, mask, ex = batch(prompts, [300, 1, 129, 64, 7], seed=prompts)
    rows, new = prompts * samples, 21
    forced = np.random.default_rng(1).integers(0, 12, (rows, new)).astype(np.int32)
    kw = dict(stop_on_end=False, forced=forced, want_logits=True)
    shared = generate_tokens(eng, ids, pos, mask, ex, new, samples=samples, **kw)
    apart = generate_tokens(eng, *(np.repeat(a, samples, 0) for a in (ids, pos, mask, ex)), new, attn_splits=1, **kw)
    assert shared.prefill_tokens * samples == apart.prefill_tokens
    assert torch.equal(shared.first_logits, shared.first_logits[::samples].repeat_interleave(samples, 0))
    scale = apart.step_logits.square().mean().sqrt()
    assert bool(torch.isfinite(shared.step_logits).all())
    assert float((shared.step_logits - apart.step_logits).square().mean().sqrt() / scale) < (2 ** -9 if act == "f16" else 2 ** -6)
    eng.close()


def test_greedy_samples_are_equal_and_samples_differ():
    eng = engine(256, 192, 2, seed=3, chain=True)
    ids, pos, mask, ex = batch(3, [200, 31, 64], seed=5)
    a = generate_tokens(eng, ids, pos, mask, ex, 40, samples=6).tokens.view(3, 6, -1)
    assert bool((a == a[:, :1]).all())
    b = generate_tokens(eng, ids, pos, mask, ex, 40, attn_splits=1).tokens
    width = min(a.shape[2], b.shape[1])
    assert torch.equal(a[:, 0, :width], b[:, :width])       # clear choices: every one the successor of a token
    kw = dict(stop_on_end=False, temperature=1.5, sample_seed=7, samples=6)
    s = generate_tokens(eng, ids, pos, mask, ex, 40, **kw).tokens
    assert torch.equal(s, generate_tokens(eng, ids, pos, mask, ex, 40, **kw).tokens)
    # every row draws from its own stream, as it does where it holds its prompt itself
    rows = [np.repeat(v, 6, 0) for v in (ids, pos, mask, ex)]
    assert torch.equal(s, generate_tokens(eng, *rows, 40, attn_splits=1, **{**kw, "samples": 1}).tokens)
    assert len({tuple(r) for r in s.tolist()}) > 3
    eng.close()


def test_rows_that_end_and_rows_that_go_on():
    """Frozen rows beside others of their group, the first row of a group among them."""
    eng = engine(256, 192, 2, seed=3, chain=True)
    ids, pos, mask, ex = batch(2, [150, 40], seed=5)
    kw = dict(temperature=2.0, sample_seed=3, samples=8)
    out = generate_tokens(eng, ids, pos, mask, ex, 60, **kw).tokens.tolist()
    free = generate_tokens(eng, ids, pos, mask, ex, 60, stop_on_end=False, **kw).tokens.tolist()
    ends = set()
    for a, b in zip(out, free):
        n = a.index(13) + 1 if 13 in a else len(a)
        ends.add(n)
        assert a[:n] == b[:n] and all(t == 13 for t in a[n:])
    assert len(ends) > 1            # rows of a group end at different steps
    eng.close()


def test_predictions_share_prompts():
    eng = engine(128, 192, 2, seed=3, chain=True)
    task = {"train": [{"input": [[1, 2], [3, 4]], "output": [[5, 6, 7]]}], "test": [{"input": [[0, 9, 8]]}]}
    kw = dict(num_color_perms=2, max_output_tokens=24, num_samples=3)
    apart = predict_with_augmentations(eng, task, 0, "cuda:0", batched=False, **kw)
    shared = predict_with_augmentations(eng, task, 0, "cuda:0", share_prompts=True, **kw)
    assert len(shared) == 8 * 2 * 3 and shared == apart
    eng.close()


def test_refusals_of_shared_prompts():
    eng = engine(128, 64, 1)
    ids, pos, mask, ex = batch(2, [5, 9])
    with pytest.raises(ValueError):
        generate_tokens(eng, ids, pos, mask, ex, 4, samples=0)
    with pytest.raises(ValueError):
        eng.new_session(7, 32, 4, 64, prefix_group=2)
    session = eng.new_session(4, 32, 4, 64)
    with pytest.raises(ValueError):
        generate_tokens(eng, ids, pos, mask, ex, 4, samples=2, session=session)
    for args in ((-1, 3, [0]), (4, 3, [0]), (0, 49, [1]), (0, -1, [1]), (0, 3, [4]), (0, 3, [1, 1]), (0, 3, [-1])):
        with pytest.raises(_lib.ArcbError):
            session.copy_rows(*args)
    session.close()
    session = eng.new_session(4, 32, 4, 64, prefix_group=2)
    with pytest.raises(_lib.ArcbError):
        session.copy_rows(1, 3, [0])          # row 0 holds the prompt of both
    session.close()
    eng.close()


def test_copied_rows_of_a_grid_session():
    eng = engine(256, 64, 3)
    session = eng.new_session(5, 40, 4, 64)
    cache = session.kv_cache.view(torch.int16)
    cache.copy_(torch.randint(-2 ** 15, 2 ** 15, cache.shape, dtype=torch.int16, device="cuda"))
    view = cache.view(6, 5, 4, session.t_max, 64)
    want = view.clone()
    session.copy_rows(2, 17, [0, 4, 2])
    for t in (0, 4):
        want[:, t, :, :17] = want[:, 2, :, :17]
    assert torch.equal(view, want)
    session.copy_rows(1, 0, [0])
    session.copy_rows(1, 5, [])
    assert torch.equal(view, want)
    session.close()
    eng.close()


CASES = [("vodavik", n) for n in sorted(vodavik_util.CONFIGS)] + [("logesun", n) for n in sorted(logesun_util.CONFIGS)]


@pytest.mark.parametrize("fmt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("family,name", CASES)
def test_forked_sequences_continue_as_prefilled_ones(family, name, fmt):
    """To the bit: what a fork holds is what its source holds, in every kind of layer."""
    util, oracle = (vodavik_util, vo) if family == "vodavik" else (logesun_util, lo)
    cfg = util.CONFIGS[name]
    eng = build_engine(cfg, oracle.random_weights(cfg, 0), "cuda:0", fmt)
    prompt, more = util.tokens(cfg, 75, 1), [util.tokens(cfg, 9, 2 + i) for i in range(3)]
    got = []
    for forked in (False, True):
        session = eng.new_session(5, 120, 1, 128)
        slots = [session.acquire() for _ in range(5)]
        use = [slots[3], slots[0], slots[4]]
        session.step([Segment(slots[1], util.tokens(cfg, 90, 9))])          # somebody else's sequence, and what a target held before
        session.step([Segment(use[2], util.tokens(cfg, 101, 10))])
        session.release(use[2])
        assert session.acquire() == use[2]
        for s in use[:1] if forked else use:
            session.step([Segment(s, prompt)])
        if forked:
            session.fork(use[0], use[1:])
            assert [session.lens[s] for s in use] == [75] * 3
        rows = []
        for t in range(4):
            rows += session.step([Segment(s, m[t:t + 1], [0]) for s, m in zip(use, more)])
        rows += session.step([Segment(s, m[4:], [0, len(m) - 5]) for s, m in zip(use, more)])
        rows += session.step([Segment(slots[1], [5], [0])])
        got.append([r.cpu() for r in rows])
        session.close()
    assert all(torch.equal(a, b) for a, b in zip(*got))
    eng.close()


@pytest.mark.parametrize("family", ["vodavik", "logesun"])
def test_generated_samples(family):
    util, oracle = (vodavik_util, vo) if family == "vodavik" else (logesun_util, lo)
    cfg = util.CONFIGS["mixed"]
    eng = build_engine(cfg, oracle.random_weights(cfg, 0), "cuda:0", "f32")
    prompts = [util.tokens(cfg, n, n) for n in (40, 1, 131)]
    want = generate(eng, [p for p in prompts for _ in range(3)], 12)
    for max_batch in (2, 3, 4, 64):
        assert generate(eng, prompts, 12, samples=3, max_batch=max_batch, prefill_tokens=64) == want
    a, b = (generate(eng, prompts, 12, samples=4, temperature=1.0, seed=5, max_batch=m) for m in (64, 5))
    assert a == b and len({tuple(r) for r in a}) > 8
    eng.close()


def test_fork_refusals():
    cfg = vodavik_util.CONFIGS["single_head"]
    eng = build_engine(cfg, vo.random_weights(cfg, 0), "cuda:0", "f32")
    with pytest.raises(ValueError):
        eng.new_session(4, 64, 4, 64, prefix_group=2)
    session = eng.new_session(4, 64, 4, 64)
    a, b, c = (session.acquire() for _ in range(3))
    session.step([Segment(a, [1, 2, 3])])
    for slot, targets in ((a, [a]), (a, [b, b]), (a, [4]), (a, [-1]), (3 - a - b - c + 3, [a]), (a, [({0, 1, 2, 3} - {a, b, c}).pop()])):
        with pytest.raises(ValueError):
            session.fork(slot, targets)
    assert session.lens[b] == 0
    session.fork(b, [c])                    # nothing held, nothing copied
    session.fork(a, [])
    assert session.lens[c] == 0
    session.close()
    eng.close()
