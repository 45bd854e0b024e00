"""Sessions whose rows share a prompt: what they refuse, and where sharing is by copies."""
import numpy as np
import pytest
import torch

from gpu_util import have_b200
from mdlarc_scale_b200 import _lib
from mdlarc_scale_b200.inference import generate_tokens
from test_gpu_step_cluster import batch, engine

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not have_b200(), reason="needs a B200")]


def test_a_number_of_splits_is_refused_not_ignored():
    eng = engine(128, 64, 1)
    ids, pos, mask, ex = batch(2, [5, 9])
    for splits in (1, 4):
        with pytest.raises(_lib.ArcbError):
            eng.new_session(4, 32, 4, 64, prefix_group=2, attn_splits=splits)
        with pytest.raises(_lib.ArcbError):
            generate_tokens(eng, ids, pos, mask, ex, 4, samples=2, attn_splits=splits)
        eng.new_session(4, 32, 4, 64, prefix_group=1, attn_splits=splits).close()
        generate_tokens(eng, ids, pos, mask, ex, 4, attn_splits=splits)
    eng.new_session(4, 32, 4, 64, prefix_group=2).close()
    eng.close()


def test_groups_of_one_are_no_groups():
    """prefix_group 0 and 1 say the same: every row holds its prompt."""
    eng = engine(128, 64, 1)
    ids, pos, mask, ex = batch(2, [5, 9])
    tokens = []
    for group in (0, 1):
        session = eng.new_session(2, 32, 4, 64, stop_on_end=False, prefix_group=group)
        tokens.append(generate_tokens(eng, ids, pos, mask, ex, 4, stop_on_end=False, session=session).tokens.clone())
        with pytest.raises(ValueError):
            generate_tokens(eng, ids[:1], pos[:1], mask[:1], ex[:1], 4, samples=2, session=session)
        session.close()
    assert torch.equal(*tokens)
    session = eng.new_session(2, 32, 4, 64, prefix_group=2)
    with pytest.raises(ValueError):
        generate_tokens(eng, ids, pos, mask, ex, 4, session=session)
    session.close()
    eng.close()


# models whose steps run in one cluster with so few rows, and ones whose do not
@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("prompts,samples", [(1, 2), (1, 3), (1, 4), (2, 2), (2, 3)])
@pytest.mark.parametrize("d,dff,layers", [(128, 192, 3), (256, 704, 4), (512, 1024, 1)])
def test_few_rows_of_the_smallest_models_keep_their_steps(d, dff, layers, prompts, samples, act):
    """Samples take the steps that as many prompts would: sharing costs no launches."""
    eng = engine(d, dff, layers, act, seed=samples)
    ids, pos, mask, ex = batch(prompts, [130, 33], seed=d)
    rows, new = prompts * samples, 30
    forced = np.random.default_rng(1).integers(0, 12, (rows, new)).astype(np.int32)
    kw = dict(stop_on_end=False, forced=forced, want_logits=True)
    lib, counts, logits = _lib.load(), [], []
    every = [np.repeat(a, samples, 0) for a in (ids, pos, mask, ex)]
    session = eng.new_session(rows, 130 + new, new, 300, forced=torch.from_numpy(forced), want_step_logits=True, stop_on_end=False, prefix_group=samples)
    for call in (lambda: generate_tokens(eng, ids, pos, mask, ex, new, samples=samples, **kw), lambda: generate_tokens(eng, *every, new, **kw),
                 lambda: generate_tokens(eng, ids, pos, mask, ex, new, samples=samples, session=session, **kw)):
        lib.arcb_launch_count(1)
        out = call()
        counts.append(lib.arcb_launch_count(1))
        logits.append(out.step_logits)
        assert torch.equal(out.first_logits, out.first_logits[::samples].repeat_interleave(samples, 0)) and bool(torch.isfinite(out.step_logits).all())
    fits = rows <= 4 and d < 512
    assert (eng.step_ctas(rows, 130 + new) > 0) == fits
    # the copies of a prompt are one launch; a session that shares steps launch by launch
    assert counts[0] <= counts[1] + prompts and counts[2] > counts[0] + new if fits else counts[0] == counts[2]
    # rows round at the same places; sums in another order turn a rounding (2^-11, bf16 2^-8) over here and there
    scale = logits[1].square().mean().sqrt()
    for other in (logits[0], logits[2]):
        assert float((other - logits[1]).square().mean().sqrt() / scale) < (2 ** -9 if act == "f16" else 2 ** -6)
    session.close()
    eng.close()
