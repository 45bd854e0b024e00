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
