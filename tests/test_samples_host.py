"""Several continuations of a prompt: scheduling on a session without a GPU, refusals, and the layout of the operators' arguments."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from mdlarc_scale_b200 import _lib, prefix
from mdlarc_scale_b200.engine import plan_prefill
from mdlarc_scale_b200.generation import Request, Scheduler, generate
from test_vodavik_host import _CpuEngine, _CpuSession, _Lens

ROOT = Path(__file__).resolve().parent.parent


class _Session(_CpuSession):
    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.prefilled, self.forks = [], []

    def prefill_segments(self, segments):
        assert sum(len(s.tokens) for s in segments) <= self.max_prefill_tokens
        self.prefilled += [(s.slot, [int(t) for t in s.tokens]) for s in segments]
        super().prefill_segments(segments)

    def fork(self, slot, targets):
        assert slot not in self.free and not set(targets) & set(self.free)
        self.forks.append((slot, list(targets)))
        for t in targets:
            self.fed[t], self.lens[t] = list(self.fed[slot]), self.lens[slot]


class _Engine(_CpuEngine):
    def new_session(self, n_slots, t_max, max_new, max_prefill_tokens, **kw):
        self.session = _Session(n_slots, t_max, max_new, max_prefill_tokens, **kw)
        self.session.lens = _Lens(self.session)
        return self.session


@pytest.mark.parametrize("max_batch", [3, 4, 64])
@pytest.mark.parametrize("samples", [1, 2, 3, 7])
@pytest.mark.parametrize("end", [None, 40])
def test_samples_prefill_a_prompt_once(max_batch, samples, end):
    prompts = [[1, 2, 36], [7], list(range(30)) + [38], [3, 4]]
    engine = _Engine()
    out, logits = generate(engine, prompts, 9, end_token=end, max_batch=max_batch, prefill_tokens=16, return_logits=True, samples=samples)
    assert len(out) == len(prompts) * samples
    for i, row in enumerate(out):
        last = prompts[i // samples][-1]
        want = list(range(last, last + 9))
        if end in want:
            want = want[:want.index(end) + 1]
        assert row == want and logits[i][:, 0].tolist() == want
    session = engine.session
    # every continuation has its own random stream and has been fed the whole prompt
    assert sorted(session.streams) == sorted((prompts[i // samples], i) for i in range(len(out)))
    # the prompt but its last token once for as many samples as run together
    families = -(-samples // max_batch)
    for p in prompts:
        assert sum(len(t) for _, t in session.prefilled) == sum(families * (len(q) - 1) + samples for q in prompts)
    sizes = [min(max_batch, samples - j) for j in range(0, samples, max_batch)]
    assert sorted(len(t) for _, t in session.forks) == sorted(n - 1 for n in sizes for p in prompts if n > 1 and len(p) > 1)


def test_samples_of_one_are_what_they_were():
    prompts = [[1, 2, 36], [5] * 30 + [38]]
    a, b = _Engine(), _Engine()
    assert generate(a, prompts, 9, prefill_tokens=16) == generate(b, prompts, 9, prefill_tokens=16, samples=1)
    assert a.session.prefilled == b.session.prefilled and not a.session.forks


def test_refusals():
    with pytest.raises(ValueError):
        generate(_Engine(), [[1, 2]], 3, samples=0)
    sched = Scheduler(_Engine(), 3, 100, 2)
    with pytest.raises(ValueError):
        sched.submit_samples([Request(i, [1, 2]) for i in range(3)])
    with pytest.raises(ValueError):
        sched.submit_samples([Request(i, []) for i in range(2)])
    assert generate(_Engine(), [[1]], 0, samples=3) == [[], [], []] and generate(_Engine(), [], 4, samples=3) == []


def test_plan_for_samples():
    g = np.random.default_rng(0)
    mask = np.arange(9)[None] < np.array([9, 1, 4])[:, None]
    ids, pos = g.integers(0, 12, (3, 9)), g.integers(0, 5, (3, 9, 3))
    one = plan_prefill(ids, pos, mask, np.array([1, 2]))
    many = one.for_samples(3)
    assert many.n_tokens == one.n_tokens and torch.equal(many.token_ids, one.token_ids) and torch.equal(many.kv_count, one.kv_count)
    assert many.seq.tolist() == [3] + [6] * 4 and many.n_first == 6
    assert many.first_seq.tolist() == [3, 4, 5, 6, 7, 8] and many.first_row.tolist() == [0, 0, 0, 4, 4, 4] and many.prompt_len.tolist() == [1] * 3 + [4] * 3
    assert all(t.dtype == torch.int32 for t in (many.seq, many.first_seq, many.first_row, many.grid_x))


def test_argument_layout_is_the_headers(tmp_path):
    fields = [f for f, _ in _lib.PrefixAttentionArgs._fields_]
    src = '#include "arcb200.h"\n#include <cstddef>\n#include <cstdio>\nint main() { printf("%zu", sizeof(arcb_prefix_attention_args));\n'
    src += "".join(f'printf(" %zu", offsetof(arcb_prefix_attention_args, {f}));\n' for f in fields)
    src += 'printf(" %zu %zu", sizeof(arcb_session_desc), offsetof(arcb_session_desc, prefix_group)); }\n'
    (tmp_path / "p.cpp").write_text(src)
    subprocess.run(["g++", "-I", str(ROOT / "include"), str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()]
    want = [C.sizeof(_lib.PrefixAttentionArgs)] + [getattr(_lib.PrefixAttentionArgs, f).offset for f in fields]
    assert got == want + [C.sizeof(_lib.SessionDesc), _lib.SessionDesc.prefix_group.offset]
    values = [0.5 if f == "scale" else 3 + i for i, f in enumerate(fields)]
    packed = _lib.PrefixAttentionArgs.from_buffer_copy(prefix._ARGS.pack(*values))
    assert prefix._ARGS.size == want[0] and [getattr(packed, f) for f in fields] == values


@pytest.fixture(scope="module")
def lib():
    from mdlarc_scale_b200 import build
    build.build()
    return _lib.load()


def prefix_args(**kw):
    base = dict(n_groups=2, n_items=5, n_heads=4, n_kv=2, dim=64, n_seqs=7, t_max=100, scale=0.125, act_format=_lib.ACT_F16, kv_format=_lib.ACT_BF16,
                d_q=4096, d_k=4096, d_v=4096, d_out=4096, d_group_first=4096, d_group_seq=4096, d_group_len=4096, d_item_end=4096)
    base.update(kw)
    return _lib.PrefixAttentionArgs(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(n_items=0), _lib.E_ARG), (dict(n_groups=-1), _lib.E_ARG), (dict(n_kv=3), _lib.E_ARG), (dict(dim=96), _lib.E_UNSUPPORTED),
    (dict(act_format=_lib.ACT_BF16, kv_format=_lib.ACT_F16), _lib.E_UNSUPPORTED), (dict(act_format=_lib.ACT_F32), _lib.E_UNSUPPORTED),
    (dict(kv_format=_lib.ACT_F32), _lib.E_UNSUPPORTED), (dict(act_format=3), _lib.E_ARG), (dict(kv_format=-1), _lib.E_ARG), (dict(t_max=0), _lib.E_ARG),
    (dict(n_groups=0, d_item_end=None), _lib.E_ARG), (dict(scale=float("nan")), _lib.E_ARG), (dict(n_seqs=1 << 20, t_max=1 << 12), _lib.E_UNSUPPORTED),
    (dict(d_q=None), _lib.E_ARG), (dict(d_group_len=None), _lib.E_ARG), (dict(d_k=4100), _lib.E_ARG), (dict(d_out=4104), _lib.E_ARG),
    (dict(q_pitch=257), _lib.E_ARG), (dict(q_pitch=-256), _lib.E_ARG), (dict(), _lib.E_ARG)])
def test_prefix_attention_refuses(lib, kw, code):
    """Without a GPU: everything that is refused is refused ahead of the first launch (the last one for want of scratch)."""
    a = prefix_args(**kw)
    assert lib.arcb_op_prefix_attention(C.byref(a), None) == code
    assert lib.arcb_last_error()
    assert lib.arcb_op_prefix_attention(None, None) == _lib.E_ARG


@pytest.mark.parametrize("kw", [dict(d_cache=None), dict(n_planes=0), dict(n_seqs=0), dict(t_max=0), dict(row_bytes=0), dict(row_bytes=6), dict(d_cache=4098),
                                dict(n_copies=-1), dict(copies=[[0, 5, 0, 1]]), dict(copies=[[0, 1, 0, 11]]), dict(copies=[[0, 1, 5, 4]]), dict(copies=[[-1, 1, 0, 1]]),
                                dict(copies=[[0, 1, 0, 1], [2, 1, 4, 5]])])
def test_cache_copy_refuses(lib, kw):
    base = dict(d_cache=4096, n_planes=2, n_seqs=5, n_heads=3, t_max=10, row_bytes=128, copies=[[0, 1, 0, 1]])
    base.update(kw)
    m = np.ascontiguousarray(base["copies"], np.int32)
    n = base.get("n_copies", len(m))
    rc = lib.arcb_op_cache_copy(base["d_cache"], base["n_planes"], base["n_seqs"], base["n_heads"], base["t_max"], base["row_bytes"], m.ctypes.data, n, None)
    assert rc == _lib.E_ARG
    assert lib.arcb_op_cache_copy(4096, 2, 5, 3, 10, 128, None, 1, None) == _lib.E_ARG
    # nothing to do needs no GPU
    assert lib.arcb_op_cache_copy(4096, 2, 5, 3, 10, 128, None, 0, None) == 0
