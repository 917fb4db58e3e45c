"""The planner's memory fit with 8-bit pools and with readouts under the whole vocabulary, on the host: what a pass
allocates beside its activations and pools is part of what has to fit."""
import ctypes

import numpy as np
import pytest
import torch

from kv8_cases import make_segments
from morj_b200 import _native as nat
from morj_b200 import kv8
from morj_b200.lean_core import KINDS, LeanGemma4, Request
from morj_b200.tree import Tree


def model(**kw):
    m = LeanGemma4.__new__(LeanGemma4)
    m.free_bytes, m.step_tokens, m.single_max, m.act_bytes, m.window = 2**34, 8192, 16384, 2000, 256
    m.geom = {'sliding_attention': (16, 128), 'full_attention': (16, 128)}
    m.types = ['sliding_attention', 'full_attention']
    m.hq, m.hidden, m.kv8 = 32, 512, True
    m.kv_bytes = sum(2 * h * d + 1 for h, d in m.geom.values())
    m.retain_budget, m.shared, m.device = 10 * 2**30, None, torch.device('cpu')
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def workspace(m, st, kind):
    """What the step's attention calls of a layer kind allocate."""
    kk = KINDS[kind]
    window = m.window if kk == 's' else 0
    _, counts = nat.kv8_attention_work(st['qo_indptr'], st['kv_indptr_' + kk], st['kv_indices_' + kk], 0, m.hq,
                                       m.geom[kind][0], window)
    return nat.kv8_attention_workspace(counts, *m.geom[kind])


@pytest.mark.parametrize('hq,hk,d', [(32, 16, 128), (4, 2, 64), (64, 1, 128), (6, 3, 64)])
def test_no_plan_needs_more_workspace_than_the_bound(hq, hk, d):
    rng = np.random.default_rng(hq)
    for _ in range(60):
        spec = []
        for _ in range(rng.integers(1, 9)):
            n = int(np.exp(rng.uniform(0, 7)))
            spec.append((n, max(n, int(np.exp(rng.uniform(0, 9.5))))))
        if rng.random() < 0.5:
            qo, kv, indices, _, _ = make_segments(rng, spec, 1)
        else:  # a shared prefix: listed by every segment, expanded once
            prefix = min(k - n for n, k in spec)
            at = np.cumsum([prefix] + [k - prefix for _, k in spec])
            lists = [np.concatenate([np.arange(prefix), np.arange(a, b)]) for a, b in zip(at[:-1], at[1:])]
            qo = np.concatenate([[0], np.cumsum([n for n, _ in spec])])
            kv, indices = np.concatenate([[0], np.cumsum([len(x) for x in lists])]), np.concatenate(lists)
        _, counts = nat.kv8_attention_work(qo, kv, indices, 0, hq, hk, int(rng.choice([0, 300])))
        most = kv8.attention_workspace_bound(len(set(indices.tolist())), hk, d, sms=148)
        assert nat.kv8_attention_workspace(counts, hk, d) <= most


def test_a_pass_over_8_bit_pools_is_cut_or_refused_when_its_workspace_does_not_fit():
    req = Request(Tree([list(range(1, 3000)) + [5], list(range(1, 3000)) + [6]]), [[0], [0]], False, [])
    seen = set()
    for available in (10_000_000, 20_000_000, 40_000_000, 60_000_000, 80_000_000):
        m = model()
        try:
            _, _, _, plan = m.plan(req, [0, 1], available=available)
        except MemoryError:
            seen.add('refused')
            continue
        steps = plan['steps']
        pools = sum(m._pool_bytes(t, plan['cap'][KINDS[t]]) for t in m.types) if len(steps) > 1 else 0
        most = max(workspace(m, st, t) for st in steps for t in m.types)
        assert pools + max(len(st['tokens']) for st in steps) * m.act_bytes + most <= available
        seen.add('whole' if len(steps) == 1 else 'steps')
    assert 'refused' in seen and 'whole' in seen


def test_bf16_pools_and_the_label_head_are_fitted_as_before():
    req = Request(Tree([list(range(1, 3000))]), [[0]], False, [])
    m = model(kv8=False, act_bytes=1000)
    _, _, _, plan = m.plan(req, [0], available=2999 * 1000)
    assert len(plan['steps']) == 1
    assert m._pass_bytes(plan, False) == 2999 * 1000
    assert m._retention(3000, True, 3000 * (1000 + m.kv_bytes)) == (True, False)


def logprobs_workspace(n, top):
    b = ctypes.c_ulonglong(0)
    nat.call('morj_token_logprobs_workspace', n, top, ctypes.byref(b))
    return b.value


@pytest.mark.parametrize('use8', [False, True])
def test_a_readout_under_the_whole_vocabulary_is_part_of_the_fit(use8):
    req = Request(Tree([list(range(1, 3000))]), [[0]], False, [])
    m = model(kv8=use8, act_bytes=1000)
    H = m.hidden
    for top in (0, 5):
        # the scored rows' residuals live through the steps, their two copies and the workspace come after them
        readout = 2 * 2998 * H + 2 * 2998 * 2 * H + logprobs_workspace(2998, top)
        with pytest.raises(MemoryError):
            m.plan(req, [0], available=readout, vocab=(2998, top))
        _, _, _, plan = m.plan(req, [0], available=readout + 2**20 if not use8 else 2**30, vocab=(2998, top))
        assert len(plan['steps']) == 1
    # the engine's calls say so
    asked = []
    m.plan = lambda req, seqs, available=None, vocab=None: asked.append(vocab) or 1 / 0
    m.embed = torch.empty(4096, 1)
    req.label_ids = [[0]]
    for call, want in [(lambda: m.token_logprobs(req, [0], top=3), (2998, 3)),
                       (lambda: m.token_logprobs(req, [0], start=[2900]), (99, 0)),
                       (lambda: m.label_logprobs(req, [0, 0], top=2), (2, 2)), (lambda: m.run(req, [0]), None)]:
        with pytest.raises(ZeroDivisionError):
            call()
        assert asked.pop() == want


def test_a_sequence_asked_for_many_times_is_read_as_often():
    req = Request(Tree([[1, 2, 3]]), [[0]], False, [])
    m = model(kv8=False, act_bytes=10)
    need = 2 * 500 * m.hidden + 4 * 500 * m.hidden + logprobs_workspace(500, 4)
    with pytest.raises(MemoryError):
        m.plan(req, [0] * 500, available=need, vocab=(500, 4))
    m.plan(req, [0] * 500, available=need + 2**16, vocab=(500, 4))


def test_retained_8_bit_requests_leave_room_for_the_workspace():
    m = model(act_bytes=1000)
    pools, act = 3000 * m.kv_bytes, 3000 * m.act_bytes
    assert m._retention(3000, True, pools + act) == (False, True)
    assert m._retention(3000, True, pools + act + 3000 * 4 * 16 * 128 + 2**25) == (True, False)
