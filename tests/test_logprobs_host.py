"""Refusals of the full-vocabulary log-probabilities, on the CPU: a call's arguments are checked before any device
access (16 stands for an aligned pointer that is never read)."""
import ctypes

import pytest
import torch

from morj_b200 import _native as nat
from morj_b200.logprobs import token_logprobs


def args(**kw):
    a = dict(h=16, ld_h=64, n=2, w=16, ld_w=64, vocab=100, H=64, softcap=30.0, targets=16, n_targets=1, logprobs=16,
             lse=16, entropy=16, top=2, top_ids=16, top_logprobs=16, ws=16, nbytes=1 << 40, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('kw,match', [
    (dict(h=None), 'null pointer'), (dict(w=None), 'null pointer'), (dict(n=-1), 'bad size'), (dict(vocab=0), 'bad size'),
    (dict(vocab=2**31 - 1), 'bad size'), (dict(H=0), 'bad size'), (dict(n_targets=-1), 'bad size'),
    (dict(targets=None), 'null pointer'), (dict(logprobs=None), 'null pointer'), (dict(top_ids=None), 'null pointer'),
    (dict(top_logprobs=None), 'null pointer'), (dict(top=-1), 'top'), (dict(top=33), 'top'),
    (dict(top=20, vocab=19), 'top'), (dict(softcap=-1.0), 'softcap'), (dict(softcap=float('nan')), 'softcap'),
    (dict(softcap=float('inf')), 'softcap'), (dict(softcap=1e-35), 'softcap'), (dict(H=60), 'multiples of 8'),
    (dict(ld_h=56), 'multiples of 8'), (dict(ld_w=68), 'multiples of 8'), (dict(h=24), '16-byte'), (dict(w=8), '16-byte'),
    (dict(ws=8), '16-byte'), (dict(ws=None), 'workspace of'), (dict(nbytes=1000), 'needed')])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        nat.call('morj_token_logprobs', *args(**kw))


def test_nothing_to_do_and_workspace_sizes():
    nat.call('morj_token_logprobs', *args(n=0))
    b = ctypes.c_ulonglong(0)
    sizes = []
    for n, top in [(0, 0), (1, 0), (1, 8), (128, 8), (129, 8), (2048, 8), (100000, 8)]:
        nat.call('morj_token_logprobs_workspace', n, top, ctypes.byref(b))
        sizes.append(b.value)
    assert sizes[0] == 0 and sizes[2] == sizes[3] and sizes[4] == 2 * sizes[3] and sizes[5] == sizes[6]
    for bad in [(-1, 0), (1, -1), (1, 33)]:
        with pytest.raises(ValueError):
            nat.call('morj_token_logprobs_workspace', *bad, ctypes.byref(b))
    with pytest.raises(ValueError):
        nat.call('morj_token_logprobs_workspace', 1, 0, None)


def test_tensors_that_are_not_on_a_cuda_device_are_refused():
    # (launched, the kernels would read host addresses)
    h, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='must be on a CUDA device, not on cpu'):
        token_logprobs(h, w, torch.zeros(2, 1, dtype=torch.int32))
