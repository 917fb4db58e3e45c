"""Log-probabilities of given tokens under the whole vocabulary, with log-sum-exp, entropy and the top alternatives
(`morj_token_logprobs`): the readout beside the label-restricted head. The [rows, vocab] logits are never stored.

`LeanGemma4.token_logprobs` and `LeanGemma4.label_logprobs` call it on the engine's readout rows.
"""
import ctypes
from typing import NamedTuple, Optional

import torch

from . import _native as nat
from .kv8 import _on

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """Per row, FP32: `logprob` of the given tokens [n, targets], `lse`, `entropy` (nats); with top > 0 the ids [n, top]
    (int32, most likely first, the lower id first among equal logits) and log-probabilities of the top alternatives."""
    logprob: torch.Tensor
    lse: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor] = None
    top_logprobs: Optional[torch.Tensor] = None


_bytes = {}  # (rows, top) -> workspace bytes (a pure function of them and the device's SM count)


def workspace_bytes(n, top):
    key = (n, top)
    if key not in _bytes:
        b = ctypes.c_ulonglong(0)
        nat.call('morj_token_logprobs_workspace', n, top, ctypes.byref(b))
        if len(_bytes) > 4096:
            _bytes.clear()
        _bytes[key] = b.value
    return _bytes[key]


def token_logprobs(h, w, targets, top=0, softcap=0.0):
    """`h`: normed rows, BF16 [n, H] (rows any multiple of 8 elements apart); `w`: the vocabulary's rows, BF16 [vocab, H];
    `targets`: int32 [n, targets per row], -1 for none (its log-probability reads 0). Launches on the current stream of
    the tensors' device and waits for nothing."""
    if h.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or h.dim() != 2 or w.dim() != 2 or h.shape[1] != w.shape[1]:
        raise ValueError(f'h and w must be BF16 [rows, H]: {h.dtype} {tuple(h.shape)}, {w.dtype} {tuple(w.shape)}')
    n, H = h.shape
    if targets.dtype != torch.int32 or targets.dim() != 2 or targets.shape[0] != n or not targets.is_contiguous():
        raise ValueError(f'targets must be contiguous int32 [{n}, targets]: {targets.dtype} {tuple(targets.shape)}')
    dev = h.device
    if w.device != dev or targets.device != dev:
        raise ValueError(f'h, w and targets are on {dev}, {w.device}, {targets.device}')
    if not 0 <= top <= min(MAX_TOP, w.shape[0]):
        raise ValueError(f'top {top} must be in [0, {min(MAX_TOP, w.shape[0])}]')
    if (n and h.stride(1) != 1) or w.stride(1) != 1:
        raise ValueError('the elements of a row must be contiguous')
    T = targets.shape[1]
    # one allocation for the outputs (several cost a small call more than its kernels)
    flat = torch.empty(n * (T + 2 + 2 * top), dtype=torch.float32, device=dev)
    logprob, lse, entropy, lps, ids = flat.split_with_sizes((n * T, n, n, n * top, n * top))
    logprob = logprob.view(n, T)
    ids, lps = (ids.view(torch.int32).view(n, top), lps.view(n, top)) if top else (None, None)
    if n:
        nbytes = workspace_bytes(n, top)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with _on(dev) as s:
            nat.call('morj_token_logprobs', h.data_ptr(), h.stride(0) if n > 1 else H, n, w.data_ptr(),
                     w.stride(0) if w.shape[0] > 1 else H, w.shape[0], H, softcap, targets.data_ptr() if T else None, T,
                     logprob.data_ptr() if T else None, lse.data_ptr(), entropy.data_ptr(), top,
                     ids.data_ptr() if top else None, lps.data_ptr() if top else None, ws.data_ptr(), nbytes, s)
    return TokenLogprobs(logprob, lse, entropy, ids, lps)
