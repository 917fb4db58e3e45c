"""The 8-bit K/V cache: e4m3 pools with one power-of-two scale per block of 64 slots and head, the store that fills them
and the tree attention that reads them (`morj_kv8_store`, `morj_kv8_gather`, `morj_tree_attention_kv8`).

A pool takes half the bytes of a BF16 one (0.5 MB instead of 1 MB per token of the 31B model's 60 layers), so twice the
kept requests fit. What a call needs of the host (which rows go to which block; which CTA takes which keys) is planned
once per step from the step's tables and serves every layer:

    pool = KV8Pool(slots, kv_heads, head_dim, device)
    store(pool, k_rows, v_rows, StorePlan(slot_of_row, pool.slots, device))
    out = tree_attention(q, pool, AttentionPlan(qo_indptr, kv_indptr, kv_indices, hq, hk, d, device=device), sm_scale)

Calls launch on the current stream of the pool's device and wait for nothing; the tensors they are given must be usable
on it. `LeanGemma4(kv_cache='e4m3')` keeps its K/V in these pools.
"""
import numpy as np
import torch

from . import _native as nat

BLOCK = 64
CODES = torch.float8_e4m3fn


class _on:
    """The device of a call made the current one while it launches (nothing when it already is). ValueError for tensors
    that are not on a CUDA device: a kernel given their addresses would fault the GPU."""

    def __init__(self, device):
        if device.type != 'cuda':
            raise ValueError(f'the tensors of a launch must be on a CUDA device, not on {device}')
        self.index, self.back = device.index, None

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self.index:
            self.back = now
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.back is not None:
            torch.cuda.set_device(self.back)


def _upload(device, *arrays):
    """int32 arrays, each 16-byte aligned in one device buffer: (buffer, views)."""
    parts, spans, at = [], [], 0
    for a in arrays:
        a = np.ascontiguousarray(a, dtype=np.int32).reshape(-1)
        spans.append((at, len(a)))
        parts += [a, np.zeros(-len(a) % 4, np.int32)]
        at += len(a) + -len(a) % 4
    buf = torch.from_numpy(np.concatenate(parts) if at else np.zeros(4, np.int32)).to(device)
    return buf, [buf[o:o + n] for o, n in spans]


class KV8Pool:
    """K and V of one layer: `k`, `v` codes [slots, heads, head_dim] (torch.float8_e4m3fn), `k_scale`, `v_scale` FP32
    [ceil(slots / 64), heads], zero while nothing is stored in a block."""

    def __init__(self, slots, heads, head_dim, device='cuda'):
        if slots < 0 or heads <= 0 or head_dim not in (64, 128):
            raise ValueError(f'unsupported 8-bit pool: {slots} slots, {heads} heads of {head_dim} (64 or 128)')
        shape, blocks = (max(slots, 1), heads, head_dim), (max(slots, 1) + BLOCK - 1) // BLOCK
        make = lambda: torch.empty(shape, dtype=torch.uint8, device=device).view(CODES)
        self.scales = torch.zeros(2, blocks, heads, device=device)  # (K's and V's, one tensor to clear)
        self._set(make(), self.scales[0], make(), self.scales[1])

    @classmethod
    def of(cls, k, k_scale, v, v_scale):
        """A pool over existing tensors (contiguous; codes as float8_e4m3fn or uint8)."""
        if k.dim() != 3 or v.shape != k.shape or k.shape[2] not in (64, 128) or k.shape[0] < 1:
            raise ValueError(f'codes must be [slots, heads, 64 or 128]: {tuple(k.shape)}, {tuple(v.shape)}')
        want = ((k.shape[0] + BLOCK - 1) // BLOCK, k.shape[1])
        for t in (k_scale, v_scale):
            if tuple(t.shape) != want or t.dtype != torch.float32:
                raise ValueError(f'scales must be FP32 {want}: {tuple(t.shape)} {t.dtype}')
        if any(t.dtype not in (CODES, torch.uint8) for t in (k, v)):
            raise ValueError(f'codes must be float8_e4m3fn or uint8: {k.dtype}, {v.dtype}')
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)) or len({t.device for t in
                                                                               (k, v, k_scale, v_scale)}) != 1:
            raise ValueError('codes and scales must be contiguous and on one device')
        self = cls.__new__(cls)
        self.scales = None
        self._set(k.view(CODES), k_scale, v.view(CODES), v_scale)
        return self

    def _set(self, k, k_scale, v, v_scale):
        self.k, self.k_scale, self.v, self.v_scale = k, k_scale, v, v_scale
        self.slots, self.heads, self.head_dim = k.shape
        self.device = k.device

    def clear(self):
        """Forget what is stored: every block is empty again."""
        if self.scales is not None:
            self.scales.zero_()
        else:
            self.k_scale.zero_()
            self.v_scale.zero_()

    def copy_head(self, other):
        """The codes and scales of a pool of the same heads into the first slots (this pool is new, or larger)."""
        n, b = min(self.slots, other.slots), min(len(self.k_scale), len(other.k_scale))
        for name in ('k', 'v'):
            getattr(self, name).view(torch.uint8)[:n].copy_(getattr(other, name).view(torch.uint8)[:n])
            getattr(self, name + '_scale')[:b].copy_(getattr(other, name + '_scale')[:b])

    @property
    def nbytes(self):
        return 2 * (self.k.numel() + 4 * self.k_scale.numel())

    def rows(self, slots):
        """The K and V rows of pool slots `slots` (int32, on the pool's device) as BF16 [n, heads, head_dim]. A slot outside
        the pool sets the device error word, and its row is left as it was allocated."""
        if slots.dtype != torch.int32 or slots.dim() != 1 or not slots.is_contiguous() or slots.device != self.device:
            raise ValueError('slots must be a contiguous int32 vector on the pool\'s device')
        out = []
        width = self.heads * self.head_dim
        for codes, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            o = torch.empty(len(slots), self.heads, self.head_dim, dtype=torch.bfloat16, device=self.device)
            with _on(self.device) as s:
                nat.call('morj_kv8_gather', codes.data_ptr(), scale.data_ptr(), self.slots, slots.data_ptr(),
                         len(slots), self.heads, self.head_dim, o.data_ptr(), width, s)
            out.append(o)
        return tuple(out)


class StorePlan:
    """Where a step's rows go: row i to pool slot slots[i] (host integers, distinct, in a pool of `pool_slots`)."""

    def __init__(self, slots, pool_slots, device='cuda'):
        work, self.blocks = nat.kv8_store_work(slots, pool_slots)
        self.n, self.pool_slots = len(np.asarray(slots).reshape(-1)), pool_slots
        self.work, _ = _upload(device, work)


def _check_rows(name, t, n, heads, head_dim, device):
    if t.dtype != torch.bfloat16 or t.dim() != 3 or tuple(t.shape) != (n, heads, head_dim):
        raise ValueError(f'{name} must be BF16 [{n}, {heads}, {head_dim}]: {t.dtype} {tuple(t.shape)}')
    if t.device != device:
        raise ValueError(f'{name} is on {t.device}, not {device}')
    if n and (t.stride(2) != 1 or t.stride(1) != head_dim):
        raise ValueError(f'the heads of a row of {name} must be contiguous: strides {t.stride()}')


def store(pool, k, v, plan):
    """Write the rows k, v (BF16 [n, heads, head_dim]; rows may be any multiple of 8 elements apart) to their slots."""
    for name, t in (('k', k), ('v', v)):
        _check_rows(name, t, plan.n, pool.heads, pool.head_dim, pool.device)
    if plan.pool_slots != pool.slots or plan.work.device != pool.device:
        raise ValueError(f'the plan is for a pool of {plan.pool_slots} slots on {plan.work.device}')
    if not plan.n:
        return
    width = pool.heads * pool.head_dim
    with _on(pool.device) as s:
        nat.call('morj_kv8_store', k.data_ptr(), k.stride(0) if plan.n > 1 else width, v.data_ptr(),
                 v.stride(0) if plan.n > 1 else width, plan.n, pool.heads, pool.head_dim, plan.work.data_ptr(),
                 plan.blocks, pool.k.data_ptr(), pool.k_scale.data_ptr(), pool.v.data_ptr(), pool.v_scale.data_ptr(),
                 pool.slots, s)


def attention_workspace_bound(slots, heads, head_dim, sms=None):
    """Workspace bytes that no attention call whose segments list at most `slots` distinct slots (page size 1) exceeds on
    a GPU of `sms` SMs (default this one's): every slot expanded, and the partial units of tiles cut until two (few rows:
    three) CTAs an SM are busy, eight units (one) a part."""
    if sms is None:
        sms = torch.cuda.get_device_properties(torch.cuda.current_device()).multi_processor_count
    counts = nat.KV8_COUNTS()
    counts[2], counts[6] = -(-(8 * 2 + 3) * sms // heads), slots
    return nat.kv8_attention_workspace(counts, heads, head_dim)


class AttentionPlan:
    """A call's key lists and work list on the device (arguments as `morj_tree_attention`'s tables: host integers)."""

    def __init__(self, qo_indptr, kv_indptr, kv_indices, hq, hk, d, page_size=1, kv_last_page_len=None, window=0,
                 n_bidir=0, device='cuda'):
        qo, kv = nat.host_int32('qo_indptr', qo_indptr), nat.host_int32('kv_indptr', kv_indptr)
        kv_indices = nat.host_int32('kv_indices', kv_indices)
        if len(qo) < 1 or len(qo) != len(kv) or qo[0] != 0 or kv[0] < 0 or len(kv_indices) < kv[-1]:
            raise ValueError('qo_indptr and kv_indptr must have one entry per segment and one more, within kv_indices')
        if d not in (64, 128):
            raise ValueError(f'head_dim {d} unsupported (64, 128)')
        last = None if kv_last_page_len is None else nat.host_int32('kv_last_page_len', kv_last_page_len)
        if last is not None and (len(last) != len(qo) - 1 or (last < 0).any() or (last > page_size).any()):
            raise ValueError('kv_last_page_len must have one entry in [0, page_size] per segment')
        work, self.counts = nat.kv8_attention_work(qo, kv, kv_indices, n_bidir, hq, hk, window, page_size, last)
        self.n_q, self.n_bidir = int(qo[-1]), n_bidir
        self.hq, self.hk, self.d, self.page_size, self.window = hq, hk, d, page_size, window
        self.workspace_bytes = nat.kv8_attention_workspace(self.counts, hk, d, page_size)
        self.buf, (self.indices, self.work) = _upload(device, kv_indices, work)


def tree_attention(q, pool, plan, sm_scale, out=None):
    """Attention of q (BF16 [n_q, hq, d]) over the pool; returns `out` (allocated when not given)."""
    shape = (plan.n_q, plan.hq, plan.d)
    if q.dtype != torch.bfloat16 or tuple(q.shape) != shape or not q.is_contiguous():
        raise ValueError(f'q must be contiguous BF16 {shape}: {q.dtype} {tuple(q.shape)}')
    if (pool.heads, pool.head_dim) != (plan.hk, plan.d):
        raise ValueError(f'the pool has {pool.heads} heads of {pool.head_dim}, the plan {plan.hk} of {plan.d}')
    if q.device != pool.device or plan.buf.device != pool.device:
        raise ValueError(f'q, the plan and the pool are on {q.device}, {plan.buf.device}, {pool.device}')
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous() or out.device != q.device:
        raise ValueError(f'out must be like q: {out.dtype} {tuple(out.shape)} on {out.device}')
    if not plan.n_q:
        return out
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=q.device) if plan.workspace_bytes else None
    with _on(pool.device) as s:
        nat.call('morj_tree_attention_kv8', q.data_ptr(), plan.n_q, pool.k.data_ptr(), pool.k_scale.data_ptr(),
                 pool.v.data_ptr(), pool.v_scale.data_ptr(), pool.slots, out.data_ptr(), plan.indices.data_ptr(),
                 plan.n_bidir, plan.hq, plan.hk, plan.d, plan.page_size, plan.window, sm_scale, plan.work.data_ptr(),
                 plan.counts, ws.data_ptr() if ws is not None else None, plan.workspace_bytes, s)
    return out
