"""Cases of the operators around an 8-bit K/V cache and the full-vocabulary readout, with their plain forms.

Three operators (`op`):

* `store`   writes K/V rows (BF16) into pools of e4m3 codes with one power-of-two scale per 64-slot block and head.
  A block's scale only grows; when it does, the block's resident codes move to the new scale.
* `attn`    tree attention over such pools: segments of queries over slot (page 1) or page lists, bottom-right causal,
  optional sliding window, grouped heads; one query per segment is the single-token form.
* `logp`    log-probabilities of given tokens under the whole vocabulary (softcapped logits of normed rows against the
  tied embedding), with log-sum-exp, entropy and the top alternatives.

`run` computes them with elementary torch operations in 32 bits; with `own` set it calls `morj_b200.kv8` and
`morj_b200.logprobs`.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 64           # slots that share a scale
CODE_MAX = 448.0     # largest e4m3 value
MIN_EXP = -100       # smallest scale is 2^-100
DEV = 'cuda'


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # 64 requests decode one token each: the smallest call of the store, where its latency counts
        dict(name='store 64 tokens', op='store', hk=16, d=128, rows=64, slots=16384, fresh=False),
        # the K/V rows of one step over the 8,704-token latency tree into a fresh pool
        dict(name='store 8704 prompt', op='store', hk=16, d=128, rows=8704, slots=8704, fresh=True),
        # the 2-layer test model (4 query / 2 KV heads of 64, window 64): the smallest tree
        dict(name='attn tiny tree', op='attn', form='tree', hq=4, hk=2, d=64, window=64, page=1, prefix=128,
             branches=4, branch=24),
        # the last layer of the 31B text tree: its 9 readout rows, one query each over 1,560 keys
        dict(name='attn 9 readouts', op='attn', form='last', hq=32, hk=16, d=128, window=0, page=1, prefix=1500,
             branches=9, branch=60),
        # single-token attention of 64 requests of uneven length in a paged cache
        dict(name='attn 64 singles 8192', op='attn', form='batch', hq=32, hk=16, d=128, window=0, page=64,
             prefix=8192, branches=64, branch=1),
        # a later pass: 8 branches of 64 tokens over an 8,192-token prefix kept in 8 bits
        dict(name='attn 8x64 on 8192', op='attn', form='branches', hq=32, hk=16, d=128, window=0, page=1, prefix=8192,
             branches=8, branch=64),
        # a sliding layer of the 31B text tree, every token computed
        dict(name='attn text sliding', op='attn', form='tree', hq=32, hk=16, d=128, window=1024, page=1, prefix=1500,
             branches=9, branch=60),
        # the op-level tree attention configuration (2048 + 8 x 64, pages of 64 slots in shuffled order), global mask
        dict(name='attn op-level paged', op='attn', form='tree', hq=32, hk=16, d=128, window=0, page=64, prefix=2048,
             branches=8, branch=64),
        # one row of the 2-layer test model: the smallest readout
        dict(name='logp 1 row 4096', op='logp', rows=1, hidden=256, vocab=4096, targets=4, top=4, softcap=30.0),
        # the text tree's 9 readout rows over the whole vocabulary, 5 labels each
        dict(name='logp 9 rows', op='logp', rows=9, hidden=5376, vocab=262144, targets=5, top=8, softcap=30.0),
        # every token of the text tree's 9 branches of 60, scored
        dict(name='logp 540 rows', op='logp', rows=540, hidden=5376, vocab=262144, targets=1, top=5, softcap=30.0),
        # every token of the text tree scored
        dict(name='logp 2040 rows', op='logp', rows=2040, hidden=5376, vocab=262144, targets=1, top=0,
             softcap=30.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['store', 'attn', 'attn', 'logp'])
    if op == 'store':
        hk, d = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128])
        rows = _log_int(rng, 1, 8704)
        fresh = rng.random() < 0.5
        slots = rows + rng.randrange(0, 64) if fresh else rows * 2 + rng.randrange(64, 4096)
        return dict(op='store', hk=hk, d=d, rows=rows, slots=slots, fresh=fresh)
    if op == 'attn':
        hk = rng.choice([1, 2, 4, 8, 16])
        case = dict(op='attn', form=rng.choice(['tree', 'branches', 'last', 'batch']), hq=hk * rng.choice([1, 2, 4, 8]),
                    hk=hk, d=rng.choice([64, 128]), window=rng.choice([0, 0, rng.randrange(16, 2048)]),
                    page=rng.choice([1, 64]))
        case['hq'] = min(case['hq'], 32) // hk * hk
        case['prefix'] = _log_int(rng, 1, 2048 if case['form'] == 'tree' else 8192)
        if case['page'] > 1 and case['form'] != 'batch':  # branches share whole pages of the prefix
            case['prefix'] = max(1, case['prefix'] // case['page']) * case['page']
        case['branches'] = _log_int(rng, 1, 64 if case['form'] in ('last', 'batch') else 9)
        case['branch'] = 1 if case['form'] == 'batch' else rng.randrange(1, 97)
        return case
    hidden, vocab = rng.choice([(8 * rng.randrange(8, 129), _log_int(rng, 100, 65536)),
                                (5376, _log_int(rng, 4096, 262144))])
    return dict(op='logp', rows=_log_int(rng, 1, 2040), hidden=hidden, vocab=vocab, targets=rng.randrange(0, 9),
                top=rng.choice([0, 1, rng.randrange(2, 21)]), softcap=rng.choice([30.0, 30.0, 0.0]))


# ---- tables of an attention case ------------------------------------------------------------------------------------

def _tables(case):
    """Host tables: per segment its queries and key list (slots or pages), the pool size and the longest list."""
    page, P, B, L = case['page'], case['prefix'], case['branches'], case['branch']
    rng = np.random.default_rng([P, B, L, page, case['hk']])
    pages_of = lambda n: (n + page - 1) // page
    q_len, kv_len, lists = [], [], []
    if case['form'] == 'batch':  # every request has its own list, lengths spread over (0, prefix]
        lens = [1] + [int(n) for n in np.exp(rng.uniform(math.log(max(1, P / 16)), math.log(P + 1), B - 1))] if B > 1 \
            else [P]
        at = 0
        for n in [min(P, max(1, n)) for n in lens]:
            q_len.append(1)
            kv_len.append(n)
            lists.append(np.arange(at, at + pages_of(n)))
            at += pages_of(n)
    else:
        head, at = np.arange(pages_of(P)), pages_of(P)
        if case['form'] == 'tree':
            q_len.append(P)
            kv_len.append(P)
            lists.append(head)
        for _ in range(B):
            lists.append(np.concatenate([head, np.arange(at, at + pages_of(L))]))
            at += pages_of(L)
            q_len.append(1 if case['form'] == 'last' else L)
            kv_len.append(P + L)
    if page > 1:  # logical page -> physical page
        perm = rng.permutation(at)
        lists = [perm[x] for x in lists]
    return dict(qo_indptr=np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32),
                kv_indptr=np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32),
                kv_indices=np.concatenate(lists).astype(np.int32),
                last_page_len=np.asarray([n - (pages_of(n) - 1) * page for n in kv_len], np.int32),
                kv_len=np.asarray(kv_len), pool_slots=int(at) * page, longest=int(max(kv_len)))


def _visible(case, t, s):
    """(first, last) visible key position of each query of segment s."""
    n = int(t['qo_indptr'][s + 1] - t['qo_indptr'][s])
    hi = int(t['kv_len'][s]) - n + np.arange(n)
    lo = np.maximum(0, hi - case['window'] + 1) if case['window'] else np.zeros(n, np.int64)
    return lo, hi


def _slots(case, t, s):
    pages = t['kv_indices'][t['kv_indptr'][s]:t['kv_indptr'][s + 1]].astype(np.int64)
    return (pages[:, None] * case['page'] + np.arange(case['page'])).reshape(-1)[:t['kv_len'][s]]


def work(case):
    if case['op'] == 'store':
        n, width = case['rows'], case['hk'] * case['d']
        return {'bytes': 2 * n * width * (2 + 1) + 2 * (n + BLOCK - 1) // BLOCK * case['hk'] * 8, 'flops': 4 * n * width}
    if case['op'] == 'attn':
        t = _tables(case)
        seen, pairs = np.zeros(t['pool_slots'], bool), 0
        for s in range(len(t['kv_len'])):
            lo, hi = _visible(case, t, s)
            pairs += int((hi - lo + 1).sum())
            seen[_slots(case, t, s)[int(lo.min()):int(hi.max()) + 1]] = True
        n_q, kv = int(t['qo_indptr'][-1]), int(seen.sum())
        return {'bytes': 2 * 2 * n_q * case['hq'] * case['d'] + 2 * kv * case['hk'] * (case['d'] + 4 / BLOCK),
                'flops': 4 * case['hq'] * case['d'] * pairs}
    n, V, H = case['rows'], case['vocab'], case['hidden']
    return {'bytes': 2 * (n + V) * H + 4 * n * (2 + 2 * case['targets'] + 2 * case['top']), 'flops': 2 * n * V * H}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _rows(g, n, hk, d, gain):
    """K or V rows as a layer makes them: per-token norms that differ, per-head gains, one strong channel."""
    x = torch.randn(n, hk, d, generator=g, device=DEV)
    x *= torch.exp(0.3 * torch.randn(n, 1, 1, generator=g, device=DEV)) * gain
    x[:, :, 5] *= 3
    return x.to(torch.bfloat16)


def _scales(a):
    """The power-of-two scale that brings |x| <= a within the code range."""
    m, e = torch.frexp(a.float())  # a = m * 2^e, m in [0.5, 1), and the largest code is 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=MIN_EXP)
    e = torch.where(a > 0, e, MIN_EXP).to(torch.int32)
    return ((e + 127) << 23).view(torch.float32)


def _quantised(x):
    """A filled pool: codes and block scales of the rows x [slots, hk, d]."""
    n, hk, d = x.shape
    blocks = (n + BLOCK - 1) // BLOCK
    padded = torch.zeros(blocks * BLOCK, hk, device=DEV)
    padded[:n] = x.abs().amax(2)
    scale = _scales(padded.view(blocks, BLOCK, hk).amax(1))
    codes = (x.float() / scale.repeat_interleave(BLOCK, 0)[:n, :, None]).to(torch.float8_e4m3fn)
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    if case['op'] == 'store':
        hk, d, n, slots = case['hk'], case['d'], case['rows'], case['slots']
        gain = torch.exp2(0.5 * torch.randn(1, hk, 1, generator=g, device=DEV))
        st['k'], st['v'] = _rows(g, n, hk, d, gain), _rows(g, n, hk, d, gain)
        if case['fresh']:  # a step's rows in tree order
            where = np.arange(n) + (slots - n)
            st['codes'] = [torch.zeros(slots, hk, d, device=DEV).to(torch.float8_e4m3fn) for _ in 'kv']
            st['scale'] = [torch.zeros((slots + BLOCK - 1) // BLOCK, hk, device=DEV) for _ in 'kv']
        else:  # rows of many requests into blocks that hold earlier tokens
            where = np.random.default_rng(seed).permutation(slots)[:n]
            pairs = [_quantised(_rows(g, slots, hk, d, gain)) for _ in 'kv']
            st['codes'], st['scale'] = [p[0] for p in pairs], [p[1] for p in pairs]
        st['slots'] = torch.as_tensor(where, device=DEV)
        if own:  # the pool and the plan a step keeps for its layers
            from morj_b200 import kv8
            st['pool'] = kv8.KV8Pool.of(st['codes'][0], st['scale'][0], st['codes'][1], st['scale'][1])
            st['plan'] = kv8.StorePlan(where, slots, DEV)
    elif case['op'] == 'attn':
        hk, d, t = case['hk'], case['d'], _tables(case)
        gain = torch.exp2(0.5 * torch.randn(1, hk, 1, generator=g, device=DEV))
        (st['k'], st['ks']), (st['v'], st['vs']) = (_quantised(_rows(g, t['pool_slots'], hk, d, gain)) for _ in 'kv')
        st['q'] = torch.randn(int(t['qo_indptr'][-1]), case['hq'], d, generator=g, device=DEV).to(torch.bfloat16)
        st['longest'] = t['longest']
        for key in ('qo_indptr', 'kv_indptr', 'kv_indices', 'last_page_len'):
            st[key] = torch.as_tensor(t[key], device=DEV).long()
        if own:
            from morj_b200 import kv8
            st['pool'] = kv8.KV8Pool.of(st['k'], st['ks'], st['v'], st['vs'])
            st['plan'] = kv8.AttentionPlan(t['qo_indptr'], t['kv_indptr'], t['kv_indices'], case['hq'], hk, d,
                                           page_size=case['page'], kv_last_page_len=t['last_page_len'],
                                           window=case['window'], device=DEV)
    else:
        n, H, V, T = case['rows'], case['hidden'], case['vocab'], case['targets']
        # Embedding of std 0.02 and unit-RMS rows that favour a few tokens, as a trained readout does. Their values are
        # multiples of 2^-10 and 2^-5, so a logit is the same number in any order of summation and the ids of the top
        # alternatives are determined.
        w = torch.empty(V, H, dtype=torch.bfloat16, device=DEV)
        for r in range(0, V, 65536):
            block = torch.randn(min(65536, V - r), H, generator=g, device=DEV) * 0.02
            w[r:r + 65536] = (block.clamp_(-0.12, 0.12) * 1024).round_() / 1024
        liked = torch.randint(V, (n, 4), generator=g, device=DEV)
        h = torch.randn(n, H, generator=g, device=DEV)
        for j in range(4):
            h += w[liked[:, j]].float() * (5 * torch.rand(n, 1, generator=g, device=DEV))
        st['h'] = ((h.clamp_(-3.5, 3.5) * 32).round_() / 32).to(torch.bfloat16)
        st['w'] = w
        ids = torch.randint(V, (n, T), generator=g, device=DEV)
        if T:
            ids[:, 0] = liked[:, 0]
        st['targets'] = ids.to(torch.int32)
    return st


# ---- the operators in their plain form ------------------------------------------------------------------------------

def _plain_store(rows, where, codes, scale):
    n, hk, d = rows.shape
    x = rows.float()
    slots = codes.shape[0]
    a = torch.zeros(slots, hk, device=DEV).index_copy(0, where, x.abs().amax(2))
    hit = torch.zeros(slots, 1, device=DEV).index_fill(0, where, 1.0)
    pad = scale.shape[0] * BLOCK - slots
    a = torch.nn.functional.pad(a, (0, 0, 0, pad)).view(-1, BLOCK, hk).amax(1)
    hit = torch.nn.functional.pad(hit, (0, 0, 0, pad)).view(-1, BLOCK, 1).amax(1) > 0
    new = torch.where(hit, torch.maximum(scale, _scales(a)), scale)
    ratio = torch.where(scale > 0, scale / new, torch.ones_like(new)).repeat_interleave(BLOCK, 0)[:slots, :, None]
    out = (codes.float() * ratio).to(codes.dtype).view(torch.uint8)
    per_row = new[where // BLOCK][:, :, None]
    out = out.index_copy(0, where, (x / per_row).to(codes.dtype).view(torch.uint8))
    codes.view(torch.uint8).copy_(out)
    scale.copy_(new)
    return codes, scale


def _plain_attention(st):
    case, q = st['case'], st['q']
    n_q, hq, d = q.shape
    hk, page, window = case['hk'], case['page'], case['window']
    slots = st['k'].shape[0]
    spread = lambda s: s.repeat_interleave(BLOCK, 0)[:slots, :, None]
    k = (st['k'].float() * spread(st['ks'])).transpose(0, 1)   # [hk, slots, d]
    v = (st['v'].float() * spread(st['vs'])).transpose(0, 1)
    qo, kv = st['qo_indptr'], st['kv_indptr']
    q_len, pages = qo[1:] - qo[:-1], kv[1:] - kv[:-1]
    kv_len = (pages - 1) * page + st['last_page_len']
    row = torch.arange(n_q, device=DEV)
    seg = torch.searchsorted(qo, row, right=True) - 1
    t = torch.arange(st['longest'], device=DEV)
    hi = (kv_len - q_len)[seg] + row - qo[seg]
    lo = (hi - window + 1).clamp(min=0) if window else torch.zeros_like(hi)
    seen = (t >= lo[:, None]) & (t <= hi[:, None])                       # [n_q, longest]
    at = (kv[:-1, None] + t // page).clamp(max=st['kv_indices'].numel() - 1)
    slot = st['kv_indices'][at] * page + t % page                          # [segments, longest]
    slot = torch.where(t < kv_len[:, None], slot, slots)
    mask = torch.zeros(n_q, slots + 1, dtype=torch.bool, device=DEV).scatter_(1, slot[seg], seen)[:, :slots]
    s = torch.matmul(q.float().view(n_q, hk, hq // hk, d).transpose(0, 1).reshape(hk, -1, d), k.transpose(1, 2))
    s = s.view(hk, n_q, hq // hk, slots) * d ** -0.5
    s = torch.where(mask[None, :, None], s, -math.inf)
    m = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p.view(hk, -1, slots), v).view(hk, n_q, hq // hk, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.transpose(0, 1).reshape(n_q, hq, d).to(torch.bfloat16)


def _plain_logprobs(h, w, targets, top, softcap):
    logits = torch.matmul(h.float(), w.float().T)
    z = softcap * torch.tanh(logits / softcap) if softcap else logits
    m = z.amax(1, keepdim=True)
    lse = (m + torch.log(torch.exp(z - m).sum(1, keepdim=True)))
    lp = z - lse
    out = dict(logprob=lp.gather(1, targets.long()), lse=lse[:, 0], entropy=-(torch.exp(lp) * lp).sum(1))
    if top:  # by logit, the lower id first among equals
        bits = (logits + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7fffffff)).long()
        V = w.shape[0]
        key = order * (1 << 32) + (V - 1 - torch.arange(V, device=DEV))
        ids = V - 1 - (torch.topk(key, top).values & 0xffffffff)
        out.update(top_ids=ids.to(torch.int32), top_logprobs=lp.gather(1, ids))
    return out


def run(state):
    case = state['case']
    if case['op'] == 'store':
        if own:
            from morj_b200 import kv8
            kv8.store(state['pool'], state['k'], state['v'], state['plan'])
        else:
            for x, codes, scale in zip((state['k'], state['v']), state['codes'], state['scale']):
                _plain_store(x, state['slots'], codes, scale)
        return dict(k=state['codes'][0], k_scale=state['scale'][0], v=state['codes'][1], v_scale=state['scale'][1])
    if case['op'] == 'attn':
        if own:
            from morj_b200 import kv8
            return kv8.tree_attention(state['q'], state['pool'], state['plan'], case['d'] ** -0.5)
        return _plain_attention(state)
    if own:
        from morj_b200 import logprobs
        got = logprobs.token_logprobs(state['h'], state['w'], state['targets'], top=case['top'],
                                      softcap=case['softcap'])
        out = dict(logprob=got.logprob, lse=got.lse, entropy=got.entropy)
        if case['top']:
            out.update(top_ids=got.top_ids, top_logprobs=got.top_logprobs)
        return out
    return _plain_logprobs(state['h'], state['w'], state['targets'], case['top'], case['softcap'])


# ---- 64 bits ---------------------------------------------------------------------------------------------------------

def _e4m3(y):
    """The nearest value with 3 mantissa bits, exponents -6..8 and subnormals, ties to even."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'store':
        out, where = {}, st['slots'].tolist()
        blocks = {}
        for row, slot in enumerate(where):
            blocks.setdefault(slot // BLOCK, []).append((slot, row))
        for name, x, codes, scale in zip('kv', (st['k'], st['v']), st['codes'], st['scale']):
            val, s = codes.double(), scale.double()
            for b, pairs in blocks.items():
                at = torch.tensor([p[0] for p in pairs], device=DEV)
                rows = x[torch.tensor([p[1] for p in pairs], device=DEV)].double()
                a = rows.abs().amax((0, 2))
                need = (a / torch.full_like(a, CODE_MAX)).clamp(min=2.0 ** MIN_EXP)
                m, e = torch.frexp(need)  # the power of two at or above it
                new = torch.maximum(s[b], torch.exp2((e - (m == 0.5).int()).double()))
                old = torch.where(s[b] > 0, s[b], new)
                lo, hi = b * BLOCK, min((b + 1) * BLOCK, val.shape[0])
                val[lo:hi] = _e4m3(val[lo:hi] * (old / new)[None, :, None])
                val[at] = _e4m3(rows / new[None, :, None])
                s[b] = new
            out[name], out[name + '_scale'] = val, s
        return out
    if case['op'] == 'attn':
        t, hk, G = _tables(case), case['hk'], case['hq'] // case['hk']
        o = torch.zeros(st['q'].shape, dtype=torch.float64, device=DEV)
        for s in range(len(t['kv_len'])):
            a, b = int(t['qo_indptr'][s]), int(t['qo_indptr'][s + 1])
            lo, hi = (torch.as_tensor(x, device=DEV) for x in _visible(case, t, s))
            slots = torch.as_tensor(_slots(case, t, s), device=DEV)
            pos = torch.arange(len(slots), device=DEV)
            hidden = (pos < lo[:, None]) | (pos > hi[:, None])
            for h in range(hk):
                k = st['k'][slots, h].double() * st['ks'][slots // BLOCK, h].double()[:, None]
                v = st['v'][slots, h].double() * st['vs'][slots // BLOCK, h].double()[:, None]
                for j in range(h * G, (h + 1) * G):
                    w = (st['q'][a:b, j].double() @ k.T * case['d'] ** -0.5).masked_fill(hidden, -math.inf)
                    o[a:b, j] = torch.softmax(w, 1) @ v
        return o
    if case['rows'] * case['vocab'] * case['hidden'] > 4e12:
        return None  # (tens of seconds in 64 bits where the card has few of those units)
    n, V, top, c = case['rows'], case['vocab'], case['top'], case['softcap']
    w = st['w'].double()
    out = dict(logprob=[], lse=[], entropy=[])
    if top:
        out.update(top_ids=[], top_logprobs=[])
    for r in range(0, n, 64):
        raw = st['h'][r:r + 64].double() @ w.T
        z = torch.tanh(raw / c) * c if c else raw
        lse = torch.logsumexp(z, 1)
        p = torch.softmax(z, 1)
        out['lse'].append(lse)
        out['entropy'].append(lse - (p * z).sum(1))
        out['logprob'].append(z.gather(1, st['targets'][r:r + 64].long()) - lse[:, None])
        if top:
            ids = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :top]
            out['top_ids'].append(ids.to(torch.int32))
            out['top_logprobs'].append(z.gather(1, ids) - lse[:, None])
    return {key: torch.cat(v) for key, v in out.items()}
