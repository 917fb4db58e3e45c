"""Host side of the 8-bit K/V cache: the store's and the attention's work lists and every refusal, on the CPU."""
import ctypes

import numpy as np
import pytest
import torch

from morj_b200 import _native as nat
from morj_b200 import kv8

ITEM = 12


def groups(work, blocks, n):
    heads = work[:3 * blocks].reshape(-1, 3)
    pairs = work[3 * blocks + (blocks & 1):].reshape(-1, 2)
    assert len(pairs) == n
    return heads.tolist(), pairs


@pytest.mark.parametrize('n,slots', [(0, 5), (1, 1), (7, 640), (64, 64), (500, 1000), (500, 60000)])
def test_store_work_groups_every_row_by_block(n, slots):
    where = np.random.default_rng(n).permutation(slots)[:n]
    work, blocks = nat.kv8_store_work(where, slots)
    heads, pairs = groups(work, blocks, n)
    assert sorted(map(tuple, pairs.tolist())) == sorted((int(s), i) for i, s in enumerate(where))
    assert [b for b, _, _ in heads] == sorted({int(s) // 64 for s in where})
    at = 0
    for b, first, count in heads:
        assert first == at and all(int(s) // 64 == b for s, _ in pairs[first:first + count])
        at += count
    assert at == n


def test_store_work_refusals():
    with pytest.raises(ValueError, match='row 1.s slot 10 is outside the pool of 10'):
        nat.kv8_store_work([3, 10], 10)
    with pytest.raises(ValueError, match='outside'):
        nat.kv8_store_work([-1], 10)
    with pytest.raises(ValueError, match='rows 0 and 2 have the same slot 4'):
        nat.kv8_store_work([4, 5, 4], 10)
    buf = np.zeros(4, np.int32)
    s = np.array([1, 2], np.int32)
    assert nat.lib().morj_kv8_store_work(s.ctypes.data_as(nat.IP), 2, 10, buf.ctypes.data_as(nat.IP), 4) == -1
    assert b'exceed capacity' in nat.lib().morj_last_error()
    assert nat.lib().morj_kv8_store_work(None, 2, 10, buf.ctypes.data_as(nat.IP), 4) == -1


def view(q_len, keys, bidir, window, j):
    diag = keys - q_len
    hi = keys - 1 if bidir else diag + j
    if window <= 0:
        lo = 0
    elif bidir:
        lo = diag + min(0, j - (window - 1))
    else:
        lo = hi - (window - 1)
    return max(0, lo), hi


CASES = [  # (segments (queries, keys), hq, hk, window, n_bidir)
    ([(1, 1)], 4, 2, 0, 0),
    ([(1, 5000), (1, 0), (0, 30), (1, 64)], 32, 16, 0, 0),
    ([(1, 3000)] * 40, 8, 8, 100, 0),
    ([(130, 130), (5, 200), (3, 1)], 8, 2, 0, 0),
    ([(40, 40), (60, 100)], 4, 4, 16, 1),
    ([(2, 9000)], 24, 8, 0, 0),
    ([(1, 20000)], 64, 1, 0, 0),
    ([(700, 1700), (1, 4000), (64, 64)], 32, 16, 1024, 0),
    ([(130, 130), (5, 200), (3, 1), (900, 2000)], 8, 2, 0, 0),
    ([(400, 400), (600, 1000)], 4, 4, 160, 1),
    ([(300, 40), (40, 0), (2, 5), (900, 1500)], 6, 2, 0, 0),
]


@pytest.mark.parametrize('spec,hq,hk,window,n_bidir', CASES)
@pytest.mark.parametrize('page', [1, 16])
def test_attention_work_covers_every_row_and_key_once(spec, hq, hk, window, n_bidir, page):
    G = hq // hk
    pages = [(n + page - 1) // page for _, n in spec]
    qo = np.concatenate([[0], np.cumsum([a for a, _ in spec])])
    kv = np.concatenate([[0], np.cumsum(pages)])
    last = [n - (p - 1) * page if p else 0 for (_, n), p in zip(spec, pages)]
    perm = np.random.default_rng(len(spec)).permutation(int(kv[-1]) + 5)[:int(kv[-1])]
    work, counts = nat.kv8_attention_work(qo, kv, perm, n_bidir, hq, hk, window, page, last)
    # few rows see few keys: everything 16 rows at a time
    few = [[view(n, keys, s < n_bidir, window, r // G) for r in range(r0, min(r0 + 16, n * G))]
           for s, (n, keys) in enumerate(spec) for r0 in range(0, n * G, 16)]
    seen = sum(max(max(hi for _, hi in rows) - min(lo for lo, _ in rows) + 1, 0) for rows in few)
    all_few = seen * hk <= 65536 and len(few) * hk <= 3 * 148
    check_work(work, counts, spec, G, window, n_bidir, kv, all_few)
    if all_few:
        return
    check_pages(work, counts, spec, G, window, n_bidir, page, kv, perm)


def check_pages(work, counts, spec, G, window, n_bidir, page, kv, indices):
    """The pages the 128-row tiles see: each once, with the number of its slots that are listed; the lists point to them;
    the blocks are the 64-slot blocks of those slots."""
    n_rows, n_joins, _, _, _, n_tiles, n_pages, n_blocks, n_list = list(counts)[:9]
    rest = work[(n_tiles + n_rows + n_joins) * ITEM:]
    pairs, blocks, lists = rest[:2 * n_pages].reshape(-1, 2), rest[2 * n_pages:2 * n_pages + n_blocks], \
        rest[2 * n_pages + n_blocks:]
    assert len(lists) == n_list and len(set(pairs[:, 0].tolist())) == n_pages
    slots = set()
    for s, (n, keys) in enumerate(spec):
        if n * G <= 16:
            continue
        seen = [view(n, keys, s < n_bidir, window, j) for j in range(n)]
        seen = [(lo, hi) for lo, hi in seen if lo <= hi]
        if not seen:
            continue
        for t in range(min(lo for lo, _ in seen), max(hi for _, hi in seen) + 1):
            at = int(kv[s]) + t // page
            p, used = pairs[lists[at]]
            assert p == indices[at] and t % page < used
            slots.add(int(p) * page + t % page)
    assert sum(u for _, u in pairs) >= len(slots) and (n_list == int(kv[-1]) or not slots)
    assert blocks.tolist() == sorted({x // 64 for p, u in pairs.tolist() for x in (p * page, p * page + u - 1)}
                                     | {x // 64 for x in slots})


def check_work(work, counts, spec, G, window, n_bidir, kv, all_few):
    n_rows, n_joins, units, few, ints, n_tiles = list(counts)[:6]
    items = work[:(n_tiles + n_rows + n_joins) * ITEM].reshape(-1, ITEM).tolist()
    assert len(work) == ints
    parts, rows_of = {}, {}
    for i, (seg, r0, t0, t1, unit, _, _, rows, q0, q_len, kv0, keys) in enumerate(items[:n_tiles + n_rows]):
        assert (q_len, keys) == spec[seg] and q0 == sum(n for n, _ in spec[:seg]) and kv0 == kv[seg]
        # segments of more than 16 rows in 128-row tiles, the others in small ones
        assert rows == (128 if i < n_tiles else few) and (not all_few and spec[seg][0] * G > 16) == (i < n_tiles)
        assert r0 % rows == 0 and t0 <= t1
        parts.setdefault((seg, r0), []).append((t0, t1, unit))
        rows_of[seg] = rows
    assert few in (8, 16) and (few == 16 or all(n * G <= 8 or (not all_few and n * G > 16) for n, _ in spec))
    assert set(parts) == {(s, r0) for s, (n, _) in enumerate(spec) if n for r0 in range(0, n * G, rows_of[s])}
    joined = {(j[0], j[1]): j for j in items[n_tiles + n_rows:]}
    assert len(joined) == n_joins
    used = set()
    for (seg, r0), got in parts.items():
        n, keys = spec[seg]
        rows = range(r0, min(r0 + rows_of[seg], n * G))
        los, his = zip(*(view(n, keys, seg < n_bidir, window, r // G) for r in rows))
        got.sort()
        if max(his) < min(los):
            assert len(got) == 1 and got[0][0] == got[0][1]
        else:
            assert got[0][0] == min(los) and got[-1][1] == max(his) + 1 <= keys
            assert all(a[1] == b[0] and a[1] % 64 == 0 for a, b in zip(got, got[1:]))
            assert all(a < b for a, b, _ in got)
        per = (rows_of[seg] + 15) // 16
        if len(got) == 1:
            assert got[0][2] == -1 and (seg, r0) not in joined
            continue
        for u in range(per):
            j = joined.pop((seg, r0 + 16 * u))
            assert j[5] == len(got) and [x[2] + u for x in got] == [j[4] + i * j[6] for i in range(len(got))]
            assert j[7] == min(16, rows_of[seg])
        for _, _, first in got:
            assert not used & set(range(first, first + per))
            used |= set(range(first, first + per))
    assert not joined and used == set(range(units))


def test_long_single_rows_are_cut_and_short_ones_are_not():
    _, long = nat.kv8_attention_work([0, 1], [0, 20000], np.arange(20000), 0, 32, 16, 0)
    assert long[1] == 1 and long[2] > 8
    _, long = nat.kv8_attention_work([0, 64], [0, 20000], np.arange(20000), 0, 32, 16, 0)
    assert long[5] > 1 and long[1] == 8 and long[2] == 8 * long[5]
    _, short = nat.kv8_attention_work([0, 1], [0, 200], np.arange(200), 0, 32, 16, 0)
    assert short[1] == 0 and short[2] == 0


def test_a_page_far_outside_any_pool_names_no_block_inside_one():
    # (page * page size passes 2^31 blocks: the device is to find the block outside the pool, not a wrapped one inside)
    work, counts = nat.kv8_attention_work([0, 300], [0, 2], [3, 2**31 - 1], 0, 4, 2, 0, 4096, [904])
    n_tiles, n_pages, n_blocks = counts[5], counts[6], counts[7]
    assert n_tiles > 0 and n_pages == 2
    at = (counts[0] + counts[1] + n_tiles) * ITEM + 2 * n_pages
    blocks = work[at:at + n_blocks].astype(np.int64)
    near = blocks[blocks < 2**25]
    assert (blocks >= 0).all() and near.tolist() == list(range(3 * 64, 4 * 64)) and n_blocks > len(near)


def test_attention_work_refusals():
    for args in [dict(hq=3, hk=2), dict(hq=0, hk=1), dict(page_size=0), dict(n_bidir=2), dict(n_bidir=-1)]:
        a = dict(qo_indptr=[0, 1], kv_indptr=[0, 4], kv_indices=range(4), n_bidir=0, hq=4, hk=2, window=0)
        with pytest.raises(ValueError):
            nat.kv8_attention_work(**{**a, **args})
    with pytest.raises(ValueError, match='out of order'):
        nat.kv8_attention_work([0, 3, 1], [0, 4, 8], range(8), 0, 4, 2, 0)
    with pytest.raises(ValueError, match='out of order'):
        nat.kv8_attention_work([0, 1, 2], [0, 4, 3], range(4), 0, 4, 2, 0)
    with pytest.raises(ValueError, match='list entries'):
        nat.kv8_attention_work([0, 1], [0, 4], range(3), 0, 4, 2, 0)
    with pytest.raises(ValueError, match='page -1'):
        nat.kv8_attention_work([0, 40], [0, 41], [-1] * 41, 0, 4, 2, 0)


# a call's arguments are refused before any device access; 16 stands for an aligned pointer that is never read
def store_args(**kw):
    a = dict(k=16, ld_k=256, v=16, ld_v=256, n=4, hk=2, d=128, work=16, n_blocks=1, k_codes=16, k_scale=16, v_codes=16,
             v_scale=16, pool_slots=64, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('kw,match', [
    (dict(k=None), 'null pointer'), (dict(v=None), 'null pointer'), (dict(work=None), 'null pointer'),
    (dict(k_scale=None), 'null pointer'), (dict(n=-1), 'bad size'), (dict(n_blocks=5), 'bad size'),
    (dict(hk=0), 'bad size'), (dict(hk=70000), 'bad size'), (dict(pool_slots=0), 'bad size'),
    (dict(ld_k=255), 'multiples of 8'), (dict(ld_v=248), 'at least 256'), (dict(k=24), '16-byte'),
    (dict(v_codes=8), '16-byte'), (dict(work=20), '8-byte'), (dict(k_scale=18), '4-byte')])
def test_store_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        nat.call('morj_kv8_store', *store_args(**kw))


def test_store_refuses_other_head_sizes_and_accepts_nothing_to_do():
    with pytest.raises(nat.NativeFailure, match='head_dim 96'):
        nat.call('morj_kv8_store', *store_args(d=96))
    nat.call('morj_kv8_store', *store_args(n=0))


def gather_args(**kw):
    a = dict(codes=16, scale=16, pool_slots=64, slots=16, n=2, hk=2, d=64, out=16, ld=128, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('kw', [dict(codes=None), dict(scale=None), dict(slots=None), dict(out=None), dict(n=-1),
                                dict(pool_slots=0), dict(d=60), dict(ld=120), dict(ld=129), dict(out=24),
                                dict(codes=8)])
def test_gather_refusals(kw):
    with pytest.raises(ValueError):
        nat.call('morj_kv8_gather', *gather_args(**kw))


def attention_args(**kw):
    counts = nat.KV8_COUNTS(*kw.pop('counts', (1, 0, 0, 8, 12, 0, 0, 0, 0, 1)))
    a = dict(q=16, n_q=1, k=16, ks=16, v=16, vs=16, pool_slots=64, out=16, idx=16, n_bidir=0, hq=4, hk=2, d=128, page=1,
             window=0, scale=1.0, work=16, counts=counts, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


PARTS = (1, 1, 2, 8, 24, 0, 0, 0, 0, 1)


@pytest.mark.parametrize('kw,match', [
    (dict(q=None), 'null pointer'), (dict(k=None), 'null pointer'), (dict(ks=None), 'null pointer'),
    (dict(v=None), 'null pointer'), (dict(vs=None), 'null pointer'), (dict(out=None), 'null pointer'),
    (dict(idx=None), 'null pointer'), (dict(work=None), 'null pointer'), (dict(n_q=0), 'bad size'),
    (dict(pool_slots=0), 'bad size'), (dict(hq=3), 'multiple'), (dict(hk=0), 'multiple'), (dict(page=0), 'page_size'),
    (dict(n_bidir=-1), 'n_bidir'), (dict(scale=0.0), 'sm_scale'), (dict(scale=-1.0), 'sm_scale'), (dict(q=24), '16-byte'),
    (dict(work=24), '16-byte'), (dict(counts=(1, 0, 0, 8, 12, 0, 0, 0, 0, 2)), 'the work list has 2'),
    (dict(counts=PARTS), 'workspace of 0 bytes'), (dict(counts=PARTS, ws=16, ws_bytes=33279), '33280 needed'),
    (dict(counts=(0, 0, 0, 8, 12, 1, 3, 1, 5, 1), ws=16, ws_bytes=100), 'needed')])
def test_attention_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        nat.call('morj_tree_attention_kv8', *attention_args(**kw))


def test_attention_refuses_other_head_sizes_and_accepts_nothing_to_do():
    with pytest.raises(nat.NativeFailure, match='head_dim 96'):
        nat.call('morj_tree_attention_kv8', *attention_args(d=96))
    nat.call('morj_tree_attention_kv8', *attention_args(counts=(0,)))


def test_pool_and_plan_refusals():
    with pytest.raises(ValueError, match='64 or 128'):
        kv8.KV8Pool(10, 2, 96, 'cpu')
    k = torch.zeros(70, 2, 64, dtype=torch.uint8)
    s = torch.zeros(2, 2)
    pool = kv8.KV8Pool.of(k, s, k.clone(), s.clone())
    assert (pool.slots, pool.heads, pool.head_dim, pool.nbytes) == (70, 2, 64, 2 * (70 * 128 + 16))
    with pytest.raises(ValueError, match='scales must be'):
        kv8.KV8Pool.of(k, s[:1], k, s)
    with pytest.raises(ValueError, match='scales must be'):
        kv8.KV8Pool.of(k, s.half(), k, s)
    with pytest.raises(ValueError, match='codes must be'):
        kv8.KV8Pool.of(k.float(), s, k.float(), s)
    with pytest.raises(ValueError, match='contiguous'):
        kv8.KV8Pool.of(torch.zeros(70, 2, 128, dtype=torch.uint8)[:, :, ::2], s, k, s)
    with pytest.raises(ValueError, match='int32'):
        pool.rows(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match='same slot'):
        kv8.StorePlan([1, 1], 70, 'cpu')
    plan = kv8.StorePlan([1, 2], 70, 'cpu')
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='k must be BF16'):
        kv8.store(pool, rows.float(), rows, plan)
    with pytest.raises(ValueError, match='v must be BF16'):
        kv8.store(pool, rows, rows[:1], plan)
    with pytest.raises(ValueError, match='contiguous'):
        kv8.store(pool, rows.transpose(0, 1), rows, plan)
    with pytest.raises(ValueError, match='pool of 80'):
        kv8.store(pool, rows, rows, kv8.StorePlan([1, 2], 80, 'cpu'))
    kv8.store(pool, rows[:0], rows[:0], kv8.StorePlan([], 70, 'cpu'))  # nothing to store: no launch
    with pytest.raises(ValueError, match='one entry per segment'):
        kv8.AttentionPlan([0, 1], [0, 1, 2], [0, 1], 2, 2, 64, device='cpu')
    with pytest.raises(ValueError, match='within kv_indices'):
        kv8.AttentionPlan([0, 1], [0, 3], [0, 1], 2, 2, 64, device='cpu')
    with pytest.raises(ValueError, match='head_dim 96'):
        kv8.AttentionPlan([0, 1], [0, 2], [0, 1], 2, 2, 96, device='cpu')
    with pytest.raises(ValueError, match='kv_last_page_len'):
        kv8.AttentionPlan([0, 1], [0, 2], [0, 1], 2, 2, 64, page_size=16, kv_last_page_len=[17], device='cpu')
    plan = kv8.AttentionPlan([0, 1], [0, 2], [0, 1], 4, 2, 64, device='cpu')
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for bad in (q.float(), q[:, :2], torch.zeros(1, 4, 128, dtype=torch.bfloat16)[:, :, ::2]):
        with pytest.raises(ValueError, match='q must be'):
            kv8.tree_attention(bad, pool, plan, 1.0)
    with pytest.raises(ValueError, match='the pool has'):
        kv8.tree_attention(torch.zeros(1, 4, 64, dtype=torch.bfloat16), kv8.KV8Pool(70, 1, 64, 'cpu'), plan, 1.0)
    with pytest.raises(ValueError, match='out must be'):
        kv8.tree_attention(q, pool, plan, 1.0, out=q.float())
    empty = kv8.AttentionPlan([0, 0], [0, 2], [0, 1], 4, 2, 64, device='cpu')
    assert kv8.tree_attention(q[:0], pool, empty, 1.0).shape == (0, 4, 64)


def test_tensors_that_are_not_on_a_cuda_device_are_refused():
    # (launched, the kernels would read host addresses)
    pool = kv8.KV8Pool(70, 2, 64, 'cpu')
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    plan = kv8.AttentionPlan([0, 1], [0, 2], [0, 1], 4, 2, 64, device='cpu')
    for bad in (lambda: kv8.store(pool, rows, rows, kv8.StorePlan([1, 2], 70, 'cpu')),
                lambda: pool.rows(torch.zeros(3, dtype=torch.int32)),
                lambda: kv8.tree_attention(torch.zeros(1, 4, 64, dtype=torch.bfloat16), pool, plan, 1.0)):
        with pytest.raises(ValueError, match='must be on a CUDA device, not on cpu'):
            bad()


@pytest.mark.parametrize('bad', [2**32 + 5, -2**32 + 5, 2**31])
def test_host_indices_past_32_bits_are_refused(bad):
    # (cast, 2^32 + 5 would be slot 5: another token's K/V overwritten, or read)
    for slots in (np.array([1, bad]), [1, bad]):
        with pytest.raises(ValueError, match='fit 32 bits'):
            nat.kv8_store_work(slots, 64)
        with pytest.raises(ValueError, match='fit 32 bits'):
            kv8.StorePlan(slots, 64, 'cpu')
    good = dict(qo_indptr=[0, 1], kv_indptr=[0, 2], kv_indices=[0, 1], kv_last_page_len=[1])
    for name in good:
        args = {**good, name: np.array(good[name][:-1] + [bad])}
        with pytest.raises(ValueError, match=f'{name} must fit 32 bits'):
            kv8.AttentionPlan(**args, hq=4, hk=2, d=64, device='cpu')
        with pytest.raises(ValueError, match=f'{name} must fit 32 bits'):
            nat.kv8_attention_work(**args, n_bidir=0, hq=4, hk=2, window=0)


def test_host_indices_that_are_not_whole_numbers_are_refused():
    with pytest.raises(ValueError, match='slots must be integers'):
        kv8.StorePlan([1.5, 2.0], 64, 'cpu')
    with pytest.raises(ValueError, match='kv_indices must be integers'):
        kv8.AttentionPlan([0, 1], [0, 2], np.array([0.0, 1.0]), 4, 2, 64, device='cpu')
    work, blocks = nat.kv8_store_work(np.array([70, 3], np.uint64), 128)
    assert blocks == 2 and work[6:].tolist() == [3, 1, 70, 0]


def test_a_last_page_holds_from_none_to_all_of_its_slots():
    # (more would list keys past the segment's pages: reads past the list)
    for page, last in [(16, 17), (16, -1), (1, 2), (1, -1)]:
        with pytest.raises(ValueError, match='the last page of segment 1 holds'):
            nat.kv8_attention_work([0, 1, 2], [0, 2, 4], range(4), 0, 4, 2, 0, page, [page, last])
    for page in (1, 16):
        for last in (0, 1):
            work, counts = nat.kv8_attention_work([0, 1], [0, 3], range(3), 0, 4, 2, 0, page, [last])
            assert counts[0] == 1 and work[11] == 2 * page + last == work[3]
    work, _ = nat.kv8_attention_work([0, 1], [0, 0], [], 0, 4, 2, 0, 16, [0])
    assert work[11] == 0


def test_queries_in_front_of_the_first_row_are_refused():
    # (their rows would be read and written in front of q and out)
    for qo in ([-3, 2], [-2**31, 2**31 - 1], [0, -1]):
        with pytest.raises(ValueError, match='out of order'):
            nat.kv8_attention_work(qo, [0, 4], range(4), 0, 4, 2, 0)
    work, counts = nat.kv8_attention_work([3, 5], [0, 4], range(4), 0, 4, 2, 0)
    assert counts[9] == 5 and work[8] == 3
