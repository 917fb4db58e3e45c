"""The 8-bit K/V cache on the GPU: the store's codes and scales exactly as the definition gives them, the attention
within the elementwise bound that `kv8_cases.attention_ref` derives from its roundings."""
import numpy as np
import pytest
import torch

from kv8_cases import (BLOCK, attention_ref, e4m3, fill, make_segments, pool_rows, segments, store_ref)
from morj_b200 import _native as nat
from morj_b200 import kv8

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    nat.lib()
    yield
    torch.cuda.synchronize()
    assert nat.device_error(torch.cuda.current_stream().cuda_stream) == 0


def values(pool):
    return (pool.k.float(), pool.k_scale), (pool.v.float(), pool.v_scale)


def random_pool(g, slots, hk, d, filled=True):
    pool = kv8.KV8Pool(slots, hk, d, DEV)
    pool.k.view(torch.uint8).zero_()
    pool.v.view(torch.uint8).zero_()
    if filled:
        kv8.store(pool, pool_rows(g, slots, hk, d, DEV), pool_rows(g, slots, hk, d, DEV),
                  kv8.StorePlan(np.arange(slots), slots, DEV))
    return pool


def check_store(pool, k, v, slots, plan=None):
    before = [(c.double(), s.clone()) for c, s in values(pool)]
    kv8.store(pool, k, v, plan or kv8.StorePlan(slots, pool.slots, DEV))
    for (c, s), (c0, s0), rows in zip(values(pool), before, (k, v)):
        want, want_s = store_ref(rows, slots, c0, s0)
        assert torch.equal(s.double(), want_s)
        assert torch.equal(c.double(), want)


@pytest.mark.parametrize('n,hk,d,slots', [(1, 1, 64, 1), (1, 16, 128, 640), (3, 2, 64, 70), (64, 2, 128, 64),
                                          (65, 3, 64, 65), (200, 5, 128, 1000), (777, 2, 64, 777)])
@pytest.mark.parametrize('filled', [False, True])
def test_store_is_the_definition(n, hk, d, slots, filled):
    g = torch.Generator(device=DEV).manual_seed(n + d)
    pool = random_pool(g, slots, hk, d, filled)
    where = np.random.default_rng(n).permutation(slots)[:n]
    check_store(pool, pool_rows(g, n, hk, d, DEV, gain=2.0), pool_rows(g, n, hk, d, DEV, 1.0), where)
    # again, larger: every touched scale grows and the resident codes move
    check_store(pool, pool_rows(g, n, hk, d, DEV, gain=300.0), pool_rows(g, n, hk, d, DEV, gain=0.01), where[::-1].copy())


@pytest.mark.parametrize('value', [0.0, -0.0, 448.0, 449.0, 3.5, 3.515625, 1e-30, 9.2e-41, 3.3895e38, -3.3895e38, 2.0 ** -109,
                                   57344.0])
def test_store_at_the_ends_of_the_range(value):
    x = torch.full((2, 2, 64), value, dtype=torch.bfloat16, device=DEV)
    x[1, :, ::3] *= 0.0007
    pool = random_pool(None, 100, 2, 64, filled=False)
    check_store(pool, x, x.flip(0).contiguous(), [99, 64])
    back = pool.rows(torch.tensor([99, 64], dtype=torch.int32, device=DEV))[0]
    assert torch.isfinite(back).all()


def test_store_moves_resident_codes_into_subnormals_and_to_zero():
    g = torch.Generator(device=DEV).manual_seed(0)
    pool = random_pool(g, 64, 1, 64)
    check_store(pool, pool_rows(g, 1, 1, 64, DEV, gain=2.0 ** 14), pool_rows(g, 1, 1, 64, DEV, gain=2.0 ** 40), [10])


def test_store_does_not_depend_on_the_order_of_its_rows_and_leaves_other_slots():
    g = torch.Generator(device=DEV).manual_seed(1)
    n, hk, d, slots = 150, 4, 128, 500
    k, v = pool_rows(g, n, hk, d, DEV), pool_rows(g, n, hk, d, DEV)
    where = np.random.default_rng(2).permutation(slots)[:n]
    pools = []
    for order in (np.arange(n), np.random.default_rng(3).permutation(n)):
        pool = random_pool(None, slots, hk, d, filled=False)
        pool.k.view(torch.uint8).fill_(0x5a)
        pool.v.view(torch.uint8).fill_(0x7f)
        idx = torch.as_tensor(order, device=DEV)
        kv8.store(pool, k[idx].contiguous(), v[idx].contiguous(), kv8.StorePlan(where[order], slots, DEV))
        pools.append(pool)
    for a, b in zip((pools[0].k, pools[0].v), (pools[1].k, pools[1].v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    other = torch.ones(slots, dtype=torch.bool, device=DEV)
    other[torch.as_tensor(where, device=DEV)] = False
    assert (pools[0].k.view(torch.uint8)[other] == 0x5a).all() and (pools[0].v.view(torch.uint8)[other] == 0x7f).all()
    assert torch.equal(pools[0].k_scale, pools[1].k_scale)
    hit = torch.zeros(len(pools[0].k_scale), dtype=torch.bool, device=DEV)
    hit[torch.as_tensor(where // BLOCK, device=DEV)] = True
    assert (pools[0].k_scale[~hit] == 0).all() and (pools[0].k_scale[hit] > 0).all()


def test_store_of_strided_rows_and_a_poisoned_fresh_pool():
    g = torch.Generator(device=DEV).manual_seed(4)
    n, hk, d = 90, 2, 128
    wide = torch.full((n, 3 * hk, d), float('nan'), dtype=torch.bfloat16, device=DEV)
    wide[:, hk:2 * hk] = pool_rows(g, n, hk, d, DEV)
    wide[:, :hk] = pool_rows(g, n, hk, d, DEV)
    pool = kv8.KV8Pool(n, hk, d, DEV)
    pool.k.view(torch.uint8).fill_(0x7f)
    pool.v.view(torch.uint8).fill_(0x7f)
    pool.k_scale.fill_(float('nan'))
    pool.v_scale.fill_(float('nan'))
    k, v = wide[:, hk:2 * hk], wide[:, :hk]
    plan = kv8.StorePlan(np.arange(n)[::-1], n, DEV)
    kv8.store(pool, k, v, plan)
    fresh = torch.zeros(n, hk, d, dtype=torch.float64, device=DEV)
    zero = torch.zeros_like(pool.k_scale)
    for (c, s), rows in zip(values(pool), (k, v)):
        want, want_s = store_ref(rows, np.arange(n)[::-1], fresh, zero)
        assert torch.equal(c.double(), want) and torch.equal(s.double(), want_s)


def test_store_reports_values_that_are_not_finite():
    g = torch.Generator(device=DEV).manual_seed(5)
    pool = random_pool(g, 64, 1, 64)
    k = pool_rows(g, 2, 1, 64, DEV)
    k[0, 0, 3], k[0, 0, 4], k[1, 0, 5] = float('nan'), float('inf'), -float('inf')
    check_store(pool, k, pool_rows(g, 2, 1, 64, DEV), [7, 9])
    assert nat.device_error(torch.cuda.current_stream().cuda_stream) == 0x303


def test_rows_are_the_codes_times_their_scale_and_bad_slots_are_reported():
    g = torch.Generator(device=DEV).manual_seed(6)
    pool = random_pool(g, 300, 3, 64)
    slots = torch.tensor([0, 299, 64, 64, 5], dtype=torch.int32, device=DEV)
    for got, codes, scale in zip(pool.rows(slots), (pool.k, pool.v), (pool.k_scale, pool.v_scale)):
        want = codes[slots.long()].double() * scale[slots.long() // BLOCK].double()[:, :, None]
        assert torch.equal(got.double(), want)
    assert pool.rows(slots[:0])[0].shape == (0, 3, 64)
    out = torch.full((2, 3, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    bad = torch.tensor([300, 1], dtype=torch.int32, device=DEV)
    s = torch.cuda.current_stream().cuda_stream
    nat.call('morj_kv8_gather', pool.k.data_ptr(), pool.k_scale.data_ptr(), 300, bad.data_ptr(), 2, 3, 64, out.data_ptr(),
             192, s)
    assert nat.device_error(s) == 0x301 and (out[0] == 7).all() and (out[1] != 7).any()


# ---- attention ------------------------------------------------------------------------------------------------------

def check_attention(pool, q, qo, kv, indices, last, page, window, n_bidir, sm_scale, out=None):
    hq, d = q.shape[1:]
    plan = kv8.AttentionPlan(qo, kv, indices, hq, pool.heads, d, page_size=page, kv_last_page_len=last, window=window,
                             n_bidir=n_bidir, device=DEV)
    got = kv8.tree_attention(q, pool, plan, sm_scale, out=out)
    want, bound = attention_ref(q, pool.k, pool.k_scale, pool.v, pool.v_scale, qo, kv, indices, last, page, window,
                                n_bidir, sm_scale)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    worst = (err / bound).max().item()
    assert worst <= 1, f'{worst:.3g} of the bound, max err {err.max().item():.3g}'
    # the same call again gives the same bits
    assert torch.equal(got, kv8.tree_attention(q, pool, plan, sm_scale))
    return got, plan


SPECS = {
    'one key': [(1, 1)],
    'singles': [(1, 5), (1, 64), (1, 1), (1, 333), (1, 32), (1, 1000)],
    'long single': [(1, 20000)],
    'long singles': [(1, 3001), (1, 2000), (1, 7), (1, 4096)],
    'nothing to see': [(1, 0), (3, 1), (2, 40), (0, 10), (5, 0)],
    'few queries': [(2, 70), (4, 4), (7, 500)],
    'prompt': [(130, 130), (60, 190), (60, 200)],
    'long and short': [(300, 1300), (1, 2500), (64, 64), (17, 900)],
}


@pytest.mark.parametrize('name', SPECS)
@pytest.mark.parametrize('hq,hk,d', [(4, 2, 64), (32, 16, 128), (3, 3, 128), (8, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize('window,page', [(0, 1), (40, 64), (1000, 5)])
def test_attention_matches_the_definition(name, hq, hk, d, window, page):
    spec = SPECS[name]
    rng = np.random.default_rng(len(name) + window)
    g = torch.Generator(device=DEV).manual_seed(len(name))
    qo, kv, indices, last, slots = make_segments(rng, spec, page)
    pool = random_pool(g, slots, hk, d)
    q = torch.randn(int(qo[-1]), hq, d, generator=g, device=DEV).to(torch.bfloat16)
    check_attention(pool, q, qo, kv, indices, last, page, window, 0, d ** -0.5)


@pytest.mark.parametrize('hq,hk', [(64, 2), (40, 1), (12, 1), (16, 1)])
def test_attention_of_large_head_groups(hq, hk):
    rng, g = np.random.default_rng(0), torch.Generator(device=DEV).manual_seed(0)
    qo, kv, indices, last, slots = make_segments(rng, [(1, 700), (3, 50), (1, 9)], 16)
    pool = random_pool(g, slots, hk, 64)
    q = torch.randn(5, hq, 64, generator=g, device=DEV).to(torch.bfloat16)
    check_attention(pool, q, qo, kv, indices, last, 16, 0, 0, 0.125)


@pytest.mark.parametrize('window', [0, 20, 500])
def test_attention_of_image_blocks(window):
    rng, g = np.random.default_rng(1), torch.Generator(device=DEV).manual_seed(1)
    qo, kv, indices, last, slots = make_segments(rng, [(50, 50), (70, 200), (40, 300)], 1)
    pool = random_pool(g, slots, 2, 128)
    q = torch.randn(int(qo[-1]), 4, 128, generator=g, device=DEV).to(torch.bfloat16)
    check_attention(pool, q, qo, kv, indices, None, 1, window, 2, 128 ** -0.5)


def test_attention_over_a_shared_prefix_in_slot_order():
    g = torch.Generator(device=DEV).manual_seed(2)
    P, B, L = 700, 5, 33
    lists = [np.arange(P)] + [np.concatenate([np.arange(P), P + b * L + np.arange(L)]) for b in range(B)]
    qo = np.concatenate([[0], np.cumsum([P] + [L] * B)]).astype(np.int32)
    kv = np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)
    pool = random_pool(g, P + B * L, 4, 128)
    q = torch.randn(int(qo[-1]), 8, 128, generator=g, device=DEV).to(torch.bfloat16)
    check_attention(pool, q, qo, kv, np.concatenate(lists).astype(np.int32), None, 1, 0, 0, 0.1)
    check_attention(pool, q, qo, kv, np.concatenate(lists).astype(np.int32), None, 1, 128, 0, 0.1)


@pytest.mark.parametrize('spec', [[(1, 2000), (1, 90)], [(130, 700)]])
def test_attention_with_scales_far_apart(spec):
    # K and V blocks whose scales differ by up to 2^20, and a few huge and tiny query rows
    rng, g = np.random.default_rng(3), torch.Generator(device=DEV).manual_seed(3)
    qo, kv, indices, last, slots = make_segments(rng, spec, 1)
    k, v = pool_rows(g, slots, 2, 64, DEV), pool_rows(g, slots, 2, 64, DEV)
    gain = torch.exp2(torch.randint(-10, 11, ((slots + 63) // 64, 1, 1), generator=g, device=DEV).float())
    v = (v.float() * gain.repeat_interleave(64, 0)[:slots]).to(torch.bfloat16)
    gain = torch.exp2(torch.randint(-6, 1, ((slots + 63) // 64, 1, 1), generator=g, device=DEV).float())
    k = (k.float() * gain.repeat_interleave(64, 0)[:slots]).to(torch.bfloat16)
    pool = kv8.KV8Pool(slots, 2, 64, DEV)
    kv8.store(pool, k, v, kv8.StorePlan(np.arange(slots), slots, DEV))
    q = torch.randn(int(qo[-1]), 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    q[0, 0] *= 2.0 ** -60
    q[0, 2] = 0
    check_attention(pool, q, qo, kv, indices, last, 1, 0, 0, 0.125)
    q[0, 1] *= 100
    check_attention(pool, q, qo, kv, indices, last, 1, 0, 0, 0.125)


def test_attention_reads_nothing_a_query_may_not_see():
    # every slot but the listed ones, and what lies past a last page's end or before the window, is NaN
    rng, g = np.random.default_rng(4), torch.Generator(device=DEV).manual_seed(4)
    for spec, window, page in [([(1, 70), (1, 129), (1, 1)], 0, 64), ([(1, 2000), (1, 300)], 100, 64),
                               ([(9, 90), (70, 1000), (1, 500)], 0, 64), ([(40, 600)], 64, 1)]:
        qo, kv, indices, last, slots = make_segments(rng, spec, page)
        good = random_pool(g, slots, 2, 64)
        codes = [torch.full_like(c.view(torch.uint8), 0x7f) for c in (good.k, good.v)]
        scales = [torch.full_like(s, float('nan')) for s in (good.k_scale, good.v_scale)]
        for s, (n, keys) in enumerate(spec):
            pages = indices[kv[s]:kv[s + 1]].astype(np.int64)
            at = (pages[:, None] * page + np.arange(page)).reshape(-1)[:keys]
            at = at[max(0, keys - n - (window - 1)) if window else 0:]
            at = torch.as_tensor(at, device=DEV)
            for new, old in zip(codes, (good.k, good.v)):
                new[at] = old.view(torch.uint8)[at]
            for new, old in zip(scales, (good.k_scale, good.v_scale)):
                new[at // BLOCK] = old[at // BLOCK]
        pool = kv8.KV8Pool.of(codes[0], scales[0], codes[1], scales[1])
        q = torch.randn(int(qo[-1]), 4, 64, generator=g, device=DEV).to(torch.bfloat16)
        plan = kv8.AttentionPlan(qo, kv, indices, 4, 2, 64, page_size=page, kv_last_page_len=last, window=window, device=DEV)
        got = kv8.tree_attention(q, pool, plan, 0.125)
        want, _ = check_attention(good, q, qo, kv, indices, last, page, window, 0, 0.125)
        assert torch.equal(got, want)


def test_attention_reports_a_slot_outside_the_pool():
    g = torch.Generator(device=DEV).manual_seed(7)
    pool = random_pool(g, 100, 2, 64)
    plan = kv8.AttentionPlan([0, 1], [0, 3], [5, 100, 7], 4, 2, 64, device=DEV)
    kv8.tree_attention(torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV), pool, plan, 1.0)
    assert nat.device_error(torch.cuda.current_stream().cuda_stream) == 0x301


def test_attention_carries_nan_and_overflow_as_the_formula_does():
    g = torch.Generator(device=DEV).manual_seed(8)
    pool = random_pool(g, 128, 1, 64)
    q = torch.randn(2, 2, 64, generator=g, device=DEV).to(torch.bfloat16)
    q[0, 0, 3] = float('nan')
    plan = kv8.AttentionPlan([0, 1, 2], [0, 64, 128], np.arange(128), 2, 1, 64, device=DEV)
    got = kv8.tree_attention(q, pool, plan, 0.125)
    assert torch.isnan(got[0, 0]).all() and torch.isfinite(got[0, 1]).all() and torch.isfinite(got[1]).all()


def test_other_streams_graphs_and_given_outputs():
    g = torch.Generator(device=DEV).manual_seed(9)
    rng = np.random.default_rng(9)
    qo, kv, indices, last, slots = make_segments(rng, [(1, 3000), (1, 900), (20, 100)], 1)
    pool = random_pool(g, slots, 2, 128)
    q = torch.randn(int(qo[-1]), 4, 128, generator=g, device=DEV).to(torch.bfloat16)
    buf = torch.full((q.shape[0] + 2, 4, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    want, plan = check_attention(pool, q, qo, kv, indices, last, 1, 0, 0, 0.1, out=buf[1:-1])
    assert (buf[0] == 5).all() and (buf[-1] == 5).all()
    k, v = pool_rows(g, 3, 2, 128, DEV), pool_rows(g, 3, 2, 128, DEV)
    where = [int(indices[0]), int(indices[kv[1]]), int(indices[kv[2]])]
    store_plan = kv8.StorePlan(where, slots, DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(kv8.tree_attention(q, pool, plan, 0.1), want)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs: each has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kv8.store(pool, k, v, store_plan)
            outs.append(kv8.tree_attention(q, pool, plan, 0.1))
        graphs.append(graph)
    torch.cuda.synchronize()
    assert torch.equal(kv8.tree_attention(q, pool, plan, 0.1), want)  # (capturing stored nothing)
    graphs[0].replay()
    torch.cuda.synchronize()
    new = kv8.tree_attention(q, pool, plan, 0.1)
    assert torch.equal(outs[0], new) and not torch.equal(new, want)
    k.mul_(0.5)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], kv8.tree_attention(q, pool, plan, 0.1))


def test_a_pool_beyond_32_bit_offsets():
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip('needs 20 GB')
    hk, d = 16, 128
    slots = (1 << 32) // (hk * d) + 200  # more than 2^32 codes in K alone
    pool = kv8.KV8Pool(slots, hk, d, DEV)
    g = torch.Generator(device=DEV).manual_seed(10)
    where = np.concatenate([np.arange(slots - 150, slots), np.arange(20), (1 << 31) // (hk * d) + np.arange(-3, 4)])
    k, v = pool_rows(g, len(where), hk, d, DEV), pool_rows(g, len(where), hk, d, DEV)
    kv8.store(pool, k, v, kv8.StorePlan(where, slots, DEV))
    at = torch.as_tensor(where, dtype=torch.int32, device=DEV)
    for got, rows in zip(pool.rows(at), (k, v)):
        # a value is off by half an e4m3 step: 2^-4 of it, or of the smallest normal code (2^-6) below that
        small = 2.0 ** -10 * pool.k_scale.max() if rows is k else 2.0 ** -10 * pool.v_scale.max()
        assert ((got.double() - rows.double()).abs() <= rows.double().abs() * 2.0 ** -4 + small).all()
    q = torch.randn(1, 32, d, generator=g, device=DEV).to(torch.bfloat16)
    plan = kv8.AttentionPlan([0, 1], [0, len(where)], where, 32, hk, d, device=DEV)
    got = kv8.tree_attention(q, pool, plan, 0.1)
    small = kv8.KV8Pool(len(where), hk, d, DEV)
    # the same rows in a small pool, their codes and scales copied
    for a, b, sa, sb in ((pool.k, small.k, pool.k_scale, small.k_scale), (pool.v, small.v, pool.v_scale, small.v_scale)):
        b.view(torch.uint8).copy_(a.view(torch.uint8)[at.long()])
    out = torch.zeros(1, 32, d, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    for h in range(hk):
        kd, vd = (c[:, h].double() * s[at.long() // BLOCK, h].double()[:, None]
                  for c, s in ((small.k, pool.k_scale), (small.v, pool.v_scale)))
        for j in (2 * h, 2 * h + 1):
            p = torch.softmax(q[0, j].double() @ kd.T * 0.1, 0)
            out[0, j] = p @ vd
            bound[0, j] = out[0, j].abs() * 2.0 ** -8 + (p @ vd.abs()) * 2.0 ** -9
    assert ((got.double() - out).abs() <= bound).all()


# ---- attention of calls with many rows (128-row tiles on expanded pages) ----------------------------------------------

MANY = {
    'nothing to see': [(300, 40), (40, 0), (0, 10), (900, 1500), (3, 1)],
    'prompts': [(700, 700), (401, 1101), (60, 1130)],
    'ends inside a tile': [(129, 2049), (640, 1999), (127, 1)],
    'with few rows': [(800, 1300), (1, 2500), (8, 8), (1, 0)],
}


@pytest.mark.parametrize('name', MANY)
@pytest.mark.parametrize('hq,hk,d', [(4, 2, 64), (16, 16, 128), (9, 3, 128), (8, 1, 64)])
@pytest.mark.parametrize('window,page', [(0, 1), (500, 64), (1000, 5)])
def test_attention_of_many_rows_matches_the_definition(name, hq, hk, d, window, page):
    spec = MANY[name]
    rng = np.random.default_rng(len(name) + window)
    g = torch.Generator(device=DEV).manual_seed(len(name))
    qo, kv, indices, last, slots = make_segments(rng, spec, page)
    pool = random_pool(g, slots, hk, d)
    q = torch.randn(int(qo[-1]), hq, d, generator=g, device=DEV).to(torch.bfloat16)
    _, plan = check_attention(pool, q, qo, kv, indices, last, page, window, 0, d ** -0.5)
    assert plan.counts[5] > 0


@pytest.mark.parametrize('window', [0, 300, 500])
def test_attention_of_large_image_blocks(window):
    rng, g = np.random.default_rng(1), torch.Generator(device=DEV).manual_seed(1)
    qo, kv, indices, last, slots = make_segments(rng, [(500, 500), (700, 1200), (400, 900)], 1)
    pool = random_pool(g, slots, 4, 128)
    q = torch.randn(int(qo[-1]), 8, 128, generator=g, device=DEV).to(torch.bfloat16)
    _, plan = check_attention(pool, q, qo, kv, indices, None, 1, window, 2, 128 ** -0.5)
    assert plan.counts[5] > 0


def test_attention_of_many_rows_with_scales_far_apart():
    rng, g = np.random.default_rng(3), torch.Generator(device=DEV).manual_seed(3)
    qo, kv, indices, last, slots = make_segments(rng, [(500, 2000)], 1)
    k, v = pool_rows(g, slots, 2, 64, DEV), pool_rows(g, slots, 2, 64, DEV)
    gain = torch.exp2(torch.randint(-10, 11, ((slots + 63) // 64, 1, 1), generator=g, device=DEV).float())
    v = (v.float() * gain.repeat_interleave(64, 0)[:slots]).to(torch.bfloat16)
    gain = torch.exp2(torch.randint(-6, 1, ((slots + 63) // 64, 1, 1), generator=g, device=DEV).float())
    k = (k.float() * gain.repeat_interleave(64, 0)[:slots]).to(torch.bfloat16)
    pool = kv8.KV8Pool(slots, 2, 64, DEV)
    kv8.store(pool, k, v, kv8.StorePlan(np.arange(slots), slots, DEV))
    q = torch.randn(int(qo[-1]), 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    q[0, 0] *= 2.0 ** -60
    q[0, 2] = 0
    q[0, 1] *= 100
    _, plan = check_attention(pool, q, qo, kv, indices, last, 1, 0, 0, 0.125)
    assert plan.counts[5] > 0


@pytest.mark.parametrize('spec,window,page', [([(9, 90), (700, 3000), (1, 500)], 0, 64), ([(6000, 6200)], 64, 1),
                                              ([(300, 4000), (200, 1111)], 700, 16)])
def test_attention_of_many_rows_reads_nothing_a_query_may_not_see(spec, window, page):
    rng, g = np.random.default_rng(4), torch.Generator(device=DEV).manual_seed(4)
    qo, kv, indices, last, slots = make_segments(rng, spec, page)
    good = random_pool(g, slots, 2, 64)
    codes = [torch.full_like(c.view(torch.uint8), 0x7f) for c in (good.k, good.v)]
    scales = [torch.full_like(s, float('nan')) for s in (good.k_scale, good.v_scale)]
    for s, (n, keys) in enumerate(spec):
        pages = indices[kv[s]:kv[s + 1]].astype(np.int64)
        at = (pages[:, None] * page + np.arange(page)).reshape(-1)[:keys]
        at = at[max(0, keys - n - (window - 1)) if window else 0:]
        if window:  # (whole pages are expanded from the first one a query sees on: its unseen slots are the caller's too)
            first = max(0, keys - n - (window - 1)) // page * page
            at = (pages[:, None] * page + np.arange(page)).reshape(-1)[first:keys]
        at = torch.as_tensor(at, device=DEV)
        for new, old in zip(codes, (good.k, good.v)):
            new[at] = old.view(torch.uint8)[at]
        for new, old in zip(scales, (good.k_scale, good.v_scale)):
            new[at // BLOCK] = old[at // BLOCK]
    pool = kv8.KV8Pool.of(codes[0], scales[0], codes[1], scales[1])
    q = torch.randn(int(qo[-1]), 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    plan = kv8.AttentionPlan(qo, kv, indices, 4, 2, 64, page_size=page, kv_last_page_len=last, window=window, device=DEV)
    assert plan.counts[5] > 0
    got = kv8.tree_attention(q, pool, plan, 0.125)
    want, _ = check_attention(good, q, qo, kv, indices, last, page, window, 0, 0.125)
    assert torch.equal(got, want)


def test_attention_of_many_rows_reports_a_slot_outside_the_pool():
    g = torch.Generator(device=DEV).manual_seed(7)
    pool = random_pool(g, 2000, 2, 64)
    where = np.arange(2000)
    where[1234] = 2000
    plan = kv8.AttentionPlan([0, 700], [0, 2000], where, 4, 2, 64, device=DEV)
    assert plan.counts[5] > 0
    kv8.tree_attention(torch.zeros(700, 4, 64, dtype=torch.bfloat16, device=DEV), pool, plan, 1.0)
    assert nat.device_error(torch.cuda.current_stream().cuda_stream) == 0x301


def test_attention_of_many_rows_on_streams_in_graphs_and_into_given_outputs():
    g = torch.Generator(device=DEV).manual_seed(9)
    qo, kv, indices, last, slots = make_segments(np.random.default_rng(9), [(500, 1500), (1, 900), (20, 100)], 1)
    pool = random_pool(g, slots, 2, 128)
    q = torch.randn(int(qo[-1]), 4, 128, generator=g, device=DEV).to(torch.bfloat16)
    buf = torch.full((q.shape[0] + 2, 4, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    want, plan = check_attention(pool, q, qo, kv, indices, last, 1, 0, 0, 0.1, out=buf[1:-1])
    assert plan.counts[5] > 0 and (buf[0] == 5).all() and (buf[-1] == 5).all()
    side, outs, graphs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    with torch.cuda.stream(side):  # two calls of one plan at once
        other = kv8.tree_attention(q, pool, plan, 0.1)
    here = kv8.tree_attention(q, pool, plan, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(other, want) and torch.equal(here, want)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kv8.tree_attention(q, pool, plan, 0.1))
        graphs.append(graph)
    q.mul_(0.5)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], kv8.tree_attention(q, pool, plan, 0.1))
    assert not torch.equal(outs[0], want)


def test_many_rows_over_a_pool_beyond_32_bit_offsets():
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip('needs 20 GB')
    hk, d = 16, 128
    slots = (1 << 32) // (hk * d) + 200  # more than 2^32 codes in K alone
    pool = kv8.KV8Pool(slots, hk, d, DEV)
    g = torch.Generator(device=DEV).manual_seed(10)
    where = np.concatenate([np.arange(slots - 150, slots), np.arange(20), (1 << 31) // (hk * d) + np.arange(-3, 4)])
    n = len(where)
    k, v = pool_rows(g, n, hk, d, DEV), pool_rows(g, n, hk, d, DEV)
    kv8.store(pool, k, v, kv8.StorePlan(where, slots, DEV))
    # the same blocks of the large pool, with their codes and scales, one after another in a small one
    blocks, index = np.unique(where // BLOCK, return_inverse=True)
    at = index * BLOCK + where % BLOCK
    near = kv8.KV8Pool(len(blocks) * BLOCK, hk, d, DEV)
    for big, small, sb, ss in ((pool.k, near.k, pool.k_scale, near.k_scale), (pool.v, near.v, pool.v_scale, near.v_scale)):
        small.view(torch.uint8)[at] = big.view(torch.uint8)[torch.as_tensor(where, device=DEV)]
        ss.copy_(sb[torch.as_tensor(blocks, device=DEV)])
    q = torch.randn(400, 32, d, generator=g, device=DEV).to(torch.bfloat16)
    out = []
    for p, slot in ((pool, where), (near, at)):
        plan = kv8.AttentionPlan([0, 400], [0, n], slot, 32, hk, d, device=DEV)
        assert plan.counts[5] > 0
        out.append(kv8.tree_attention(q, p, plan, 0.1))
    assert torch.equal(out[0], out[1])


def test_a_rounded_value_is_the_nearest_code():
    # every e4m3 value and the midpoints between neighbours, against the reference rounding
    bits = torch.arange(256, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).float()
    vals = torch.sort(bits[torch.isfinite(bits)]).values
    mid = torch.cat([vals, (vals[1:] + vals[:-1]) / 2])
    mid = mid[mid == mid.to(torch.bfloat16).float()]
    n = (len(mid) + 63) // 64
    x = torch.zeros(n, 1, 64, device=DEV)
    x.view(-1)[:len(mid)] = mid
    x[:, 0, 0] = 448  # scale 1 in every block
    pool = random_pool(None, n * 64, 1, 64, filled=False)
    x = x.to(torch.bfloat16)
    check_store(pool, x, x, np.arange(n) * 64)
    assert (pool.k_scale == 1).all()
    assert torch.equal(pool.k.double()[::64][:, 0], e4m3(x[:, 0].double()))


# ---- what no query, or another tile's queries only, may see -----------------------------------------------------------

def hidden_as_nan(good, qo, kv, indices, last, page, window):
    """A copy of the pool whose codes and scales are NaN except in the slots that some query sees (a block's scale stays
    where one of its slots does)."""
    pool = kv8.KV8Pool(good.slots, good.heads, good.head_dim, DEV)
    for t in (pool.k, pool.v):
        t.view(torch.uint8).fill_(0x7f)
    pool.scales.fill_(float('nan'))
    for s, (_, n, keys) in enumerate(segments(qo, kv, last, page)):
        pages = indices[kv[s]:kv[s + 1]].astype(np.int64)
        at = (pages[:, None] * page + np.arange(page)).reshape(-1)[:keys]
        at = torch.as_tensor(at[max(0, keys - n - (window - 1)) if window else 0:], device=DEV)
        for new, old in ((pool.k, good.k), (pool.v, good.v)):
            new.view(torch.uint8)[at] = old.view(torch.uint8)[at]
        for new, old in ((pool.k_scale, good.k_scale), (pool.v_scale, good.v_scale)):
            new[at // BLOCK] = old[at // BLOCK]
    return pool


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('spec,window,page', [([(300, 4000), (200, 1111)], 700, 16), ([(300, 4000), (200, 1111)], 701, 64),
                                              ([(500, 2000), (1, 900), (400, 3333)], 333, 256), ([(2000, 6200)], 65, 1000),
                                              ([(300, 4000), (200, 1111)], 700, 1)])
def test_attention_of_many_rows_ignores_a_window_s_first_page_before_the_window(spec, window, page, d):
    rng, g = np.random.default_rng(page), torch.Generator(device=DEV).manual_seed(page)
    qo, kv, indices, last, slots = make_segments(rng, spec, page)
    good = kv8.KV8Pool(slots, 2, d, DEV)
    fill(good, pool_rows(g, slots, 2, d, DEV), pool_rows(g, slots, 2, d, DEV), np.arange(slots), kv8.store, kv8.StorePlan)
    pool = hidden_as_nan(good, qo, kv, indices, last, page, window)
    q = torch.randn(int(qo[-1]), 4, d, generator=g, device=DEV).to(torch.bfloat16)
    plan = kv8.AttentionPlan(qo, kv, indices, 4, 2, d, page_size=page, kv_last_page_len=last, window=window, device=DEV)
    assert plan.counts[5] > 0
    got = kv8.tree_attention(q, pool, plan, d ** -0.5)
    want, _ = check_attention(good, q, qo, kv, indices, last, page, window, 0, d ** -0.5)
    assert torch.equal(got, want)


def test_attention_of_many_rows_keeps_another_segment_s_nan_out():
    # two segments list the same pages; the shorter one ends inside a page whose further slots hold NaN
    g = torch.Generator(device=DEV).manual_seed(12)
    good = random_pool(g, 2048, 2, 64)
    lists = np.random.default_rng(12).permutation(32)
    qo, kv, indices, last = [0, 400, 900], [0, 24, 48], np.concatenate([lists[:24], lists[:24]]), [10, 64]
    q = torch.randn(900, 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    plan = kv8.AttentionPlan(qo, kv, indices, 4, 2, 64, page_size=64, kv_last_page_len=last, device=DEV)
    assert plan.counts[5] > 0
    want = kv8.tree_attention(q, good, plan, 0.125)
    good.k.view(torch.uint8)[int(lists[23]) * 64 + 10:int(lists[23]) * 64 + 64] = 0x7f
    good.v.view(torch.uint8)[int(lists[23]) * 64 + 10:int(lists[23]) * 64 + 64] = 0x7f
    got = kv8.tree_attention(q, good, plan, 0.125)
    assert torch.equal(got[:400], want[:400]) and torch.isnan(got[-1]).all()


# ---- V scales of a call further apart than one FP16 range -------------------------------------------------------------

def scaled_segments(spec, gains, page, d, seed):
    """Segments over private pages, the V rows of segment s times 2^gains[s] in head 1 (head 0 stays as it is)."""
    rng, g = np.random.default_rng(seed), torch.Generator(device=DEV).manual_seed(seed)
    qo, kv, indices, last, slots = make_segments(rng, spec, page)
    k, v = pool_rows(g, slots, 2, d, DEV), pool_rows(g, slots, 2, d, DEV)
    for s, gain in enumerate(gains):
        pages = torch.as_tensor(indices[kv[s]:kv[s + 1]].astype(np.int64), device=DEV)
        at = (pages[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
        v[at, 1] = (v[at, 1].float() * 2.0 ** gain).to(torch.bfloat16)
    pool = kv8.KV8Pool(slots, 2, d, DEV)
    fill(pool, k, v, np.arange(slots), kv8.store, kv8.StorePlan)
    q = torch.randn(int(qo[-1]), 4, d, generator=g, device=DEV).to(torch.bfloat16)
    return pool, q, qo, kv, indices, last


@pytest.mark.parametrize('gains', [(0, -30, 0, 0), (-70, 0, 40, 3), (0, 0, 60, -60), (0, 20, 10, -10)])
@pytest.mark.parametrize('window,d,page', [(0, 128, 64), (0, 64, 128), (400, 128, 64)])
def test_attention_of_many_rows_over_segments_whose_v_scales_are_far_apart(gains, window, d, page):
    # (pages of whole scale blocks; each segment is held to its own largest V, `attention_ref`)
    spec = [(300, 1500), (500, 3900), (40, 700), (260, 260)]
    args = scaled_segments(spec, gains, page, d, 21)
    _, plan = check_attention(*args, page, window, 0, d ** -0.5)
    assert plan.counts[5] > 0 and (window or plan.counts[1] > 0)


def test_attention_of_many_rows_within_a_segment_whose_v_scales_are_far_apart():
    for d, span in ((64, 30), (128, 60)):
        rng, g = np.random.default_rng(22), torch.Generator(device=DEV).manual_seed(22)
        qo, kv, indices, last, slots = make_segments(rng, [(500, 2000), (9, 1500)], 1)
        k, v = pool_rows(g, slots, 2, d, DEV), pool_rows(g, slots, 2, d, DEV)
        gain = torch.exp2(torch.randint(-span, span + 1, ((slots + 63) // 64, 2, 1), generator=g, device=DEV).float())
        v = (v.float() * gain.repeat_interleave(64, 0)[:slots]).to(torch.bfloat16)
        pool = kv8.KV8Pool(slots, 2, d, DEV)
        fill(pool, k, v, np.arange(slots), kv8.store, kv8.StorePlan)
        q = torch.randn(int(qo[-1]), 4, d, generator=g, device=DEV).to(torch.bfloat16)
        for window in (0, 333):
            _, plan = check_attention(pool, q, qo, kv, indices, last, 1, window, 0, d ** -0.5)
            assert plan.counts[5] > 0 or window  # (with the window the call is small enough to go 16 rows at a time)


def test_another_segment_s_v_scales_move_no_bit():
    spec = [(300, 1500), (500, 3900), (260, 260)]
    got = []
    for gain in (30, 45, 60):
        pool, q, qo, kv, indices, last = scaled_segments(spec, (0, gain, 0), 64, 128, 23)
        plan = kv8.AttentionPlan(qo, kv, indices, 4, 2, 128, page_size=64, kv_last_page_len=last, device=DEV)
        got.append(kv8.tree_attention(q, pool, plan, 128 ** -0.5))
    own = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    own[300:800] = False
    assert torch.equal(got[0][own], got[1][own]) and torch.equal(got[0][own], got[2][own])
    assert got[0][own].abs().amin((0, 2)).max() > 0 or (got[0][own] != 0).float().mean() > 0.99
