"""The engine over 8-bit K/V pools and its full-vocabulary readouts, used together: requests kept in 8 bits, later passes
over them, the shared head, and the log-probabilities read from both kinds of pools."""
import numpy as np
import pytest
import torch

from kv8_cases import BLOCK, e4m3, scale_for
from morj_b200 import _native as nat
from test_gpu_engine import CASES, TOL, check_contract, engine, flat, full_width_model, state  # noqa: F401

pytestmark = pytest.mark.gpu


def quantised(pool):
    """A pool as the 8-bit cache holds it: every block and head scaled by its largest magnitude."""
    out = pool.double().clone()
    for b in range(0, pool.shape[0], BLOCK):
        for h in range(pool.shape[1]):
            x = out[b:b + BLOCK, h]
            s = scale_for(float(x.abs().max()))
            out[b:b + BLOCK, h] = e4m3(x / s) * s
    return out.float()


@pytest.fixture
def oracle8(monkeypatch):
    """The CPU oracle with its attention reading quantised pools."""
    import oracle.lean_oracle as lo
    plain = lo.tree_attention
    monkeypatch.setattr(lo, 'tree_attention', lambda q, k, v, *a, **kw: plain(q, quantised(k), quantised(v), *a, **kw))
    return lo.OracleModel


def images_of(state, c):  # noqa: F811
    if not c['images']:
        return None
    from make_forward_golden import tiny_images
    return [f.cuda() for f in tiny_images(state[0])]


@pytest.mark.parametrize('name', ['tiny', 'tiny-nested', 'tiny-steps'])
def test_engine_over_8_bit_pools_matches_the_oracle_over_them(state, oracle8, name):  # noqa: F811
    from morj_b200.tree import Tree
    c = CASES[name]
    m = engine(state, single_max=c['single_max'], step_tokens=c['step_tokens'], kv_cache='e4m3')
    got = m.run(m.prepare(c['seqs'], c['label_ids']), list(range(len(c['seqs']))))
    check_contract(got, c['label_ids'])
    want = oracle8(*state).forward_tree(Tree, c['seqs'], c['label_ids'], 'bf16', c['single_max'], c['step_tokens'])
    assert np.abs(flat(got) - flat(want)).max() <= TOL


@pytest.mark.parametrize('name', ['tiny-steps', 'tiny-retain-two-pass', 'tiny-pinned-two-pass', 'tiny-images',
                                  'tiny-images-steps'])
@pytest.mark.parametrize('poison', [False, True])
def test_every_way_of_keeping_8_bit_kv_gives_one_pass_s_probabilities(state, monkeypatch, name, poison):  # noqa: F811
    """Steps, retained and pinned passes read the same 8-bit K/V as one pass over the whole tree."""
    import morj_b200.lean_core as lc
    monkeypatch.setattr(lc, 'POISON', poison)
    c = CASES[name]
    whole = engine(state, kv_cache='e4m3')
    want = whole.run(whole.prepare(c['seqs'], c['label_ids'], images=images_of(state, c)), list(range(len(c['seqs']))))
    m = engine(state, single_max=c['single_max'], step_tokens=c['step_tokens'], retain_budget=c['retain_budget'],
               kv_cache='e4m3')
    req = m.prepare(c['seqs'], c['label_ids'], retain=c['retain'], images=images_of(state, c))
    assert (req.retain, req.pinned) == (c['retained'], c['pinned'])
    for p in c['passes']:
        got = m.run(req, list(p))
        assert np.abs(flat(got) - flat([want[b] for b in p])).max() <= TOL
    if len(c['passes']) > 1:
        assert m.timing['tokens'] < req.tree.num_tokens


def test_the_shared_head_in_8_bits(state):  # noqa: F811
    c = CASES['tiny']
    plain = engine(state, kv_cache='e4m3')
    want = plain.run(plain.prepare(c['seqs'], c['label_ids']), [0, 1, 2, 3])
    for retain in (False, True):
        m = engine(state, kv_cache='e4m3')
        m.set_shared_prefix(c['seqs'][0][:40])
        req = m.prepare(c['seqs'], c['label_ids'], retain=retain)
        assert req.head_nodes
        got = m.run(req, [0, 1, 2, 3])
        assert not set(req.head_nodes) & set(m.last_need)
        assert np.abs(flat(got) - flat(want)).max() <= TOL


def test_8_bit_pools_take_half_the_memory(state):  # noqa: F811
    a, b = engine(state), engine(state, kv_cache='e4m3')
    # 2 layers x (K, V) x 2 heads x (64 codes + 4 bytes of scale per 64 slots)
    assert a.kv_bytes == 2 * 2 * 2 * 2 * 64 and b.kv_bytes == 2 * 2 * 2 * 64 + 2 * 2 * 2 * 4 // 64 + 1
    c = CASES['tiny']
    req = b.prepare(c['seqs'], c['label_ids'], retain=True)
    assert sum(p.nbytes for p in req.pools) <= req.tree.num_tokens * b.kv_bytes + 2 * 2 * 2 * 4
    with pytest.raises(ValueError, match='kv_cache'):
        engine(state, kv_cache='int8')


def test_full_width_layers_over_8_bit_pools(oracle8):
    from morj_b200.tree import Tree
    from morj_b200.workloads import text_tree
    top, st = full_width_model()
    t = text_tree(seed=0, prefix=200, questions=2, rotations=2, branch=20, vocab=4096)
    m = engine((top, st), kv_cache='e4m3')
    got = m.run(m.prepare(t['seqs'], t['label_ids']), list(range(4)))
    want = oracle8(top, st).forward_tree(Tree, t['seqs'], t['label_ids'], 'bf16')
    assert np.abs(flat(got) - flat(want)).max() <= TOL


# ---- full-vocabulary readouts ---------------------------------------------------------------------------------------

def vocabulary(m, rows):
    """Float64 log-probabilities of residual rows: final norm rounded to BF16 as the engine rounds it, softcap."""
    x = rows.double()
    h = (x * torch.rsqrt((x * x).mean(1, keepdim=True) + m.eps) * m.norm.double()).to(torch.bfloat16).double()
    z = h @ m.embed.double().T
    z = torch.tanh(z / m.softcap) * m.softcap
    return torch.log_softmax(z, 1)


@pytest.mark.parametrize('kv_cache', ['bf16', 'e4m3'])
def test_label_logprobs_are_run_s_readout_under_the_whole_vocabulary(state, kv_cache):  # noqa: F811
    c = CASES['tiny-nested']
    m = engine(state, kv_cache=kv_cache)
    seqs = list(range(len(c['seqs'])))
    probs = m.run(m.prepare(c['seqs'], c['label_ids']), seqs)
    req = m.prepare(c['seqs'], c['label_ids'])
    got = m.label_logprobs(req, seqs, top=5)
    p = m.prepare_pass(req, seqs)
    lp = vocabulary(m, m._execute_steps(p)[p['ro']['t']['seq_row'].long()])
    for i, (g, q, ids) in enumerate(zip(got, probs, c['label_ids'])):
        soft = np.exp(g['logprob'].astype(np.float64))
        assert np.abs(soft / soft.sum() - q).max() <= 1e-3
        # rows normed in FP32 and rounded to BF16: a rounding that falls the other way moves a logit by 2^-8 |h w|
        want = lp[i].cpu().numpy()
        assert np.abs(g['logprob'] - want[list(ids)]).max() <= 0.02
        assert abs(g['entropy'] + (np.exp(want) * want).sum()) <= 0.02
        assert (np.diff(g['top_logprobs']) <= 0).all() and len(set(g['top_ids'].tolist())) == 5
        assert np.abs(g['top_logprobs'] - np.sort(want)[::-1][:5]).max() <= 0.02
    assert nat.device_error(torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.parametrize('kv_cache', ['bf16', 'e4m3'])
@pytest.mark.parametrize('pruned', [False, True])
def test_token_logprobs_score_every_token_given_the_ones_before(state, monkeypatch, kv_cache, pruned):  # noqa: F811
    import morj_b200.lean_core as lc
    monkeypatch.setattr(lc, 'MAX_PRUNED_ROWS', 10**9 if pruned else 0)
    c = CASES['tiny-nested']
    seqs = list(range(len(c['seqs'])))
    m = engine(state, kv_cache=kv_cache)
    got = m.token_logprobs(m.prepare(c['seqs'], c['label_ids']), seqs, top=3)
    for b, g in zip(seqs, got):
        s = c['seqs'][b]
        assert g['start'] == 1 and g['tokens'].tolist() == list(s[1:])
        # the sequence alone, its last row only, at a few lengths: the same next-token distribution
        alone = engine(state, kv_cache=kv_cache)
        for t in (1, len(s) // 2, len(s) - 1):
            one = alone.label_logprobs(alone.prepare([s[:t]], [[s[t]]]), [0])[0]
            assert abs(np.exp(one['logprob'][0]) - np.exp(g['logprob'][t - 1])) <= TOL
            assert abs(one['entropy'] - g['entropy'][t - 1]) <= 0.05
    # shared tokens have one value
    same = [i for i in range(1, min(len(s) for s in c['seqs'])) if len({tuple(s[:i + 1]) for s in c['seqs']}) == 1]
    for t in same:
        assert len({float(g['logprob'][t - 1]) for g in got}) == 1
    # a later start is the same pass read from there on
    part = m.token_logprobs(m.prepare(c['seqs'], c['label_ids']), [1, 0], start=[5, None])
    assert part[0]['start'] == 5 and np.abs(part[0]['logprob'] - got[1]['logprob'][4:]).max() <= 0.05
    assert part[1]['start'] == 1


@pytest.mark.parametrize('kv_cache', ['bf16', 'e4m3'])
def test_answers_scored_against_a_kept_prompt(state, kv_cache):  # noqa: F811
    """One pass keeps the prompt with a first answer; a later pass scores the other answers over the kept K/V."""
    c = CASES['tiny-retain-two-pass']
    m = engine(state, kv_cache=kv_cache)
    whole = m.token_logprobs(m.prepare(c['seqs'], c['label_ids']), list(range(len(c['seqs']))))
    req = m.prepare(c['seqs'], c['label_ids'], retain=True)
    assert req.retain
    first, later = [0], list(range(1, len(c['seqs'])))
    m.run(req, first)
    got = m.token_logprobs(req, later, top=2)
    assert m.timing['tokens'] < req.tree.num_tokens
    for b, g in zip(later, got):
        shared = next(i for i, (x, y) in enumerate(zip(c['seqs'][0], c['seqs'][b])) if x != y)
        assert g['start'] == shared + 1  # the token after the prompt is predicted by a row the first pass computed
        assert np.abs(np.exp(g['logprob']) - np.exp(whole[b]['logprob'][g['start'] - 1:])).max() <= TOL
    with pytest.raises(ValueError, match='an earlier pass computed'):
        m.token_logprobs(req, later, start=[1] * len(later))


@pytest.mark.parametrize('kv_cache', ['bf16', 'e4m3'])
def test_a_sequence_may_be_asked_for_twice(state, kv_cache):  # noqa: F811
    c = CASES['tiny-nested']
    m = engine(state, kv_cache=kv_cache)
    a, b, again = m.token_logprobs(m.prepare(c['seqs'], c['label_ids']), [1, 0, 1], start=[None, None, 3], top=2)
    assert np.array_equal(a['logprob'][2:], again['logprob']) and np.array_equal(a['top_ids'][2:], again['top_ids'])
    x, y = m.label_logprobs(m.prepare(c['seqs'], c['label_ids']), [1, 1], top=2)
    assert np.array_equal(x['logprob'], y['logprob']) and x['lse'] == y['lse']


def test_scoring_refusals(state):  # noqa: F811
    c = CASES['tiny']
    m = engine(state)
    req = m.prepare(c['seqs'], c['label_ids'])
    for bad, match in [(lambda: m.token_logprobs(req, [0], top=33), 'top'),
                       (lambda: m.token_logprobs(req, []), 'sequences'),
                       (lambda: m.token_logprobs(req, [9]), 'sequences'),
                       (lambda: m.token_logprobs(req, [0, 1], start=[1]), '1 starts for 2'),
                       (lambda: m.token_logprobs(req, [0], start=[0]), 'to score'),
                       (lambda: m.token_logprobs(req, [0], start=[len(c['seqs'][0]) + 1]), 'to score'),
                       (lambda: m.token_logprobs(req, [0], start=[len(c['seqs'][0])]), 'no token'),
                       (lambda: m.label_logprobs(req, [0], top=-1), 'top'),
                       (lambda: m.label_logprobs(m.prepare(c['seqs'], [[4096]] * 4), [0]), 'vocabulary')]:
        with pytest.raises(ValueError, match=match):
            bad()


def test_scoring_over_image_blocks(state):  # noqa: F811
    c = CASES['tiny-images']
    m = engine(state, kv_cache='e4m3')
    req = m.prepare(c['seqs'], c['label_ids'], images=images_of(state, c))
    after = int(req.blocks.end[-1]) + 2  # text only
    seqs = list(range(len(c['seqs'])))
    got = m.token_logprobs(req, seqs, start=[after] * len(seqs))
    want = m.label_logprobs(m.prepare(c['seqs'], c['label_ids'], images=images_of(state, c)), seqs)
    assert all(np.isfinite(g['logprob']).all() and np.isfinite(w['lse']) for g, w in zip(got, want))


@pytest.mark.parametrize('name', ['tiny-images', 'tiny-images-steps'])
@pytest.mark.parametrize('kv_cache', ['bf16', 'e4m3'])
def test_with_images_the_text_behind_them_is_scored(state, monkeypatch, name, kv_cache):  # noqa: F811
    """Without a start scoring begins behind the last block; its values are those of the truncated sequences' readouts,
    with the last layer run for the scored rows only or for all."""
    import morj_b200.lean_core as lc
    c = CASES[name]
    make = lambda **kw: engine(state, kv_cache=kv_cache, **kw)
    m = make(single_max=c['single_max'], step_tokens=c['step_tokens'])
    images, seqs = images_of(state, c), list(range(len(c['seqs'])))
    got = []
    for pruned in (10**9, 0):
        monkeypatch.setattr(lc, 'MAX_PRUNED_ROWS', pruned)
        req = m.prepare(c['seqs'], c['label_ids'], images=images)
        got.append(m.token_logprobs(req, seqs, top=2))
    end = int(req.blocks.end[-1])
    for b, g, whole in zip(seqs, *got):
        s = req.blocks.seqs[b]
        assert g['start'] == whole['start'] == end + 1 and g['tokens'].tolist() == s[end + 1:]
        assert m.image_id not in g['tokens'].tolist()
        assert np.abs(np.exp(g['logprob']) - np.exp(whole['logprob'])).max() <= TOL
        for t in (end + 1, len(s) - 1):
            alone = make()
            r = alone.prepare([c['seqs'][b][:len(c['seqs'][b]) - (len(s) - t)]], [[s[t]]], images=images)
            assert r.blocks.seqs[0] == s[:t]
            one = alone.label_logprobs(r, [0])[0]
            assert abs(np.exp(one['logprob'][0]) - np.exp(g['logprob'][t - g['start']])) <= TOL
            assert abs(one['lse'] - g['lse'][t - g['start']]) <= 0.05
            assert abs(one['entropy'] - g['entropy'][t - g['start']]) <= 0.05
    for start in (1, end):
        with pytest.raises(ValueError, match=f'from {end + 1} on, not from {start}'):
            m.token_logprobs(req, seqs, start=[start] * len(seqs))


@pytest.mark.parametrize('kv_cache', ['bf16', 'e4m3'])
def test_scoring_through_the_tensor_parallel_path(state, monkeypatch, tmp_path, kv_cache):  # noqa: F811
    """A group of one rank takes the peer exchange's path (partials, reductions, waits; all on one stream): the same
    probabilities and scores, with the last layer run for a few rows and for all of them (where the last site returns the
    residual rows)."""
    import torch.distributed as dist
    import morj_b200.lean_core as lc
    c = CASES['tiny-nested']
    seqs = list(range(len(c['seqs'])))
    plain = engine(state, kv_cache=kv_cache)
    want = plain.run(plain.prepare(c['seqs'], c['label_ids']), seqs)
    scores = plain.token_logprobs(plain.prepare(c['seqs'], c['label_ids']), seqs, top=2)
    dist.init_process_group('gloo', init_method=f'file://{tmp_path}/store', world_size=1, rank=0)
    try:
        m = engine(state, kv_cache=kv_cache, tp_group=dist.group.WORLD, single_max=1024, step_tokens=1024)
        assert m.peer is not None
        for pruned in (10**9, 0):
            monkeypatch.setattr(lc, 'MAX_PRUNED_ROWS', pruned)
            assert np.abs(flat(m.run(m.prepare(c['seqs'], c['label_ids']), seqs)) - flat(want)).max() <= TOL
            for g, w in zip(m.token_logprobs(m.prepare(c['seqs'], c['label_ids']), seqs, top=2), scores):
                assert g['start'] == w['start']
                assert np.abs(np.exp(g['logprob']) - np.exp(w['logprob'])).max() <= TOL
                assert np.abs(g['entropy'] - w['entropy']).max() <= 0.05
        m.peer.close()
    finally:
        dist.destroy_process_group()
