"""Full-vocabulary log-probabilities on the GPU against 64 bits.

Bounds, absolute. A logit off by dl: 0 where the inputs are multiples of 2^-5 and 2^-10 (every partial sum is a multiple
of 2^-15 below 2^9, which FP32 holds exactly), else (H + 8) roundings or truncations of 2^-23 of sum |h||w|. The softcap
adds dc = softcap * 2^-21 (2^-22 of it beyond a quarter of the cap, 8 roundings of z below). An exponential is off by
|u| 2^-23 + 2^-22 with |u| = m - z, a sum by one rounding per 32 terms and one per CTA: at most 2^-16 for the sizes here.
So lse is off by d = dl + dc + 2^-15, a log-probability by 2 d, and the entropy by 2 d (1 + E|u|)."""
import numpy as np
import pytest
import torch

from morj_b200 import _native as nat
from morj_b200.logprobs import token_logprobs

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


def reference(h, w, targets, top, softcap):
    l = h.double() @ w.double().T
    z = torch.tanh(l / softcap) * softcap if softcap else l
    lse = torch.logsumexp(z, 1)
    lp = z - lse[:, None]
    p = torch.exp(lp)
    order = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top]
    spread = (p * (z.amax(1, keepdim=True) - z)).sum(1)
    got = torch.where(targets >= 0, lp.gather(1, targets.clamp(min=0).long()), 0.0) if targets.shape[1] else lp[:, :0]
    return dict(logprob=got, lse=lse, entropy=-(p * lp).sum(1), top_ids=order, top_logprobs=lp.gather(1, order),
                spread=spread)


def check(h, w, targets, top, softcap, dl=0.0):
    got = token_logprobs(h, w, targets, top=top, softcap=softcap)
    want = reference(h, w, targets, top, softcap)
    d = dl + softcap * 2.0 ** -21 + 2.0 ** -15
    assert ((got.lse.double() - want['lse']).abs() <= d + want['lse'].abs() * 2.0 ** -23).all()
    if targets.shape[1]:
        assert ((got.logprob.double() - want['logprob']).abs() <= 2 * d + want['logprob'].abs() * 2.0 ** -22).all()
    assert ((got.entropy.double() - want['entropy']).abs() <= 2 * d * (1 + want['spread'])).all()
    if top:
        if dl == 0:
            assert torch.equal(got.top_ids.long(), want['top_ids'])
        assert ((got.top_logprobs.double() - want['top_logprobs']).abs()
                <= 2 * d + want['top_logprobs'].abs() * 2.0 ** -22).all()
    again = token_logprobs(h, w, targets, top=top, softcap=softcap)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a, b)
    return got


def grid(g, n, H, V, like=0.0):
    w = ((torch.randn(V, H, generator=g, device=DEV) * 0.02).clamp(-0.12, 0.12) * 1024).round() / 1024
    h = torch.randn(n, H, generator=g, device=DEV)
    if like:
        h += like * w[torch.randint(V, (n,), generator=g, device=DEV)]
    return (h.clamp(-3.5, 3.5) * 32).round().div(32).to(torch.bfloat16), w.to(torch.bfloat16)


@pytest.mark.parametrize('n,H,V', [(1, 8, 1), (1, 64, 33), (3, 72, 255), (5, 256, 4096), (17, 200, 257), (64, 136, 1000),
                                   (127, 64, 8193), (128, 64, 300), (129, 520, 5000), (300, 256, 20001), (9, 5376, 9001)])
@pytest.mark.parametrize('top,T,softcap', [(0, 1, 30.0), (1, 0, 0.0), (5, 3, 30.0), (32, 2, 4.0)])
def test_against_64_bits(n, H, V, top, T, softcap):
    g = torch.Generator(device=DEV).manual_seed(n + V)
    h, w = grid(g, n, H, V, like=5.0)
    targets = torch.randint(-1, V, (n, T), generator=g, device=DEV, dtype=torch.int32)
    check(h, w, targets, min(top, V), softcap)


def test_more_rows_than_a_chunk_holds():
    g = torch.Generator(device=DEV).manual_seed(0)
    h, w = grid(g, 4500, 64, 700)
    check(h, w, torch.randint(700, (4500, 2), generator=g, device=DEV, dtype=torch.int32), 4, 30.0)


def test_ordinary_values_and_strided_rows():
    g = torch.Generator(device=DEV).manual_seed(1)
    n, H, V = 70, 640, 3001
    hb = torch.randn(n, H + 24, generator=g, device=DEV).to(torch.bfloat16)
    wb = (torch.randn(V, 2 * H, generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    h, w = hb[:, 24:], wb[:, :H]
    dl = (H + 8) * 2.0 ** -23 * float((h.double().abs() @ w.double().abs().T).max())
    t = torch.randint(V, (n, 1), generator=g, device=DEV, dtype=torch.int32)
    check(h, w, t, 6, 30.0, dl=dl)
    check(h, w, t, 6, 0.0, dl=dl)


def test_equal_logits_are_ranked_by_id():
    h = torch.ones(3, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(2000, 64, dtype=torch.bfloat16, device=DEV)
    w[7] = 0.25
    w[1500] = 0.25
    w[300:310] = 0.125
    got = check(h, w, torch.tensor([[7], [0], [-1]], dtype=torch.int32, device=DEV), 32, 30.0)
    rest = [i for i in range(21) if i != 7]
    assert got.top_ids[0].tolist() == [7, 1500] + list(range(300, 310)) + rest
    assert got.logprob[2, 0] == 0


@pytest.mark.parametrize('V', [40000, 9001])
def test_more_equal_logits_than_fit_in_shared_memory(V):
    h, w = torch.ones(3, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(V, 64, device=DEV, dtype=torch.bfloat16)
    w[:, 0] = 0.5
    w[V - 1, 0] = 0.75  # the one that comes first
    got = check(h, w, torch.tensor([[V - 1], [0], [-1]], device=DEV, dtype=torch.int32), 32, 30.0)
    assert got.top_ids.tolist() == [[V - 1] + list(range(31))] * 3


@pytest.mark.parametrize('V', [700, 40000])
def test_a_row_s_numbers_do_not_depend_on_its_neighbours(V):
    g = torch.Generator(device=DEV).manual_seed(3)
    h, w = grid(g, 64, 128, V)
    targets = torch.randint(V, (64, 2), generator=g, device=DEV, dtype=torch.int32)
    loud = h.clone()
    loud[1::2] *= 32  # far beyond a quarter of the softcap, in the same warps
    a, b = (token_logprobs(x, w, targets, top=4, softcap=20.0) for x in (h, loud))
    for x, y in zip(a, b):
        assert torch.equal(x[::2], y[::2])


def test_candidates_in_rising_and_falling_order():
    V = 6000
    h = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    h[0, 0], h[1, 0] = 1, -1
    w = torch.zeros(V, 64, dtype=torch.bfloat16, device=DEV)
    w[:, 0] = (torch.arange(V, device=DEV) // 32).to(torch.bfloat16) / 64  # (multiples of 1/64 below 3: exact)
    got = check(h, w, torch.zeros(2, 0, dtype=torch.int32, device=DEV), 32, 0.0)
    assert got.top_ids[1].tolist() == list(range(32))


def test_peaked_and_flat_rows():
    V, H = 5000, 64
    w = torch.zeros(V, H, dtype=torch.bfloat16, device=DEV)
    w[123] = 1
    h = torch.zeros(3, H, dtype=torch.bfloat16, device=DEV)
    h[0] = 4    # logit 256: all the mass with no cap, a cap of 30 in its flat part
    h[1] = 0.5  # logit 32
    for c in (0.0, 30.0):
        got = check(h, w, torch.full((3, 1), 123, dtype=torch.int32, device=DEV), 1, c)
        assert got.top_ids[:2, 0].tolist() == [123, 123] and got.top_ids[2, 0] == 0
    h[0] = -4
    check(h, w, torch.full((3, 1), 123, dtype=torch.int32, device=DEV), 2, 0.0)


def test_the_softcap_from_its_linear_to_its_flat_part():
    V = 4001
    h = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    h[0, 0], h[1, 0] = 1, 16
    w = torch.zeros(V, 64, dtype=torch.bfloat16, device=DEV)
    w[:, 0] = ((torch.arange(V, device=DEV) - V // 2) / 128).to(torch.bfloat16)
    for c in (1.0, 30.0, 1000.0):
        check(h, w, torch.tensor([[0, V - 1, V // 2], [5, 6, 7]], dtype=torch.int32, device=DEV), 3, c)


def test_rows_with_values_that_are_not_finite():
    g = torch.Generator(device=DEV).manual_seed(2)
    h, w = grid(g, 4, 64, 500)
    h[1, 3] = float('nan')
    t = torch.full((4, 1), 9, dtype=torch.int32, device=DEV)
    got = token_logprobs(h, w, t, top=2, softcap=30.0)
    assert torch.isnan(got.lse[1]) and torch.isnan(got.logprob[1, 0]) and torch.isnan(got.entropy[1])
    assert (got.top_ids[1] == -1).all() and torch.isnan(got.top_logprobs[1]).all()
    keep = torch.tensor([0, 2, 3], device=DEV)
    want = token_logprobs(h[keep].contiguous(), w, t[keep], top=2, softcap=30.0)
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b)


def test_a_target_outside_the_vocabulary_is_reported():
    g = torch.Generator(device=DEV).manual_seed(3)
    h, w = grid(g, 2, 64, 100)
    t = torch.tensor([[100, 5], [-2, -1]], dtype=torch.int32, device=DEV)
    got = token_logprobs(h, w, t, softcap=30.0)
    assert nat.device_error(torch.cuda.current_stream().cuda_stream) == 0x301
    assert torch.isnan(got.logprob[0, 0]) and torch.isnan(got.logprob[1, 0])
    assert torch.isfinite(got.logprob[0, 1]) and got.logprob[1, 1] == 0


def test_streams_and_graphs():
    g = torch.Generator(device=DEV).manual_seed(4)
    h, w = grid(g, 40, 128, 3000)
    t = torch.randint(3000, (40, 1), generator=g, device=DEV, dtype=torch.int32)
    want = check(h, w, t, 3, 30.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = token_logprobs(h, w, t, top=3, softcap=30.0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(token_logprobs(h, w, t, top=3, softcap=30.0))
        graphs.append(graph)
    h.copy_(h.flip(0).contiguous())
    side.wait_stream(torch.cuda.default_stream())
    with torch.cuda.stream(side):
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    new = token_logprobs(h, w, t, top=3, softcap=30.0)
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, new))


def test_it_agrees_with_the_label_head():
    """The label head's softmax over a few labels is this operator's log-probabilities renormalised over them."""
    g = torch.Generator(device=DEV).manual_seed(5)
    H, V, n = 256, 4096, 6
    x = torch.randn(n, H, generator=g, device=DEV).to(torch.bfloat16)
    w = (torch.randn(V, H, generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    norm = (1 + 0.1 * torch.randn(H, generator=g, device=DEV)).to(torch.bfloat16)
    labels = torch.randint(V, (n, 5), generator=g, device=DEV, dtype=torch.int32)
    s = torch.cuda.current_stream().cuda_stream
    rows = torch.arange(n, dtype=torch.int32, device=DEV)
    indptr = torch.arange(0, 5 * n + 1, 5, dtype=torch.int32, device=DEV)
    probs = torch.empty(n, 5, device=DEV)
    nat.call('morj_label_head', x.data_ptr(), H, rows.data_ptr(), indptr.data_ptr(), labels.data_ptr(), n,
             norm.data_ptr(), w.data_ptr(), H, 1e-6, 30.0, probs.data_ptr(), s)
    h = torch.empty_like(x)
    nat.call('morj_rmsnorm_rows', x.data_ptr(), norm.data_ptr(), n, H, 1e-6, h.data_ptr(), s)
    got = token_logprobs(h, w, labels, softcap=30.0)
    assert ((torch.softmax(got.logprob, 1) - probs).abs() <= 1e-4).all()


def test_a_vocabulary_beyond_32_bit_offsets():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 40 GB')
    H, V = 16384, 140000  # 2.3e9 elements
    w = torch.zeros(V, H, dtype=torch.bfloat16, device=DEV)
    h = torch.zeros(2, H, dtype=torch.bfloat16, device=DEV)
    h[0, :64], h[1, -64:] = 1, 1
    w[V - 1, :64] = 0.25
    w[V - 3, -64:] = 0.125
    t = torch.tensor([[V - 1], [V - 3]], dtype=torch.int32, device=DEV)
    got = token_logprobs(h, w, t, top=2, softcap=0.0)
    z = torch.tensor([16.0, 8.0], dtype=torch.float64, device=DEV)
    lse = torch.log(torch.exp(z) + V - 1)
    assert got.top_ids.tolist() == [[V - 1, 0], [V - 3, 0]]
    assert ((got.lse.double() - lse).abs() <= 2.0 ** -14).all()
    assert ((got.logprob[:, 0].double() - (z - lse)).abs() <= 2.0 ** -13).all()


def test_refusals():
    g = torch.Generator(device=DEV).manual_seed(6)
    h, w = grid(g, 2, 64, 100)
    t = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    for bad, match in [(lambda: token_logprobs(h.float(), w, t), 'BF16'),
                       (lambda: token_logprobs(h, w[:, :56], t), 'BF16'),
                       (lambda: token_logprobs(h, w, t.long()), 'int32'),
                       (lambda: token_logprobs(h, w, t[:1]), 'int32'),
                       (lambda: token_logprobs(h, w, t, top=33), 'top'),
                       (lambda: token_logprobs(h, w[:5], t, top=6), 'top'),
                       (lambda: token_logprobs(h, w, t, softcap=-1.0), 'softcap'),
                       (lambda: token_logprobs(h, w, t, softcap=float('nan')), 'softcap'),
                       (lambda: token_logprobs(h, w, t.cpu()), 'are on'),
                       (lambda: token_logprobs(h[:, ::2], w[:, ::2], t), 'contiguous'),
                       (lambda: token_logprobs(h[:, :60].contiguous(), w[:, :60].contiguous(), t), 'multiples of 8')]:
        with pytest.raises(ValueError, match=match):
            bad()
    empty = token_logprobs(h[:0], w, t[:0], top=2)
    assert empty.lse.shape == (0,) and empty.top_ids.shape == (0, 2)
    assert np.isfinite(token_logprobs(h, w, t[:, :0].contiguous()).lse.cpu().numpy()).all()


@pytest.mark.parametrize('V', [50, 300, 9001])
def test_logits_of_minus_infinity_have_no_probability(V):
    """Vocabulary rows masked by -infinity in a column where every h is 1: their probability is 0, and so is their part of
    the entropy (p log p -> 0)."""
    g = torch.Generator(device=DEV).manual_seed(V)
    h, w = grid(g, 5, 64, V, like=5.0)
    h[:, 7] = 1
    masked = torch.arange(V, device=DEV) % 3 == 1
    masked[:32] = True  # (the whole first group of a tile)
    w[masked, 7] = float('-inf')
    assert not masked.all()
    live = torch.nonzero(~masked)[:, 0]
    t = torch.stack([live[:5], live[-5:], masked.nonzero()[:5, 0]], 1).to(torch.int32)
    top = min(8, len(live))
    got = token_logprobs(h, w, t, top=top, softcap=0.0)
    l = h.double() @ w[live].double().T  # the definition over the rows that are left
    lse = torch.logsumexp(l, 1)
    lp = l - lse[:, None]
    d = 2.0 ** -15
    assert ((got.lse.double() - lse).abs() <= d + lse.abs() * 2.0 ** -23).all()
    spread = (lp.exp() * (l.amax(1, keepdim=True) - l)).sum(1)
    assert ((got.entropy.double() + (lp.exp() * lp).sum(1)).abs() <= 2 * d * (1 + spread)).all()
    order = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids.long(), live[order])
    place = torch.searchsorted(live, t[:, :2].long())
    assert ((got.logprob[:, :2].double() - lp.gather(1, place)).abs() <= 2 * d + lp.abs().max() * 2.0 ** -22).all()
    assert (got.logprob[:, 2] == float('-inf')).all()
    # all masked: nothing is left
    w[:, 7] = float('-inf')
    got = token_logprobs(h, w, t, top=1, softcap=0.0)
    assert (got.lse == float('-inf')).all() and (got.top_ids == -1).all() and torch.isnan(got.top_logprobs).all()
