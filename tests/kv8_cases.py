"""References in 64 bits for the 8-bit K/V cache: the store's codes and scales (exact) and the attention over them with
its elementwise error bound. They run on the device of their inputs and share no code with the package."""
import math

import numpy as np
import torch

BLOCK = 64


def e4m3(y):
    """The e4m3 value nearest to y (float64, |y| <= 448), ties to even."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def scale_for(a):
    """The smallest power of two s >= 2^-100 with a <= 448 s."""
    s = 2.0 ** -100
    while a > 448 * s:
        s *= 2
    return s


def store_ref(rows, slots, values, scale):
    """(codes as values, scales) after storing `rows` [n, hk, d] at `slots` into codes `values` with `scale`, float64.
    NaN rows are stored as 0 and infinite ones as the largest value; neither counts in the scale."""
    values, scale = values.double().clone(), scale.double().clone()
    rows = rows.double()
    for b in sorted({int(s) // BLOCK for s in slots}):
        at = [(int(s), i) for i, s in enumerate(slots) if int(s) // BLOCK == b]
        lo, hi = b * BLOCK, min((b + 1) * BLOCK, values.shape[0])
        for h in range(rows.shape[1]):
            x = torch.stack([rows[i, h] for _, i in at])
            a = x[torch.isfinite(x)].abs()
            old = float(scale[b, h])
            new = max(old if old > 0 else 0.0, scale_for(float(a.max()) if a.numel() else 0.0))
            if old > 0 and new > old:
                values[lo:hi, h] = e4m3(values[lo:hi, h] * (old / new))
            y = torch.nan_to_num(x / new, nan=0.0, posinf=448.0, neginf=-448.0)
            values[torch.tensor([s for s, _ in at], device=values.device), h] = e4m3(y)
            scale[b, h] = new
    return values, scale


def fill(pool, k, v, slots, store, plan):
    store(pool, k, v, plan(slots, pool.slots, pool.device))


def segments(qo, kv, last, page):
    """(first query, queries, keys) of each segment."""
    out = []
    for s in range(len(qo) - 1):
        pages = int(kv[s + 1] - kv[s])
        n = pages if page == 1 or not pages else (pages - 1) * page + (int(last[s]) if last is not None else page)
        out.append((int(qo[s]), int(qo[s + 1] - qo[s]), n))
    return out


def attention_ref(q, k, ks, v, vs, qo, kv, indices, last, page, window, n_bidir, sm_scale):
    """(out, bound): float64 attention over the dequantised pool and how far a kernel may be from it, elementwise.

    The bound counts: the output's rounding to BF16 (2^-8 of it); each probability's rounding to FP16 (2^-11) and the
    sum's and exponential's FP32 errors (2^-11 with room); the scores' FP32 sums (d + 2 roundings of 2^-24 of
    sum |q||k|, as an exponent's absolute error); FP16's smallest step for a probability: 2^-24 of 2^7 p (tiles) or 2^10 p
    (few rows), so half of it is at most 2^-32 of a key's largest value (the largest V scale times the largest code)."""
    n_q, hq, d = q.shape
    hk = ks.shape[1]
    G = hq // hk
    out = torch.zeros(n_q, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for s, (a, n, keys) in enumerate(segments(qo, kv, last, page)):
        if not n:
            continue
        pages = torch.as_tensor(np.asarray(indices[int(kv[s]):int(kv[s + 1])]), device=q.device).long()
        slot = (pages[:, None] * page + torch.arange(page, device=q.device)).reshape(-1)[:keys]
        j = torch.arange(n, device=q.device)
        t = torch.arange(keys, device=q.device)
        diag = keys - n
        if s < n_bidir:
            hi = torch.full_like(j, keys - 1)
            lo = diag + (j - (window - 1)).clamp(max=0) if window > 0 else torch.zeros_like(j)
        else:
            hi = diag + j
            lo = hi - (window - 1) if window > 0 else torch.zeros_like(j)
        seen = (t >= lo[:, None]) & (t <= hi[:, None])
        any_seen = seen.any(1)
        for h in range(hk):
            kd = k[slot, h].double() * ks[slot // BLOCK, h].double()[:, None]
            vd = v[slot, h].double() * vs[slot // BLOCK, h].double()[:, None]
            # what no query sees takes no part
            dead = ~seen.any(0)
            kd[dead], vd[dead] = 0, 0
            for g in range(G):
                x = q[a:a + n, h * G + g].double()
                w = (x @ kd.T * sm_scale).masked_fill(~seen, -math.inf)
                mag = float((x.abs() @ kd.abs().T * abs(sm_scale)).masked_fill(~seen, 0).max()) if keys else 0.0
                p = torch.where(any_seen[:, None], torch.softmax(w, 1), 0.0) if keys else w
                p = torch.nan_to_num(p, nan=0.0) if not any_seen.all() else p
                o = p @ vd
                out[a:a + n, h * G + g] = o
                top = float(vs[slot // BLOCK, h].max()) * 448 if keys else 0.0
                bound[a:a + n, h * G + g] = (o.abs() * 2.0 ** -8 + (p @ vd.abs()) * (2.0 ** -10 + 2 * (d + 2) * 2.0 ** -24 * mag)
                                             + keys * 2.0 ** -32 * top + 1e-38)
    return out, bound


def pool_rows(g, n, hk, d, device, spread=0.3, gain=1.0):
    x = torch.randn(n, hk, d, generator=g, device=device)
    x *= torch.exp(spread * torch.randn(n, 1, 1, generator=g, device=device)) * gain
    return x.to(torch.bfloat16)


def make_segments(rng, spec, page):
    """Segments (queries, keys) with private key lists in shuffled pages: (qo, kv, indices, last, pool slots)."""
    need = [(n + page - 1) // page for _, n in spec]
    perm = rng.permutation(sum(need) + 3)[:sum(need)] if sum(need) else np.zeros(0, np.int64)
    qo = np.concatenate([[0], np.cumsum([a for a, _ in spec])]).astype(np.int32)
    kv = np.concatenate([[0], np.cumsum(need)]).astype(np.int32)
    last = np.asarray([n - (p - 1) * page if p else 0 for (_, n), p in zip(spec, need)], np.int32)
    return qo, kv, perm.astype(np.int32), last, (sum(need) + 3) * page
