"""GPU tests of the draws and of clipping on random calls: sizes, types, strides, settings, masks and non-finite entries together,
each call against numpy in float64.

Draws: an index may differ from numpy's only where the random number lies within the roundings of a border between two kept entries:
numpy's running sum of V <= 3e5 positive weights is off by at most V half steps, 3e5 x 2^-53 < 4e-11 of the sum (the kernel's, in
trees and short chains, by far less).  Rows with a running sum that near to top_p's share, or a weight within 1e-12 (of which each is
off by a few half steps) of min_p, are left out.  The log-probabilities are z - log Z: z carries 2 roundings of
|z|, Z the sum's, bounded by 2^-53 (8 |z| + 40 + V / 32 + 8 |log Z|).  Clipping: the bounds of tests/test_gpu_gradients.py.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from pgmuvi_amd import gradients as G
from pgmuvi_amd.sampling import draw_indices

TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]
SIGNALLING = {torch.float64: (torch.int64, 0x7FF0000000000001), torch.float32: (torch.int32, 0x7F800001), torch.bfloat16: (torch.int16, 0x7F81),
             torch.float16: (torch.int16, 0x7C01)}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("-m gpu tests need the MI355X")
    return torch.device("cuda:0")


# ---- draws ---------------------------------------------------------------------------------------------------------------
def _kept(l, temperature, top_k, top_p, min_p):
    """(kept indices in order, weights, z, is a truncation's border within 1e-12 of an entry?)"""
    alive = np.flatnonzero(l > -np.inf)
    if alive.size == 0:
        return alive, np.zeros(0), np.zeros(0), False
    order = alive[np.argsort(-l[alive], kind="stable")]
    best = l[order[0]]
    if not temperature > 0:
        return order[:1], np.ones(1), np.zeros(1), False
    with np.errstate(all="ignore"):
        z = np.where(l[order] == best, 0.0, (l[order] - best) / temperature)
    w, n, edge = np.exp(z), len(order), False
    if top_k:
        n = min(n, top_k)
    if top_p <= 0.0:
        n = 1
    elif top_p < 1.0:
        c = np.cumsum(w[:n])
        edge = bool(np.abs(c - top_p * c[-1]).min() < 4e-11 * c[-1])
        n = min(n, 1 + int(np.searchsorted(c, top_p * c[-1], side="left")))
    if min_p > 0.0:
        edge = edge or (min_p < 1.0 and bool((np.abs(w[:n] - min_p) < 1e-12 * min_p).any()))
        n = max(1, int(np.count_nonzero(w[:n] >= min_p)))
    at = np.argsort(order[:n])
    return order[:n][at], w[:n][at], z[:n][at], edge


def _row(rng, V, dtype):
    low, kind = float(torch.finfo(dtype).min), rng.integers(0, 14)
    l = (rng.normal(0, rng.choice([0.1, 3, 100]), V) if kind == 0 else rng.integers(0, rng.choice([2, 5, 50]), V).astype(float) if kind == 1
         else np.full(V, rng.normal()) if kind == 2 else rng.normal(0, 1, V) * (-low / 8) if kind == 3 else rng.exponential(size=V) if kind == 4
         else np.sort(rng.normal(0, 4, V)) if kind == 5 else -np.sort(rng.normal(0, 4, V)) * 1e-3 if kind == 6
         else rng.choice([0.0, -0.0, 1e-310, -1e-310, 5e-324], V) if kind == 7 else np.where(rng.random(V) < 0.02, rng.normal(0, 2, V), -np.inf) if kind == 8
         else np.where(rng.random(V) < 0.5, rng.normal(0, 2, V), low) if kind == 9 else rng.normal(1e6, 1e-3, V) if kind == 10
         else np.full(V, -np.inf) if kind == 11 else low * (1 - rng.random(V) * rng.choice([1e-15, 1e-3, 0.5])) if kind == 12 else rng.standard_cauchy(V))
    if kind == 4:
        l[rng.integers(0, V, 3)] += rng.uniform(0, 60, 3)
    if kind == 11:
        a = rng.integers(0, V)
        l[a:a + rng.integers(1, 300)] = rng.normal()
    if rng.random() < 0.25:
        l[rng.random(V) < 0.05] = np.nan
    if rng.random() < 0.1:
        l[rng.integers(0, V, rng.integers(1, 4))] = np.inf
    if rng.random() < 0.15:
        l[rng.random(V) < rng.choice([0.1, 0.9, 0.999])] = -np.inf
    return l


def _settings(rng, V):
    return dict(temperature=float(rng.choice([1, 1, 0.3, 3, 0, 1e-5, 1e5, 1e290, 1e-300])),
                top_k=int(rng.choice([0, 0, 1, 3, 20, 64, 200, 256, 257, 500, 513, 1024, 5000, V, V + 3])),
                top_p=float(rng.choice([1, 1, rng.random(), 0.9, 0.999999, 1e-9, 0])), min_p=float(rng.choice([0, 0, 0, rng.random(), 1e-3, 1e-12, 1])))


@pytest.mark.parametrize("seed", range(8))
def test_random_draws(dev, seed):
    rng = np.random.default_rng([seed, 51])
    for _ in range(100):
        dtype = TYPES[rng.integers(0, 4)]
        V = int(np.exp(rng.uniform(0, np.log(rng.choice([300, 3000, 30_000, 300_000])))))
        B = min(int(rng.choice([1, 1, 2, 3, 7, 130, 520, 1030])), max(1, 3_000_000 // V))
        S = min(int(rng.choice([1, 1, 2, 5, 20, 40, 90, 300, 1500])), max(1, 200_000 // B))
        rows = [_row(rng, V, dtype) for _ in range(min(B, 5))]
        with np.errstate(all="ignore"):
            l = torch.as_tensor(np.stack([rows[b % len(rows)] for b in range(B)])).to(dtype)
        if rng.random() < 0.2:                                   # NaNs of the signalling kind, by their bits
            ints, pattern = SIGNALLING[dtype]
            l.view(ints)[torch.as_tensor(rng.random((B, V)) < 0.03)] = pattern
        per_row = rng.random() < 0.3
        settings = [_settings(rng, V) for _ in range(B)] if per_row else [_settings(rng, V)] * B
        lengths = rng.integers(-2, V + 3, B) if rng.random() < 0.3 else None
        u = rng.random((B, S))
        if rng.random() < 0.3:
            u[:, 0], u[:, -1] = 0.0, 1.0 - 2.0 ** -53
        d = l.to(dev)
        if rng.random() < 0.15:
            d = d.t().contiguous().t()
        elif rng.random() < 0.15:
            wide = torch.zeros(B, V + 5, dtype=dtype, device=dev)
            wide[:, 3:V + 3] = d
            d = wide[:, 3:V + 3]
        if per_row:
            kw = {k: torch.tensor([s[k] for s in settings], dtype=torch.int64 if k == "top_k" else torch.float64, device=dev) for k in settings[0]}
        else:
            kw = dict(settings[0], top_k=settings[0]["top_k"] or None)
        index, logp = draw_indices(d, torch.as_tensor(u, device=dev), lengths=None if lengths is None else torch.as_tensor(lengths, device=dev),
                                   return_logprob=True, **kw)
        index, logp = index.cpu().numpy(), logp.cpu().numpy()
        for b in sorted({0, 1 % B, 2 % B, 3 % B, 4 % B, B // 2, B - 1}):
            n = V if lengths is None else int(max(0, min(V, lengths[b])))
            case = (dtype, B, V, S, n, settings[b])
            kept, w, z, edge = _kept(l[b].double().numpy()[:n], **settings[b])
            if len(kept) == 0:
                assert (index[b] == -1).all() and (logp[b] == -np.inf).all(), case
                continue
            if edge:
                continue
            c = np.cumsum(w)
            at = np.minimum(np.searchsorted(c, u[b] * c[-1], side="right"), np.flatnonzero(w > 0)[-1])
            same = index[b] == kept[at]
            pos = np.minimum(np.searchsorted(kept, index[b]), len(kept) - 1)
            before, slack = np.where(pos > 0, c[np.maximum(pos - 1, 0)], 0.0), 4e-11 * c[-1]
            border = (kept[pos] == index[b]) & (w[pos] > 0) & (u[b] * c[-1] >= before - slack) & (u[b] * c[-1] <= c[pos] + slack)
            assert (same | border).all(), (case, u[b][~(same | border)][:3], index[b][~(same | border)][:3])
            log_z = math.log(math.fsum(w))
            off = np.abs(logp[b] - (z[pos] - log_z))
            assert (off <= 2.0 ** -53 * (8 * np.abs(z[pos]) + 40 + V / 32 + 8 * abs(log_z))).all(), case


# ---- clipping ------------------------------------------------------------------------------------------------------------
HALF_STEP = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float64: 2.0 ** -1074, torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _norm(a, p):
    a = np.abs(a)
    if a.size == 0 or np.isnan(a).any() or np.isinf(a).any() or a.max() == 0.0:
        return 0.0 if a.size == 0 else float(a.max())            # (max: NaN before infinity before zero)
    if p == math.inf:
        return float(a.max())
    if p == 1:
        return math.fsum(a.tolist())
    m = math.frexp(float(a.max()))[1]
    return math.ldexp(math.sqrt(math.fsum((np.ldexp(a, -m) ** 2).tolist())), m)


def _view_of(rng, x):
    """x itself, or a strided view that holds it."""
    kind = rng.integers(0, 9)
    if kind < 5 or x.dim() == 0:
        return x.clone()
    if kind == 5:
        return x.transpose(-1, -2).contiguous().transpose(-1, -2) if x.dim() >= 2 else x.clone()
    buf = torch.zeros(*x.shape[:-1], x.shape[-1] * 2 + 6, dtype=x.dtype, device=x.device)
    v = buf[..., 1:2 * x.shape[-1] + 1:2] if kind == 6 else buf[..., 2:2 + x.shape[-1]]
    if kind == 8:
        v = torch.zeros(x.numel() + 3, dtype=x.dtype, device=x.device)[1:1 + x.numel()].view(x.shape)
    return v.copy_(x)


@pytest.mark.parametrize("seed", range(8))
def test_random_clips(dev, seed):
    rng = np.random.default_rng([seed, 52])
    for _ in range(60):
        members = rng.random() < 0.45
        lead = int(rng.choice([1, 2, 3, 17, 130, 600, 3000])) if members else None
        count, one_type, p = int(rng.choice([1, 2, 5, 8, 9, 20, 70, 150])), rng.random() < 0.75, [2, 2, 2, 1, math.inf][rng.integers(0, 5)]
        most, kind = 200_000 // (lead or 1) // count + 2, rng.integers(0, 4)
        grads = []
        for _ in range(count):
            n = int(np.exp(rng.uniform(0, np.log(most))))
            side = max(1, int(n ** 0.5))
            shape = ((lead,) if members else ()) + [(), (n,), (side, max(1, n // side)), (side, max(1, n // side), int(rng.integers(1, 4))), (0,)][
                rng.choice(5, p=[0.2, 0.25, 0.3, 0.22, 0.03])]
            dtype = TYPES[kind if one_type else rng.integers(0, 4)]
            scale = 10.0 ** (rng.uniform(-320, 300) if dtype is torch.float64 and rng.random() < 0.5 else rng.uniform(-4, 2))
            x = torch.as_tensor(rng.normal(size=shape) * scale).to(dtype)
            if x.numel() and rng.random() < 0.02:
                x.view(-1)[rng.integers(0, x.numel())] = [math.nan, math.inf, -math.inf][rng.integers(0, 3)]
            grads.append(_view_of(rng, x.to(dev)))
        before = [g.double().cpu().numpy() for g in grads]
        limit, in_place = float(rng.choice([0.0, 1e-3, 1.0, 50.0, 1e30, math.inf])), rng.random() < 0.5
        outs = grads if in_place else [_view_of(rng, torch.full(g.shape, 7.0, dtype=g.dtype, device=dev)) for g in grads]
        total = G.total_norm(grads, p, members)
        norm = G.clip_grads_(grads, limit, p, out=None if in_place else outs, members=members)
        wide = any(g.dtype is torch.float64 for g in grads)
        assert norm.dtype is (torch.float64 if wide else torch.float32)
        # (a tensor that is one run by itself may be none together with its output: another order of summation)
        assert not in_place or torch.equal(torch.nan_to_num(total), torch.nan_to_num(norm))
        norms = [x.double().cpu().numpy().reshape(-1) for x in (norm, total)]
        after = [o.double().cpu().numpy() for o in outs]
        for b in sorted({0, lead // 2, lead - 1}) if members else (None,):
            pick = lambda a: a if b is None else a[b]
            flat = np.concatenate([np.asarray(pick(a)).reshape(-1) for a in before])
            case = (members, lead, count, p, limit, in_place, [(g.dtype, tuple(g.shape), g.stride()) for g in grads][:4], b)
            want = _norm(flat, p)
            tol = (72 + flat.size / 1024) * 2.0 ** -53
            for got in (x[b or 0] for x in norms):
                near = (tol + (0.0 if wide else 2.0 ** -24)) * want + (2.0 ** -1073 if wide else 2.0 ** -148)
                assert got == want or (math.isnan(want) and math.isnan(got)) or abs(got - want) <= near, (case, want, got)
            c = 1.0 if limit == math.inf else math.nan if math.isnan(want) else min(1.0, limit / (want + 1e-6))
            for a, o in zip(before, after):
                with np.errstate(all="ignore"):
                    exact, o = c * np.asarray(pick(a)), np.asarray(pick(o))
                    t = grads[[x is a for x in before].index(True)].dtype
                    # (a factor below 2^-1022 has steps of 2^-1074)
                    bound = (tol + 6 * 2.0 ** -53 + HALF_STEP[t] * (1 + 2.0 ** -10) + (2.0 ** -1074 / c if 0.0 < c < 2.0 ** -1022 else 0.0)) * np.abs(exact) + TINY[t]
                    ok = (np.abs(o - exact) <= bound) | (np.isnan(exact) & np.isnan(o)) | (o == exact)
                assert ok.all(), case
        if not in_place:
            for g, a in zip(grads, before):
                assert np.array_equal(g.double().cpu().numpy(), a, equal_nan=True)
