"""GPU tests of gradient limits and drawn starts where the framework uses them: the three optimiser loops, a batch of
evaluations, the periodogram's frequency posterior, the sampler's starts, and all of them in one multi-start fit.

``train`` against a loop of torch's own ``clip_grad_norm_``, and the device-resident loops against ``train``, are held to the
tolerances those loops are held to without a limit (tests/test_gpu_parity.py: 1e-9 on the losses): clipping multiplies the
gradient by a factor that both sides form in float64 to a few roundings.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import os, sys
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _draw_oracle as oracle
from pgmuvi_amd import gpytorch as g, lombscargle as L, mcmc, synthetic as syn
from pgmuvi_amd.batch import evaluate_batch
from pgmuvi_amd.gradients import clip_grads_
from pgmuvi_amd.trainers import train, train_device, train_native

D = torch.float64


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("-m gpu tests need the MI355X")
    return torch.device("cuda:0")


def _model(dev, n, learn_noise=False, two_d=False):
    if two_d:
        x, y, e = syn.cfg4(n_per_band=n)
        h = syn.cfg_hypers(4, y.double())
        q, d = 3, 2
    else:
        x, y, e = syn.cfg2(n_obs=n)
        h = syn.cfg_hypers(2, y.double())
        q, d = 4, 1
    x, y, nz = x.double().to(dev), y.double().to(dev), (e.double() ** 2).to(dev)
    lik = g.likelihoods.GaussianLikelihood().double().to(dev) if learn_noise else g.likelihoods.FixedNoiseGaussianLikelihood(nz)

    class Model(g.models.ExactGP):
        def __init__(self):
            super().__init__(x, y, lik)
            self.mean_module = g.means.ConstantMean()
            self.covar_module = g.kernels.SpectralMixtureKernel(num_mixtures=q, **({"ard_num_dims": d} if d > 1 else {}))

        def forward(self, v):
            return g.distributions.MultivariateNormal(self.mean_module(v), self.covar_module(v))

    m = Model().double().to(dev)
    m.initialize(**{"covar_module.mixture_weights": h["w"].to(dev) * 0.7, "covar_module.mixture_means": h["mu"].to(dev) * 1.02,
                    "covar_module.mixture_scales": h["v"].to(dev) * 1.5, "mean_module.constant": torch.tensor(0.1, dtype=D, device=dev)})
    if learn_noise:
        lik.noise = torch.tensor(0.02, dtype=D, device=dev)
    return m, lik, x, y


def _losses(r):
    return np.array(r["loss"], dtype=float)


def _raw(m):
    return torch.cat([p.detach().reshape(-1) for p in m.parameters()])


@pytest.mark.parametrize("n", [60, 300])
@pytest.mark.parametrize("optim", ["SGD", "Adam"])
def test_the_loop_clips_like_torch(dev, n, optim):
    m, lik, x, y = _model(dev, n)
    r = train(model=m, likelihood=lik, train_x=x, train_y=y, maxiter=12, lr=0.02, optim=optim, progress=False, max_grad_norm=0.05)
    m2, lik2, _, _ = _model(dev, n)
    m2.train(); lik2.train()
    mll = g.mlls.ExactMarginalLogLikelihood(lik2, m2)
    opt = (torch.optim.SGD if optim == "SGD" else torch.optim.Adam)(m2.parameters(), lr=0.02)
    losses, clipped = [], 0
    for _ in range(12):
        opt.zero_grad()
        loss = -mll(m2(x), y)
        loss.backward()
        clipped += float(torch.nn.utils.clip_grad_norm_(m2.parameters(), 0.05)) > 0.05
        opt.step()
        losses.append(float(loss.detach()))
    assert clipped >= 3                                          # (the limit does something here)
    assert np.allclose(_losses(r), losses, rtol=0, atol=1e-9)
    assert torch.allclose(_raw(m), _raw(m2), rtol=1e-8, atol=1e-10)


@pytest.mark.parametrize("n, learn_noise, two_d", [(60, False, False), (60, True, False), (300, True, False), (1300, False, False), (10, False, True)])
def test_device_resident_loops_follow_the_loop(dev, n, learn_noise, two_d):
    for optim, limit in (("SGD", 0.03), ("AdamW", 0.03), ("SGD", 0.0), ("Adam", 1e12)):
        runs = []
        for loop, kw in ((train, dict(progress=False)), (train_native, {}), (train_device, {})):
            m, lik, x, y = _model(dev, n, learn_noise, two_d)
            start = _raw(m).clone()
            r = loop(model=m, likelihood=lik, train_x=x, train_y=y, maxiter=30, lr=0.01, optim=optim, max_grad_norm=limit, **kw)
            runs.append((_losses(r), _raw(m), start))
        tol = 1e-9 if optim == "SGD" else 2e-5                   # (torch's capturable Adam counts its steps in float32: train_device)
        assert np.allclose(runs[0][0], runs[1][0], rtol=0, atol=1e-9), (optim, limit)
        assert np.allclose(runs[0][0], runs[2][0], rtol=0, atol=tol), (optim, limit)
        if limit == 0.0:
            for _, raw, start in runs:
                assert torch.equal(raw, start)                   # (no step at all)


def test_one_native_step_has_the_limit_as_its_length(dev):
    for n in (60, 300):
        m, lik, x, y = _model(dev, n)
        start = _raw(m).clone()
        train_native(model=m, likelihood=lik, train_x=x, train_y=y, maxiter=1, lr=0.5, optim="SGD", max_grad_norm=0.01)
        step = float((_raw(m) - start).norm()) / 0.5
        assert 0.01 * (1 - 1e-3) < step <= 0.01 * (1 + 1e-12)    # (norm / (norm + 1e-6) of the limit)


def test_without_a_limit_nothing_changes(dev):
    for n in (60, 300):
        runs = []
        for kw in ({}, dict(max_grad_norm=None), dict(max_grad_norm=math.inf)):
            m, lik, x, y = _model(dev, n)
            r = train_native(model=m, likelihood=lik, train_x=x, train_y=y, maxiter=30, lr=0.01, optim="AdamW", **kw)
            runs.append(_losses(r))
        assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


def test_limits_are_checked(dev):
    m, lik, x, y = _model(dev, 40)
    for loop in (train, train_device, train_native):
        for bad in (-1.0, math.nan):
            with pytest.raises(ValueError, match="max_grad_norm"):
                loop(model=m, likelihood=lik, train_x=x, train_y=y, maxiter=2, max_grad_norm=bad)


def _curves(dev, B, n, Q=2):
    rows = []
    for b in range(B):
        (t, y, e), per = syn.cfg3_lightcurve(900 + b, n_obs=n)
        rows.append((t.double(), y.double(), e.double()))
    return tuple(torch.stack(c).to(dev) for c in zip(*rows))


def test_a_batch_of_evaluations_clips_each_light_curve(dev):
    B, n, Q = 6, 150, 2
    t, y, e = _curves(dev, B, n)
    w = torch.full((B, Q), 0.5, dtype=D, device=dev)
    mu = (torch.tensor([[1 / 150.0], [1 / 60.0]], dtype=D, device=dev)).expand(B, Q, 1).contiguous()
    v = torch.full((B, Q, 1), 1 / 900.0, dtype=D, device=dev)
    args = (t.unsqueeze(-1), y, y.mean(-1, keepdim=True).expand(B, n).contiguous(), e ** 2, w, mu, v)
    free = evaluate_batch(*args)
    flat = torch.cat([free[k].reshape(B, -1) for k in ("g_w", "g_mu", "g_v")], 1)
    norms = flat.norm(dim=1)
    limit = float(norms.median())
    out = evaluate_batch(*args, max_grad_norm=limit)
    assert torch.allclose(out["grad_norm"], norms, rtol=1e-13) and torch.equal(out["mll"], free["mll"])
    got = torch.cat([out[k].reshape(B, -1) for k in ("g_w", "g_mu", "g_v")], 1)
    assert torch.allclose(got, flat * torch.clamp(limit / (norms + 1e-6), max=1.0)[:, None], rtol=1e-13)
    assert torch.equal(out["g_noise"], free["g_noise"])          # (not among the clipped ones)
    both = evaluate_batch(*args, max_grad_norm=limit, clip=("g_w", "g_mu", "g_v", "g_noise", "g_mean"), chunk=4)
    assert bool((both["grad_norm"] >= norms * (1 - 1e-12)).all())
    with pytest.raises(ValueError, match="need_grad"):
        evaluate_batch(*args, need_grad=False, max_grad_norm=1.0)


def test_frequencies_are_drawn_from_the_periodogram(dev):
    B, n = 3, 120
    t, y, e = _curves(dev, B, n)
    u = torch.as_tensor(np.random.default_rng(0).random((B, 16)), device=dev)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=5, temperature=3.0), dict(min_p=0.1)):
        f, lp, grid = L.draw_frequencies(t, y, e, u, **kw)
        P = L.periodogram_batched(t, y, e, grid)
        odds = (-0.5 * (n - 3) * torch.log1p(-P.clamp(max=1 - 2.0 ** -52))).cpu().numpy()
        for b in range(B):
            idx, want = oracle.draw_row(odds[b], u[b].cpu().numpy(), **kw)
            assert torch.equal(f[b].cpu(), grid.cpu()[idx])
            assert np.allclose(lp[b].cpu().numpy(), want, rtol=1e-9, atol=1e-9)     # (odds of hundreds, log1p on two machines)
    fap = torch.exp(-torch.as_tensor(odds))                      # the odds are the reciprocal of the single-frequency false-alarm probability
    assert torch.allclose(fap, (1 - P.cpu()) ** (0.5 * (n - 3)), rtol=1e-9)
    best, _, _ = L.draw_frequencies(t, y, e, u[:, :1], temperature=0.0)
    seeds, _, _ = L.seed_frequencies(t, y, e, num_peaks=1)
    assert np.allclose(best[:, 0].cpu().numpy(), seeds[:, 0])    # temperature zero: the highest peak
    dead, lp, _ = L.draw_frequencies(t, torch.zeros_like(y), e, u)                  # a constant light curve has no periodogram (0 / 0)
    assert bool(torch.isnan(dead).all()) and bool((lp == -math.inf).all())


def test_chains_start_on_the_periodogram(dev):
    t, y, e = _curves(dev, 1, 100)
    kw = dict(noise=e[0] ** 2, num_mixtures=2, num_chains=3, num_samples=2, warmup_steps=2, max_tree_depth=2, seed=5, group_by_chain=True)
    a = mcmc.run_mcmc(t[0], y[0], initial_values="periodogram", **kw)
    b = mcmc.run_mcmc(t[0], y[0], initial_values="periodogram", **kw)
    f = a["covar_module.mixture_means_prior"]
    assert f.shape == (3, 2, 2, 1, 1) and np.isfinite(f).all() and (f > 0).all()
    assert np.array_equal(f, b["covar_module.mixture_means_prior"])
    with pytest.raises(ValueError, match="initial_values"):
        mcmc.run_mcmc(t[0], y[0], initial_values="prior", **kw)
    with pytest.raises(NotImplementedError, match="one input dimension"):
        mcmc.run_mcmc(torch.stack([t[0], t[0]], -1), y[0], initial_values="periodogram", **kw)


def test_a_multi_start_fit(dev):
    """Eight starts for one light curve: frequencies drawn from its periodogram, all starts evaluated in one batch, every start's
    gradient limited on its own, steps taken in the logarithms."""
    S, n, Q = 8, 140, 2
    t, y, e = _curves(dev, 1, n)
    u = torch.as_tensor(np.random.default_rng(3).random((1, S * Q)), device=dev)
    f, lp, _ = L.draw_frequencies(t, y, e, u, top_p=0.95, temperature=2.0)
    assert bool(torch.isfinite(f).all()) and bool((lp <= 0).all())
    theta = dict(w=torch.full((S, Q), 0.4, dtype=D, device=dev), mu=f.reshape(S, Q, 1).clone(), v=torch.full((S, Q, 1), 1 / 1000.0, dtype=D, device=dev))
    rows = lambda a: a.expand(S, n).contiguous()
    for _ in range(5):
        out = evaluate_batch(rows(t).unsqueeze(-1), rows(y), rows(y.mean(-1, keepdim=True)), rows(e ** 2), theta["w"], theta["mu"], theta["v"])
        logs = [out["g_" + k] * theta[k] for k in ("w", "mu", "v")]
        before = torch.cat([z.reshape(S, -1) for z in logs], 1).norm(dim=1)
        norm = clip_grads_(logs, 0.2, members=True)
        after = torch.cat([z.reshape(S, -1) for z in logs], 1).norm(dim=1)
        assert torch.allclose(norm, before, rtol=1e-13) and bool((after <= 0.2 * (1 + 1e-12)).all())
        assert torch.allclose(after, torch.minimum(before, 0.2 * before / (before + 1e-6)), rtol=1e-12)
        for k, z in zip(("w", "mu", "v"), logs):
            theta[k] = theta[k] * torch.exp(0.5 * z)
    assert all(bool(torch.isfinite(x).all()) and bool((x > 0).all()) for x in theta.values())


def test_a_limit_is_set_before_the_first_step(dev):
    from pgmuvi_amd.trainers import _native_fit_handle
    m, lik, x, y = _model(dev, 60)
    fit = _native_fit_handle(m, lik, x, y, 4, 1e-3, "Adam", 1e-8)[0]
    for bad in (-1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError):
            fit.set_clip(bad)
    fit.set_clip(0.5)
    fit.set_clip(0.25)
    fit.run(2)
    with pytest.raises(RuntimeError):
        fit.set_clip(1.0)


def test_chains_without_a_periodogram_and_with_spans_of_their_own(dev):
    t, y, e = _curves(dev, 3, 100)
    t = t.clone()
    t[1] *= 1.5                                                  # (its own span, so its own grid)
    both = mcmc._start_frequencies(t, y, e, 4, 7, range(5, 8))
    alone = [mcmc._start_frequencies(t[c:c + 1], y[c:c + 1], e[c:c + 1], 4, 7, range(5 + c, 6 + c)) for c in range(3)]
    assert np.array_equal(both, np.concatenate(alone)) and np.isfinite(both).all()
    y = y.clone()
    y[2] = 0.0
    dead = mcmc._start_frequencies(t, y, e, 4, 7, range(5, 8))
    assert np.array_equal(dead[:2], both[:2]) and np.isnan(dead[2]).all()
    kw = dict(noise=e ** 2, num_mixtures=2, num_samples=2, warmup_steps=2, max_tree_depth=2, seed=5, group_by_chain=True)
    with pytest.raises(ValueError, match=r"chains \[2\]"):
        mcmc.run_mcmc(t.unsqueeze(-1), y, initial_values="periodogram", **kw)


@pytest.mark.parametrize("n", [60, 300, 1300])
@pytest.mark.parametrize("optim", ["SGD", "Adam"])
def test_an_infinite_gradient_gives_every_loop_the_same_step(dev, n, optim):
    """A prior so narrow that its derivative overflows while its logarithm does not ((1e-10 / 2^-535)^2 / 2 = 6e301, and the
    variance 2^-1070 is exact): the norm is infinite, the factor zero, and only the infinite entry's parameter becomes NaN."""
    ends = []
    for loop, kw in ((train, dict(progress=False)), (train_native, {}), (train_device, {})):
        m, lik, x, y = _model(dev, n)
        m.initialize(**{"mean_module.constant": torch.tensor(1e-10, dtype=D, device=dev)})
        scale = torch.tensor(2.0 ** -535, dtype=D, device=dev)
        m.mean_module.register_prior("narrow", g.priors.NormalPrior(torch.zeros_like(scale), scale), "constant")
        start = {k: p.detach().clone() for k, p in m.named_parameters()}
        r = loop(model=m, likelihood=lik, train_x=x, train_y=y, maxiter=1, lr=0.01, optim=optim, max_grad_norm=0.1, **kw)
        assert np.isfinite(_losses(r)).all()
        for k, p in m.named_parameters():
            if k == "mean_module.raw_constant":
                assert bool(torch.isnan(p).all()), loop
            else:
                assert torch.equal(p.detach(), start[k]), (loop, k)
        ends.append(_losses(r))
    assert np.allclose(ends[0], ends[1], rtol=1e-9, atol=0) and np.allclose(ends[0], ends[2], rtol=1e-9, atol=0)


def _apart(f, baseline):
    """Smallest distance of two frequencies of each row, in peak widths (1 / baseline)."""
    f = np.sort(np.asarray(f), axis=-1)
    return np.diff(f, axis=-1).min(-1) * baseline


@pytest.mark.parametrize("n", [89, 300, 1000])
def test_distinct_frequencies_are_drawn_from_what_the_earlier_ones_leave(dev, n):
    """The light curves have a clear period: 0.95 of the odds lie in one or two grid points."""
    B, S = 3, 6
    t, y, e = _curves(dev, B, n)
    t = (t - t.amin(1, keepdim=True)) / (t.amax(1, keepdim=True) - t.amin(1, keepdim=True)) * 3450.0     # (one span)
    u = torch.as_tensor(np.random.default_rng(n).random((B, S)), device=dev)
    plain, _, grid = L.draw_frequencies(t, y, e, u, top_p=0.95)
    assert (_apart(plain.cpu(), 3450.0) < 1.0).all()             # (with repetition: the same peak again)
    odds = (-0.5 * (n - 3) * torch.log1p(-L.periodogram_batched(t, y, e, grid).clamp(max=1 - 2.0 ** -52))).cpu().numpy()
    for kw in (dict(top_p=0.95), dict(temperature=5.0, min_p=1e-3), dict(temperature=0.0)):
        f, lp, _ = L.draw_frequencies(t, y, e, u, distinct=True, **kw)
        assert (_apart(f.cpu(), 3450.0) > 1.0).all()
        for b in range(B):
            left = odds[b].copy()
            for s in range(S):
                idx, want = oracle.draw_row(left, u[b, s:s + 1].cpu().numpy(), **kw)
                assert float(f[b, s]) == float(grid[int(idx[0])]), (b, s)
                assert abs(float(lp[b, s]) - want[0]) <= 1e-9 * max(1.0, abs(want[0]))       # (odds of hundreds, log1p on two machines)
                left[max(0, idx[0] - 5):idx[0] + 6] = -math.inf
    assert L.draw_frequencies(t, y, e, u[:, :0], distinct=True)[0].shape == (B, 0)
    dead, lp, _ = L.draw_frequencies(t, torch.zeros_like(y), e, u, distinct=True)
    assert bool(torch.isnan(dead).all()) and bool((lp == -math.inf).all())


def test_more_distinct_frequencies_than_there_are_begin_again(dev):
    t, y, e = _curves(dev, 2, 8)
    t = (t - t.amin(1, keepdim=True)) / (t.amax(1, keepdim=True) - t.amin(1, keepdim=True)) * 100.0
    u = torch.as_tensor(np.random.default_rng(1).random((2, 60)), device=dev)
    f, lp, grid = L.draw_frequencies(t, y, e, u, distinct=True)
    assert grid.numel() < 60 * 6 and bool(torch.isfinite(f).all()) and bool((lp <= 0).all())
    first = grid.numel() // 11                                   # (a draw takes at most eleven grid points away)
    assert (_apart(f[:, :first].cpu(), 100.0) > 1.0).all()


@pytest.mark.parametrize("n", [89, 300, 1000])
def test_the_mixtures_of_a_chain_start_on_different_peaks(dev, n):
    t, y, e = _curves(dev, 3, n)
    span = (t.amax(1) - t.amin(1)).cpu().numpy()
    chains, Q = 8, 4
    for b in range(3):
        f = mcmc._start_frequencies(t[b].expand(chains, n), y[b].expand(chains, n), e[b].expand(chains, n), Q, 5, range(chains))
        assert f.shape == (chains, Q) and (_apart(f, span[b]) > 1.0).all()


def test_chains_differ_where_the_data_leave_a_choice(dev):
    """Noise alone: 0.95 of the odds of the first draw are spread over 260 of 750 grid points, the largest share is 0.36."""
    n, chains, Q = 60, 8, 4
    rng = np.random.default_rng(4)
    t = torch.as_tensor(np.sort(rng.uniform(0, 1000.0, n)), device=dev).expand(chains, n)
    y = torch.as_tensor(rng.normal(size=n), device=dev).expand(chains, n)
    f = mcmc._start_frequencies(t, y, None, Q, 5, range(chains))
    assert len(np.unique(f[:, 0])) >= 3 and len(np.unique(np.sort(f, axis=1), axis=0)) >= 6
    assert (_apart(f, float(t.max() - t.min())) > 1.0).all()
