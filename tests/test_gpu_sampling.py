"""GPU tests of the draws against numpy in float64.

The indices are compared exactly: the inputs are fixed, and a draw or a cut would have to lie within the ~1e-13 relative
difference of two orders of summation to come out differently.  The log-probabilities are z - log Z: z carries two roundings
(difference, quotient) and Z the sum of up to V weights, each with an error of at most 2 steps of the exponential and one of its
argument's: |error| <= 2 |z| 2^-53 + (4 + V / 64) 2^-53 + 2 |log Z| 2^-53.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import os, sys
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _draw_oracle as oracle
from pgmuvi_amd.sampling import draw_indices

TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("-m gpu tests need the MI355X")
    return torch.device("cuda:0")


def _rows(B, V, dtype, seed, peaks=2):
    """Log odds like a periodogram's: exponential noise and a few peaks."""
    rng = np.random.default_rng(seed)
    l = rng.exponential(size=(B, V))
    for b in range(B):
        for _ in range(peaks):
            l[b, rng.integers(0, V)] += rng.uniform(0, 12)
    return torch.as_tensor(l).to(dtype)


def _check(logits, u, got, lengths=None, **settings):
    idx, logp = got
    l = logits.double().cpu().numpy()
    idx, logp, u = idx.cpu().numpy(), logp.cpu().numpy(), u.double().cpu().numpy()
    assert idx.dtype == np.int64 and logp.dtype == np.float64 and idx.shape == u.shape
    if u.ndim == 1:
        idx, logp, u = idx[:, None], logp[:, None], u[:, None]
    for b in range(l.shape[0]):
        row = {k: (v[b] if isinstance(v, (list, np.ndarray)) else v) for k, v in settings.items()}
        n = l.shape[1] if lengths is None else max(0, min(l.shape[1], lengths[b]))
        want, wlp = oracle.draw_row(l[b, :n], u[b], **row)
        if idx[b].tolist() != want.tolist() and 0.0 < row.get("top_p", 1.0) < 1.0:
            # A cut exactly on the border.  Weights k/5 (test_ties_go_to_the_lower_index) can put a running sum at top_p Z in real
            # arithmetic; whether the computed sum reaches the computed product is then a matter of roundings.  Each weight is off by
            # at most 4 half steps (exponential and argument), a sum of V of them by V half steps more, the product by one: cuts of
            # top_p (1 +- e) with e = (V + 5) 2^-53 enclose every correctly rounded one.
            e = (n + 5) * 2.0 ** -53
            near = [oracle.draw_row(l[b, :n], u[b], **dict(row, top_p=row["top_p"] * f)) for f in (1 - e, 1 + e)]
            want, wlp = next((r for r in near if idx[b].tolist() == r[0].tolist()), (want, wlp))
        assert idx[b].tolist() == want.tolist(), (b, row)
        live = want >= 0
        z = l[b, idx[b][live]] - np.nanmax(l[b, :n]) if live.any() else np.zeros(0)
        t = row.get("temperature", 1.0)
        t = t if t > 0 else 1.0                                  # (0, negative, NaN: the best entry, z = 0)
        with np.errstate(invalid="ignore"):
            tol = 2.0 ** -53 * (4 * np.abs(np.nan_to_num(z) / t) + 4 + l.shape[1] / 64 + 2 * np.abs(wlp[live]) + 8)
        assert (np.abs(logp[b][live] - wlp[live]) <= tol).all()
        assert (logp[b][~live] == -math.inf).all()


SETTINGS = [dict(), dict(temperature=0.3), dict(temperature=4.0), dict(top_k=1), dict(top_k=7), dict(top_k=10 ** 9), dict(top_p=0.9), dict(top_p=0.05), dict(top_p=0.0),
            dict(top_p=1.0), dict(min_p=0.1), dict(min_p=1.0), dict(top_k=40, top_p=0.8, min_p=0.02, temperature=1.7), dict(temperature=0.0), dict(top_p=0.999, min_p=1e-9)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
@pytest.mark.parametrize("dtype", TYPES)
def test_draws(dev, dtype, settings):
    for B, V, S in ((1, 1, 3), (3, 2, 5), (2, 63, 9), (2, 65, 1), (5, 1113, 8), (2, 9001, 33)):
        l = _rows(B, V, dtype, 100 * V + B)
        u = torch.as_tensor(np.random.default_rng(V).random((B, S)))
        _check(l, u, draw_indices(l.to(dev), u.to(dev), return_logprob=True, **settings), **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=300), dict(top_p=0.6), dict(top_k=5000, top_p=0.97), dict(min_p=0.3)], ids=str)
@pytest.mark.parametrize("dtype, V", [(torch.float64, 51200), (torch.float64, 204800), (torch.float32, 70001), (torch.bfloat16, 140001), (torch.float64, 1_300_001)])
def test_long_rows(dev, dtype, V, settings):
    l = _rows(1, V, dtype, V)
    u = torch.as_tensor(np.random.default_rng(V).random((1, 40)))
    _check(l, u, draw_indices(l.to(dev), u.to(dev), return_logprob=True, **settings), **settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 3000, 30_000])
def test_ties_go_to_the_lower_index(dev, dtype, V):
    rng = np.random.default_rng(V)
    for levels in (1, 2, 5):
        l = torch.as_tensor(np.log(rng.integers(1, levels + 1, size=(3, V)).astype(float)) if levels > 1 else np.full((3, V), -7.5)).to(dtype)
        u = torch.as_tensor(rng.random((3, 20)))
        for settings in (dict(top_k=V // 3), dict(top_k=V - 1), dict(top_p=0.5), dict(top_p=0.37, temperature=0.8), dict(top_k=V // 2 + 1, top_p=0.25), dict(temperature=0.0)):
            _check(l, u, draw_indices(l.to(dev), u.to(dev), return_logprob=True, **settings), **settings)
    uniform = torch.zeros(1, V, dtype=dtype, device=dev)
    u = (torch.arange(V, dtype=torch.float64, device=dev)[None] + 0.5) / V
    assert torch.equal(draw_indices(uniform, u)[0], torch.arange(V, device=dev))
    half = draw_indices(uniform, u, top_p=0.5)[0]
    assert int(half.max()) == (V + 1) // 2 - 1 and int(half.min()) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_and_nonfinite_entries(dev, dtype):
    low = torch.finfo(dtype).min
    V = 700
    base = _rows(7, V, dtype, 5)
    base[0, :] = -math.inf                                       # nothing to draw
    base[1, :] = math.nan
    base[2, ::2] = -math.inf
    base[2, 1::4] = math.nan
    base[3, 5:] = low                                            # masked with the type's lowest value
    base[4, :] = low                                             # ... all of them: equal weights
    base[5, 3], base[5, 90] = math.inf, math.inf                 # two certain ones
    base[6, 1:] = -math.inf                                      # a single entry
    u = torch.as_tensor(np.random.default_rng(1).random((7, 12)))
    for settings in (dict(), dict(top_k=4), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0), dict(top_k=699, top_p=0.99), dict(temperature=1e6)):
        got = draw_indices(base.to(dev), u.to(dev), return_logprob=True, **settings)
        assert (got[0][:2] == -1).all() and (got[1][:2] == -math.inf).all()
        sub = [2, 3, 4, 6]
        _check(base[sub], u[sub], (got[0][sub], got[1][sub]), **settings)
        assert set(got[0][5].tolist()) <= {3, 90}
        keep = 1 if settings.get("temperature") == 0.0 else 2
        assert float((got[1][5] + math.log(keep)).abs().max()) < 1e-15
    signed = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], dtype=dtype, device=dev)       # equal values
    assert draw_indices(signed, torch.tensor([[0.1, 0.9]], device=dev), top_k=2).tolist() == [[0, 1]]


def test_random_numbers_at_their_limits(dev):
    l = torch.tensor([[-2000.0, 0.0, 1.0, -2000.0, 0.5, -2000.0]], dtype=torch.float64, device=dev)
    u = torch.tensor([[0.0, 1.0 - 2.0 ** -53, 1.0, 5.0, -1.0, math.nan, -0.0]], dtype=torch.float64, device=dev)
    assert draw_indices(l, u).tolist() == [[1, 4, 4, 4, 1, 4, 1]]                # (entries without weight are never drawn)
    u32 = torch.tensor([[0.0, 0.25, 1.0 - 2.0 ** -24]], device=dev)
    assert draw_indices(l, u32).tolist() == [[1, 2, 4]]


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_settings_per_row_and_strides(dev, dtype):
    B, V, S = 9, 1500, 6
    l = _rows(B, V, dtype, 77)
    u = torch.as_tensor(np.random.default_rng(2).random((B, S)))
    lengths = [0, 1, 2, 64, 700, 1499, 1500, 5000, -3]
    poisoned = l.clone()
    for b, n in enumerate(lengths):
        poisoned[b, max(0, n):] = math.inf                       # (never read)
    per = dict(temperature=np.array([1.0, 0.5, 0.0, -1.0, 2.0, 1.0, 3.0, math.nan, 1.0]), top_k=np.array([0, 3, 5, 0, -2, 40, 1000, 3, 1]),
               top_p=np.array([1.0, 0.5, 0.9, 0.0, 0.8, 2.0, math.nan, 0.3, 0.5]), min_p=np.array([0.0, 0.1, 0.0, 0.0, -1.0, 0.05, 0.0, 7.0, math.nan]))
    on = {k: torch.as_tensor(v).to(dev) for k, v in per.items()}
    got = draw_indices(poisoned.to(dev), u.to(dev), lengths=torch.as_tensor(lengths), return_logprob=True, **on)
    _check(l, u, got, lengths=lengths, **per)
    assert got[0][0].tolist() == [-1] * S and got[0][8].tolist() == [-1] * S
    wide = torch.zeros(B, 2 * V + 7, dtype=dtype, device=dev)
    views = [wide[:, 3:V + 3], wide[:, 1:2 * V:2], torch.zeros(V, B, dtype=dtype, device=dev).t()]
    plain = draw_indices(l.to(dev), u.to(dev), top_k=50, top_p=0.9)
    for v in views:
        v.copy_(l)
        assert torch.equal(draw_indices(v, u.to(dev), top_k=50, top_p=0.9), plain)
    one = draw_indices(l[4].to(dev), u[4].to(dev), top_k=50, top_p=0.9)
    assert torch.equal(one, plain[4]) and one.shape == (S,)
    assert torch.equal(draw_indices(l.to(dev), u[:, 2].to(dev), top_k=50, top_p=0.9), plain[:, 2])
    assert draw_indices(l[4].to(dev), u[4, 1].to(dev), top_k=50, top_p=0.9).item() == int(plain[4, 1])
    assert torch.equal(draw_indices(l[4].to(dev).expand(3, V), u[4:5].to(dev).expand(3, S), top_k=50, top_p=0.9), plain[4:5].expand(3, S))


def test_empty_shapes_and_refusals(dev):
    l = torch.zeros(4, 10, device=dev)
    assert draw_indices(l, torch.zeros(4, 0, device=dev)).shape == (4, 0)
    assert draw_indices(l[:0], torch.zeros(0, 3, device=dev)).shape == (0, 3)
    i, p = draw_indices(l[:, :0], torch.zeros(4, 2, device=dev), return_logprob=True)
    assert (i == -1).all() and (p == -math.inf).all()
    for args, kw in (((l, torch.zeros(3, 2, device=dev)), {}), ((l, torch.zeros((), device=dev)), {}), ((l[0], torch.zeros(2, 2, device=dev)), {}),
                     ((l[None], torch.zeros(4, 2, device=dev)), {}), ((l, torch.zeros(4, 2)), {}), ((l, torch.zeros(4, 2, device=dev)), dict(top_p=1.5)),
                     ((l, torch.zeros(4, 2, device=dev)), dict(lengths=torch.zeros(3, dtype=torch.int64))), ((l, torch.zeros(4, 2, device=dev)), dict(top_k=0)),
                     ((l, torch.zeros(4, 2, device=dev)), dict(temperature=torch.ones(3, device=dev)))):
        with pytest.raises((ValueError, RuntimeError)):
            draw_indices(*args, **kw)


def test_a_row_does_not_depend_on_its_company_or_on_the_call(dev):
    l, u = _rows(300, 2000, torch.float64, 3).to(dev), torch.rand(300, 4, dtype=torch.float64, device=dev)
    all_rows = draw_indices(l, u, top_p=0.8, return_logprob=True)
    for _ in range(2):
        again = draw_indices(l, u, top_p=0.8, return_logprob=True)
        assert torch.equal(again[0], all_rows[0]) and torch.equal(again[1], all_rows[1])
    some = draw_indices(l[17:19], u[17:19], top_p=0.8, return_logprob=True)
    assert torch.equal(some[0], all_rows[0][17:19]) and torch.equal(some[1], all_rows[1][17:19])


def test_streams_and_a_replayed_graph(dev):
    l, u = _rows(20, 3001, torch.float32, 8).to(dev), torch.rand(20, 5, dtype=torch.float64, device=dev)
    want = draw_indices(l, u, top_k=30, top_p=0.9, return_logprob=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = draw_indices(l, u, top_k=30, top_p=0.9, return_logprob=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = draw_indices(l, u, top_k=30, top_p=0.9, return_logprob=True)
    for k in range(3):
        u.copy_(torch.rand(20, 5, dtype=torch.float64, device=dev))
        l.copy_(_rows(20, 3001, torch.float32, 50 + k))
        graph.replay()
        eager = draw_indices(l, u, top_k=30, top_p=0.9, return_logprob=True)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_frequencies_of_draws_follow_the_weights(dev):
    w = np.array([0.05, 0.3, 0.15, 0.4, 0.1])
    u = (torch.arange(1000, dtype=torch.float64, device=dev)[None] + 0.5) / 1000
    idx = draw_indices(torch.as_tensor(np.log(w))[None].to(dev), u)[0]
    assert torch.bincount(idx, minlength=5).tolist() == [50, 300, 150, 400, 100]


def test_more_than_32_bits_of_offset(dev):
    V = 4_000_000
    rows = torch.zeros(1100, V, dtype=torch.bfloat16, device=dev)
    rows[1099, V - 2] = 30.0
    u = torch.full((1100, 1), 0.75, dtype=torch.float64, device=dev)
    idx = draw_indices(rows, u, min_p=0.5)
    assert int(idx[1099]) == V - 2 and int(idx[0]) == 3 * V // 4


@pytest.mark.parametrize("settings", [dict(), dict(top_k=20), dict(top_k=3000), dict(top_p=0.9), dict(top_k=900, top_p=0.6, min_p=0.01), dict(min_p=0.05)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B, V, S", [(2, 60_000, 3), (2, 60_000, 100), (64, 20_001, 1), (70, 20_001, 70), (600, 20_001, 2), (600, 3000, 90), (1100, 1500, 3)])
def test_every_division_of_the_work(dev, B, V, S, dtype, settings):
    """Rows shared by workgroups, one workgroup per row in its builds, draws apart from the rest: a few rows of each against numpy."""
    l = _rows(B, V, dtype, B + V)
    u = torch.as_tensor(np.random.default_rng(B).random((B, S)))
    lengths = [V] * B
    lengths[1] = V - 777 if V > 1000 else V
    idx, logp = draw_indices(l.to(dev), u.to(dev), lengths=torch.as_tensor(lengths), return_logprob=True, **settings)
    assert int(idx.min()) >= 0
    some = sorted({0, 1, B // 2, B - 1})
    _check(l[some], u[some], (idx[some], logp[some]), lengths=[lengths[b] for b in some], **settings)


@pytest.mark.parametrize("V", [30_000, 300_000])
def test_long_rows_with_settings_per_row(dev, V):
    B = 5
    l = _rows(B, V, torch.float64, 4)
    l[3] = l[3].round()                                          # (many ties)
    l[4, :] = 0.0
    u = torch.as_tensor(np.random.default_rng(9).random((B, 20)))
    per = dict(temperature=np.array([1.0, 0.0, 0.5, 2.0, 1.0]), top_k=np.array([0, 7, 0, V // 3, 0]), top_p=np.array([1.0, 0.5, 0.9, 0.4, 0.3]),
               min_p=np.array([0.01, 0.0, 0.0, 0.0, 0.0]))
    got = draw_indices(l.to(dev), u.to(dev), return_logprob=True, **{k: torch.as_tensor(v).to(dev) for k, v in per.items()})
    _check(l, u, got, **per)
    wide = l.to(dev).t().contiguous().t()                        # a column per frequency: strided rows
    assert torch.equal(draw_indices(wide, u.to(dev), top_p=0.8), draw_indices(l.to(dev), u.to(dev), top_p=0.8))


def test_negated_views(dev):
    """The imaginary part of a conjugate is a view whose memory holds the opposite sign."""
    z = torch.complex(torch.zeros(2, 500, dtype=torch.float64), torch.as_tensor(np.random.default_rng(1).normal(0, 3, (2, 500)))).to(dev).conj()
    l, u = z.imag, torch.as_tensor(np.random.default_rng(2).random((2, 8)), device=dev)
    assert l.is_neg() and torch.equal(draw_indices(l, u), draw_indices(l.clone(), u))


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_k=700), dict(top_p=0.4, min_p=0.1), dict(min_p=0.05)])
def test_many_draws_of_many_short_rows(dev, dtype, kw):
    """A row's draws do not depend on how many there are, nor on the rows beside it."""
    g = np.random.default_rng(11)
    l = torch.as_tensor(g.normal(0, 3, (1030, 777))).to(dtype).to(dev)
    l[5] = -math.inf
    u = torch.as_tensor(g.random((1030, 130)), device=dev)
    index, logp = draw_indices(l, u, return_logprob=True, **kw)
    assert bool((index[5] == -1).all())
    for s in (slice(0, 40), slice(90, 130)):
        few, lp = draw_indices(l, u[:, s], return_logprob=True, **kw)
        assert torch.equal(few, index[:, s]) and torch.equal(lp, logp[:, s])
    for b in (0, 1029):
        want, lp = oracle.draw_row(l[b].double().cpu().numpy(), u[b].cpu().numpy(), **kw)
        assert torch.equal(index[b].cpu(), torch.as_tensor(want)) and np.allclose(logp[b].cpu().numpy(), lp, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, lengths", [(30, 5000, None), (100, 9000, [9000, 0, 1, 4097, 777]), (2, 300_000, None), (1, 40_000, None)])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_k=3000), dict(top_p=0.4, min_p=0.1), dict(min_p=0.05)])
def test_many_draws_of_long_rows(dev, dtype, rows, cols, lengths, kw):
    l = _rows(rows, cols, dtype, 21).to(dev)
    g = np.random.default_rng(12)
    S = 3000 if rows < 30 else 300
    u = torch.as_tensor(g.random((rows, S)), device=dev)
    u[:, 0], u[:, 1], u[:, 2] = 0.0, 1.0 - 2.0 ** -53, 1.0
    n = None if lengths is None else torch.as_tensor((lengths * rows)[:rows], device=dev)
    index, logp = draw_indices(l, u, lengths=n, return_logprob=True, **kw)
    few, lp = draw_indices(l, u[:, :60], lengths=n, return_logprob=True, **kw)
    assert torch.equal(few[:, 3:], index[:, 3:60]) and torch.allclose(lp[:, 3:], logp[:, 3:60], rtol=1e-12, atol=1e-12)
    for b in {0, 1 % rows, 2 % rows, 4 % rows, rows - 1}:
        v = cols if n is None else int(n[b])
        want, wl = oracle.draw_row(l[b, :v].double().cpu().numpy(), u[b, :2].cpu().numpy().tolist() + u[b, 3:].cpu().numpy().tolist(), **kw)
        got, gl = index[b].cpu().numpy(), logp[b].cpu().numpy()
        assert np.array_equal(np.delete(got, 2), want) and np.allclose(np.delete(gl, 2), wl, rtol=1e-12, atol=1e-12)
        if v:
            assert got[2] == oracle.kept_entries(l[b, :v].double().cpu().numpy(), **kw)[0].max()           # (u outside [0, 1): the last kept one)


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("kw", [dict(), dict(min_p=0.05), dict(temperature=0.0), dict(top_p=0.0), dict(top_k=3), dict(top_k=600), dict(top_p=0.5), dict(top_k=5000, top_p=0.8)])
@pytest.mark.parametrize("cols", [13_000, 90_000, 210_000])
def test_a_setting_per_row_is_the_same_as_one_for_all(dev, rows, kw, cols):
    """One number and a tensor of it may take other launches: the same draws."""
    l = _rows(rows, cols, torch.float64, 5).to(dev)
    u = torch.as_tensor(np.random.default_rng(6).random((rows, 12)), device=dev)
    index, logp = draw_indices(l, u, return_logprob=True, **kw)
    each = {k: torch.full((rows,), v, dtype=torch.int64 if k == "top_k" else torch.float64, device=dev) for k, v in kw.items()}
    i2, l2 = draw_indices(l, u, return_logprob=True, **each)
    assert torch.equal(index, i2) and torch.allclose(logp, l2, rtol=1e-12, atol=1e-12)
    want, wl = oracle.draw_row(l[-1].cpu().numpy(), u[-1].cpu().numpy(), **kw)
    assert np.array_equal(index[-1].cpu().numpy(), want) and np.allclose(logp[-1].cpu().numpy(), wl, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("rows, cols, per", [(1030, 777, 40), (3, 777, 700), (3, 5000, 20), (3, 5000, 40), (2, 60_000, 700), (2, 60_000, 5000), (200, 5000, 60)])
@pytest.mark.parametrize("kw", [dict(min_p=0.3), dict(top_k=30), dict(top_k=900, min_p=0.2)])
def test_draws_at_the_borders_of_the_kept_entries(dev, rows, cols, per, kw):
    """Random numbers within a few steps of every border between two kept entries, with entries that weigh nothing between them: one
    of the two is drawn, whatever the roundings of the running sums."""
    rng = np.random.default_rng(31)
    l = rng.normal(-60.0, 1.0, cols)
    l[rng.choice(cols, 60, replace=False)] = rng.uniform(-1.0, 0.0, 60)
    idx, w, _ = oracle.kept_entries(l, **kw)
    c = np.cumsum(w)
    at = rng.integers(0, len(idx) - 1, rows * per)
    u = c[at] / c[-1] * (1.0 + rng.integers(-6, 7, rows * per) * 2.0 ** -53)
    got = draw_indices(torch.as_tensor(l, device=dev).expand(rows, cols), torch.as_tensor(u.reshape(rows, per), device=dev), **kw).cpu().numpy().ravel()
    pos = np.searchsorted(idx, got)
    assert (got >= 0).all() and np.array_equal(idx[np.minimum(pos, len(idx) - 1)], got)
    assert ((pos == at) | (pos == at + 1)).all()


def test_the_most_rows(dev):
    n = (1 << 23) - 1
    u = torch.rand(n, dtype=torch.float64, device=dev)
    l = torch.zeros(2, dtype=torch.float64, device=dev)
    assert torch.equal(draw_indices(l.expand(n, 2), u), (u >= 0.5).to(torch.int64))
    with pytest.raises(ValueError, match="rows"):
        draw_indices(l.expand(n + 1, 2), torch.zeros(1, dtype=torch.float64, device=dev).expand(n + 1))


@pytest.mark.parametrize("rows, cols, S", [(40, 9000, 300), (2, 80_000, 20), (2, 80_000, 5000), (1100, 900, 100)])
def test_graphs_of_several_launches_replayed(dev, rows, cols, S):
    """Two captured calls that share a memory pool, replayed in turn with new inputs and eager calls on another stream between."""
    l, u = _rows(rows, cols, torch.float64, 3).to(dev), torch.rand(rows, S, dtype=torch.float64, device=dev)
    kws = (dict(top_p=0.8), dict(top_k=700, min_p=0.01))
    for kw in kws:
        draw_indices(l, u, **kw)
    graphs, outs = [], []
    for kw in kws:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(draw_indices(l, u, return_logprob=True, **kw))
        graphs.append(g)
    side = torch.cuda.Stream()
    for k in range(3):
        l.copy_(_rows(rows, cols, torch.float64, 60 + k))
        u.copy_(torch.rand(rows, S, dtype=torch.float64, device=dev))
        for g, out, kw in zip(graphs, outs, kws):
            g.replay()
            got = [x.clone() for x in out]
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                eager = draw_indices(l, u, return_logprob=True, **kw)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def _mostly_masked(B, V, dtype, seed, values):
    """Rows of -inf but for 40 neighbouring entries near the beginning and 40 near the end: fewer cells with an entry than any top_k below."""
    rng = np.random.default_rng(seed)
    l = np.full((B, V), -math.inf)
    for b in range(B):
        for at in (rng.integers(0, 60), V - 100 + rng.integers(0, 60)):
            l[b, at:at + 40] = values(rng, 40)
    return torch.as_tensor(l).to(dtype)


@pytest.mark.parametrize("settings", [dict(top_k=5), dict(top_k=30, top_p=0.7), dict(top_k=79, min_p=0.2), dict(top_k=250)], ids=str)
@pytest.mark.parametrize("B, V", [(3, 9001), (520, 80_000), (1030, 2000), (1, 300_000), (2, 60_000)])
def test_fewer_cells_with_an_entry_than_top_k(dev, B, V, settings):
    """... at the lowest end of float64 (the difference to the type's lowest value is below 1e300), where the row's entries are counted in
    the bins that counted the cells, and in the usual range of every type."""
    u = torch.as_tensor(np.random.default_rng(V).random((B, 9)))
    some = sorted({0, B // 2, B - 1})
    low, step = np.finfo(np.float64).min, 2.0 ** 971             # (the distance of two float64 there)
    cases = [(torch.float64, lambda rng, n: low + step * rng.integers(0, 1 << 20, n), dict(temperature=2e296)),
             (torch.float64, lambda rng, n: low + step * rng.integers(0, 3, n), dict(temperature=2e293))]
    cases += [(dtype, lambda rng, n: rng.normal(0, 3, n), {}) for dtype in TYPES]
    for dtype, values, kw in cases:
        l = _mostly_masked(B, V, dtype, B, values)
        kw = dict(settings, **kw)
        idx, logp = draw_indices(l.to(dev), u.to(dev), return_logprob=True, **kw)
        assert int(idx.min()) >= 0
        _check(l[some], u[some], (idx[some], logp[some]), **kw)
        each = {k: torch.full((B,), v, dtype=torch.int64 if k == "top_k" else torch.float64, device=dev) for k, v in kw.items()}
        assert torch.equal(draw_indices(l.to(dev), u.to(dev), **each), idx)


def test_settings_that_are_negated_views(dev):
    """(One row's view is contiguous as it is, so that nothing on the way copies it.)"""
    for rows in (1, 3):
        l = _rows(rows, 600, torch.float64, 8).to(dev)
        u = torch.as_tensor(np.random.default_rng(2).random((rows, 40)), device=dev)
        for name, v in (("temperature", [0.5, 2.0, 1.0]), ("top_p", [0.5, 0.9, 0.3]), ("min_p", [0.1, 0.02, 0.5])):
            v = torch.tensor(v[:rows], dtype=torch.float64, device=dev)
            view = torch.complex(torch.zeros_like(v), -v).conj().imag
            assert view.is_neg() and torch.equal(view, v)
            assert torch.equal(draw_indices(l, u, **{name: view}), draw_indices(l, u, **{name: v}))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, S", [(1, 500, 12), (3, 77, 12), (1030, 900, 12), (9, 30_000, 1200), (2, 90_000, 5000)])
def test_the_last_kept_entry_at_the_end_of_the_weight(dev, rows, cols, S, dtype):
    """u within twelve steps of one, and entries that weigh nothing behind the last kept one: that one is drawn, whatever the roundings
    of the running sums behind it (the one in front of it ends a whole weight, more than 2^-18 of all, earlier)."""
    u = torch.as_tensor(1.0 - 2.0 ** -53 * (1 + np.arange(S) % 12)[None] * np.ones((rows, 1)), device=dev)
    rng = np.random.default_rng(cols)
    flat = torch.full((rows, cols), -7.5, dtype=dtype)
    few = torch.full((rows, cols), -math.inf, dtype=dtype)
    few[:, :cols // 3] = torch.as_tensor(np.log(rng.uniform(0.5, 1.0, (rows, cols // 3)))).to(dtype)
    for l, settings in ((flat, [dict(top_p=0.9), dict(top_p=0.23, temperature=0.3), dict(top_k=cols // 2 + 1), dict(top_k=17)]),
                        (few, [dict(), dict(min_p=0.7), dict(temperature=1e5), dict(top_p=0.999), dict(top_k=cols // 5)])):
        for kw in settings:
            got = draw_indices(l.to(dev), u, **kw)
            for b in (0, rows - 1):
                idx, w, _ = oracle.kept_entries(l[b].double().numpy(), **kw)
                assert (got[b] == int(idx[-1])).all(), (kw, b, int(idx[-1]), got[b][:12].tolist())


@pytest.mark.parametrize("settings", [dict(), dict(top_k=4), dict(top_k=300), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_signalling_nans_are_never_drawn_and_hide_nothing(dev, dtype, settings):
    """Every NaN bit pattern is a masked entry: the hardware's maximum returns a NaN of a signalling one instead of its other operand."""
    bits, patterns = {torch.float64: (torch.int64, (0x7FF0000000000001, -0x000FFFFFFFFFFFFF)), torch.float32: (torch.int32, (0x7F800001, -0x007FFFFF)),
                      torch.bfloat16: (torch.int16, (0x7F81, -0x007F)), torch.float16: (torch.int16, (0x7C01, -0x03FF))}[dtype]
    for B, V in ((1, 5), (3, 700), (2, 9000), (520, 20_001), (1030, 900), (1, 300_000)):
        rng = np.random.default_rng(V)
        l = _rows(B, V, dtype, V)
        for share, pattern in ((0.05, patterns[0]), (0.3, patterns[1])):
            l.view(bits)[torch.as_tensor(rng.random((B, V)) < share)] = pattern
        l[0, 3] = 2.0                                            # (not all of a short row)
        u = torch.as_tensor(rng.random((B, 6)))
        d = torch.empty(B, V, dtype=dtype, device=dev)
        d.view(bits).copy_(l.view(bits))
        idx, logp = draw_indices(d, u.to(dev), return_logprob=True, **settings)
        assert torch.equal(d.view(bits).cpu(), l.view(bits)) and int(idx[0].min()) >= 0
        some = sorted({0, B // 2, B - 1})
        _check(l[some], u[some], (idx[some], logp[some]), **settings)
