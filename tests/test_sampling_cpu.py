"""CPU tests of the draws: argument checks of the Python layer, the refusals of ``pgm_draw_indices`` (before any launch; addresses
are made up) and the oracle against hand-made distributions."""
import math

import numpy as np
import pytest
import torch

from pgmuvi_amd import _hip, sampling
import os, sys
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _draw_oracle as oracle


def test_cpu_tensors_and_wrong_types_are_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sampling.draw_indices(torch.zeros(3), torch.zeros(2))
    for l, u in ((torch.zeros(3, dtype=torch.int32), torch.zeros(2)), (torch.zeros(3), torch.zeros(2, dtype=torch.int64)), ([0.0], torch.zeros(1)),
                 (torch.zeros(3), [0.5])):
        with pytest.raises(TypeError):
            sampling.draw_indices(l, u)


@pytest.mark.parametrize("name, off, lo, hi, dtype, bad", [
    ("temperature", 1.0, 0.0, 1e300, torch.float64, [-1.0, math.nan, math.inf]), ("top_k", 0, 1, 1 << 62, torch.int64, [0, -3, 2.5]),
    ("top_p", 1.0, 0.0, 1.0, torch.float64, [-0.1, 1.1, math.nan]), ("min_p", 0.0, 0.0, 1.0, torch.float64, [-0.1, 1.1, math.nan])])
def test_settings(name, off, lo, hi, dtype, bad):
    assert sampling._setting(None, off, lo, hi, name, 4, "cpu", dtype) == (off, None, None)
    assert sampling._setting(1, off, lo, hi, name, 4, "cpu", dtype)[0] == 1
    for b in bad:
        with pytest.raises(ValueError, match=name):
            sampling._setting(b, off, lo, hi, name, 4, "cpu", dtype)
    with pytest.raises(ValueError, match="one per row"):
        sampling._setting(torch.ones(3), off, lo, hi, name, 4, "cpu", dtype)


def _call(**kw):
    a = dict(logits=64, type=0, rows=2, cols=5, row_stride=5, col_stride=1, lengths=None, u=64, draws=1, t=1.0, tp=None, k=0, kp=None, p=1.0, pp=None,
             m=0.0, mp=None, index=64, logp=None, scratch=64, doubles=1 << 40, stream=None)
    a.update(kw)
    return _hip.load().pgm_draw_indices(*a.values())


@pytest.mark.parametrize("code, kw", [
    (-1, dict(logits=None)), (-2, dict(type=4)), (-2, dict(type=-1)), (-3, dict(rows=0)), (-3, dict(rows=1 << 31)), (-3, dict(rows=1 << 23)), (-4, dict(cols=0)), (-4, dict(cols=1 << 24)),
    (-5, dict(row_stride=-1)), (-6, dict(col_stride=-1)), (-8, dict(u=None)), (-9, dict(draws=0)), (-10, dict(t=-1.0)), (-10, dict(t=math.nan)), (-10, dict(t=math.inf)),
    (-12, dict(k=-1)), (-14, dict(p=1.5)), (-14, dict(p=math.nan)), (-16, dict(m=-0.5)), (-16, dict(m=2.0)), (-18, dict(index=None)),
    (-20, dict(cols=200_000, scratch=None)), (-21, dict(cols=200_000, doubles=3)), (-21, dict(draws=1000, doubles=3))])
def test_refusals_come_before_any_launch(code, kw):
    assert _call(**kw) == code


def test_oracle_on_small_distributions():
    l = np.log(np.array([0.1, 0.4, 0.1, 0.3, 0.1]))
    assert oracle.kept_entries(l)[0].tolist() == [0, 1, 2, 3, 4]
    assert oracle.kept_entries(l, top_k=3)[0].tolist() == [0, 1, 3]                       # (the first of the equal ones)
    assert oracle.kept_entries(l, top_p=0.75)[0].tolist() == [0, 1, 3]
    assert oracle.kept_entries(l, top_p=0.69)[0].tolist() == [1, 3]
    assert oracle.kept_entries(l, top_k=2, top_p=0.5)[0].tolist() == [1]                 # (4/7 of what top_k left)
    assert oracle.kept_entries(l, min_p=0.5)[0].tolist() == [1, 3]
    assert oracle.draw_row(l, [0.0, 0.15, 0.55, 0.95])[0].tolist() == [0, 1, 2, 4]
    assert oracle.draw_row([-math.inf, math.nan], [0.5])[0].tolist() == [-1]
    idx, lp = oracle.draw_row(l, [0.3], top_k=2)
    assert idx[0] == 1 and abs(lp[0] - math.log(4 / 7)) < 1e-15


def test_light_curves_too_short_for_odds_are_refused():
    from pgmuvi_amd.lombscargle import draw_frequencies
    with pytest.raises(ValueError, match="at least four points"):
        draw_frequencies(torch.zeros(1, 3), torch.zeros(1, 3), None, torch.zeros(1, 1))


def test_a_start_that_does_not_exist_is_refused():
    from pgmuvi_amd import mcmc
    with pytest.raises(ValueError, match="initial_values"):
        mcmc.run_mcmc(torch.zeros(5), torch.zeros(5), initial_values="peaks")


def test_distinct_frequencies_need_numbers_per_light_curve():
    from pgmuvi_amd.lombscargle import draw_frequencies
    with pytest.raises(ValueError, match=r"\(B, S\)"):
        draw_frequencies(torch.zeros(2, 9), torch.zeros(2, 9), None, torch.zeros(2), distinct=True)
