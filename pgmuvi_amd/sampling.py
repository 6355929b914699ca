"""Draws from log-weights on the MI355X (``pgm_draw_indices``): temperature, top-k, top-p and min-p truncation, from random
numbers the caller gives.

The reference seeds a fit from the highest peaks of a periodogram (``pgmuvi/lightcurve.py:5516-5541``), so every start is the
same one.  A periodogram is also a posterior over the frequency (:func:`pgmuvi_amd.lombscargle.draw_frequencies`), and starts
drawn from it differ in proportion to what the data say: top-p keeps the highest-density set, min-p a likelihood ratio,
top-k the best grid points, and a temperature above one flattens it.  The sampler's chains start on such draws
(:func:`pgmuvi_amd.mcmc.run_mcmc`, ``initial_values="periodogram"``).

There is no CPU path: tensors on the GPU or an error.  Nothing synchronises the host but a setting given as a 0-dim tensor on the
device (it is read as a number) and ``lengths`` given on the host (they are copied): a call that is captured gives numbers or (B,)
tensors on the device.  Neither the indices nor the log-probabilities carry a gradient.
"""
from __future__ import annotations

import torch

from . import _hip

_TYPE = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}


def _setting(value, off, lo, hi, name, rows, dev, dtype):
    """(scalar, device pointer or None, tensor kept alive) of a truncation argument: a number for all rows, or one per row."""
    if value is None:
        return off, None, None
    if torch.is_tensor(value) and value.dim() > 0:
        if tuple(value.shape) != (rows,):
            raise ValueError(f"draw_indices: {name} must be a number or one per row ({rows}), got {tuple(value.shape)}")
        _hip.require_gpu(value, "draw_indices")
        if dtype is torch.int64 and value.dtype.is_floating_point:
            raise TypeError(f"draw_indices: {name} takes whole numbers")
        t = value.detach().to(device=dev, dtype=dtype).resolve_neg().contiguous()
        return off, t.data_ptr(), t
    number = int(value) if dtype is torch.int64 else float(value)
    if not lo <= number <= hi or (dtype is torch.int64 and number != value):
        raise ValueError(f"draw_indices: {name} must be in [{lo}, {hi}], got {value}")
    return number, None, None


def draw_indices(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=None, top_p=None, min_p=None, lengths=None,
                 return_logprob: bool = False):
    """Indices drawn from rows of unnormalised log-probabilities.

    ``logits`` (B, V) or (V,), float64 / float32 / bfloat16 / float16, any strides; ``u`` uniform numbers in [0, 1), (B, S) or
    (B,) -- (S,) or () for one row -- each of which draws one index.  With ``w = exp((l - max l) / temperature)`` and the order
    (value descending, index ascending): ``top_k`` keeps the first k entries, ``top_p`` the shortest beginning of those that
    holds at least that share of their weight, ``min_p`` the entries of that with a weight of at least ``min_p`` times the
    best one's.  The index is the first kept one, in index order, whose running weight exceeds ``u`` times the kept weight.
    ``temperature`` 0 takes the best entry.  Each of the four is a number (``None``: off) or a (B,) tensor.  ``lengths`` (B,)
    whole numbers, on the device or the host: entries of each row; the rest is not read.  Entries of -inf or NaN are never drawn.

    Returns int64 indices of the shape of ``u`` (-1 where a row has nothing to draw), with ``return_logprob`` also the
    float64 log-probabilities of the draws under the truncated distribution (-inf there), outside any autograd graph: a loss on
    them differentiates its own expression of the logits at the indices."""
    if not torch.is_tensor(logits) or logits.dtype not in _TYPE or logits.layout is not torch.strided:
        raise TypeError("draw_indices: logits must be a dense float64, float32, bfloat16 or float16 tensor")
    if not torch.is_tensor(u) or u.dtype not in _TYPE:
        raise TypeError("draw_indices: u must be a floating-point tensor of random numbers")
    _hip.require_gpu(logits, "draw_indices")
    dev, logits, u = logits.device, logits.resolve_neg(), u.resolve_neg()
    if u.device != dev:
        raise ValueError(f"draw_indices: u is on {u.device}, the logits on {dev}")
    single = logits.dim() == 1
    if logits.dim() not in (1, 2):
        raise ValueError(f"draw_indices: logits must be (B, V) or (V,), got {tuple(logits.shape)}")
    B, V = (1, logits.shape[0]) if single else logits.shape
    row_stride, col_stride = (0, logits.stride(0)) if single else logits.stride()
    if u.dim() > 2 - single or (not single and (u.dim() == 0 or u.shape[0] != B)):
        raise ValueError(f"draw_indices: u must be {'(S,) or ()' if single else f'({B}, S) or ({B},)'}, got {tuple(u.shape)}")
    ud = u if u.dtype is torch.float64 and u.is_contiguous() else u.detach().to(torch.float64).contiguous()
    S = ud.numel() // B if B else 0
    settings = [_setting(temperature, 1.0, 0.0, 1e300, "temperature", B, dev, torch.float64),
                _setting(top_k, 0, 1, (1 << 62), "top_k", B, dev, torch.int64),
                _setting(top_p, 1.0, 0.0, 1.0, "top_p", B, dev, torch.float64),
                _setting(min_p, 0.0, 0.0, 1.0, "min_p", B, dev, torch.float64)]
    ln = None
    if lengths is not None:
        if not torch.is_tensor(lengths):
            lengths = torch.as_tensor(lengths)
        if tuple(lengths.shape) != (B,) or lengths.dtype.is_floating_point:
            raise ValueError(f"draw_indices: lengths must be {B} whole numbers")
        ln = lengths.to(device=dev, dtype=torch.int64).contiguous()
    index = torch.empty(u.shape, dtype=torch.int64, device=dev)
    logp = torch.empty(u.shape, dtype=torch.float64, device=dev) if return_logprob else None
    if V == 0:                                                   # rows without entries
        index.fill_(-1)
        if return_logprob:
            logp.fill_(float("-inf"))
    elif B and S:
        if B >= 1 << 23:
            raise ValueError(f"draw_indices: at most {(1 << 23) - 1} rows, got {B}")
        if V >= 1 << 24:
            raise ValueError(f"draw_indices: rows of at most {(1 << 24) - 1} entries, got {V}")
        (t, tp, _t), (k, kp, _k), (p, pp, _p), (m, mp, _m) = settings
        lib, kind = _hip.load(), _TYPE[logits.dtype]
        n = int(lib.pgm_draw_scratch_doubles(kind, B, V, S))
        scratch = torch.empty(n, dtype=torch.float64, device=dev) if n else None
        with _hip.on_device(dev.index):
            rc = lib.pgm_draw_indices(logits.data_ptr(), kind, B, V, row_stride, col_stride, None if ln is None else ln.data_ptr(),
                                      ud.data_ptr(), S, t, tp, k, kp, p, pp, m, mp, index.data_ptr(), None if logp is None else logp.data_ptr(),
                                      None if scratch is None else scratch.data_ptr(), n, _hip.stream_of(dev.index))
        _hip._check(rc, "pgm_draw_indices")
    return (index, logp) if return_logprob else index
