"""Norm and clipping of gradients on the MI355X (``pgm_grad_clip``): what stands between ``loss.backward()`` and
``optimizer.step()`` of the loops in :mod:`pgmuvi_amd.trainers` (``max_grad_norm=``) and behind a batch of evaluations
(:func:`pgmuvi_amd.batch.evaluate_batch`, one norm per light curve).

The reference's loop (``pgmuvi/trainers.py:177-182``) takes every step in full.  A fit that starts far from a peak, or whose
covariance is nearly singular, meets gradients many orders of magnitude above the usual ones; bounding the step by the
gradient's norm is the common remedy.  Names and formulas are those of ``torch.nn.utils``::

    n = (sum |g|^p)^(1/p) over every entry of every tensor,    g <- min(1, max_norm / (n + 1e-6)) g

There is no CPU path: tensors on the GPU or an error.  Nothing synchronises the host unless ``error_if_nonfinite`` asks for it.
"""
from __future__ import annotations

import math
from array import array

import torch

from . import _hip

_TYPE = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}
_BYTES = (8, 4, 2, 2)
_POWER = {1.0: 1, 2.0: 2, math.inf: 0}


def _coalesced(sizes, *strides):
    """Neighbouring dimensions that are one run in every stride list, merged: [(size, stride, ...)], outermost first."""
    dims = []
    for size, *st in zip(sizes, *strides):
        if size == 1:
            continue
        if dims and all(prev == s * size for prev, s in zip(dims[-1][1:], st)):
            dims[-1] = (dims[-1][0] * size, *st)
        else:
            dims.append((size, *st))
    return dims


def _overlaps_itself(sizes, strides):
    """Can two entries of a tensor share an address?  (Sufficient, not necessary, for "no": each stride clears all smaller dimensions.)"""
    reach = 0
    for st, size in sorted((st, size) for size, st in zip(sizes, strides) if size > 1):
        if st <= reach:
            return True
        reach += (size - 1) * st
    return False


def _dense_order(t):
    """Dimensions of ``t`` from the slowest to the fastest in memory (a permuted tensor read in its own order is one run)."""
    return sorted(range(t.dim()), key=lambda k: -t.stride(k))


def _describe(tensors, outs, batch):
    """Host arrays of ``pgm_grad_clip``: (in, out | None, numel, type, member strides | None, layouts | None).  (A training step calls
    this between two launches: one C call per tensor and property, no array library.)"""
    T = torch.Tensor
    numel = array("q", map(T.numel, tensors))
    kinds = {t.dtype for t in tensors}
    types = bytearray(_TYPE[k] for k in kinds) * len(tensors) if len(kinds) == 1 else bytearray(_TYPE[t.dtype] for t in tensors)
    src = array("Q", map(T.data_ptr, tensors))
    dst = src if outs is tensors else None if outs is None else array("Q", map(T.data_ptr, outs))
    member = layout = None
    if batch is not None:
        numel = array("q", [n // batch for n in numel])
        member = array("q", [n for n in numel for _ in (0, 1)])
    if all(map(T.is_contiguous, tensors)) and (dst is src or dst is None or all(map(T.is_contiguous, outs))):
        return src, dst, numel, types, member, layout
    first = 0 if batch is None else 1
    for i, t in enumerate(tensors):
        o = t if outs is None else outs[i]
        if t.numel() == 0 or (t.is_contiguous() and o.is_contiguous()):
            continue
        if outs is not None and _overlaps_itself(o.shape, o.stride()):
            raise ValueError(f"gradient {i}: a tensor whose entries share memory (an expanded view) cannot be written")
        order = [k for k in _dense_order(t) if first == 0 or k != 0]
        dims = _coalesced([t.shape[k] for k in order], [t.stride(k) for k in order], [o.stride(k) for k in order])
        if batch is not None:
            member[2 * i], member[2 * i + 1] = t.stride(0), o.stride(0)
        if len(dims) == 0 or (len(dims) == 1 and dims[0][1] == 1 and dims[0][2] == 1):
            continue                                             # (permuted, padded between members, ...: one run per member)
        if len(dims) > 4:
            raise ValueError(f"gradient {i}: more than four strided dimensions; make it contiguous")
        if layout is None:
            layout = array("q", bytes(96 * len(tensors)))
        dims = [(1, 0, 0)] * (4 - len(dims)) + dims
        layout[12 * i:12 * i + 12] = array("q", [d[k] for k in range(3) for d in dims])
    return src, dst, numel, types, member, layout


def _sparse(t):
    return t.layout is not torch.strided


_PLAIN = {torch.Tensor, torch.nn.Parameter}


def _tensors(tensors, what):
    """The tensors as a list, checked: dense, of the four types, on one GPU."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not _PLAIN.issuperset(map(type, tensors)):
        for t in tensors:
            if not torch.is_tensor(t):
                raise TypeError(f"{what}: tensors expected, got {type(t).__name__}")
    if any(map(_sparse, tensors)) or not _TYPE.keys() >= {t.dtype for t in tensors}:
        raise TypeError(f"{what}: dense float64, float32, bfloat16 or float16 tensors expected, got "
                        f"{sorted({str(t.dtype) + ' ' + str(t.layout) for t in tensors})}")
    if tensors:
        _hip.require_gpu(tensors[0], what)
        if len(set(map(torch.Tensor.get_device, tensors))) != 1:
            raise ValueError(f"{what}: all tensors must be on one device")
    return tensors


def _address(a):
    return None if a is None else a.buffer_info()[0]


def _run(tensors, outs, max_norm, norm_type, members, what):
    p = _POWER.get(float(norm_type))
    if p is None:
        raise ValueError(f"{what}: norm_type must be 1, 2 or inf, got {norm_type}")
    if not tensors:
        if members:
            raise ValueError(f"{what}: no tensors, so no members")
        return torch.zeros((), dtype=torch.float32, device=torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else None)
    batch = None
    if members:
        if any(t.dim() == 0 for t in tensors) or len({t.shape[0] for t in tensors}) != 1:
            raise ValueError(f"{what}: with members=True every tensor needs the same leading size, got {[tuple(t.shape) for t in tensors]}")
        batch = tensors[0].shape[0]
        if batch >= 1 << 22:
            raise ValueError(f"{what}: at most {(1 << 22) - 1} members, got {batch}")
    dev = tensors[0].device
    if batch == 0:
        return torch.empty(0, dtype=torch.float64 if any(t.dtype is torch.float64 for t in tensors) else torch.float32, device=dev)
    src, dst, numel, types, member, layout = _describe(tensors, outs, batch)
    f64 = 0 in types
    norm = torch.empty(() if batch is None else (batch,), dtype=torch.float64 if f64 else torch.float32, device=dev)
    lib = _hip.load()
    members, count = batch or 1, len(tensors)
    same = types.count(types[0]) == count
    bytes_ = sum(numel) * _BYTES[types[0]] if same else sum(n * _BYTES[k] for n, k in zip(numel, types))
    n = lib.pgm_grad_scratch_doubles(members, count, bytes_, layout is not None)
    scratch = torch.empty(n, dtype=torch.float64, device=dev) if n else None
    with _hip.on_device(dev.index):
        rc = lib.pgm_grad_clip(members, count, _address(src), _address(dst), _address(numel), bytes(types), _address(member), _address(layout), p,
                               max_norm, norm.data_ptr(), f64, None if scratch is None else scratch.data_ptr(), n, _hip.stream_of(dev.index))
    if rc == -12:
        raise ValueError(f"{what}: tensors that share memory, or mesh in ways other than columns, rows and blocks of one buffer, cannot be clipped "
                         "together (the same gradient given twice?)")
    _hip._check(rc, "pgm_grad_clip")
    return norm


def total_norm(tensors, norm_type: float = 2.0, members: bool = False) -> torch.Tensor:
    """Norm over every entry of every tensor (on the device; no synchronisation): a 0-dim tensor, float64 if any of the
    tensors is, else float32.  ``members``: the tensors share a leading axis of independent fits and each gets its own norm,
    (B,).  ``norm_type``: 1, 2 or ``inf``."""
    return _run(_tensors(tensors, "total_norm"), None, 0.0, norm_type, members, "total_norm")


def clip_grads_(grads, max_norm: float, norm_type: float = 2.0, out=None, members: bool = False,
                error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales gradients to a norm of at most ``max_norm``, in place or into ``out`` (tensors of the same shapes and types),
    and returns the norm they had (see :func:`total_norm`).  ``members``: one norm and one factor for every index of the
    leading axis.  The factor is ``min(1, max_norm / (norm + 1e-6))``; a NaN norm makes the gradients NaN, an infinite one
    zero (NaN where the gradient is infinite).  An infinite ``max_norm`` is no limit: the gradients stay as they are, whatever
    their norm.  ``error_if_nonfinite``: raise where the norm is not finite, with the gradients untouched (waits for the norm)."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads_: max_norm must not be negative, got {max_norm}")
    grads = _tensors(grads, "clip_grads_")
    outs = grads
    if out is not None:
        outs = _tensors(out, "clip_grads_")
        if len(outs) != len(grads) or any(o.shape != g.shape or o.dtype is not g.dtype for o, g in zip(outs, grads)):
            raise ValueError("clip_grads_: out must hold one tensor of the same shape and type for every gradient")
        if grads and outs[0].device != grads[0].device:
            raise ValueError("clip_grads_: all tensors must be on one device")
        if any(o.is_neg() for o in outs):
            raise ValueError("clip_grads_: out must not be a negated view")
        grads = [g.resolve_neg() for g in grads]                 # (in place the kernel scales the memory behind the view: the same)
    if error_if_nonfinite:
        norm = _run(grads, None, 0.0, norm_type, members, "clip_grads_")
        if not bool(torch.isfinite(norm).all()):
            raise RuntimeError("clip_grads_: the norm of the gradients is not finite, so they were not clipped")
    norm = _run(grads, outs, max_norm, norm_type, members, "clip_grads_")
    if outs:
        torch.autograd.graph.increment_version(outs)             # (autograd does not see the kernel's writes by itself)
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` on the HIP kernels: clips the gradients of ``parameters`` (those without one are left
    out) in place and returns their norm."""
    parameters = [parameters] if torch.is_tensor(parameters) else list(parameters)
    return clip_grads_([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, error_if_nonfinite=error_if_nonfinite)
