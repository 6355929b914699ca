"""CPU tests of gradient norms and clipping: argument checks of the Python layer, the description of strided tensors, and the
refusals of ``pgm_grad_clip`` that come before any launch (addresses are made up: nothing is run)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from pgmuvi_amd import _hip, gradients as G


def test_cpu_tensors_and_wrong_arguments_are_refused():
    g = torch.ones(3, dtype=torch.float64)
    for call in (lambda: G.total_norm([g]), lambda: G.clip_grads_([g], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            G.clip_grads_([g], bad)
    for t in (torch.ones(3, dtype=torch.int64), torch.ones(3, dtype=torch.complex64), torch.ones(3).to_sparse()):
        with pytest.raises(TypeError):
            G.total_norm([t])
    with pytest.raises(TypeError, match="tensors expected"):
        G.total_norm([1.0])


def test_parameters_without_gradients_are_left_out():
    p = torch.nn.Parameter(torch.ones(3))
    assert float(G.clip_grad_norm_([p], 1.0)) == 0.0             # (nothing to do: no device is touched)
    assert float(G.clip_grad_norm_(p, 1.0)) == 0.0
    with pytest.raises(ValueError, match="no members"):
        G.total_norm([], members=True)


def _walk(layout_row, base, numel):
    """Entry offsets a described tensor stands for, sorted."""
    if layout_row is None or layout_row[0] == 0:
        return list(range(numel))
    s, st = layout_row[:4], layout_row[4:8]
    return sorted(int(i * st[0] + j * st[1] + k * st[2] + l * st[3]) for i in range(s[0]) for j in range(s[1]) for k in range(s[2]) for l in range(s[3]))


@pytest.mark.parametrize("make", [lambda: torch.zeros(4, 6)[:, 1:3], lambda: torch.zeros(6, 4).t(), lambda: torch.zeros(5, 4, 3).permute(2, 0, 1),
                                  lambda: torch.zeros(12)[::3], lambda: torch.zeros(3, 4, 5, 6)[::2, :, 1:4, ::3], lambda: torch.zeros(7, 1)[:, 0],
                                  lambda: torch.zeros(2, 1, 3).expand(2, 5, 3)])
def test_strided_tensors_are_described_entry_by_entry(make):
    t = make()
    _, dst, numel, _, member, layout = G._describe([t, torch.zeros(3)], None, None)
    assert dst is None and member is None and numel.tolist() == [t.numel(), 3]
    want = sorted(sum(i * s for i, s in zip(idx, t.stride())) for idx in np.ndindex(*t.shape))
    assert _walk(None if layout is None else layout[:12], 0, t.numel()) == want


def test_members_of_columns_are_runs_with_the_buffer_as_distance():
    buf = torch.zeros(6, 11)
    cols = [buf[:, :4], buf[:, 4:5], buf[:, 5:]]
    src, dst, numel, _, member, layout = G._describe(cols, cols, 6)
    assert numel.tolist() == [4, 1, 6] and member.tolist() == [11, 11] * 3 and layout is None
    t = torch.zeros(6, 5, 4).transpose(1, 2)                     # permuted inside the member: still one run, read in memory order
    _, _, numel, _, member, layout = G._describe([t], [t], 6)
    assert numel.tolist() == [20] and member.tolist() == [20, 20] and layout is None
    _, _, _, _, _, layout = G._describe([t], [torch.zeros(6, 4, 5)], 6)
    assert layout is not None and sorted(layout[:4].tolist()) == [1, 1, 4, 5]


def test_expanded_outputs_are_refused():
    g = torch.zeros(3).expand(4, 3)
    with pytest.raises(ValueError, match="share memory"):
        G._describe([g], [g], None)
    with pytest.raises(ValueError, match="four strided dimensions"):
        t = torch.zeros(3, 3, 3, 3, 3, 2)[::2, ::2, ::2, ::2, ::2, 0]
        G._describe([t], None, None)


def _clip(src, dst, numel, types, member=None, layout=None, batch=1, p=2, max_norm=1.0, norm=64, scratch=64, doubles=1 << 20):
    arr = lambda a, t: None if a is None else np.ascontiguousarray(np.asarray(a, dtype=t))
    a = [arr(src, np.uint64), arr(dst, np.uint64), arr(numel, np.int64), arr(types, np.uint8), arr(member, np.int64), arr(layout, np.int64)]
    at = [None if x is None else x.ctypes.data_as(ctypes.c_void_p) for x in a]
    return _hip.load().pgm_grad_clip(batch, len(src), at[0], at[1], at[2], at[3], at[4], at[5], p, max_norm, norm, 1, scratch, doubles, None)


A = 1 << 20


@pytest.mark.parametrize("code, kw", [
    (-1, dict(src=[A], dst=None, numel=[8], types=[0], batch=0)),
    (-1, dict(src=[A], dst=None, numel=[8], types=[0], batch=1 << 22, member=[[8, 8]])),
    (-3, dict(src=[0], dst=None, numel=[8], types=[0])),
    (-4, dict(src=[A], dst=[0], numel=[8], types=[0])),
    (-5, dict(src=[A], dst=None, numel=[-8], types=[0])),
    (-6, dict(src=[A], dst=None, numel=[8], types=[7])),
    (-7, dict(src=[A], dst=None, numel=[8], types=[0], batch=2)),
    (-7, dict(src=[A], dst=None, numel=[8], types=[0], batch=2, member=[[-1, 8]])),
    (-8, dict(src=[A], dst=None, numel=[8], types=[0], layout=[[1, 1, 2, 3, 0, 0, 3, 1, 0, 0, 3, 1]])),      # six entries, not eight
    (-8, dict(src=[A], dst=None, numel=[6], types=[0], layout=[[1, 1, 2, 3, 0, 0, -3, 1, 0, 0, 3, 1]])),
    (-9, dict(src=[A], dst=None, numel=[8], types=[0], p=3)),
    (-10, dict(src=[A], dst=[A], numel=[8], types=[0], max_norm=-1.0)),
    (-10, dict(src=[A], dst=[A], numel=[8], types=[0], max_norm=math.nan)),
    (-11, dict(src=[A], dst=None, numel=[8], types=[0], norm=None)),
    (-13, dict(src=[A], dst=None, numel=[1 << 24], types=[0], scratch=None)),
    (-14, dict(src=[A], dst=None, numel=[1 << 24], types=[0], doubles=3)),
    (-12, dict(src=[A, A], dst=[A, A], numel=[8, 8], types=[0, 0])),                                        # the same gradient twice
    (-12, dict(src=[A, A + 56], dst=[A, A + 56], numel=[8, 8], types=[0, 0])),                              # overlapping by one entry
    (-12, dict(src=[A, A + 4096], dst=[A + 4096, A], numel=[8, 8], types=[0, 0])),                          # one's output is the other's input
    (-12, dict(src=[A], dst=[A + 8], numel=[8], types=[0])),                                                # an output shifted by one entry
    (-12, dict(src=[A], dst=[A], numel=[8], types=[0], batch=3, member=[[4, 4]])),                          # members written over each other
    (-12, dict(src=[A, A + 32], dst=[A, A + 32], numel=[5, 4], types=[0, 0], batch=3, member=[[9, 9], [9, 9]])),   # columns 0-4 and 4-7 of nine
    (-12, dict(src=[A, A + 32], dst=[A, A + 32], numel=[4, 6], types=[0, 0], batch=3, member=[[9, 9], [9, 9]])),   # columns 4-9 reach into the next row
])
def test_refusals_come_before_any_launch(code, kw):
    assert _clip(**kw) == code


def test_scratch_covers_every_launch():
    need = _hip.load().pgm_grad_scratch_doubles
    assert need(0, 3, 8, 0) == 0 and need(1, -1, 8, 0) == 0 and need(1, 3, -8, 0) == 0
    assert need(1, 5, 112, 0) == 0 and need(4096, 5, 90_000, 0) == 0            # (one launch: no partial sums)
    for batch in (1, 7, 300, 4096):
        for count in (1, 64, 65, 5000):
            assert need(batch, count, 1 << 24, 0) >= 3 * (2048 + batch * (count // 64 + 1))
            assert need(batch, count, 64, 1) >= 3 * (2048 + batch * (count // 24 + 1))


# ---- what may share memory (layouts are never one launch, so that a call without scratch ends with -13 where it is not refused) -------
SHARED, DISTINCT = -12, -13


@pytest.mark.parametrize("kw", [
    dict(src=[A], dst=[A], numel=[4], types=[0], layout=[[1, 1, 1, 4, 0, 0, 0, 1, 0, 0, 0, 1]], batch=3, member=[[2, 2]]),     # members two apart, of four entries
    dict(src=[A], dst=[A], numel=[4], types=[0], layout=[[1, 1, 2, 2, 0, 0, 1, 8, 0, 0, 1, 8]], batch=9, member=[[1, 1]]),     # ... reaching each other's second column
    dict(src=[A], dst=[A], numel=[6], types=[0], layout=[[1, 1, 2, 3, 0, 0, 3, 1, 0, 0, 0, 1]]),                               # an expanded output
    dict(src=[A], dst=[A], numel=[6], types=[0], layout=[[1, 1, 2, 3, 0, 0, 2, 1, 0, 0, 2, 1]]),                               # rows that overlap by one
    dict(src=[A], dst=[A], numel=[4], types=[0], layout=[[1, 1, 1, 4, 0, 0, 0, 2, 0, 0, 0, 2]], batch=3, member=[[8, 0]]),     # one output for all members
])
def test_outputs_written_over_themselves_are_refused(kw):
    assert _clip(scratch=None, **kw) == SHARED


def _addresses(base, size, stride, batch, member):
    n = [batch] + list(size)
    st = [member] + list(stride)
    at = np.zeros(1, dtype=np.int64) + base
    for k, s in zip(n, st):
        at = (at[:, None] + np.arange(k) * s).ravel()
    return at


def _strided_call(boxes, batch):
    """In-place clip of (first entry, sizes, strides, member stride) of one fp64 buffer; an output given twice or overlapping -> SHARED."""
    layout = [list(size) + list(stride) + list(stride) for _, size, stride, _ in boxes]
    src = [A + 8 * b for b, _, _, _ in boxes]
    numel = [int(np.prod(size)) for _, size, _, _ in boxes]
    return _clip(src=src, dst=src, numel=numel, types=[0] * len(boxes), layout=layout, batch=batch, member=[[m, m] for _, _, _, m in boxes], scratch=None)


def test_no_two_entries_at_one_address_are_let_through():
    """Random layouts against the addresses themselves.  (The check may refuse entries that mesh without meeting, never the reverse.)"""
    rng = np.random.default_rng(0)
    let = met = 0
    for _ in range(20_000):
        batch = int(rng.choice([1, 1, 2, 3]))
        boxes = []
        for _ in range(int(rng.integers(1, 4))):
            size = [int(v) for v in rng.integers(1, 4, 4) * (rng.random(4) < 0.5) + 1]
            stride = [int(v) for v in rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 48, 49], 4, p=[0.02] + [0.098] * 10)]
            boxes.append((int(rng.integers(0, 200)), size, stride, int(rng.choice([1, 5, 24, 96, 200, 400]))))
        at = np.concatenate([_addresses(b, s, st, batch, m) for b, s, st, m in boxes])
        meets = len(np.unique(at)) < len(at)
        rc = _strided_call(boxes, batch)
        assert rc in (SHARED, DISTINCT)
        assert rc == SHARED or not meets, (batch, boxes)
        let += rc == DISTINCT
        met += meets
    assert let > 2000 and met > 2000                             # (the test reaches both)


def test_columns_rows_and_blocks_of_one_buffer_are_let_through():
    rng = np.random.default_rng(1)
    for _ in range(500):
        # a grid cut along every axis, all blocks of it (sizes of one and whole axes among them), the members' axis first or last
        dims = [int(v) for v in rng.integers(1, 7, 3)]
        batch = int(rng.choice([1, 1, 4]))
        inner = int(np.prod(dims))
        if batch > 1 and rng.random() < 0.5:
            stride, member = [dims[1] * dims[2] * batch, dims[2] * batch, batch], 1                # [..., member]
        else:
            stride, member = [dims[1] * dims[2], dims[2], 1], inner                                # [member, ...]
        cuts = [sorted({0, n, *(int(v) for v in rng.integers(0, n + 1, 2))}) for n in dims]
        boxes = []
        for a, b in zip(cuts[0], cuts[0][1:]):
            for c, d in zip(cuts[1], cuts[1][1:]):
                for e, f in zip(cuts[2], cuts[2][1:]):
                    boxes.append((a * stride[0] + c * stride[1] + e * stride[2], [1, b - a, d - c, f - e], [0] + stride, member))
        order = rng.permutation(len(boxes))
        assert _strided_call([boxes[k] for k in order], batch) == DISTINCT, (dims, cuts, batch)
        twice = boxes + [boxes[int(rng.integers(0, len(boxes)))]]
        assert _strided_call(twice, batch) == SHARED
    even, odd = (0, [1, 1, 5, 8], [0, 0, 16, 1], 0), (8, [1, 1, 5, 8], [0, 0, 16, 1], 0)
    assert _strided_call([even, odd], 1) == DISTINCT             # every other row each
    # columns of two types in one buffer of bytes (the size of an entry differs, the row does not)
    layout = [[1, 1, 6, 4, 0, 0, 6, 1, 0, 0, 6, 1], [1, 1, 6, 4, 0, 0, 12, 1, 0, 0, 12, 1]]
    assert _clip(src=[A, A + 32], dst=[A, A + 32], numel=[24, 24], types=[0, 1], layout=layout, scratch=None) == DISTINCT
    assert _clip(src=[A, A + 28], dst=[A, A + 28], numel=[24, 24], types=[0, 1], layout=layout, scratch=None) == SHARED
