"""Objectives without a GPU: their arguments, their layouts, and the formulas their tests compare with."""

import ctypes as C

import numpy as np
import pytest
import torch

import objective_util as ref
from packboost_b200 import backends as B
from packboost_b200 import objectives as O


def _differences(f, s, h=1e-6):
    out = np.zeros_like(s)
    for i in range(len(s)):
        if not np.isfinite(s[i]):
            continue
        up, down = s.copy(), s.copy()
        up[i] += h
        down[i] -= h
        out[i] = (f(up) - f(down)) / (2 * h)
    return out


# central differences: h^2 / 6 of the third derivative (below 10 here) and 2^-53 of the loss (below 1e3) over h
_DIFF = 1e-6


@pytest.mark.parametrize("kind,smoothing", [("logistic", 0.0), ("logistic", 0.1), ("squared", 0.0)])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_pair_formula_against_differences(kind, smoothing, reduction):
    rng = np.random.default_rng(3)
    s, r = rng.normal(size=12), rng.normal(size=12)
    c = rng.integers(0, 12, 40)
    j = (c + 1 + rng.integers(0, 11, 40)) % 12
    w = rng.random(40).astype(np.float32)
    args = dict(weight=w, reference=r, beta=0.7, smoothing=smoothing, kind=kind, reduction=reduction)
    grad = ref.pair_loss(s, c, j, **args)[1]
    np.testing.assert_allclose(grad, _differences(lambda v: ref.pair_loss(v, c, j, **args)[0], s), rtol=0, atol=_DIFF)


@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_group_formulas_against_differences(reduction):
    rng = np.random.default_rng(4)
    group = np.array([0, 0, 0, 2, 2, 3, 3, 3, 3, 5, 5, 2])
    s = rng.normal(size=12)
    s[[1, 9, 10]] = -np.inf
    t = np.where(np.isfinite(s), rng.random(12), 0)
    grad = ref.choice(s, group, 6, t, reduction)[1]
    np.testing.assert_allclose(grad, _differences(lambda v: ref.choice(v, group, 6, t, reduction)[0], s), rtol=0, atol=_DIFF)
    a = rng.normal(size=12)
    a[4] = 0.0
    old = ref.log_probs(np.where(np.isfinite(s), s + 0.2 * rng.normal(size=12), s), group, 6)
    prior = ref.log_probs(np.where(np.isfinite(s), rng.normal(size=12), s), group, 6)
    old[~np.isfinite(s)] = prior[~np.isfinite(s)] = np.nan
    old[4] = np.nan

    def loss(v):
        return ref.policy(v, group, 6, a, old, prior, (0.1, 0.2), 0.3, reduction)

    assert 0 < loss(s)[3] < 8          # some ratios are beyond their borders, some are not
    np.testing.assert_allclose(loss(s)[1], _differences(lambda v: loss(v)[0], s), rtol=0, atol=_DIFF)


@pytest.mark.parametrize("ids,in_order", [([], True), ([4], True), ([0, 0, 3, 3, 3, 7], True), ([3, 0, 3, 7, 0, 3], False)])
def test_layout_of_groups(ids, in_order):
    lay = O._lay_out_groups(torch.tensor(ids, dtype=torch.int64))
    rows = np.arange(len(ids)) if lay["rows"] is None else lay["rows"].numpy()
    assert (lay["rows"] is None) == in_order
    off = lay["offsets"].numpy()
    got = [sorted(rows[a:b]) for a, b in zip(off[:-1], off[1:])]
    assert got == [np.flatnonzero(np.array(ids) == g).tolist() for g in sorted(set(ids))]
    assert off[0] == 0 and off[-1] == len(ids)


@pytest.mark.parametrize("args,kw,error", [
    (([0.0], [1], 3), {}, TypeError), (([True], [1], 3), {}, TypeError), (([[0]], [[1]], 3), {}, ValueError),
    (([0, 1], [1], 3), {}, ValueError), (([0], [3], 3), {}, ValueError), (([-1], [0], 3), {}, ValueError),
    (([1], [1], 3), {}, ValueError), (([0], [1], -1), {}, ValueError), (([0], [1], 2.0), {}, TypeError),
    (([0], [1], 1 << 31), {}, ValueError), (([0], [1], True), {}, TypeError),
    (([0], [1], 2), {"weight": [-1.0]}, ValueError), (([0], [1], 2), {"weight": [float("nan")]}, ValueError),
    (([0], [1], 2), {"weight": [1.0, 2.0]}, ValueError), (([0], [1], 2), {"weight": [1e300]}, ValueError),
    (([0], [1], 2), {"reference": [1.0]}, ValueError), (([0], [1], 2), {"reference": [1j, 2]}, TypeError),
    (([0], [1], 2), {"device": "cpu"}, ValueError),
])
def test_refused_pairs(args, kw, error):
    with pytest.raises(error):
        O.RowPairs(*args, **kw)


@pytest.mark.parametrize("args,kw,error", [
    (([0.5],), {}, TypeError), (([[0]],), {}, ValueError), (([-1, 0],), {}, ValueError), (([0, 3], 3), {}, ValueError),
    (([0], 1.5), {}, TypeError), (([0], -2), {}, ValueError), (([0],), {"device": "cpu"}, ValueError),
])
def test_refused_groups(args, kw, error):
    with pytest.raises(error):
        O.RowGroups(*args, **kw)


class _Stub:
    """A layout as far as the checks look at it."""

    def __init__(self, n_rows, **kw):
        self.n_rows, self.device, self._struct = n_rows, torch.device("cpu"), kw.pop("struct", None)
        self.__dict__.update(kw)


def test_refused_scores_and_rows():
    lay = _Stub(4)
    for scores, error in ((torch.zeros(4, dtype=torch.float64), TypeError), (np.zeros(4, np.float32), TypeError),
                          (torch.zeros(5), ValueError), (torch.zeros(4, 1), ValueError),
                          (torch.zeros(4, device="meta"), ValueError)):
        with pytest.raises(error):
            O._check_scores(scores, lay)
    for rows, error in (([0.0] * 4, TypeError), (torch.zeros(3), ValueError), (torch.zeros(4, dtype=torch.complex64), TypeError),
                        (torch.zeros(4, dtype=torch.bool), TypeError), (torch.zeros(4, device="meta"), ValueError)):
        with pytest.raises(error):
            O._per_row(rows, "target", lay)
    strided = O._check_scores(torch.arange(8.0)[::2], lay)
    assert strided.is_contiguous() and strided.tolist() == [0.0, 2.0, 4.0, 6.0]


@pytest.mark.parametrize("kw", [
    dict(beta=0.0), dict(beta=-1.0), dict(beta=float("inf")), dict(beta=float("nan")), dict(smoothing=0.5),
    dict(smoothing=-0.1), dict(kind="hinge"), dict(kind="squared", smoothing=0.1), dict(reduction="none"),
])
def test_refused_preference_options(kw):
    pairs = _Stub(2, struct=B.Pairs(2, 0), total_weight=1.0)
    with pytest.raises(ValueError):
        O._preference_struct(pairs, kw.get("beta", 1.0), kw.get("smoothing", 0.0), kw.get("kind", "logistic"),
                             kw.get("reduction", "sum"))


def test_refused_means_over_nothing():
    with pytest.raises(ValueError, match="not defined"):
        O._preference_struct(_Stub(2, struct=B.Pairs(2, 0), total_weight=0.0), 1.0, 0.0, "logistic", "mean")
    with pytest.raises(ValueError, match="not defined"):
        O._choice_struct(_Stub(0, struct=B.Groups(0, 0), n_groups=0), torch.zeros(0), "mean")


@pytest.mark.parametrize("clip,kl,with_reference", [((-0.1, 0.2), 0.0, True), ((1.1, 0.2), 0.0, True), ((0.2, -0.1), 0.0, True),
                                                    ((float("nan"), 0.2), 0.0, True), ((0.2, 0.2), float("nan"), True),
                                                    ((0.2, 0.2), 0.1, False)])
def test_refused_policy_options(clip, kl, with_reference):
    groups = _Stub(2, struct=B.Groups(2, 1), n_groups=1)
    rows = torch.zeros(2)
    with pytest.raises(ValueError):
        O._policy_struct(groups, rows, rows, rows if with_reference else None, clip, kl, "sum")


def test_library_refuses_bad_descriptors():
    """No launch: the checks come before it."""
    lib = B.lib()

    def refused(o, match):
        with pytest.raises(ValueError, match=match):
            B.check(lib.pb_objective_evaluate(C.byref(o), 1, 0, 1, None, None, None, None, 0, None))
        assert lib.pb_objective_workspace_bytes(C.byref(o)) < 0

    ok = B.Pairs(4, 2, 1, 1, None, None)
    refused(B.Objective(kind=9), "unknown objective")
    refused(B.Objective(kind=0), "pairs are null")
    refused(B.Objective(kind=1), "groups are null")
    for p, match in ((B.Pairs(-1, 0), "n_rows"), (B.Pairs(1 << 31, 0), "n_rows"), (B.Pairs(4, 1 << 31), "n_items"),
                     (B.Pairs(4, 2, None, 1), "offsets"), (B.Pairs(4, 2, 1, None), "items"), (B.Pairs(1, 2, 1, 1), "items")):
        refused(B.Objective(kind=0, pairs=C.pointer(p), beta=1.0), match)
    for kw, match in ((dict(beta=0.0), "beta"), (dict(beta=1.0, smoothing=0.5), "smoothing"),
                      (dict(beta=1.0, scale=float("nan")), "scale")):
        refused(B.Objective(kind=0, pairs=C.pointer(ok), **kw), match)
    for g, match in ((B.Groups(-1, 0), "n_rows"), (B.Groups(3, 4, 1), "n_groups"), (B.Groups(3, 0, 1), "without a group"),
                     (B.Groups(3, 1, None), "offsets")):
        refused(B.Objective(kind=1, groups=C.pointer(g)), match)
    good = B.Groups(3, 1, 1)
    refused(B.Objective(kind=1, groups=C.pointer(good)), "target")
    rows = dict(groups=C.pointer(good), advantage=1, old=1)
    refused(B.Objective(kind=2, groups=C.pointer(good), advantage=1), "old")
    for kw, match in ((dict(clip_low=1.5), "clip_low"), (dict(clip_high=-1.0), "clip_high"), (dict(kl_coef=0.1), "reference")):
        refused(B.Objective(kind=2, **rows, **kw), match)
    # scores, types and scratch
    o = B.Objective(kind=0, pairs=C.pointer(ok), beta=1.0, scale=1.0)
    for scores, typ, grad, loss, match in ((None, 0, 1, None, "null"), (1, 0, None, None, "null"), (1, 7, 1, None, "type"),
                                           (1, 0, 1, 1, "workspace is null")):
        with pytest.raises(ValueError, match=match):
            B.check(lib.pb_objective_evaluate(C.byref(o), scores, typ, grad, loss, None, None, None, 0, None))
    with pytest.raises(RuntimeError, match="bytes given"):
        B.check(lib.pb_objective_evaluate(C.byref(o), 1, 0, 1, 1, None, None, 8, 8, None))
    with pytest.raises(ValueError, match="null"):
        B.check(lib.pb_group_log_probs(C.byref(good), None, 0, 1, None))
    with pytest.raises(ValueError, match="type"):
        B.check(lib.pb_group_log_probs(C.byref(good), 1, 5, 1, None))
    with pytest.raises(ValueError):
        B.check(lib.pb_round_begin_objective(C.byref(B.TrainState()), C.byref(o), 0, None, 0, None))
    with pytest.raises(ValueError):
        B.check(lib.pb_loop_submit_objective(None, C.byref(B.TrainState()), None, None, 0, 0, None, None, 1, None, 0, 0, None))


def test_structs_mirror_the_library():
    for i, t in enumerate((B.Pairs, B.Groups, B.Objective)):
        assert B.lib().pb_objective_struct_bytes(i) == C.sizeof(t)
