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


def _pairs(rng, rows, pairs, hubs, touched):
    c = rng.integers(0, hubs or touched, pairs)
    j = rng.integers(0, max(touched - 1, 1), pairs)
    return c, j + (j >= c)


@pytest.mark.parametrize("rows,pairs,hubs,touched", [(1, 0, 0, 1), (9, 23, 0, 7), (5000, 2000, 0, 5000), (400, 9000, 1, 300),
                                                     (30_000, 40_000, 2, 30_000), (2, 20_000, 0, 2), (8192, 0, 0, 8192),
                                                     (60, 1100, 0, 60), (20_000, 100_000, 0, 20_000)])
def test_layout_of_pairs(rows, pairs, hubs, touched):
    rng = np.random.default_rng(rows + pairs)
    c, j = _pairs(rng, rows, pairs, hubs, touched)
    w, r = rng.random(pairs).astype(np.float32), rng.normal(size=rows)
    lay = O._lay_out_pairs(torch.from_numpy(c), torch.from_numpy(j), rows, torch.from_numpy(w), torch.from_numpy(r))
    n_c, n_j = np.bincount(c, minlength=rows), np.bincount(j, minlength=rows)
    other, offset, weight = (lay[k].numpy() for k in ("other", "offset", "weight"))
    assert ((0 <= other) & (other < rows)).all()
    used, done, got = np.zeros(len(other), int), np.zeros(rows, int), []

    def take(row, items, chosen):
        used[items] += 1
        np.testing.assert_array_equal(offset[items], (r[row] - r[other[items]]).astype(np.float32))
        for o, x in zip(other[items].tolist(), weight[items].tolist()):
            got.append((row, o, x) if chosen else (o, row, x))

    slices, lanes = lay["slices"].numpy(), lay["slice_rows"].numpy().reshape(-1, 64, 2)
    for (column, tall), slice_rows in zip(slices, lanes):
        chosen, rejected = tall & 0xFFFF, tall >> 16
        assert 64 * (column + chosen + rejected) <= len(other) or chosen + rejected == 0
        for lane, (row, have) in enumerate(slice_rows):
            if row < 0:
                assert have == 0
                continue
            done[row] += 1
            assert have & 0xFFFF == n_c[row] <= chosen <= 32 and have >> 16 == n_j[row] <= rejected <= 32
            take(int(row), 64 * (column + np.arange(n_c[row])) + lane, True)
            take(int(row), 64 * (column + chosen + np.arange(n_j[row])) + lane, False)
    assert len(slices) == lay["n_slices"] == len(lanes)
    left = {}
    chunks = lay["chunks"].numpy() if "chunks" in lay else np.zeros((0, 8), np.int32)
    for k, (row, begin, count, better, number, first, n_of, zero) in enumerate(chunks):
        assert 0 < count <= O._CHUNK_ITEMS and 0 <= better <= count and first <= k < first + n_of and zero == 0
        assert chunks[first: first + n_of, 0].tolist() == [row] * n_of and chunks[first: first + n_of, 2].sum() == n_c[row] + n_j[row]
        if n_of > 1:
            assert left.setdefault(int(row), int(number)) == number and 0 <= number < lay["n_split"]
        assert begin + count <= len(other)
        done[row] += k == first
        take(int(row), begin + np.arange(better), True)
        take(int(row), begin + np.arange(better, count), False)
    assert len(set(left.values())) == len(left) == lay.get("n_split", 0) and len(chunks) == lay.get("n_chunks", 0)
    assert (done == 1).all() and used.max(initial=0) <= 1
    assert sorted(got) == sorted([(int(a), int(b), float(x)) for a, b, x in zip(c, j, w)] * 2)


@pytest.mark.parametrize("lengths", [[], [1], [1] * 5000, [128] * 40, [256, 257, 129, 1, 128, 2048, 2049, 3, 4096, 4097, 8192, 8193, 5, 2048 * 9, 1, 16384, 16385],
                                     [7, 13, 127, 2] * 400, [20_000], [895, 1, 1, 128, 900, 128]])
@pytest.mark.parametrize("mixed", [False, True])
def test_layout_of_groups(lengths, mixed):
    rng = np.random.default_rng(len(lengths))
    ids = np.repeat(np.arange(len(lengths)) * 3, lengths)       # (ids without rows between)
    if mixed:
        ids = rng.permutation(ids)
    lay = O._lay_out_groups(torch.from_numpy(ids.astype(np.int64)))
    n = len(ids)
    assert lay["n_groups"] == len(lengths)
    if n == 0:
        return
    rows = np.arange(n) if lay["rows"] is None else lay["rows"].numpy()
    assert (lay["rows"] is None) == bool((np.diff(ids) >= 0).all())
    starts = np.cumsum([0] + lengths)[:-1]
    length_of = dict(zip(starts.tolist(), lengths))
    for a, size in length_of.items():
        assert len(set(ids[rows[a: a + size]])) == 1
    done = np.zeros(n, int)                                     # every place is somebody's, once

    def take(table, low, high):
        for begin, size in table:
            assert length_of[begin] == size and low < size <= high
            done[begin: begin + size] += 1

    teams, seen = lay["teams"].numpy(), np.zeros(len(lay["teams"]), int)
    for first, word in lay["team_warps"].numpy():
        c, most = word & 0xFF, word >> 8
        own = teams[first: first + (32 >> c)]
        seen[first: first + (32 >> c)] += 1
        real = own[own[:, 1] > 0]
        take(real.tolist(), O._TEAM_ROWS[c - 1] if c else 0, O._TEAM_ROWS[c])
        assert most == -(-real[:, 1].max() // (1 << c)) and 1 <= most <= 8 and (own[own[:, 1] == 0] == 0).all()
    assert (seen == 1).all() and len(lay["team_warps"]) == lay["n_team_warps"]
    blocks = lay["blocks"].numpy().tolist()
    take(blocks, O._TEAM_ROWS[-1], O._BLOCK_ROWS)
    assert len(blocks) == lay["n_blocks"] and lay["block_rows"] == max([s for _, s in blocks], default=0)
    for i, (begin, size, first, count) in enumerate(lay["pieces"].numpy()):
        start = begin - (i - first) * O._PIECE
        assert 0 < size <= O._PIECE and first <= i < first + count and length_of[start] > O._BLOCK_ROWS
        assert (i == first + count - 1) == (begin + size == start + length_of[start])
        done[begin: begin + size] += 1
    assert (done == 1).all() and lay["n_pieces"] == len(lay["pieces"])


@pytest.mark.parametrize("args,kw,error", [
    (([0.0], [1], 3), {}, TypeError), (([True], [1], 3), {}, TypeError), (([[0]], [[1]], 3), {}, ValueError),
    (([0, 1], [1], 3), {}, ValueError), (([0], [3], 3), {}, ValueError), (([-1], [0], 3), {}, ValueError),
    (([1], [1], 3), {}, ValueError), (([0], [1], -1), {}, ValueError), (([0], [1], 2.0), {}, TypeError),
    (([0], [1], 1 << 31), {}, ValueError), (([0], [1], O._MOST + 1), {}, ValueError), (([0], [1], True), {}, TypeError),
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
        self.n_rows, self.device, self._struct, self._structs = n_rows, torch.device("cpu"), kw.pop("struct", None), {}
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
    dict(beta=0.0), dict(beta=-1.0), dict(beta=float("inf")), dict(beta=float("nan")), dict(beta=1e39), dict(beta=1e-40), dict(smoothing=0.5),
    dict(smoothing=-0.1), dict(kind="hinge"), dict(kind="squared", smoothing=0.1), dict(reduction="none"),
])
def test_refused_preference_options(kw):
    pairs = _Stub(2, struct=B.Pairs(n_rows=2), total_weight=1.0)
    with pytest.raises(ValueError):
        O._preference_struct(pairs, kw.get("beta", 1.0), kw.get("smoothing", 0.0), kw.get("kind", "logistic"),
                             kw.get("reduction", "sum"))


def test_refused_means_over_nothing():
    with pytest.raises(ValueError, match="not defined"):
        O._preference_struct(_Stub(2, struct=B.Pairs(n_rows=2), total_weight=0.0), 1.0, 0.0, "logistic", "mean")
    with pytest.raises(ValueError, match="not defined"):
        O._choice_struct(_Stub(0, struct=B.Groups(0, 0), n_groups=0), torch.zeros(0), "mean")


@pytest.mark.parametrize("clip,kl,with_reference", [((-0.1, 0.2), 0.0, True), ((1.1, 0.2), 0.0, True), ((0.2, -0.1), 0.0, True),
                                                    ((float("nan"), 0.2), 0.0, True), ((0.2, 0.2), float("nan"), True), ((0.2, 0.2), 1e39, True),
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

    def pairs(**kw):
        return B.Pairs(**dict(dict(n_rows=4, n_slices=1, slices=16, slice_rows=16, other=16), **kw))

    def groups(**kw):
        return B.Groups(**dict(dict(n_rows=3, n_groups=1, n_team_warps=1, team_warps=16, teams=16), **kw))

    ok, good = pairs(), groups()
    refused(B.Objective(kind=9), "unknown objective")
    refused(B.Objective(kind=0), "pairs are null")
    refused(B.Objective(kind=1), "groups are null")
    for kw, match in ((dict(n_rows=-1), "n_rows"), (dict(n_rows=O._MOST + 1), "n_rows"), (dict(n_slices=1 << 26), "range"),
                      (dict(n_slices=0), "not laid out"), (dict(slices=None), "null"), (dict(slice_rows=None), "null"),
                      (dict(other=None), "null"), (dict(n_chunks=1), "null"), (dict(n_chunks=-1), "range"),
                      (dict(n_split=1), "range"), (dict(slices=20), "aligned"), (dict(offset=20), "aligned"), (dict(n_chunks=1, chunks=24), "aligned")):
        refused(B.Objective(kind=0, pairs=C.pointer(pairs(**kw)), beta=1.0), match)
    for kw, match in ((dict(beta=0.0), "beta"), (dict(beta=1e31), "beta"), (dict(beta=1.0, smoothing=0.5), "smoothing"),
                      (dict(beta=1.0, scale=float("nan")), "scale"), (dict(beta=1.0, scale=1e40), "scale")):
        refused(B.Objective(kind=0, pairs=C.pointer(ok), **kw), match)
    for kw, match in ((dict(n_rows=-1), "n_rows"), (dict(n_groups=4), "n_groups"), (dict(n_groups=0), "without a group"),
                      (dict(n_team_warps=0), "not laid out"), (dict(teams=None), "null"), (dict(team_warps=None), "null"),
                      (dict(teams=20), "aligned"), (dict(n_blocks=1, block_rows=300), "null"), (dict(n_blocks=-1), "range"),
                      (dict(n_blocks=2), "range"), (dict(n_blocks=1, block_rows=8193, blocks=16), "range"),
                      (dict(n_blocks=1, blocks=16), "range"), (dict(n_pieces=1), "null"), (dict(n_pieces=-1), "range")):
        refused(B.Objective(kind=1, groups=C.pointer(groups(**kw))), match)
    refused(B.Objective(kind=1, groups=C.pointer(good)), "target")
    rows = dict(groups=C.pointer(good), advantage=16, old=16)
    refused(B.Objective(kind=2, groups=C.pointer(good), advantage=16), "old")
    for kw, match in ((dict(clip_low=1.5), "clip_low"), (dict(clip_high=-1.0), "clip_high"), (dict(kl_coef=0.1), "reference"),
                      (dict(kl_coef=1e40, reference=16), "kl_coef")):
        refused(B.Objective(kind=2, **rows, **kw), match)
    # scores, types and scratch
    o = B.Objective(kind=0, pairs=C.pointer(ok), beta=1.0, scale=1.0)
    for scores, typ, grad, scratch, match in ((None, 0, 16, 16, "null"), (16, 0, None, 16, "null"), (16, 7, 16, 16, "type"),
                                              (16, 0, 16, None, "workspace is null")):
        with pytest.raises(ValueError, match=match):
            B.check(lib.pb_objective_evaluate(C.byref(o), scores, typ, grad, 16, None, None, scratch, 1 << 20, None))
    with pytest.raises(RuntimeError, match="bytes given"):
        B.check(lib.pb_objective_evaluate(C.byref(o), 16, 0, 16, 16, None, None, 16, 8, None))
    with pytest.raises(ValueError, match="null"):
        B.check(lib.pb_group_log_probs(C.byref(good), None, 0, 16, None, 0, None))
    with pytest.raises(ValueError, match="type"):
        B.check(lib.pb_group_log_probs(C.byref(good), 16, 5, 16, None, 0, None))
    long = groups(n_team_warps=0, n_pieces=1, pieces=16)
    with pytest.raises(ValueError, match="workspace"):
        B.check(lib.pb_group_log_probs(C.byref(long), 16, 0, 16, None, 0, None))
    with pytest.raises(RuntimeError, match="bytes given"):
        B.check(lib.pb_group_log_probs(C.byref(long), 16, 0, 16, 16, 8, None))
    with pytest.raises(ValueError):
        B.check(lib.pb_round_begin_objective(C.byref(B.TrainState()), C.byref(o), 0, None, 0, None))
    with pytest.raises(ValueError):
        B.check(lib.pb_loop_submit_objective(None, C.byref(B.TrainState()), None, None, 0, 0, None, None, 1, None, 0, 0, None))


def test_structs_mirror_the_library():
    for i, t in enumerate((B.Pairs, B.Groups, B.Objective)):
        assert B.lib().pb_objective_struct_bytes(i) == C.sizeof(t)


def test_drawn_performance_cases_pass_the_checks(monkeypatch):
    """Every call that a drawn case makes gets past the checks of its options."""
    import random
    from perf import operators as cases
    taken = []

    def preference(scores, pairs, *, beta, label_smoothing, kind, reduction):
        taken.append((kind, O._preference_struct(pairs, beta, label_smoothing, kind, reduction).smoothing))
        return None, None

    def choice(scores, groups, target, *, reduction):
        O._choice_struct(groups, target, reduction)
        return None, None

    def policy(scores, groups, advantage, old, *, reference_log_probs, clip, kl_coef, reduction):
        O._policy_struct(groups, advantage, old, reference_log_probs, clip, kl_coef, reduction)
        return None, None

    for name, stand_in in (("preference_loss", preference), ("choice_loss", choice), ("policy_loss", policy),
                           ("group_log_probs", lambda scores, groups: None)):
        monkeypatch.setattr(O, name, stand_in)
    rng, rows = random.Random(5), torch.zeros(1)
    for case in cases.listed() + [cases.draw(rng) for _ in range(2000)]:
        if case["op"] == "preference":
            struct = B.Pairs(n_rows=case["rows"], n_slices=1, slices=16, slice_rows=16, other=16)
            plan = _Stub(case["rows"], struct=struct, total_weight=1.0)
        else:
            struct = B.Groups(n_rows=case["rows"], n_groups=1, n_team_warps=1, team_warps=16, teams=16)
            plan = _Stub(case["rows"], struct=struct, n_groups=case["groups"])
        state = dict(case=case, scores=rows, plan=plan, target=rows, advantage=rows, old=rows,
                     reference=rows if case["reference"] else None)
        cases._run_own(state)
    assert {kind for kind, _ in taken} == {"logistic", "squared"} and not any(e for kind, e in taken if kind == "squared")
    assert any(e for _, e in taken)


@pytest.mark.parametrize("n_rows", [3, 1 << 16, (1 << 30) + 1, O._MOST])
def test_items_are_ordered_for_any_number_of_rows(n_rows):
    """Owners go up to twice the number of rows, the rejected rows at the end of the largest tables among them."""
    rng = np.random.default_rng(n_rows)
    near = np.array([0, 1, 2, n_rows - 2, n_rows - 1], np.int64).clip(0)
    other = rng.choice(near, 400)
    owner = rng.choice(near, 400) + n_rows * rng.integers(0, 2, 400)
    order = O._item_order(torch.from_numpy(owner), torch.from_numpy(other), n_rows).numpy()
    np.testing.assert_array_equal(order, np.lexsort((other, owner)))   # (stable, like the sort)


def test_refused_squared_forms_of_tiny_beta():
    """1 / (2 beta) squared is a float32 number."""
    pairs = B.Pairs(n_rows=2, n_slices=1, slices=16, slice_rows=16, other=16)
    for beta in (9e-16, 1e-20, 1e-30):
        with pytest.raises(ValueError, match="squared"):
            O._preference_struct(_Stub(2, struct=pairs, total_weight=1.0), beta, 0.0, "squared", "sum")
        o = B.Objective(kind=0, pairs=C.pointer(pairs), beta=beta, squared=1, scale=1.0)
        with pytest.raises(ValueError, match="squared"):
            B.check(B.lib().pb_objective_evaluate(C.byref(o), 16, 0, 16, 16, None, None, 16, 1 << 20, None))
        assert B.lib().pb_objective_workspace_bytes(C.byref(o)) < 0
        o.squared = 0
        assert B.lib().pb_objective_workspace_bytes(C.byref(o)) > 0
        O._preference_struct(_Stub(2, struct=pairs, total_weight=1.0), beta, 0.0, "logistic", "sum")
    O._preference_struct(_Stub(2, struct=pairs, total_weight=1.0), 1e-15, 0.0, "squared", "sum")


def test_public_functions_where_torch_has_no_quicker_ones():
    def public():
        return 7
    assert O._quick("_a_name_that_is_not_there", public) is public
    for name in ("_device_now", "_stream_now", "_capturing"):
        assert callable(getattr(O, name))


def test_library_refuses_results_in_the_place_of_scores():
    """A row's score is read for other rows after its own result is written."""
    lib = B.lib()
    pairs = B.Pairs(n_rows=4, n_slices=1, slices=16, slice_rows=16, other=16)
    groups = B.Groups(n_rows=4, n_groups=1, n_team_warps=1, team_warps=16, teams=16)
    for o in (B.Objective(kind=0, pairs=C.pointer(pairs), beta=1.0, scale=1.0),
              B.Objective(kind=1, groups=C.pointer(groups), target=16, scale=1.0)):
        for typ, grad in ((0, 1024), (0, 1024 + 12), (0, 1024 - 12), (1, 1024 + 6), (2, 1024 - 6)):
            with pytest.raises(ValueError, match="overlaps"):
                B.check(lib.pb_objective_evaluate(C.byref(o), 1024, typ, grad, None, None, None, 4096, 1 << 20, None))
    for typ, out in ((0, 1024), (0, 1036), (2, 1018)):
        with pytest.raises(ValueError, match="overlaps"):
            B.check(lib.pb_group_log_probs(C.byref(groups), 1024, typ, out, None, 0, None))
