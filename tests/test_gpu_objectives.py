"""Objectives on the GPU against their definitions in float64 (objective_util.py derives the bounds)."""

import numpy as np
import pytest
import torch

import objective_util as ref
from objective_util import assert_close
from packboost_b200 import PackBoost, PackBoostConfig, PackBoostRegressor
from packboost_b200 import objectives as O

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _scores(rng, n, dtype, spread=1.0):
    """Scores of the type, and the same numbers in float64."""
    s = torch.from_numpy((rng.normal(size=n) * spread).astype(np.float32)).to(dtype)
    return s.cuda(), s.double().numpy()


# ---- preferences ---------------------------------------------------------------------------------

# rows, pairs, rows that pairs choose from (hubs), rows that pairs touch
SHAPES = [(2, 1, 0, 2), (5, 0, 0, 5), (7, 40, 0, 4), (257, 500, 0, 257), (1000, 4095, 1, 1000), (4099, 4096, 3, 4099),
          (3000, 100_003, 2, 900), (70_001, 150_000, 0, 70_001), (100_000, 333, 0, 100_000), (20_000, 300_000, 1, 20_000)]


def _pairs(rng, rows, pairs, hubs, touched):
    c = rng.integers(0, hubs or touched, pairs)
    j = rng.integers(0, max(touched - 1, 1), pairs)
    return c, j + (j >= c)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_preference(shape, dtype):
    rows, pairs = shape[:2]
    rng = np.random.default_rng(rows + pairs)
    c, j = _pairs(rng, *shape)
    x, s = _scores(rng, rows, dtype)
    w, r = rng.random(pairs).astype(np.float32), rng.normal(size=rows)
    for opts in (dict(beta=0.5, smoothing=0.1), dict(beta=2.0, kind="squared"), dict(weight=w, reference=r),
                 dict(weight=w, kind="squared"), dict(reference=r, reduction="mean")):
        if opts.get("reduction") == "mean" and pairs == 0:
            continue
        plan = O.RowPairs(c, j, rows, weight=opts.get("weight"), reference=opts.get("reference"))
        kw = {k: v for k, v in opts.items() if k in ("beta", "kind", "reduction")}
        got = O.preference_loss(x, plan, label_smoothing=opts.get("smoothing", 0.0), **kw)
        loss, grad, err_l, err_g = ref.pair_loss(s, c, j, **opts)
        assert got.grad.dtype == dtype and got.loss.dtype == torch.float32 and got.loss.shape == ()
        assert_close(got.loss, loss, err_l)
        assert_close(got.grad, grad, err_g)


def test_preference_far_scores_and_infinities():
    """Differences in the tails of the sigmoid, and scores that are not finite: only rows compared with them feel it."""
    s = np.array([0.0, 30.0, -30.0, 200.0, -np.inf, np.inf, np.nan, 1.0, 2.0, 5.0])
    c = np.array([1, 2, 3, 0, 7, 5, 8, 7])
    j = np.array([0, 0, 0, 3, 4, 8, 7, 8])
    plan = O.RowPairs(np.r_[c, 6], np.r_[j, 0], 10)
    got = O.preference_loss(_cuda(s.astype(np.float32)), plan)
    assert torch.isnan(got.loss) and torch.isnan(got.grad[6]) and torch.isnan(got.grad[0])
    plan = O.RowPairs(c, j, 10)
    got = O.preference_loss(_cuda(s.astype(np.float32)), plan)
    finite = np.array([1, 2, 3, 0, 8, 7])   # the pairs (7, 4) and (5, 8) are settled beyond doubt: no loss, no gradient
    keep = np.array([0, 1, 2, 3, 6, 7])
    with np.errstate(invalid="ignore"):
        loss, grad, err_l, err_g = ref.pair_loss(np.where(np.isfinite(s), s, 0.0), c[keep], j[keep])
    assert_close(got.loss, loss, err_l)
    assert_close(got.grad[finite.tolist()], grad[finite], err_g[finite])
    assert got.grad[[4, 5, 6, 9]].tolist() == [0.0] * 4


def test_preference_does_not_depend_on_the_run():
    rng = np.random.default_rng(0)
    c, j = _pairs(rng, 30_000, 400_000, 2, 30_000)
    x, _ = _scores(rng, 30_000, torch.float32)
    a = O.preference_loss(x, O.RowPairs(c, j, 30_000))
    for _ in range(3):
        b = O.preference_loss(x, O.RowPairs(c, j, 30_000))
        assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)


# ---- groups ----------------------------------------------------------------------------------------

LENGTHS = [
    [1], [2], [1, 1, 1], [0, 3, 0, 0, 2, 0], [31, 32, 33], [127, 128, 129, 1, 1], [255, 256, 257], [511, 512, 513],
    [1023], [1024], [1025], [1, 1023, 1, 1024, 1025, 3], [2047, 2048, 2049], [4095, 4096, 4097, 5], [5000] * 3,
    [8191], [8192, 8193], [16383, 16384, 16385], [1, 70_001, 2], [32_768, 1, 33_000], list(range(1, 90)) * 3,
    [4] * 5000, [300_000], [1] * 3000 + [9000] + [7] * 500,
]


def _groups(rng, lengths, mixed):
    group = np.repeat(np.arange(len(lengths)), lengths)
    return rng.permutation(group) if mixed else group


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
def test_groups(lengths, dtype, mixed):
    n, n_groups = sum(lengths), len(lengths)
    rng = np.random.default_rng(n + n_groups)
    group = _groups(rng, lengths, mixed)
    plan = O.RowGroups(group, n_groups)
    assert (plan.n_rows, plan.n_groups) == (n, n_groups)
    for masked in (0.0, 0.3):
        x, s = _scores(rng, n, dtype, 2.0)
        off = rng.random(n) < masked
        if masked:
            off |= group == group[0]            # a group with nothing left
            x[_cuda(off)] = -np.inf
            s[off] = -np.inf
        l = ref.log_probs(s, group, n_groups)
        got = O.group_log_probs(x, plan)
        assert got.dtype == dtype
        assert_close(got, l, ref.U * np.where(np.isfinite(l), np.abs(l), 0))

        t = np.where(off | (rng.random(n) < 0.5), 0.0, rng.random(n)).astype(np.float32)
        for reduction in ("sum", "mean"):
            got = O.choice_loss(x, plan, _cuda(t), reduction=reduction)
            loss, grad, err_l, err_g = ref.choice(s, group, n_groups, t, reduction)
            assert got.grad.dtype == dtype
            assert_close(got.loss, loss, err_l)
            assert_close(got.grad, grad, err_g)

        a = np.where(rng.random(n) < 0.4, 0.0, rng.normal(size=n)).astype(np.float32)
        live = np.where(off, 0.0, s)
        old = ref.log_probs(live + 0.3 * rng.normal(size=n), group, n_groups).astype(np.float32)
        prior = ref.log_probs(live + 0.5 * rng.normal(size=n), group, n_groups).astype(np.float32)
        old[off | (a == 0)] = np.nan            # never looked at
        prior[off] = np.nan
        a[off & (rng.random(n) < 0.5)] = np.nan
        for opts in (dict(), dict(reference=prior, kl_coef=0.1, clip=(0.1, 0.3), reduction="mean"),
                     dict(reference=prior), dict(clip=(1.0, np.inf)), dict(clip=(0.0, 0.0)), dict(clip=(0.5, 1e39))):
            kw = {k: v for k, v in opts.items() if k != "reference"}
            got = O.policy_loss(x, plan, _cuda(a), _cuda(old),
                                reference_log_probs=_cuda(prior) if "reference" in opts else None, **kw)
            loss, grad, kl, clipped, err_l, err_g, err_k = ref.policy(s, group, n_groups, np.where(off, 0, a), old, **opts)
            assert int(got.clipped) == clipped and got.clipped.dtype == torch.int64
            assert_close(got.loss, loss, err_l)
            assert_close(got.kl, kl, err_k)
            assert_close(got.grad, grad, err_g)


@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
def test_more_groups_than_ctas(mixed):
    """CTAs that take one group after the other."""
    rng = np.random.default_rng(12)
    lengths = rng.integers(257, 420, 3000).tolist() + [5000] * 3
    n, n_groups = sum(lengths), len(lengths)
    group = _groups(rng, lengths, mixed)
    plan = O.RowGroups(group)
    x, s = _scores(rng, n, torch.float32, 2.0)
    l = ref.log_probs(s, group, n_groups)
    assert_close(O.group_log_probs(x, plan), l, ref.U * np.abs(l))
    t = rng.random(n).astype(np.float32)
    got = O.choice_loss(x, plan, _cuda(t))
    loss, grad, err_l, err_g = ref.choice(s, group, n_groups, t)
    assert_close(got.loss, loss, err_l)
    assert_close(got.grad, grad, err_g)
    a, old = rng.normal(size=n).astype(np.float32), (l + 0.3 * rng.normal(size=n)).astype(np.float32)
    got = O.policy_loss(x, plan, _cuda(a), _cuda(old), reference_log_probs=_cuda(old), kl_coef=0.1)
    loss, grad, kl, clipped, err_l, err_g, err_k = ref.policy(s, group, n_groups, a, old, old, kl_coef=0.1)
    assert int(got.clipped) == clipped
    assert_close(got.loss, loss, err_l)
    assert_close(got.kl, kl, err_k)
    assert_close(got.grad, grad, err_g)


def test_ratios_at_their_borders():
    """Ratios a few steps of float32 from a border fall on the side on which the definition has them."""
    n = 4096
    rng = np.random.default_rng(1)
    s = rng.normal(size=n).astype(np.float32)
    group = np.repeat(np.arange(8), n // 8)
    l = ref.log_probs(s, group, 8)
    a = np.where(np.arange(n) % 2 == 0, 1.0, -1.0).astype(np.float32)
    old = (l - np.where(a > 0, np.log1p(0.2), np.log1p(-0.2))).astype(np.float32)
    old = np.where(np.arange(n) % 3 == 0, np.nextafter(old, np.float32(9)), old)
    plan = O.RowGroups(group)
    got = O.policy_loss(_cuda(s), plan, _cuda(a), _cuda(old))
    loss, grad, _, clipped, err_l, err_g, _ = ref.policy(s, group, 8, a, old)
    assert 0 < clipped < n and int(got.clipped) == clipped
    assert_close(got.loss, loss, err_l)
    assert_close(got.grad, grad, err_g)


def test_reference_equal_to_the_policy():
    """The divergence from itself is 0 but for the rounding of the given log-probabilities."""
    rng = np.random.default_rng(2)
    group = np.repeat(np.arange(3), 5000)
    s = rng.normal(size=15_000).astype(np.float32)
    prior = ref.log_probs(s, group, 3).astype(np.float32)
    a = np.zeros(15_000, np.float32)
    got = O.policy_loss(_cuda(s), O.RowGroups(group), _cuda(a), _cuda(a), reference_log_probs=_cuda(prior), kl_coef=1.0)
    loss, grad, kl, clipped, err_l, err_g, err_k = ref.policy(s, group, 3, a, a, prior, kl_coef=1.0)
    assert clipped == int(got.clipped) == 0
    assert_close(got.kl, kl, err_k)
    assert_close(got.grad, grad, err_g)


def test_scores_that_are_not_finite_stay_in_their_group():
    group = np.repeat(np.arange(4), 300)
    s = np.random.default_rng(3).normal(size=1200).astype(np.float32)
    s[5], s[310], s[311] = np.nan, np.inf, -np.inf
    t = np.zeros(1200, np.float32)
    t[[7, 320, 700, 1000]] = 1.0
    plan, x = O.RowGroups(group), _cuda(s)
    l = O.group_log_probs(x, plan).cpu().numpy()
    want = ref.log_probs(s[600:], group[600:] - 2, 2)
    assert_close(torch.from_numpy(l[600:]), want, ref.U * np.abs(want))
    assert np.isnan(l[:300]).all() and np.isnan(np.delete(l[300:600], 11)).all()
    got = O.choice_loss(x, plan, _cuda(t))
    assert torch.isnan(got.loss) and torch.isnan(got.grad[:300]).all()
    _, grad, _, err = ref.choice(s[600:], group[600:] - 2, 2, t[600:])
    assert_close(got.grad[600:], grad, err)
    # a target on a masked row
    s = np.zeros(4, np.float32)
    s[0] = -np.inf
    got = O.choice_loss(_cuda(s), O.RowGroups([0] * 4), _cuda(np.array([1, 0, 0, 0], np.float32)))
    assert got.loss.item() == np.inf and got.grad[0].item() == -1.0


def test_far_scores():
    """Scores far apart, far from zero and at the ends of the type."""
    for s in ([1e30, 0.0, -1e30], [-1e30, -1e30, -3e38], [800.0, 100.0, 799.0, -700.0], [-5e4, -5e4 + 1.0], [3e38, 3e38, -3e38]):
        s = np.array(s, np.float32)
        group = np.zeros(len(s), int)
        l = ref.log_probs(s, group, 1)
        plan = O.RowGroups(group)
        assert_close(O.group_log_probs(_cuda(s), plan), l, ref.U * np.abs(l))
        t = np.ones(len(s), np.float32)
        got = O.choice_loss(_cuda(s), plan, _cuda(t))
        loss, grad, err_l, err_g = ref.choice(s, group, 1, t)
        assert_close(got.loss, loss, err_l)
        assert_close(got.grad, grad, err_g)


def test_no_rows():
    plan = O.RowGroups([], 3)
    e = torch.empty(0, device="cuda")
    assert O.group_log_probs(e, plan).shape == (0,)
    got = O.policy_loss(e, plan, e, e, reference_log_probs=e, kl_coef=0.5, reduction="mean")
    assert (got.loss.item(), got.kl.item(), got.clipped.item()) == (0.0, 0.0, 0) and got.grad.shape == (0,)
    got = O.preference_loss(e, O.RowPairs([], [], 0))
    assert got.loss.item() == 0.0 and got.grad.shape == (0,)


# ---- calls ---------------------------------------------------------------------------------------------


def _problem(seed, n=50_000):
    rng = np.random.default_rng(seed)
    group = np.sort(rng.integers(0, 40, n))
    group[:9000] = 0
    x, _ = _scores(rng, n, torch.float32)
    a, old = _cuda(rng.normal(size=n).astype(np.float32)), _cuda(rng.normal(size=n).astype(np.float32) - 7)
    c, j = _pairs(rng, n, 90_000, 3, n)
    return x, O.RowGroups(group), a, old, O.RowPairs(c, j, n)


def _all(x, groups, a, old, pairs):
    return [*O.preference_loss(x, pairs), *O.choice_loss(x, groups, a.abs()), *O.policy_loss(x, groups, a, old, reference_log_probs=old, kl_coef=0.1),
            O.group_log_probs(x, groups)]


def test_strided_and_offset_arguments():
    x, groups, a, old, pairs = _problem(5)
    want = _all(x, groups, a, old, pairs)
    wide = torch.stack([x, -x], 1)
    shifted = torch.cat([x.new_zeros(1), x])[1:]
    for scores in (wide[:, 0], shifted):
        got = _all(scores, groups, a.double(), torch.stack([old, old], 1)[:, 1], pairs)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    h = x.half()
    want = _all(h, groups, a, old, pairs)
    got = _all(torch.cat([h.new_zeros(1), h])[1:], groups, a, old, pairs)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_streams_and_graphs():
    x, groups, a, old, pairs = _problem(6)
    y = x * 0.7 - 0.1
    want_x, want_y = _all(x, groups, a, old, pairs), _all(y, groups, a, old, pairs)
    torch.cuda.synchronize()
    # two streams at once, the layouts shared
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, (s, v) in enumerate(zip(streams, (x, y))):
            with torch.cuda.stream(s):
                got[i].append(_all(v, groups, a, old, pairs))
    torch.cuda.synchronize()
    for runs, want in zip(got, (want_x, want_y)):
        for run in runs:
            assert all(torch.equal(g, w) for g, w in zip(run, want))
    # two captured graphs of the same layouts, replayed in turn and at once
    graphs, outs, ins = [], [], [x.clone(), y.clone()]
    for v in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all(v, groups, a, old, pairs))
        graphs.append(g)
    for _ in range(3):
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, (want_x, want_y)):
            assert all(torch.equal(o, w) for o, w in zip(out, want))
    ins[0].copy_(y)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs[0], want_y))


def test_threads_share_layouts():
    import threading
    x, groups, a, old, pairs = _problem(8)
    want = _all(x, groups, a, old, pairs)
    torch.cuda.synchronize()
    wrong = []

    def work(stream):
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = _all(x, groups, a, old, pairs)
                stream.synchronize()
                if not all(torch.equal(g, w) for g, w in zip(got, want)):
                    wrong.append(1)

    shared = torch.cuda.Stream()
    threads = [threading.Thread(target=work, args=(s,)) for s in (shared, shared, torch.cuda.Stream(), torch.cuda.Stream())]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_arguments_of_other_kinds():
    """Lists, arrays and tensors of any integer type, on the host or the GPU, make the same layouts; sizes on both sides of
    where a layout is made on the host."""
    for n in (700, 40_000):
        rng = np.random.default_rng(n)
        c, j = _pairs(rng, n, 2 * n, 0, n)
        group = rng.integers(0, 40, n)
        w, r = rng.integers(0, 3, 2 * n), rng.normal(size=n)
        x, _ = _scores(rng, n, torch.float32)
        want_p = O.preference_loss(x, O.RowPairs(c, j, n, weight=w, reference=r), reduction="mean")
        want_l = O.group_log_probs(x, O.RowGroups(group))
        for make in (list, lambda v: torch.from_numpy(v.astype(np.int32)).cuda(), lambda v: v.astype(np.uint16), torch.from_numpy):
            got = O.preference_loss(x, O.RowPairs(make(c), make(j), np.int64(n), weight=_cuda(w), reference=_cuda(r)), reduction="mean")
            assert torch.equal(got.loss, want_p.loss) and torch.equal(got.grad, want_p.grad)
            assert torch.equal(O.group_log_probs(x, O.RowGroups(make(group), 50)), want_l)
        leaf = x.clone().requires_grad_()
        got = O.preference_loss(leaf, O.RowPairs(c, j, n, weight=w, reference=r), reduction="mean")
        assert torch.equal(got.grad, want_p.grad) and not got.loss.requires_grad and not got.grad.requires_grad


def test_fit_without_eras():
    X, _, rng = _table(n=3000, seed=8)
    n = len(X)
    c, j = _pairs(rng, n, 5000, 0, n)
    t = rng.random(n).astype(np.float32)
    for objective, other in ((O.PreferenceObjective(_cuda(c), _cuda(j)), O.PreferenceObjective(c.tolist(), j.tolist())),
                             (O.ChoiceObjective(t), O.ChoiceObjective(_cuda(t), group=np.zeros(n, np.int64)))):
        a = PackBoost(PackBoostConfig(**CFG)).fit(X, None, None, num_rounds=3, objective=objective)
        b = PackBoost(PackBoostConfig(**CFG)).fit(torch.from_numpy(X).cuda(), np.ones(n, np.float32), None, num_rounds=3, objective=other)
        _same_trees(a, b)


def test_many_options_and_streams():
    """More descriptors and more streams than a layout keeps."""
    x, groups, a, old, pairs = _problem(9, 9500)
    want = O.preference_loss(x, pairs, beta=1.0)
    for i in range(70):
        O.preference_loss(x, pairs, beta=0.5 + i / 100)
    for _ in range(20):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = O.preference_loss(x, pairs, beta=1.0)
        torch.cuda.synchronize()
        assert torch.equal(got.loss, want.loss) and torch.equal(got.grad, want.grad)


def test_a_layout_may_go_while_its_call_runs():
    want = _all(*_problem(7))
    side = torch.cuda.Stream()
    args = _problem(7)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = _all(*args)
    del args
    torch.cuda.current_stream().synchronize()
    junk = [torch.full((200_000,), 7, dtype=torch.int32, device="cuda") for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and len(junk) == 20


# ---- fits ------------------------------------------------------------------------------------------------

CFG = dict(pack_size=4, max_depth=4, learning_rate=0.1, lambda_l2=1.0, lambda_dro=0.3, min_samples_leaf=5, max_bins=32,
           random_state=11, layer_feature_fraction=0.7)


def _table(n=6000, f=12, eras=7, mixed=False, seed=0):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(n, f)).astype(np.float32)
    era = np.sort(rng.integers(0, eras, n)).astype(np.int16)
    if mixed:
        era = rng.permutation(era)
    return X, era, rng


def _objectives(n, era, rng):
    c = rng.integers(0, n, 3 * n)
    j = (c + rng.integers(1, n, 3 * n)) % n
    group = rng.integers(0, n // 9, n)
    t, a = rng.random(n).astype(np.float32), rng.normal(size=n).astype(np.float32)
    old = ref.log_probs(rng.normal(size=n) * 0.3, group, n // 9 + 1).astype(np.float32)
    r, w = rng.normal(size=n) * 0.2, rng.random(3 * n).astype(np.float32)
    era_ids = np.unique(era, return_inverse=True)[1]
    old_era = ref.log_probs(rng.normal(size=n) * 0.3, era_ids, era_ids.max() + 1).astype(np.float32)

    def preference(s):
        return ref.pair_loss(s, c, j, weight=w, reference=r, beta=0.8)[:2]

    def choice(s):
        return ref.choice(s, era_ids, era_ids.max() + 1, t)[:2]

    def policy(s):
        return ref.policy(s, group, n // 9 + 1, a, old, old, (0.2, 0.2), 0.2)[:2]

    def policy_era(s):
        return ref.policy(s, era_ids, era_ids.max() + 1, a, old_era)[:2]

    return [(O.PreferenceObjective(c, j, weight=w, reference=r, beta=0.8), preference), (O.ChoiceObjective(t), choice),
            (O.PolicyObjective(a, old, group=group, reference_log_probs=old, kl_coef=0.2), policy),
            (O.PolicyObjective(_cuda(a), _cuda(old_era)), policy_era)]


def _same_trees(a, b):
    assert len(a.trees) == len(b.trees)
    for x, y in zip(a.trees, b.trees):
        p, q = x.arrays(), y.arrays()
        assert all(np.array_equal(p[k], q[k]) for k in p)


@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
@pytest.mark.parametrize("which", range(4))
def test_fit_learns_from_the_objective(mixed, which):
    """Every round's leaves hold the mean negative gradient of the objective at the predictions before it, and the first
    tree is, bit for bit, that of the squared loss on those gradients."""
    X, era, rng = _table(mixed=mixed)
    objective, formula = _objectives(len(X), era, rng)[which]
    seen = []
    b = PackBoost(PackBoostConfig(**CFG))
    b.fit(X, None, era, num_rounds=3, objective=objective, round_callback=lambda r, m: seen.append(m["train_loss"]))
    bins = torch.from_numpy(np.stack([np.searchsorted(b._binner.bin_edges[:, k], X[:, k]) for k in range(X.shape[1])], 1)
                            .clip(0, 31).astype(np.uint8)).cuda()
    preds = np.zeros(len(X))
    for r, (tree, repeat) in enumerate(b._distinct):
        loss, grad = formula(preds)
        value = tree.predict_bins(bins).cpu().numpy()
        for v in np.unique(value):
            rows = value == v
            g, size = grad[rows].sum(), np.abs(grad[rows]).sum()
            # rows whose leaves have the same value by chance share a check; 1e-5: the predictions and the quantised
            # gradients of earlier rounds are float32
            lam = CFG["lambda_l2"]
            assert abs(v * (rows.sum() + lam) + g) <= 1e-5 * size + 1e-6 or _several_leaves(tree, v)
        preds = preds + CFG["learning_rate"] * repeat * value.astype(np.float64)
        assert abs(seen[r] - formula(preds)[0]) <= 1e-5 * (abs(seen[r]) + len(X) * 1e-2)
    np.testing.assert_allclose(b.train_predictions(), preds, rtol=1e-5, atol=1e-6)

    one = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=1, objective=objective)
    plain = PackBoost(PackBoostConfig(**CFG))
    plain._start(X, np.zeros(len(X), np.float32), era)
    bound = objective._bind(len(X), *_order(era), torch.device("cuda", 0))
    g = O._evaluate(bound.struct, bound.layout, torch.zeros(len(X), device="cuda")).grad
    plain._trainer.y.copy_(-g)
    plain._boost_one_round(0, 1)
    plain._finish()
    _same_trees(one, plain)


def _order(era):
    from packboost_b200.data import sort_eras
    _, offsets, order = sort_eras(era, len(era))
    return offsets, order


def _several_leaves(tree, v):
    a = tree.arrays()
    return ((a["value"] == np.float32(v)) & (a["is_leaf"] != 0)).sum() > 1


@pytest.mark.parametrize("env", [{"PACKBOOST_CUDA_GRAPH": "0"}, {"PACKBOOST_RUN_AHEAD": "0"}, {"PACKBOOST_TRAIN_METRICS": "1"}])
@pytest.mark.parametrize("which", [0, 2])
def test_fit_is_the_same_however_it_is_launched(env, which, monkeypatch):
    X, era, rng = _table(seed=3)
    objective, _ = _objectives(len(X), era, rng)[which]
    want = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=6, objective=objective)
    for k, v in env.items():
        monkeypatch.setenv(k, v)
    got = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=6, objective=objective)
    _same_trees(want, got)
    assert np.array_equal(want.train_predictions(), got.train_predictions())


def test_fit_phase_by_phase_is_the_loop():
    """The launches of several GPUs' ranks, which go phase by phase, on one."""
    X, era, rng = _table(seed=4)
    objective, _ = _objectives(len(X), era, rng)[0]
    want = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=4, objective=objective)
    got = PackBoost(PackBoostConfig(**CFG))
    got._start(X, None, era, objective=objective)
    tr = got._trainer
    loop, tr.loop, tr.use_graph = tr.loop, None, False
    tr.log_event = [torch.cuda.Event() for _ in range(len(tr.log_host))]
    for r in range(4):
        got._boost_one_round(r, 4)
    got._finish()
    tr.loop = loop
    _same_trees(want, got)


def test_fit_that_stops_early_is_taken_again():
    """Frontiers that empty before the last depth make the round after them be enqueued twice."""
    X, era, rng = _table(n=300, seed=5)
    objective, _ = _objectives(len(X), era, rng)[0]
    cfg = dict(CFG, min_samples_leaf=70, max_depth=5)
    got = PackBoost(PackBoostConfig(**cfg)).fit(X, None, era, num_rounds=5, objective=objective)
    calm = PackBoost(PackBoostConfig(**cfg))
    calm.fit(X, None, era, num_rounds=5, objective=objective, round_callback=lambda r, m: None)
    assert min(got._round_depths) < 5
    _same_trees(got, calm)


def test_from_choices_to_preferences_to_a_policy():
    """The three one after the other, as they are used: log-probabilities of a model are the reference of the next."""
    X, era, rng = _table(n=4000, seed=6)
    n = len(X)
    group = rng.integers(0, 500, n)
    quality = X[:, 0] + 0.5 * X[:, 1] ** 2
    first = PackBoostRegressor(num_rounds=5, **CFG).fit(X, None, era, objective=O.ChoiceObjective((quality > 1).astype(np.float32), group=group))
    prior = first.booster_.predict_log_probs(X, group)
    want = ref.log_probs(first.predict(X), group, 500)
    assert_close(torch.from_numpy(prior), want, ref.U * np.abs(want))
    c = rng.integers(0, n, 8000)
    j = (c + rng.integers(1, n, 8000)) % n
    c, j = np.where(quality[c] > quality[j], c, j), np.where(quality[c] > quality[j], j, c)
    second = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=5, objective=O.PreferenceObjective(c, j, reference=prior, beta=0.5))
    old = second.predict_log_probs(X, group)
    a = np.where(rng.random(n) < 0.3, quality - quality.mean(), 0).astype(np.float32)
    third = PackBoost(PackBoostConfig(**CFG))
    third.fit(X, quality, era, num_rounds=5, objective=O.PolicyObjective(a, old, group=group, reference_log_probs=prior, kl_coef=0.05),
              eval_sets=[("valid", X[:500], quality[:500], era[:500])], round_callback=lambda r, m: None)
    assert all(np.isfinite(m["train_loss"]) and "valid_corr" in m for m in third.round_metrics)
    with pytest.raises(ValueError):
        third.predict_log_probs(X, group[:-1])
    # and the squared loss after them, on the same booster, as ever
    third._rng.manual_seed(CFG["random_state"])
    third.fit(X, quality, era, num_rounds=3)
    _same_trees(third, PackBoost(PackBoostConfig(**CFG)).fit(X, quality, era, num_rounds=3))
    assert "train_loss" not in third.round_metrics[0]


def test_refused_fits():
    X, era, rng = _table(n=200)
    b = PackBoost(PackBoostConfig(**CFG))
    for objective, error in ((O.PreferenceObjective([0], [200]), ValueError), (O.ChoiceObjective(np.zeros(199)), ValueError),
                             (O.ChoiceObjective(np.zeros(200), group=[0] * 199), ValueError),
                             (O.PolicyObjective(np.zeros(200), np.zeros(200), kl_coef=1.0), ValueError),
                             (O.PreferenceObjective([0], [1], beta=-1), ValueError)):
        with pytest.raises(error):
            b.fit(X, None, era, num_rounds=1, objective=objective)
    with pytest.raises(ValueError):
        b.fit(X, None, era, num_rounds=1)
    with pytest.raises(TypeError):
        b.fit(X, None, era, num_rounds=1, objective="preference")
    z, one, bad = np.zeros(200), np.ones(200), np.full(200, np.nan)
    for objective in (O.ChoiceObjective(bad), O.ChoiceObjective(-one), O.PolicyObjective(bad, z), O.PolicyObjective(one, bad),
                      O.PolicyObjective(z, z, reference_log_probs=bad), O.PolicyObjective(z, z, reference_log_probs=bad, kl_coef=1.0)):
        with pytest.raises(ValueError):
            b.fit(X, None, era, num_rounds=1, objective=objective)
    b.fit(X, None, era, num_rounds=2, objective=O.PolicyObjective(z, bad))    # (nothing was taken: nothing is looked at)
    x = torch.zeros(200, device="cuda")
    with pytest.raises(ValueError):
        O.choice_loss(x, O.RowGroups([0] * 200), x.cpu())
    with pytest.raises(ValueError):
        O.preference_loss(x.cpu(), O.RowPairs([0], [1], 200))


# ---- numbers that 32 bits do not hold, kernels that take many groups ------------------------------------

# how many groups of which lengths: lanes of a warp, CTAs of 512 and of 256 threads, CTAs that take several, pieces
KINDS = {"teams": [1 + k % 256 for k in range(600)], "few": [257, 900, 8192], "blocks": [257 + k * 13 % 644 for k in range(500)],
         "many": [257 + k * 7 % 160 for k in range(2500)], "pieces": [8193, 20_001]}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_ratios_beyond_float32(kind, mixed, sign):
    """exp(l - old) above the largest float32 is infinite: never a number that is none, and in no other group.  (95 and 100: just
    beyond; what the 2^x unit's argument leaves out is of either sign.)"""
    lengths = KINDS[kind]
    n, n_groups = sum(lengths), len(lengths)
    rng = np.random.default_rng(n)
    group = _groups(rng, lengths, mixed)
    x, s = _scores(rng, n, torch.float32)
    l = ref.log_probs(s, group, n_groups)
    a = np.where(rng.random(n) < 0.5, 0.0, rng.normal(size=n)).astype(np.float32)
    old = (l + 0.3 * rng.normal(size=n)).astype(np.float32)
    plan = O.RowGroups(group, n_groups)
    over = np.zeros(n_groups, bool)
    over[::2] = True
    rows = np.array([np.flatnonzero(group == g)[-1] for g in np.flatnonzero(over)])
    clip = (0.2, 0.2) if sign < 0 else (0.2, np.inf)      # (a gain is cut off, a loss is not)
    for far in (95.0, 97.3, 100.0, 1e3, 1e30, np.inf):
        b, o = a.copy(), old.copy()
        b[over[group]] = 0.0
        b[rows], o[rows] = sign * 0.7, l[rows] - far
        got = O.policy_loss(x, plan, _cuda(b), _cuda(o.astype(np.float32)), reference_log_probs=_cuda(old), kl_coef=0.1, clip=clip)
        assert got.loss.item() == -sign * np.inf
        rest = ~over[group]
        ids = np.unique(group[rest], return_inverse=True)[1]
        _, grad, _, clipped, _, err_g, _ = ref.policy(s[rest], ids, ids.max() + 1, b[rest], o[rest], old[rest], clip, 0.1)
        g = got.grad.cpu()
        assert int(got.clipped) == clipped
        assert_close(g[torch.from_numpy(rest)], grad, err_g)
        own = np.zeros(n, bool)
        own[rows] = True
        assert (g[torch.from_numpy(own)] == -sign * np.inf).all()
        assert (g[torch.from_numpy(over[group] & ~own)] == sign * np.inf).all()
        assert torch.isfinite(got.kl)


def test_an_old_log_probability_that_is_no_number():
    """Of a taken row it makes the loss and its group's gradients no numbers, and no other group's."""
    group, s = np.repeat([0, 1], 40), np.random.default_rng(1).normal(size=80)
    a, old = np.full(80, -0.5, np.float32), ref.log_probs(s, group, 2).astype(np.float32)
    old[3] = np.nan
    x = _cuda(s.astype(np.float32))
    got = O.policy_loss(x, O.RowGroups(group), _cuda(a), _cuda(old))
    assert torch.isnan(got.loss) and torch.isnan(got.grad[:40]).all() and torch.isfinite(got.grad[40:]).all()


def test_long_groups_one_call_after_the_other():
    """The sums that a long group's launches hand on are those of their own call: calls in a row whose sums differ."""
    rng = np.random.default_rng(21)
    lengths = [70_001, 300, 9001, 5, 120_000]
    n, group = sum(lengths), np.repeat(np.arange(5), lengths)
    plan = O.RowGroups(group)
    x, s = _scores(rng, n, torch.float32)
    l = ref.log_probs(s, group, 5)
    old = (l + 0.2 * rng.normal(size=n)).astype(np.float32)
    base = np.abs(rng.normal(size=n)).astype(np.float32)
    t = rng.random(n).astype(np.float32)
    scales = [1.0, -3.0, 0.01, 50.0] * 8
    rows = [_cuda(base * np.float32(k)) for k in scales]
    o, target = _cuda(old), [_cuda(t), _cuda(3 * t)]
    torch.cuda.synchronize()
    got = [(O.policy_loss(x, plan, a, o), O.choice_loss(x, plan, target[i % 2]), O.group_log_probs(x, plan)) for i, a in enumerate(rows)]
    for i, (policy, choice, log_probs) in enumerate(got):
        loss, grad, _, clipped, err_l, err_g, _ = ref.policy(s, group, 5, base * np.float32(scales[i]), old)
        assert int(policy.clipped) == clipped
        assert_close(policy.loss, loss, err_l)
        assert_close(policy.grad, grad, err_g)
        loss, grad, err_l, err_g = ref.choice(s, group, 5, t if i % 2 == 0 else 3 * t)
        assert_close(choice.loss, loss, err_l)
        assert_close(choice.grad, grad, err_g)
        assert_close(log_probs, l, ref.U * np.abs(l))


def test_pairs_of_scores_that_the_call_before_makes():
    """Log-probabilities as the scores of pairs: the launch of the pairs may begin before they are written."""
    rng = np.random.default_rng(31)
    lengths = [40, 3000, 60_000, 7] * 3
    n, group = sum(lengths), np.repeat(np.arange(12), lengths)
    groups = O.RowGroups(group)
    c, j = _pairs(rng, n, 400_000, 2, n)
    pairs = O.RowPairs(c, j, n)
    inputs = [_scores(rng, n, torch.float32, spread) for spread in (1.0, 3.0, 0.1)]
    torch.cuda.synchronize()
    got = [O.preference_loss(O.group_log_probs(x, groups), pairs, beta=0.5) for _ in range(6) for x, _ in inputs]
    for i, (loss, grad) in enumerate(got):
        l = O.group_log_probs(inputs[i % 3][0], groups).double().cpu().numpy()
        want, want_grad, err_l, err_g = ref.pair_loss(l, c, j, beta=0.5)
        assert_close(loss, want, err_l)
        assert_close(grad, want_grad, err_g)


@pytest.mark.parametrize("hubs", [0, 1], ids=["slices", "chunks"])
@pytest.mark.parametrize("beta,size,kind", [(1e20, 1e-24, "logistic"), (1e30, 1e-25, "logistic"), (1e-30, 1e30, "logistic"), (1e-15, 1e-25, "squared")])
def test_factors_beyond_float32(beta, size, kind, hubs):
    """Beta, the weights and a mean over them are float32 numbers, their product need not be one: the gradients are still the
    definition's, and 0 for rows in no pair."""
    rng = np.random.default_rng(41)
    rows, pairs = 3000, 4000
    c, j = _pairs(rng, rows, pairs, hubs, 2000)
    # whole numbers: differences are 0 or beyond what the sigmoid notices at a large beta
    s = rng.integers(-3, 4, rows).astype(np.float64)
    w = (rng.integers(1, 5, pairs) * size).astype(np.float32)
    got = O.preference_loss(_cuda(s.astype(np.float32)), O.RowPairs(c, j, rows, weight=w), beta=beta, kind=kind, reduction="mean")
    loss, grad, err_l, err_g = ref.pair_loss(s, c, j, weight=w, beta=beta, kind=kind, reduction="mean")
    if beta > 1:
        # (a step of d = 0, and differences that are exact: only the sigmoid's roundings and the sums' are left, 23 of them)
        z = beta * (s[c] - s[j])
        slope = np.where(z == 0, -0.5, np.where(z > 0, 0.0, -1.0)) * beta
        w64 = w.astype(np.float64)
        grad = (np.bincount(c, w64 * slope, rows) - np.bincount(j, w64 * slope, rows)) / w64.sum()
        err_g = 24 * ref.U * (np.bincount(c, w64, rows) + np.bincount(j, w64, rows)) * beta / w64.sum()
    assert_close(got.grad, grad, err_g)
    assert_close(got.loss, loss, err_l)
    assert (got.grad[2000:] == 0).all()


@pytest.mark.parametrize("env", [{}, {"PACKBOOST_CUDA_GRAPH": "0"}, {"PACKBOOST_RUN_AHEAD": "0"}, {"PACKBOOST_TRAIN_METRICS": "1"}])
@pytest.mark.parametrize("both", [False, True], ids=["infinite", "no number"])
def test_fit_with_a_gradient_that_is_not_finite(env, both, monkeypatch):
    """A ratio beyond float32 (two of either sign in a group: infinity less infinity) ends the fit."""
    for k, v in env.items():
        monkeypatch.setenv(k, v)
    X, era, rng = _table(seed=9)
    n = len(X)
    group = np.arange(n) // 12
    a, old = rng.normal(size=n), np.full(n, -np.log(12.0))
    a[120], old[120] = -1.0, -120.0
    if both:
        a[121], old[121] = 1.0, -120.0
    objective = O.PolicyObjective(a, old, group=group, clip=(0.2, np.inf))
    b = PackBoost(PackBoostConfig(**CFG))
    with pytest.raises(RuntimeError, match="round 1: .*not finite"):
        b.fit(X, None, era, num_rounds=5, objective=objective)
    assert len(b.trees) == 0
    # and the same booster goes on to other fits
    b._rng.manual_seed(CFG["random_state"])
    b.fit(X, a, era, num_rounds=3)
    _same_trees(b, PackBoost(PackBoostConfig(**CFG)).fit(X, a, era, num_rounds=3))


def test_fit_whose_gradient_overflows_later_keeps_the_trees_before():
    """Tiny gains of a ratio near the end of float32 (e^87.5) raise the chosen rows' scores until it is beyond."""
    n = 1200
    group, chosen = np.arange(n) // 12, np.arange(n) % 12 == 0
    X = np.random.default_rng(10).normal(size=(n, 4)).astype(np.float32)
    X[:, 0] = chosen                                  # a leaf of its own: all chosen rows, with a slope of -10 (1 - 1/12) each
    a = np.where(chosen, 1e-37, 0.0)
    old = np.full(n, -np.log(12.0) - 87.5)
    b = PackBoost(PackBoostConfig(**dict(CFG, layer_feature_fraction=1.0)))
    with pytest.raises(RuntimeError, match="not finite") as e:
        b.fit(X, None, np.zeros(n, np.int16), num_rounds=50, objective=O.PolicyObjective(a, old, group=group, clip=(0.2, np.inf)))
    done = int(str(e.value).split(":")[0].split()[1]) - 1
    assert done >= 1 and len(b.trees) == done * CFG["pack_size"]
    value = b.trees[0].arrays()["value"]
    # (the leaf of the chosen rows: 10 (1 - 1/12) 100 / (100 + lambda), up to the float32 of advantage and old)
    want = 1e-37 * np.exp(87.5) * (11 / 12) * 100 / 101
    assert abs(value.max() / want - 1) < 1e-4


def test_a_refused_round_leaves_the_state_as_it_was():
    """Too small a workspace: nothing is launched, in particular not the last round's step of the predictions."""
    import ctypes as C
    from packboost_b200 import backends as B
    X, era, rng = _table(seed=12)
    objective, _ = _objectives(len(X), era, rng)[0]
    want = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=4, objective=objective)
    got = PackBoost(PackBoostConfig(**CFG))
    got._start(X, None, era, objective=objective)
    tr = got._trainer
    for r in range(4):
        got._boost_one_round(r, 4)
        before = tr.preds.clone()
        struct, scratch, nbytes = tr._objective_args()
        for address, size, error in ((scratch, nbytes - 1, RuntimeError), (None, nbytes, ValueError), (scratch + 4, nbytes, ValueError)):
            with pytest.raises(error, match="workspace"):
                B.check(B.lib().pb_round_begin_objective(C.byref(tr.st), struct, 1, address, size, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(tr.preds, before)
    got._finish()
    _same_trees(want, got)


def test_a_descriptor_that_changes_in_its_place(monkeypatch):
    """Rounds that are replayed learn from what the descriptor says now, not from what it said when one was captured."""
    X, era, rng = _table(seed=13)
    objective, _ = _objectives(len(X), era, rng)[0]

    def fit(change, graphs):
        monkeypatch.setenv("PACKBOOST_CUDA_GRAPH", graphs)
        b = PackBoost(PackBoostConfig(**CFG))
        b._start(X, None, era, objective=objective)
        for r in range(8):
            if change and r == 4:
                b._trainer.objective.struct.beta = 0.05
            b._boost_one_round(r, 8)
        replays = b._trainer.graph_replays
        b._finish()
        return b, replays

    (plain, none), (replayed, some), (other, _) = fit(True, "0"), fit(True, "1"), fit(False, "1")
    assert none == 0 and some >= 6
    _same_trees(plain, replayed)
    assert not np.array_equal(plain.train_predictions(), other.train_predictions())


def test_calls_through_the_public_functions(monkeypatch):
    """Where torch has no quicker ones."""
    args = _problem(14, 9500)
    want = _all(*args)
    monkeypatch.setattr(O, "_device_now", O._quick("_not_there", torch.cuda.current_device))
    monkeypatch.setattr(O, "_stream_now", O._quick("_not_there", lambda index: torch.cuda.current_stream(index).cuda_stream))
    monkeypatch.setattr(O, "_capturing", O._quick("_not_there", torch.cuda.is_current_stream_capturing))
    got = _all(*args)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _all(*args)
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        _all(*args)


@pytest.mark.parametrize("kind", ["blocks", "many"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
def test_kernels_of_many_groups(kind, dtype, mixed):
    """Tables of some hundred eras: CTAs of 256 threads for a group each, and for one group after the other; a group with nothing
    left, and arrays that do not begin on the border of a word."""
    lengths = KINDS[kind] + ([8192, 5000, 8191] if kind == "blocks" else [])
    n, n_groups = sum(lengths), len(lengths)
    rng = np.random.default_rng(n + 1)
    group = _groups(rng, lengths, mixed)
    plan = O.RowGroups(group, n_groups)
    x, s = _scores(rng, n, dtype, 2.0)
    off = (rng.random(n) < 0.1) | (group == 7)
    x[_cuda(off)] = -np.inf
    s[off] = -np.inf
    t = np.where(off | (rng.random(n) < 0.5), 0.0, rng.random(n)).astype(np.float32)
    a = np.where(off, np.nan, np.where(rng.random(n) < 0.4, 0.0, rng.normal(size=n))).astype(np.float32)
    live = np.where(off, 0.0, s)
    old = ref.log_probs(live + 0.3 * rng.normal(size=n), group, n_groups).astype(np.float32)
    prior = ref.log_probs(live + 0.5 * rng.normal(size=n), group, n_groups).astype(np.float32)
    old[off | (a == 0)] = np.nan
    prior[off] = np.nan
    l = ref.log_probs(s, group, n_groups)
    opts = dict(kl_coef=0.1, clip=(0.1, 0.3))
    want_c = ref.choice(s, group, n_groups, t, "mean")
    loss_p, grad_p, kl, clipped, err_l, err_g, err_k = ref.policy(s, group, n_groups, np.where(off, 0, a), old, prior, **opts)
    for shift in (0, 1):
        def put(v):
            v = v if isinstance(v, torch.Tensor) else _cuda(v)
            return torch.cat([v.new_zeros(shift), v])[shift:]
        y = put(x)
        assert_close(O.group_log_probs(y, plan), l, ref.U * np.where(np.isfinite(l), np.abs(l), 0))
        got = O.choice_loss(y, plan, put(t), reduction="mean")
        assert got.grad.dtype == dtype
        assert_close(got.loss, want_c[0], want_c[2])
        assert_close(got.grad, want_c[1], want_c[3])
        got = O.policy_loss(y, plan, put(a), put(old), reference_log_probs=put(prior), **opts)
        assert int(got.clipped) == clipped
        assert_close(got.loss, loss_p, err_l)
        assert_close(got.kl, kl, err_k)
        assert_close(got.grad, grad_p, err_g)


def test_log_probs_of_whatever_predict_takes():
    X, era, rng = _table(n=500, seed=15)
    group = rng.integers(0, 40, 500)
    b = PackBoost(PackBoostConfig(**CFG)).fit(X, None, era, num_rounds=2, objective=O.ChoiceObjective(rng.random(500), group=group))
    want = b.predict_log_probs(X, group)
    for other in (X.tolist(), torch.from_numpy(X), torch.from_numpy(X).cuda(), np.asfortranarray(X)):
        np.testing.assert_array_equal(b.predict_log_probs(other, group.tolist()), want)
        with pytest.raises(ValueError, match="align"):
            b.predict_log_probs(other, group[1:])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
@pytest.mark.parametrize("offset,step,dtype", [(1e5, 2.0 ** -7, torch.float32), (-3e6, 0.25, torch.float32), (1e8, 8.0, torch.float32),
                                               (-1e9, 64.0, torch.float32), (5e4, 32.0, torch.float16), (-1e9, 2.0 ** 23, torch.bfloat16)])
def test_groups_far_from_zero(kind, mixed, offset, step, dtype):
    """Only differences within a group count: scores at the 1e9 below zero of a mask that is a number, or with a large offset.
    Every other group lies there, the others do not."""
    lengths = KINDS[kind]
    n, n_groups = sum(lengths), len(lengths)
    rng = np.random.default_rng(n + 2)
    group = _groups(rng, lengths, mixed)
    far = group % 2 == 0
    # near its offset a score is a whole number of steps of the type, of which half of the rows take none
    base = float(torch.tensor(offset).to(dtype))
    more = np.where(rng.random(n) < 0.5, 0, rng.integers(0, max(2, int(4 / step)), n)) * step
    x = torch.from_numpy(np.where(far, base + more, rng.normal(size=n)).astype(np.float32)).to(dtype)
    s = x.double().numpy() - np.where(far, base, 0.0)          # (exact: what the formulas see)
    if dtype is torch.float32:
        np.testing.assert_array_equal(s[far], more[far])
    x = x.cuda()
    # The log of the sum is a 64-bit number near the offset: off by half a step of those, twice with the sum's own, relative to
    # each p and ratio; the bounds have at least two roundings (2 U) for each of them
    grow = 1 + 2 * abs(base) * 2.0 ** -53 / (2 * ref.U)
    l = ref.log_probs(s, group, n_groups)
    plan = O.RowGroups(group, n_groups)
    assert_close(O.group_log_probs(x, plan), l, ref.U * np.abs(l) + 2 * abs(base) * 2.0 ** -53)
    t = np.where(rng.random(n) < 0.5, 0.0, rng.random(n)).astype(np.float32)
    got = O.choice_loss(x, plan, _cuda(t))
    loss, grad, err_l, err_g = ref.choice(s, group, n_groups, t)
    assert_close(got.loss, loss, err_l + 2 * abs(base) * 2.0 ** -53 * t.sum())
    assert_close(got.grad, grad, err_g * grow)
    # (rows far behind in their group are not taken: their ratio is one of two float32 numbers that are not exact)
    a = np.where((rng.random(n) < 0.4) | (l < -50), 0.0, rng.normal(size=n)).astype(np.float32)
    old, prior = ((l + k * rng.normal(size=n)).astype(np.float32) for k in (0.3, 0.5))
    got = O.policy_loss(x, plan, _cuda(a), _cuda(old), reference_log_probs=_cuda(prior), kl_coef=0.1)
    loss, grad, kl, clipped, err_l, err_g, err_k = ref.policy(s, group, n_groups, a, old, prior, kl_coef=0.1)
    off = 2 * abs(base) * 2.0 ** -53 * n          # (of a group's divergence: sum p is 1)
    assert int(got.clipped) == clipped
    assert_close(got.loss, loss, err_l * grow + 0.1 * off)
    assert_close(got.kl, kl, err_k * grow + off)
    assert_close(got.grad, grad, err_g * grow + 0.1 * 2 * abs(base) * 2.0 ** -53 * 2)


def test_pairs_behind_whatever_is_in_front():
    """The launch of the pairs may begin before the kernel in front has ended, not before anything else: a wait for another stream,
    a copy from the host, a graph."""
    rng = np.random.default_rng(51)
    n = 50_000
    c, j = _pairs(rng, n, 200_000, 2, n)
    pairs = O.RowPairs(c, j, n)
    x, y = (_scores(rng, n, torch.float32)[0] for _ in range(2))
    want_x, want_y = O.preference_loss(x, pairs), O.preference_loss(y, pairs)
    host = y.cpu().pin_memory()
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    buffer, source = x.clone(), y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.cuda._sleep(300_000)
        buffer.copy_(source * 1.0)
    torch.cuda.synchronize()

    def from_another_stream():
        side.wait_stream(main)          # (the first call reads what is overwritten)
        with torch.cuda.stream(side):
            torch.cuda._sleep(3_000_000)
            buffer.copy_(y * 1.0)
        main.wait_stream(side)

    def from_the_host():
        torch.cuda._sleep(300_000)
        buffer.copy_(host, non_blocking=True)

    for fill in (from_another_stream, from_the_host, graph.replay):
        for _ in range(3):
            buffer.copy_(x)
            torch.cuda.synchronize()
            with torch.cuda.stream(main):
                first = O.preference_loss(buffer, pairs)      # (a kernel that lets the next one begin)
                fill()
                got = O.preference_loss(buffer, pairs)
            torch.cuda.synchronize()
            for g, w in ((first, want_x), (got, want_y)):
                assert torch.equal(g.loss, w.loss) and torch.equal(g.grad, w.grad)


@pytest.mark.parametrize("ahead", ["0", "1"])
def test_a_fit_that_ended_answers_with_the_trees_it_has(ahead, monkeypatch):
    """The predictions of the training rows hold a step of the round that is not there; they are gone with it."""
    monkeypatch.setenv("PACKBOOST_RUN_AHEAD", ahead)
    n = 1200
    group, chosen = np.arange(n) // 12, np.arange(n) % 12 == 0
    X = np.random.default_rng(10).normal(size=(n, 4)).astype(np.float32)
    X[:, 0] = chosen
    args = dict(group=group, clip=(0.2, np.inf))
    a, old = np.where(chosen, 1e-37, 0.0), np.full(n, -np.log(12.0) - 87.5)
    cfg, era = PackBoostConfig(**dict(CFG, layer_feature_fraction=1.0)), np.zeros(n, np.int16)
    b = PackBoost(cfg)
    with pytest.raises(RuntimeError, match="not finite") as e:
        b.fit(X, None, era, num_rounds=50, objective=O.PolicyObjective(a, old, **args))
    done = int(str(e.value).split(":")[0].split()[1]) - 1
    want = PackBoost(cfg).fit(X, None, era, num_rounds=done, objective=O.PolicyObjective(a, old, **args))
    _same_trees(b, want)
    np.testing.assert_array_equal(b.predict(X), want.predict(X))
    with pytest.raises(RuntimeError):
        b.train_predictions()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mixed", [False, True], ids=["ordered", "mixed"])
@pytest.mark.parametrize("low", [-5e3, -1e5, -1e7, -1e9])
def test_taken_rows_far_behind_in_their_group(kind, mixed, low):
    """Rows under a mask that is a number and that were taken all the same: their ratio is that of the two log-probabilities,
    however little of their floats is left in the difference."""
    lengths = [k + 1 for k in KINDS[kind]]
    n, n_groups = sum(lengths), len(lengths)
    rng = np.random.default_rng(n + 3)
    group = _groups(rng, lengths, mixed)
    x, s = _scores(rng, n, torch.float32)
    behind = rng.random(n) < 0.3
    first = np.array([np.flatnonzero(group == g)[0] for g in range(n_groups)])
    behind[first] = False                       # (a group keeps a row)
    x[_cuda(behind)] = low
    s[behind] = float(np.float32(low))
    l = ref.log_probs(s, group, n_groups)
    a = np.where(rng.random(n) < 0.4, 0.0, rng.normal(size=n)).astype(np.float32)
    near = np.where(behind, rng.choice([0.0, 1.0, -1.0, 3.0], n) * float(np.spacing(np.float32(abs(low)))), 0.3 * rng.normal(size=n))
    old = (l + np.where(np.abs(near) > 60, 0, near)).astype(np.float32)
    got = O.policy_loss(x, O.RowGroups(group, n_groups), _cuda(a), _cuda(old))
    loss, grad, _, clipped, err_l, err_g, _ = ref.policy(s, group, n_groups, a, old)
    # what the float of l leaves out is a float32 number of up to half a step of l's, 32 at 1e9: off by a rounding of it in each of four sums
    lost = 4 * ref.U * np.where(behind, float(np.spacing(np.float32(abs(low)))), 0.0).max() + 2 * abs(low) * 2.0 ** -53
    grow = 1 + lost / (2 * ref.U)
    assert int(got.clipped) == clipped and 0 < clipped
    assert_close(got.loss, loss, err_l * grow)
    assert_close(got.grad, grad, err_g * grow)
