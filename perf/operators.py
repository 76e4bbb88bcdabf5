"""Performance cases of the objectives: losses on the scores of rows, each with its gradient.

``preference_loss``   paired log ratios: which of two rows was preferred, relative to a reference model
``choice_loss``       log-likelihood of targets under the softmax of each group of rows
``policy_loss``       clipped policy loss over groups of candidates, with the KL divergence from a reference
``group_log_probs``   the normalised scores alone

A case is one evaluation, as a boosting round or a training step makes it: scores change from call to call, the pairs or
groups stay and are laid out before.  Rows and eras follow the repository's benchmark configurations
(``packboost_b200/workloads.py``): 20 000 rows in 20 eras, 500 000 in 100, 2.7 million in 574; candidate lists are ragged.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# rows, eras (pairs stay within an era), pairs; hubs: chosen rows come from so many rows only (0: any)
_PREFERENCE = dict(op="preference", rows=20_000, eras=20, pairs=60_000, hubs=0, type="fp32", kind="logistic", beta=1.0,
                   smoothing=0.0, weighted=False, reference=False, reduction="sum")
# groups: rows are split into that many; ragged: lengths spread (empty groups among them); mixed: rows in no order
_GROUPED = dict(op="choice", rows=20_000, groups=20, ragged=False, mixed=False, type="fp32", masked=0.0, taken=0.25,
                reference=False, kl=0.0, low=0.2, high=0.2, reduction="sum")


def listed():
    return [
        # the comparisons of one prompt batch: latency
        dict(_PREFERENCE, name="pairs_small", rows=257, eras=1, pairs=500, beta=0.1, reference=True, reduction="mean"),
        # the configuration with 20 eras, three comparisons a row
        dict(_PREFERENCE, name="pairs_eras", beta=0.5, smoothing=0.1, reference=True),
        # the largest table, with weights
        dict(_PREFERENCE, name="pairs_large", rows=2_700_000, eras=574, pairs=8_100_000, weighted=True, reference=True),
        # every row compared with a few baselines, 16-bit scores, squared form
        dict(_PREFERENCE, name="pairs_hubs_bf16", rows=500_001, eras=1, pairs=2_000_003, hubs=3, type="bf16", kind="squared",
             beta=2.0, weighted=True),
        # candidate lists of a ranking, 16-bit scores
        dict(_GROUPED, name="choice_lists_bf16", rows=2_700_000, groups=90_001, ragged=True, type="bf16", masked=0.05),
        # eras as groups, 5 000 rows each
        dict(_GROUPED, name="choice_eras", rows=500_000, groups=100, reduction="mean"),
        # one batch of a few candidate lists: latency
        dict(_GROUPED, name="policy_small", op="policy", rows=203, groups=25, ragged=True, reference=True, kl=0.1, taken=1.0),
        # eras as groups on the largest table
        dict(_GROUPED, name="policy_eras", op="policy", rows=2_700_000, groups=574, reference=True, kl=0.05),
        # lists whose rows are interleaved
        dict(_GROUPED, name="policy_lists_mixed", op="policy", rows=999_983, groups=12_345, ragged=True, mixed=True,
             masked=0.02, reference=True, kl=0.01, low=0.1, high=0.3, reduction="mean"),
        # no eras: all rows are one group
        dict(_GROUPED, name="policy_one_group", op="policy", rows=500_000, groups=1, taken=1.0),
        # one query's candidates, and the scores of a whole table
        dict(_GROUPED, name="log_probs_small", op="log_probs", rows=1_000, groups=1),
        dict(_GROUPED, name="log_probs_eras", op="log_probs", rows=2_700_000, groups=574, ragged=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _reduction(rng, kind):
    # (a mean over a million pairs has gradients below the smallest 16-bit numbers)
    return rng.choice(["sum", "mean"]) if kind == "fp32" else "sum"


def draw(rng):
    kind = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    rows = _spread(rng, 200, 2_500_000)
    if rng.random() < 0.4:
        return dict(_PREFERENCE, rows=rows, eras=_spread(rng, 1, max(1, rows // 100)), pairs=_spread(rng, 1, 3 * rows),
                    hubs=rng.choice([0, 0, 1, 7]), type=kind, kind=rng.choice(["logistic", "logistic", "squared"]),
                    beta=rng.choice([0.1, 0.5, 1.0, 2.0]), smoothing=rng.choice([0.0, 0.0, 0.05]),
                    weighted=rng.random() < 0.5, reference=rng.random() < 0.5, reduction=_reduction(rng, kind))
    op = rng.choice(["choice", "policy", "policy", "log_probs"])
    reference = op == "policy" and rng.random() < 0.6
    return dict(_GROUPED, op=op, rows=rows, groups=_spread(rng, 1, max(1, rows // 3)), ragged=rng.random() < 0.7,
                mixed=rng.random() < 0.3, type=kind, masked=rng.choice([0.0, 0.0, 0.05]),
                taken=rng.choice([0.05, 0.3, 1.0]), reference=reference, kl=rng.choice([0.01, 0.1]) if reference else 0.0,
                low=rng.choice([0.1, 0.2]), high=rng.choice([0.2, 0.3]), reduction=_reduction(rng, kind))


# ---- inputs ---------------------------------------------------------------------------------------


def _lengths(case, gen):
    rows, groups = case["rows"], case["groups"]
    if not case["ragged"]:
        return torch.diff(torch.arange(groups + 1, device="cuda", dtype=torch.int64) * rows // groups)
    weight = torch.rand(groups, generator=gen, device="cuda", dtype=torch.float64) ** 2
    ends = torch.floor(torch.cumsum(weight, 0) / weight.sum() * rows).to(torch.int64)
    ends[-1] = rows
    return torch.diff(ends, prepend=torch.zeros(1, dtype=torch.int64, device="cuda"))


def _log_probs64(scores, group, groups):
    s = scores.double()
    top = torch.full((groups,), -math.inf, device=s.device, dtype=torch.float64).scatter_reduce_(0, group, s, "amax")
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    total = torch.zeros(groups, device=s.device, dtype=torch.float64).index_add_(0, group, torch.exp(s - top[group]))
    return s - (top + torch.log(total))[group]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1_000_003 + 17)
    rows, typ = case["rows"], _TYPES[case["type"]]

    def normal(n, std=1.0):
        return std * torch.randn(n, generator=gen, device="cuda")

    if case["op"] == "preference":
        eras, pairs = case["eras"], case["pairs"]
        scores = normal(rows)
        start = torch.arange(eras + 1, device="cuda", dtype=torch.int64) * rows // eras
        era = torch.randint(eras, (pairs,), generator=gen, device="cuda")
        first, length = start[era], start[era + 1] - start[era]
        a = (torch.rand(pairs, generator=gen, device="cuda", dtype=torch.float64) * length).to(torch.int64)
        if case["hubs"]:
            a = torch.minimum(a % case["hubs"], length - 1)
        b = (torch.rand(pairs, generator=gen, device="cuda", dtype=torch.float64) * (length - 1)).to(torch.int64)
        b = b + (b >= a)
        weight = 0.5 + torch.rand(pairs, generator=gen, device="cuda") if case["weighted"] else None
        reference = normal(rows, 0.7) if case["reference"] else None
        return dict(scores=scores.to(typ), chosen=first + a, rejected=first + b, weight=weight, reference=reference)
    groups = case["groups"]
    group = torch.repeat_interleave(torch.arange(groups, device="cuda"), _lengths(case, gen), output_size=rows)
    if case["mixed"]:
        group = group[torch.randperm(rows, generator=gen, device="cuda")]
    scores = normal(rows)
    masked = torch.rand(rows, generator=gen, device="cuda") < case["masked"]
    if case["masked"] > 0:
        masked |= group == groups // 2          # one group with nothing left
    scores = torch.where(masked, torch.full_like(scores, -math.inf), scores).to(typ)
    d = dict(scores=scores, group=group)
    if case["op"] == "choice":
        t = torch.rand(rows, generator=gen, device="cuda")
        keep = (torch.rand(rows, generator=gen, device="cuda") < case["taken"]) & ~masked
        d["target"] = torch.where(keep, t, torch.zeros_like(t))
    if case["op"] == "policy":
        base = scores.float()
        old = _log_probs64(base + normal(rows, 0.3), group, groups).float()
        taken = (torch.rand(rows, generator=gen, device="cuda") < case["taken"]) & ~masked
        advantage = normal(rows)
        d["advantage"] = torch.where(taken, advantage, torch.zeros_like(advantage))
        d["old"] = torch.where(masked, torch.full_like(old, math.nan), old)
        d["reference"] = None
        if case["reference"]:
            ref = _log_probs64(base + normal(rows, 0.5), group, groups).float()
            d["reference"] = torch.where(masked, torch.full_like(ref, math.nan), ref)
    return d


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["op"] == "preference":
        state["total_weight"] = float(case["pairs"]) if state["weight"] is None else float(state["weight"].double().sum())
    if own:
        from packboost_b200 import objectives
        if case["op"] == "preference":
            state["plan"] = objectives.RowPairs(state["chosen"], state["rejected"], case["rows"], weight=state["weight"],
                                                reference=state["reference"])
        else:
            state["plan"] = objectives.RowGroups(state["group"], case["groups"])
    return state


# ---- the operators ----------------------------------------------------------------------------------


def _run_own(state):
    from packboost_b200 import objectives
    case = state["case"]
    if case["op"] == "preference":
        # (the squared form has no smoothing: neither the plain form nor the definition looks at it there)
        smoothing = case["smoothing"] if case["kind"] == "logistic" else 0.0
        return objectives.preference_loss(state["scores"], state["plan"], beta=case["beta"], label_smoothing=smoothing,
                                          kind=case["kind"], reduction=case["reduction"])
    if case["op"] == "choice":
        return objectives.choice_loss(state["scores"], state["plan"], state["target"], reduction=case["reduction"])
    if case["op"] == "policy":
        return objectives.policy_loss(state["scores"], state["plan"], state["advantage"], state["old"],
                                      reference_log_probs=state["reference"], clip=(case["low"], case["high"]),
                                      kl_coef=case["kl"], reduction=case["reduction"])
    return objectives.group_log_probs(state["scores"], state["plan"])


def _plain_preference(state):
    case, s = state["case"], state["scores"].float()
    c, j, beta, smooth = state["chosen"], state["rejected"], case["beta"], case["smoothing"]
    margin = s if state["reference"] is None else s - state["reference"]
    diff = margin[c] - margin[j]
    if case["kind"] == "logistic":
        z = beta * diff
        loss = torch.clamp_min(-z, 0.0) + torch.log1p(torch.exp(-z.abs())) + smooth * z
        slope = beta * (smooth - 1.0 / (1.0 + torch.exp(z)))
    else:
        off = diff - 1.0 / (2.0 * beta)
        loss, slope = off * off, 2.0 * off
    if state["weight"] is not None:
        loss, slope = loss * state["weight"], slope * state["weight"]
    scale = 1.0 / state["total_weight"] if case["reduction"] == "mean" else 1.0
    grad = torch.zeros(case["rows"], device=s.device, dtype=torch.float64)
    slope = slope.double()
    grad.index_add_(0, c, slope)
    grad.index_add_(0, j, slope, alpha=-1.0)
    return (loss.double().sum() * scale).float(), (grad * scale).to(state["scores"].dtype)


def _plain_log_probs(s, group, groups):
    top = torch.full((groups,), -math.inf, device=s.device, dtype=s.dtype).scatter_reduce_(0, group, s, "amax")
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    total = torch.zeros(groups, device=s.device, dtype=s.dtype).index_add_(0, group, torch.exp(s - top[group]))
    log_total = torch.where(total > 0, top + torch.log(total), torch.zeros_like(total))
    return s - log_total[group]


def _plain_choice(state):
    case, s, group, groups, t = state["case"], state["scores"].float(), state["group"], state["case"]["groups"], state["target"]
    logp = _plain_log_probs(s, group, groups)
    mass = torch.zeros(groups, device=s.device, dtype=s.dtype).index_add_(0, group, t)
    scale = 1.0 / groups if case["reduction"] == "mean" else 1.0
    loss = torch.where(t > 0, -t * logp, torch.zeros_like(t)).double().sum() * scale
    grad = (torch.exp(logp) * mass[group] - t) * scale
    return loss.float(), grad.to(state["scores"].dtype)


def _plain_policy(state):
    # in 64 bits: whether a ratio is beyond its border, and differences of nearly equal log-probabilities
    case, s, group, groups = state["case"], state["scores"].double(), state["group"], state["case"]["groups"]
    live = s > -math.inf
    logp = _plain_log_probs(s, group, groups)
    p = torch.exp(logp)
    zero = torch.zeros_like(s)
    adv = torch.where(live, state["advantage"].double(), zero)
    taken = adv != 0
    ratio = torch.exp(torch.where(taken, logp - state["old"].double(), zero))
    beyond = torch.where(adv > 0, ratio > 1.0 + case["high"], ratio < 1.0 - case["low"]) & taken
    bound = torch.where(adv > 0, 1.0 + case["high"], 1.0 - case["low"])
    policy = -adv * torch.where(beyond, bound, ratio)
    slope = torch.where(beyond, zero, -adv * ratio)
    scale = 1.0 / groups if case["reduction"] == "mean" else 1.0
    grad = slope - p * torch.zeros(groups, device=s.device, dtype=s.dtype).index_add_(0, group, slope)[group]
    loss, kl = policy.sum(), zero.sum()
    if state["reference"] is not None:
        gap = torch.where(live, logp - state["reference"].double(), zero)
        per_group = torch.zeros(groups, device=s.device, dtype=s.dtype).index_add_(0, group, p * gap)
        kl = per_group.sum()
        loss = loss + case["kl"] * kl
        grad = grad + case["kl"] * p * (gap - per_group[group])
    return (loss * scale).float(), (grad * scale).to(state["scores"].dtype), (kl * scale).float(), beyond.sum()


def run(state):
    if own:
        return tuple(_run_own(state)) if state["case"]["op"] != "log_probs" else _run_own(state)
    op = state["case"]["op"]
    if op == "preference":
        return _plain_preference(state)
    if op == "choice":
        return _plain_choice(state)
    if op == "policy":
        return _plain_policy(state)
    logp = _plain_log_probs(state["scores"].float(), state["group"], state["case"]["groups"])
    return logp.to(state["scores"].dtype)


def work(case):
    n, t = case["rows"], 2 if case["type"] != "fp32" else 4
    if case["op"] == "preference":
        per_pair = 8 + 4 * case["weighted"]
        return {"bytes": n * (2 * t + 4 * case["reference"]) + case["pairs"] * per_pair, "flops": 24 * case["pairs"]}
    inputs = {"choice": 4, "policy": 8 + 4 * case["reference"], "log_probs": 0}[case["op"]]
    return {"bytes": n * (2 * t + inputs + 4 * case["mixed"]) + 4 * case["groups"],
            "flops": n * {"choice": 16, "policy": 40, "log_probs": 12}[case["op"]]}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    d = {k: None if v is None else (v.double() if v.is_floating_point() else v).cpu().numpy() for k, v in _inputs(case, seed).items()}
    s = d["scores"]
    if case["op"] == "preference":
        c, j = d["chosen"], d["rejected"]
        r = d["reference"] if d["reference"] is not None else np.zeros_like(s)
        w = d["weight"] if d["weight"] is not None else np.ones(len(c))
        delta = (s[c] - r[c]) - (s[j] - r[j])
        if case["kind"] == "logistic":
            z, e = case["beta"] * delta, case["smoothing"]
            loss = (1 - e) * np.logaddexp(0.0, -z) + e * np.logaddexp(0.0, z)
            sig = np.where(z >= 0, 1.0 / (1.0 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1.0 + np.exp(-np.abs(z))))
            miss = np.where(z >= 0, np.exp(-np.abs(z)) / (1.0 + np.exp(-np.abs(z))), 1.0 / (1.0 + np.exp(-np.abs(z))))
            slope = case["beta"] * (e * sig - (1 - e) * miss)
        else:
            tau = 0.5 / case["beta"]
            loss, slope = np.square(delta - tau), 2 * (delta - tau)
        norm = w.sum() if case["reduction"] == "mean" else 1.0
        grad = np.bincount(c, weights=w * slope, minlength=len(s)) - np.bincount(j, weights=w * slope, minlength=len(s))
        return np.float64(np.sum(w * loss) / norm), grad / norm
    n_groups, order = case["groups"], np.argsort(d["group"], kind="stable")
    g = d["group"][order]
    starts = np.flatnonzero(np.r_[True, g[1:] != g[:-1]])
    sizes = np.diff(np.r_[starts, len(g)])

    def per_row(v):
        return np.repeat(v, sizes)

    s = s[order]
    top = np.maximum.reduceat(s, starts)
    top = np.where(np.isinf(top), 0.0, top)
    with np.errstate(divide="ignore"):
        lse = top + np.log(np.add.reduceat(np.exp(s - per_row(top)), starts))
    lse = np.where(np.isinf(lse), 0.0, lse)
    logp = s - per_row(lse)
    p, live = np.exp(logp), s > -np.inf
    norm = n_groups if case["reduction"] == "mean" else 1

    def back(v):
        out = np.empty_like(v)
        out[order] = v
        return out

    if case["op"] == "log_probs":
        return back(logp)
    if case["op"] == "choice":
        t = d["target"][order]
        on = t > 0
        loss = -np.sum(t[on] * logp[on])
        return np.float64(loss / norm), back((p * per_row(np.add.reduceat(t, starts)) - t) / norm)
    adv = np.where(live, d["advantage"][order], 0.0)
    on = adv != 0
    ratio = np.ones_like(s)
    ratio[on] = np.exp(logp[on] - d["old"][order][on])
    clipped = np.clip(ratio, 1 - case["low"], 1 + case["high"])
    loss = -np.sum(np.minimum(ratio * adv, clipped * adv))
    flat = on & (clipped * adv < ratio * adv)
    slope = np.where(flat, 0.0, -adv * ratio)
    grad = slope - p * per_row(np.add.reduceat(slope, starts))
    kl = 0.0
    if d["reference"] is not None:
        gap = np.zeros_like(s)
        gap[live] = logp[live] - d["reference"][order][live]
        each = np.add.reduceat(p * gap, starts)
        kl = each.sum()
        grad = grad + case["kl"] * p * (gap - per_row(each))
        loss = loss + case["kl"] * kl
    return np.float64(loss / norm), back(grad / norm), np.float64(kl / norm), int(flat.sum())
