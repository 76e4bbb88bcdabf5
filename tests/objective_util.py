"""The objectives from their definitions in float64 numpy, and how far a float32 kernel may be off.

Bounds count roundings.  u = 2^-24 is half a step of float32 relative to the value; the GPU's 2^x is documented with 2 ulp
(4 u) and its 1 / x with 1 ulp (2 u).  Each function returns values and bounds of the same shape; the bounds of
gradients do not hold the rounding to the scores' type, which `assert_close` adds (half a step, or half the smallest
number of the type)."""

import numpy as np
import torch

U = 2.0 ** -24


def pair_loss(scores, chosen, rejected, *, weight=None, reference=None, beta=1.0, smoothing=0.0, kind="logistic",
              reduction="sum"):
    s = np.asarray(scores, np.float64)
    c, j = np.asarray(chosen, np.int64), np.asarray(rejected, np.int64)
    w = np.ones(len(c)) if weight is None else np.asarray(weight, np.float32).astype(np.float64)
    r = np.zeros(len(s)) if reference is None else np.asarray(reference, np.float64)
    step, off = s[c] - s[j], r[c] - r[j]
    d = step - off
    # the difference of scores, the offset in 32 bits, and their difference: a rounding each
    err_d = U * (np.abs(step) + np.abs(off) + np.abs(d) * 2)
    if kind == "logistic":
        z = beta * d
        err_z = beta * err_d + 2 * U * np.abs(z)             # beta and the product
        loss = (1 - smoothing) * np.logaddexp(0, -z) + smoothing * np.logaddexp(0, z)
        slope = beta * (smoothing - 1 / (1 + np.exp(np.clip(z, -700, 700))))
        # sigmoid has a slope of at most 1/4; 2^x 4 u of a value whose share of 1 + 2^x is below 1, sum, 1 / x,
        # difference, product, beta and smoothing in 32 bits
        err_s = beta * (err_z / 4 + 12 * U)
        err_l = err_z + 12 * U * (1 + np.abs(loss))
    else:
        tau = 0.5 / beta
        loss, slope = (d - tau) ** 2, 2 * (d - tau)
        err_o = err_d + 2 * U * (np.abs(d) + tau)
        err_s, err_l = 2 * err_o, 2 * np.abs(d - tau) * err_o + err_o ** 2 + 2 * U * loss
    norm = 1.0 if reduction == "sum" else 1.0 / w.sum()
    n = len(s)
    grad = np.bincount(c, w * slope, n) - np.bincount(j, w * slope, n)
    size = np.bincount(c, w * np.abs(slope), n) + np.bincount(j, w * np.abs(slope), n)
    err = np.bincount(c, w * err_s, n) + np.bincount(j, w * err_s, n)
    # weight times slope, eight terms of a thread in 32 bits at most (sums across threads have 64), scale
    err_g = err + 11 * U * size + 2 * U * np.abs(grad)
    total = (w * loss).sum()
    err_t = (w * err_l).sum() + 11 * U * (w * np.abs(loss)).sum() + U * abs(total)
    return total * norm, grad * norm, err_t * norm, err_g * norm


def _by_group(group, n_groups):
    group = np.asarray(group, np.int64)

    def total(v):
        return np.bincount(group, v, n_groups)[group]

    return group, total


def log_probs(scores, group, n_groups):
    s = np.asarray(scores, np.float64)
    group, total = _by_group(group, n_groups)
    top = np.full(n_groups, -np.inf)
    np.maximum.at(top, group, s)
    top = np.where(np.isinf(top), 0.0, top)[group]
    z = total(np.exp(s - top))
    with np.errstate(divide="ignore"):
        lse = top + np.log(z)
    return s - np.where(np.isneginf(lse), 0.0, lse)


def choice(scores, group, n_groups, target, reduction="sum"):
    l = log_probs(scores, group, n_groups)
    group, total = _by_group(group, n_groups)
    t = np.asarray(target, np.float32).astype(np.float64)
    norm = 1.0 if reduction == "sum" else 1.0 / n_groups
    on = t != 0
    loss = -(t[on] * l[on]).sum()
    p, mass = np.exp(l), total(t)
    grad = p * mass - t
    # p: 2^x and the correction of its argument; the group's sum in 32 bits; product, difference, scale
    err_g = 10 * U * p * mass + 3 * U * np.abs(grad)
    return loss * norm, grad * norm, 2 * U * abs(loss * norm) + 1e-12 * np.abs(t[on] * l[on]).sum() * norm, err_g * norm


def policy(scores, group, n_groups, advantage, old, reference=None, clip=(0.2, 0.2), kl_coef=0.0, reduction="sum"):
    s = np.asarray(scores, np.float64)
    l = log_probs(s, group, n_groups)
    group, total = _by_group(group, n_groups)
    live = s != -np.inf
    a = np.where(live, np.asarray(advantage, np.float32).astype(np.float64), 0.0)
    on = a != 0
    x = np.zeros_like(s)
    x[on] = l[on] - np.asarray(old, np.float32).astype(np.float64)[on]
    with np.errstate(over="ignore"):
        ratio = np.exp(x)
    beyond = on & np.where(a > 0, ratio > 1 + clip[1], ratio < 1 - clip[0])
    bound = np.where(a > 0, 1 + clip[1], 1 - clip[0])
    each = np.where(on, -a * np.where(beyond, bound, ratio), 0.0)
    slope = np.where(on & ~beyond, each, 0.0)
    p = np.exp(l)
    h, size = total(slope), total(np.abs(slope))
    loss, kl, grad = each.sum(), 0.0, slope - p * h
    err_kl_row = np.zeros_like(s)
    gap, kl_group = np.zeros_like(s), np.zeros_like(s)
    if reference is not None:
        gap[live] = l[live] - np.asarray(reference, np.float32).astype(np.float64)[live]
        kl_group, err_kl_row = total(p * gap), 8 * U * total(p * np.abs(gap))
        kl = (p * gap).sum()
        grad = grad + kl_coef * p * (gap - kl_group)
    norm = 1.0 if reduction == "sum" else 1.0 / n_groups
    inner = np.abs(kl_coef * (gap - kl_group) - h)
    # ratio: 2^x (4 u), correction, product with the advantage; the sum in brackets rounded once to 32 bits;
    # p as above, product, sum, scale
    err_g = 8 * U * np.abs(slope) + p * (8 * U * size + abs(kl_coef) * err_kl_row + 10 * U * inner) + 4 * U * np.abs(grad)
    err_kl = 8 * U * (p * np.abs(gap)).sum() + 2 * U * abs(kl)
    err_t = 8 * U * np.abs(each).sum() + abs(kl_coef) * err_kl + 2 * U * abs(loss + kl_coef * kl)
    return ((loss + kl_coef * kl) * norm, grad * norm, kl * norm, int(beyond.sum()), err_t * norm, err_g * norm,
            err_kl * norm)


def assert_close(got: torch.Tensor, want, bound):
    info = torch.finfo(got.dtype)
    got = got.detach().double().cpu().numpy()
    want, bound = np.asarray(want, np.float64), np.asarray(bound, np.float64)
    # a number beyond the type's largest rounds to infinity
    want = np.where(np.abs(want) - bound > info.max * (1 + info.eps / 4), np.copysign(np.inf, want), want)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    step = info.smallest_normal * info.eps
    room = bound + (np.abs(want) + bound) * info.eps / 2 + step
    off = np.abs(got[finite] - want[finite])
    worst = np.argmax(off / room[finite]) if off.size else 0
    assert not off.size or (off <= room[finite]).all(), (
        f"{(off > room[finite]).sum()} of {off.size} off, the worst {off[worst]} with {room[finite][worst]} allowed "
        f"at {want[finite][worst]}")
