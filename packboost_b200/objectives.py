"""Losses on the scores of rows, each with its gradient, and the objectives that ``PackBoost.fit`` takes.

The booster's own loss is half the squared difference to a target.  The ones here are those a model of scores
is trained on after or instead of that: which of two rows was preferred, which rows of a group were chosen, and
what a policy that chooses among the rows of a group earned.  All are differentiated with respect to the
scores; hessians are 1, as everywhere in the booster, so a leaf's value is the mean of its rows' negative
gradients (with ``lambda_l2``).

As operators on CUDA tensors::

    pairs = RowPairs(chosen, rejected, n_rows, reference=reference_scores)     # laid out once
    loss, grad = preference_loss(scores, pairs, beta=0.1)
    groups = RowGroups(group_of_row)
    loss, grad = choice_loss(scores, groups, target)
    loss, grad, kl, clipped = policy_loss(scores, groups, advantage, old_log_probs,
                                          reference_log_probs=reference, kl_coef=0.05)
    log_probs = group_log_probs(scores, groups)

and as what a fit learns from::

    booster.fit(X, None, era, num_rounds=100, objective=PreferenceObjective(chosen, rejected, beta=1.0))

Scores are float32, float16 or bfloat16 and gradients have their type; sums are held in 64 bits, of up to eight terms
each in 32, in an order that does not change from run to run.  The log of a group's sum of exponentials is one
64-bit number: scores of a group beyond some 1e9 lose digits of their probabilities, and a group whose rows all
have the type's lowest number has none; what masks a row is -inf.  The results are not attached to an
autograd graph: the gradient is there already.  Calls only enqueue work on the current stream of the scores'
device and may be captured into a CUDA graph; ``RowPairs`` and ``RowGroups`` wait for their own layout, may be
used from any stream, and have to outlive the graphs that use them.  A layout takes 0.4 to 2 ms (millions of
pairs: up to 5), what some 1 to 10 evaluations save against the same losses in torch operations: it is for sets
that are evaluated many times.

In a fit, ``reduction="mean"`` divides the gradients by the number of pairs or groups while hessians stay 1, so
leaves shrink by as much and the model hardly moves: ``"sum"`` is what a learning rate of usual size goes with.
"""

from __future__ import annotations

import ctypes as C
import threading
from typing import NamedTuple

import numpy as np
import torch

from . import backends as B


def _quick(name: str, public):
    """torch's own binding behind a public function (a call of ten microseconds notices the rest), or that function."""
    return getattr(torch._C, name, None) or public


_device_now = _quick("_cuda_getDevice", torch.cuda.current_device)
_stream_now = _quick("_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)
_capturing = _quick("_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)

_SCORE_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MOST = (1 << 31) - (1 << 16)    # rows, and items (two per pair): 32-bit numbers
_PREFERENCE, _CHOICE, _POLICY = 0, 1, 2


class LossAndGradient(NamedTuple):
    loss: torch.Tensor       # float32, no dimensions
    grad: torch.Tensor       # like the scores


class PolicyLoss(NamedTuple):
    loss: torch.Tensor       # float32, no dimensions
    grad: torch.Tensor       # like the scores
    kl: torch.Tensor         # float32, no dimensions: divergence from the reference, reduced like the loss
    clipped: torch.Tensor    # int64, no dimensions: taken rows whose ratio is beyond its border


# ---- arguments -----------------------------------------------------------------------------------


def _indices(values, name: str) -> torch.Tensor:
    t = values.detach() if isinstance(values, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(np.asarray(values)))
    if t.numel() == 0 and not isinstance(values, torch.Tensor):
        t = t.to(torch.int64)   # (an empty list has no integer type)
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{name} must hold integers")
    if t.dim() != 1:
        raise ValueError(f"{name} must be 1-D")
    return t.to(torch.int64)


def _numbers(values, name: str, length: int, device) -> torch.Tensor:
    """1-D numbers of a caller, in the type they have."""
    t = values.detach() if isinstance(values, torch.Tensor) else torch.from_numpy(np.array(values, ndmin=1))
    if t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{name} must hold real numbers")
    if t.dim() != 1 or t.shape[0] != length:
        raise ValueError(f"{name} must be 1-D with {length} entries")
    return t.to(device)


def _count(value, name: str) -> int:
    if isinstance(value, bool) or not isinstance(value, (int, np.integer)):
        raise TypeError(f"{name} must be an integer")
    if not 0 <= value <= _MOST:
        raise ValueError(f"{name}={value} outside [0, {_MOST}]")
    return int(value)


def _home(*values, device=None) -> torch.device:
    """Where a layout lives: the given device, that of a CUDA tensor among the values, or the current one."""
    if device is None:
        device = next((v.device for v in values if isinstance(v, torch.Tensor) and v.is_cuda), None)
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError("objectives live on a CUDA device")
    if not B.cuda_available():
        raise RuntimeError("packboost_b200: libpackboost_b200.so is not built or no sm_100 device is visible")
    return torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)


# ---- layouts ---------------------------------------------------------------------------------------


def _check_pairs(chosen, rejected, n_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    chosen, rejected = _indices(chosen, "chosen"), _indices(rejected, "rejected")
    if chosen.shape[0] != rejected.shape[0]:
        raise ValueError("chosen and rejected differ in length")
    if 2 * chosen.shape[0] > _MOST:
        raise ValueError(f"more than {_MOST // 2} pairs")
    rejected = rejected.to(chosen.device)
    if chosen.shape[0]:
        both = torch.cat([chosen, rejected])
        low, high, same = torch.stack([both.min(), both.max(), (chosen == rejected).any().to(torch.int64)]).tolist()
        if low < 0 or high >= n_rows:
            raise ValueError(f"pairs name rows outside [0, {n_rows})")
        if same:
            raise ValueError("a pair compares a row with itself")
    return chosen, rejected


def _check_weight(weight, n_pairs: int, device) -> torch.Tensor:
    weight = _numbers(weight, "weight", n_pairs, device).to(torch.float32)
    if n_pairs and not bool((torch.isfinite(weight) & (weight >= 0)).all()):
        raise ValueError("weights must be finite and not negative")
    return weight


# (the layouts below are the ones of include/packboost_b200.h; they are made by torch, on any device: small ones on the host,
# where a step costs less than a launch)
_SLICE_ROWS, _SLICE_ITEMS, _CHUNK_ITEMS = 64, 32, 512
_WINDOW = 8192   # rows whose order a slice may change: its rows stay near the ones they are compared with
_HOST_PAIRS, _HOST_ROWS = 4096, 32768   # 500 pairs 0.4 ms there and 0.75 on the GPU, 5 000 pairs 1.3 and 0.8; 20 groups of 1 000 rows 0.3 and 0.5


def _lay_out_pairs(chosen, rejected, n_rows, weight, reference) -> dict:
    """The items of every row: by columns of 64 rows with equally many, in chunks where there are many."""
    dev, n_pairs = chosen.device, chosen.shape[0]
    if n_rows == 0:
        return {}
    # both sides in one: the items of row r that chose it have the owner r, those that rejected it n_rows + r
    owner, other = torch.cat([chosen, rejected + n_rows]), torch.cat([rejected, chosen])
    counts = torch.zeros(2 * n_rows, dtype=torch.int64, device=dev).index_add_(0, owner, torch.ones_like(owner))
    n_chosen, n_rejected = counts[:n_rows], counts[n_rows:]
    few = torch.maximum(n_chosen, n_rejected) <= _SLICE_ITEMS
    all_few = n_pairs == 0 or bool(few.all())
    row = torch.arange(n_rows, device=dev) if all_few else torch.nonzero(few)[:, 0]
    # (by turns up and down: rows on either side of a step differ by one item)
    key_c, key_r = n_chosen[row], n_rejected[row]
    key = ((row // _WINDOW) * (_SLICE_ITEMS + 1) + key_c) * (_SLICE_ITEMS + 1) + torch.where(key_c % 2 == 0, key_r, _SLICE_ITEMS - key_r)
    row = row[torch.sort(key, stable=True).indices]
    n_few = row.shape[0]
    n_slices = -(-n_few // _SLICE_ROWS)
    have = torch.zeros((_SLICE_ROWS * n_slices, 2), dtype=torch.int64, device=dev)
    have[:n_few, 0], have[:n_few, 1] = n_chosen[row], n_rejected[row]
    tall = have.view(n_slices, _SLICE_ROWS, 2).amax(1) if n_slices else have
    column = tall.sum(1).cumsum(0) - tall.sum(1)
    lanes = torch.full((_SLICE_ROWS * n_slices,), -1, dtype=torch.int64, device=dev)
    lanes[:n_few] = row
    out = {"n_slices": n_slices,
           "slices": torch.stack([column, tall[:, 0] | (tall[:, 1] << 16)], 1).to(torch.int32),
           "slice_rows": torch.stack([lanes, have[:, 0] | (have[:, 1] << 16)], 1).to(torch.int32)}
    n_items = _SLICE_ROWS * int(tall.sum())
    # where an item goes: base + stride * its rank among its owner's items
    base = torch.zeros(2 * n_rows, dtype=torch.int64, device=dev)
    at = torch.arange(n_few, device=dev)
    first = column[at // _SLICE_ROWS] * _SLICE_ROWS + at % _SLICE_ROWS
    base[row], base[row + n_rows] = first, first + tall[at // _SLICE_ROWS, 0] * _SLICE_ROWS
    stride = None
    if not all_few:
        many = torch.nonzero(~few)[:, 0]
        size = n_chosen[many] + n_rejected[many]
        begin = n_items + size.cumsum(0) - size
        n_items += int(size.sum())
        stride = torch.where(few, _SLICE_ROWS, 1).repeat(2)
        base[many], base[many + n_rows] = begin, begin + n_chosen[many]
        out.update(_lay_out_chunks(many, n_chosen[many], size, begin))
    if n_items > _MOST:
        raise ValueError("more items than 32-bit numbers count")
    order = _item_order(owner, other, n_rows)
    owner = owner[order]
    rank = torch.arange(2 * n_pairs, device=dev) - (counts.cumsum(0) - counts)[owner]
    place = base[owner] + rank * (_SLICE_ROWS if stride is None else stride[owner])
    out["other"] = torch.zeros(max(n_items, 1), dtype=torch.int32, device=dev)
    out["other"][place] = other[order].to(torch.int32)
    if reference is not None:
        r = reference.to(torch.float64)
        away = (r[chosen] - r[rejected]).to(torch.float32)
        out["offset"] = torch.zeros(max(n_items, 1), dtype=torch.float32, device=dev)
        out["offset"][place] = torch.cat([away, -away])[order]
    if weight is not None:
        out["weight"] = torch.zeros(max(n_items, 1), dtype=torch.float32, device=dev)
        out["weight"][place] = weight.repeat(2)[order]
    return out


def _item_order(owner: torch.Tensor, other: torch.Tensor, n_rows: int) -> torch.Tensor:
    """Items by owner (below 2 n_rows), those of an owner in the order of the other rows: neighbouring items of a row then look
    up neighbouring scores (rows of 670 000 items among 500 000 rows: 25 us with the items as given, 19 so)."""
    # (at most 2 n_rows^2 - 1, which 63 bits hold for all rows that are allowed; two halves of 32 bits would not hold the owner)
    return torch.sort(owner * n_rows + other, stable=True).indices


def _lay_out_chunks(row, n_chosen, size, begin) -> dict:
    """Chunks of rows with ``size`` items from ``begin`` on, of which the first ``n_chosen`` chose the row."""
    n_of = -(-size // _CHUNK_ITEMS)                      # chunks of a row
    which = torch.repeat_interleave(torch.arange(row.shape[0], device=row.device), n_of)
    first = n_of.cumsum(0) - n_of
    step = (torch.arange(which.shape[0], device=row.device) - first[which]) * _CHUNK_ITEMS
    split = (n_of > 1).to(torch.int64)
    count = torch.minimum(size[which] - step, torch.full_like(step, _CHUNK_ITEMS))
    better = (n_chosen[which] - step).clamp(min=0).minimum(count)
    chunks = torch.stack([row[which], begin[which] + step, count, better, (split.cumsum(0) - split)[which], first[which],
                          n_of[which], torch.zeros_like(step)], 1).to(torch.int32)
    return {"n_chunks": which.shape[0], "n_split": int(split.sum()), "chunks": chunks}


def _check_groups(group, n_groups) -> tuple[torch.Tensor, int]:
    group = _indices(group, "group")
    if group.shape[0] > _MOST:
        raise ValueError(f"more than {_MOST} rows")
    low, high = torch.stack([group.min(), group.max()]).tolist() if group.shape[0] else (0, -1)
    n_groups = high + 1 if n_groups is None else _count(n_groups, "n_groups")
    if low < 0 or high >= n_groups:
        raise ValueError(f"group ids outside [0, {n_groups})")
    if n_groups > _MOST:
        raise ValueError(f"more than {_MOST} groups")
    return group, n_groups


_TEAM_ROWS = (8, 16, 32, 64, 128, 256)            # of 1, 2, 4 ... 32 lanes
_BLOCK_ROWS, _PIECE = 8192, 2048


def _lay_out_groups(group: torch.Tensor) -> dict:
    """The rows by group where they are in another order, and the groups by length: teams of lanes for short ones, a CTA, pieces
    of long ones."""
    n, dev = group.shape[0], group.device
    if n == 0:
        return {"n_groups": 0}
    rows = None
    if not bool((group[1:] >= group[:-1]).all()):
        group, order = torch.sort(group, stable=True)
        rows = order.to(torch.int32)
    heads = torch.ones(n, dtype=torch.bool, device=dev)
    heads[1:] = group[1:] != group[:-1]
    starts = torch.nonzero(heads)[:, 0]
    lengths = torch.diff(starts, append=starts.new_full((1,), n))
    # short ones by length (a warp's groups should be alike), a CTA's longest first, long ones in the order of their rows
    limits = torch.tensor(_TEAM_ROWS + (_BLOCK_ROWS,), device=dev)
    kind = torch.bucketize(lengths, limits)
    key = torch.where(kind < len(_TEAM_ROWS), lengths,
                      torch.where(kind == len(_TEAM_ROWS), 2 * _BLOCK_ROWS - lengths, 2 * _BLOCK_ROWS))
    table = torch.stack([starts, lengths], 1).to(torch.int32)[torch.sort(key, stable=True).indices]
    count = torch.bincount(kind, minlength=len(limits) + 1).tolist()
    parts = list(torch.split(table, count))
    teams, warps, entry = [], [], 0
    for c in range(len(_TEAM_ROWS)):
        n_warps = -(-count[c] // (32 >> c))
        if n_warps == 0:
            continue
        own = torch.cat([parts[c], table.new_zeros((n_warps * (32 >> c) - count[c], 2))]).view(n_warps, 32 >> c, 2)
        most = (own[:, :, 1].amax(1) + (1 << c) - 1) >> c
        first = entry + torch.arange(n_warps, device=dev) * (32 >> c)
        warps.append(torch.stack([first, c | (most << 8)], 1).to(torch.int32))
        teams.append(own.view(-1, 2))
        entry += n_warps * (32 >> c)
    none = table.new_zeros((0, 2))
    out = {"rows": rows, "n_groups": starts.shape[0], "teams": torch.cat(teams or [none]),
           "team_warps": torch.cat(warps or [none]).flip(0),     # (the warps with most to do first)
           "n_blocks": count[6], "blocks": parts[6], "block_rows": int(parts[6][:, 1].max()) if count[6] else 0}
    out["n_team_warps"] = out["team_warps"].shape[0]
    begin, length = parts[7].cpu().numpy().astype(np.int64).T
    n_of = -(-length // _PIECE)
    first = np.cumsum(n_of) - n_of
    which = np.repeat(np.arange(len(n_of)), n_of)
    step = (np.arange(len(which)) - first[which]) * _PIECE
    pieces = np.stack([begin[which] + step, np.minimum(length[which] - step, _PIECE), first[which], n_of[which]], 1)
    out["n_pieces"] = len(which)
    out["pieces"] = torch.from_numpy(pieces.astype(np.int32)).to(dev)
    return out


class _Layout:
    """Tensors on one device that calls from any stream may read, and the structure that points at them."""

    def _point(self, struct: type, tables: dict, **numbers):
        fields = dict(numbers)
        for name, _ in struct._fields_:
            v = tables.get(name)
            if v is not None:
                fields[name] = (v.data_ptr() or None) if isinstance(v, torch.Tensor) else v
        return struct(**fields)

    def _settle(self, device: torch.device, tensors: dict) -> None:
        for name, t in tensors.items():   # (of a layout made on the host)
            if isinstance(t, torch.Tensor):
                tensors[name] = t.to(device)
        self.device = device
        self._tensors = [t for t in tensors.values() if isinstance(t, torch.Tensor)]
        self._structs: dict = {}   # descriptors of objectives on this layout, by their options
        self._rooms: dict = {}     # scratch of evaluations, by thread and stream
        self._scratch_bytes = 0
        # (empty_like of these takes half as long as empty, which has more to look at)
        self._number = torch.empty((), dtype=torch.float32, device=device)
        self._count = torch.empty((), dtype=torch.int64, device=device)
        stream = torch.cuda.current_stream(device)
        self._stream = stream.cuda_stream
        self._streams = {self._stream}
        stream.synchronize()

    def _used_now(self) -> int:
        """The current stream of the layout's device, which must be the current one."""
        stream = _stream_now(self.device.index)
        if stream not in self._streams:
            if len(self._streams) >= 64:
                self._streams = {self._stream}
            current = torch.cuda.current_stream()
            for t in self._tensors:   # (once for a stream: what counts is where it stands when they are freed)
                t.record_stream(current)
            self._streams.add(stream)
        return stream

    def _room(self, stream: int) -> torch.Tensor:
        """Scratch that no other evaluation uses at the same time: one per thread and stream, which a call leaves as the
        next needs it.  A captured call has its own, since its graph may run beside anything."""
        if not _capturing():
            room = self._rooms.get((threading.get_ident(), stream))
            if room is not None:
                return room
            if len(self._rooms) >= 16:
                self._rooms = {}
        room = torch.zeros(self._scratch_bytes, dtype=torch.uint8, device=self.device)
        if not _capturing():
            self._rooms[threading.get_ident(), stream] = room
        return room


class RowPairs(_Layout):
    """Pairs of rows, the first preferred to the second, laid out for :func:`preference_loss`.

    ``weight`` counts a pair so many times (its product with the pair's loss or slope is a float32);
    ``reference`` holds the scores of a reference model for all rows (those of compared rows finite; what two
    rows differ by is kept as a float32, as the difference of their scores is), so that differences of scores
    become differences of log ratios: where the scores are log-probabilities, or differ from them by something
    the two rows share, that is the paired log
    ratio of the model to the reference.  A pair may occur more than once; a row is not compared with itself."""

    def __init__(self, chosen, rejected, n_rows: int, *, weight=None, reference=None, device=None) -> None:
        n_rows = _count(n_rows, "n_rows")
        c, r = _check_pairs(chosen, rejected, n_rows)
        if weight is not None:
            weight = _check_weight(weight, c.shape[0], c.device)
        if reference is not None:
            reference = _numbers(reference, "reference", n_rows, c.device)
        home = _home(chosen, rejected, weight, reference, device=device)
        where = torch.device("cpu") if 2 * c.shape[0] + n_rows <= _HOST_PAIRS else home
        with torch.cuda.device(home):
            parts = _lay_out_pairs(c.to(where), r.to(where), n_rows, None if weight is None else weight.to(where),
                                   None if reference is None else reference.to(where))
            if parts.get("offset") is not None and not bool(torch.isfinite(parts["offset"]).all()):
                raise ValueError("reference scores of compared rows must be finite")
            self.n_rows, self.n_pairs = n_rows, int(c.shape[0])
            self.total_weight = float(self.n_pairs) if weight is None else float(weight.to(torch.float64).sum())
            self._settle(home, parts)
        self._struct = self._point(B.Pairs, parts, n_rows=n_rows)


class RowGroups(_Layout):
    """Groups of rows (the candidates among which one chooses, the rows of an era), laid out for
    :func:`choice_loss`, :func:`policy_loss` and :func:`group_log_probs`.  ``group`` holds the group id of
    every row, in any order; groups without rows are allowed and count in means (``n_groups``, by default one
    more than the largest id)."""

    def __init__(self, group, n_groups: int | None = None, *, device=None) -> None:
        g, n_groups = _check_groups(group, n_groups)
        home = _home(group, device=device)
        with torch.cuda.device(home):
            parts = _lay_out_groups(g.to("cpu" if g.shape[0] <= _HOST_ROWS else home))
            self.n_rows, self.n_groups = int(g.shape[0]), n_groups
            self._settle(home, parts)
        self._struct = self._point(B.Groups, parts, n_rows=self.n_rows)
        self._log_probs_bytes: int | None = None


# ---- operators --------------------------------------------------------------------------------------


def _check_scores(scores, layout) -> torch.Tensor:
    if not isinstance(scores, torch.Tensor) or scores.dtype not in _SCORE_TYPES:
        raise TypeError("scores must be a float32, float16 or bfloat16 tensor")
    if scores.device != layout.device:
        raise ValueError(f"scores are on {scores.device}, the layout on {layout.device}")
    if scores.dim() != 1 or scores.shape[0] != layout.n_rows:
        raise ValueError(f"scores must be 1-D with {layout.n_rows} entries")
    return scores if scores.is_contiguous() else scores.detach().contiguous()


def _per_row(values, name: str, layout) -> torch.Tensor:
    if not isinstance(values, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if values.device != layout.device:
        raise ValueError(f"{name} is on {values.device}, the layout on {layout.device}")
    if values.dtype == torch.float32 and values.dim() == 1 and values.shape[0] == layout.n_rows and values.is_contiguous():
        return values
    return _numbers(values, name, layout.n_rows, layout.device).to(torch.float32).contiguous()


def _scale(reduction: str, total: float, what: str) -> float:
    if reduction == "sum":
        return 1.0
    if reduction != "mean":
        raise ValueError(f"unknown reduction {reduction!r}")
    if not total > 0:
        raise ValueError(f"the mean over no {what} is not defined")
    return 1.0 / total


def _preference_struct(pairs: RowPairs, beta, label_smoothing, kind, reduction) -> B.Objective:
    beta, smoothing = float(beta), float(label_smoothing)
    options = (beta, smoothing, kind, reduction)
    kept = pairs._structs.get(options)
    if kept is not None:
        return kept
    if not 1e-30 <= beta <= 1e30:
        raise ValueError("beta must be positive, and between 1e-30 and 1e30")
    if not 0 <= smoothing < 0.5:
        raise ValueError("label_smoothing outside [0, 0.5)")
    if kind not in ("logistic", "squared"):
        raise ValueError(f"unknown kind {kind!r}")
    if kind == "squared" and smoothing:
        raise ValueError("the squared form has no label smoothing")
    if kind == "squared" and beta < 1e-15:
        raise ValueError("beta of the squared form below 1e-15: float32 does not hold the square of 1 / (2 beta)")
    struct = B.Objective(kind=_PREFERENCE, pairs=C.pointer(pairs._struct), beta=beta, smoothing=smoothing,
                         squared=int(kind == "squared"), scale=_scale(reduction, pairs.total_weight, "pairs"))
    return _kept_struct(pairs, options, struct)


def _choice_struct(groups: RowGroups, target: torch.Tensor, reduction) -> B.Objective:
    options = (_CHOICE, reduction)
    kept = groups._structs.get(options)
    if kept is None:
        kept = _kept_struct(groups, options, B.Objective(kind=_CHOICE, groups=C.pointer(groups._struct), target=16,
                                                         scale=_scale(reduction, groups.n_groups, "groups")))
    struct = B.Objective.from_buffer_copy(kept)
    struct.target = target.data_ptr()
    return struct


def _policy_struct(groups: RowGroups, advantage, old, reference, clip, kl_coef, reduction) -> B.Objective:
    low, high = clip
    low, high, kl = float(low), float(high), float(kl_coef)
    options = (_POLICY, low, high, kl, reduction)
    kept = groups._structs.get(options)
    if kept is None:
        if not (0 <= low <= 1 and high >= 0):
            raise ValueError("clip must be (low, high) with low in [0, 1] and high not negative")
        if not abs(kl) <= 1e30:
            raise ValueError("kl_coef must be finite, and at most 1e30")
        kept = _kept_struct(groups, options, B.Objective(
            kind=_POLICY, groups=C.pointer(groups._struct), advantage=16, old=16, reference=16, clip_low=low, clip_high=high,
            kl_coef=kl, scale=_scale(reduction, groups.n_groups, "groups")))
    if reference is None and kl:
        raise ValueError("kl_coef needs reference_log_probs")
    struct = B.Objective.from_buffer_copy(kept)
    struct.advantage, struct.old = advantage.data_ptr(), old.data_ptr()
    struct.reference = None if reference is None else reference.data_ptr()
    return struct


def _kept_struct(layout: _Layout, options: tuple, struct: B.Objective) -> B.Objective:
    """Keeps a descriptor (with addresses of rows still to be put in) and the size of its scratch."""
    nbytes = int(B.lib().pb_objective_workspace_bytes(C.byref(struct)))
    if nbytes < 0:
        B.check(nbytes)
    layout._scratch_bytes = nbytes    # (the layout alone decides it)
    if len(layout._structs) >= 64:    # (options that change from call to call: start again)
        layout._structs = {}
    layout._structs[options] = struct
    return struct


def _evaluate(struct: B.Objective, layout: _Layout, scores: torch.Tensor, policy: bool = False):
    if _device_now() != layout.device.index:
        with torch.cuda.device(layout.device):
            return _evaluate(struct, layout, scores, policy)
    stream = layout._used_now()
    room = layout._room(stream)
    grad, loss = torch.empty_like(scores), torch.empty_like(layout._number)
    if policy:
        kl, clipped = torch.empty_like(layout._number), torch.empty_like(layout._count)
        rc = B.lib().pb_objective_evaluate(struct, scores.data_ptr(), _SCORE_TYPES[scores.dtype], grad.data_ptr(), loss.data_ptr(),
                                           kl.data_ptr(), clipped.data_ptr(), room.data_ptr(), layout._scratch_bytes, stream)
    else:
        rc = B.lib().pb_objective_evaluate(struct, scores.data_ptr(), _SCORE_TYPES[scores.dtype], grad.data_ptr(), loss.data_ptr(),
                                           None, None, room.data_ptr(), layout._scratch_bytes, stream)
    if rc:
        layout._rooms = {}    # (a call that broke off may not have left its scratch in order)
        B.check(rc)
    return PolicyLoss(loss, grad, kl, clipped) if policy else LossAndGradient(loss, grad)


def preference_loss(scores: torch.Tensor, pairs: RowPairs, *, beta: float = 1.0, label_smoothing: float = 0.0,
                    kind: str = "logistic", reduction: str = "sum") -> LossAndGradient:
    """Loss of paired log ratios and its gradient with respect to the scores.

    With ``d = (s_c - r_c) - (s_j - r_j)`` for a pair of chosen row c and rejected row j (r: the reference
    scores, or 0), a pair costs, times its weight,

    * ``"logistic"``: ``-(1 - e) log sigmoid(beta d) - e log sigmoid(-beta d)``, e the label smoothing: the
      share of pairs taken to be the wrong way round;
    * ``"squared"``: ``(d - 1 / (2 beta))^2``.

    ``reduction``: ``"sum"``, or ``"mean"`` over the weights.  Rows in no pair get the gradient 0."""
    struct = _preference_struct(pairs, beta, label_smoothing, kind, reduction)
    return _evaluate(struct, pairs, _check_scores(scores, pairs))


def choice_loss(scores: torch.Tensor, groups: RowGroups, target: torch.Tensor, *, reduction: str = "sum") -> LossAndGradient:
    """Negative log-likelihood ``-sum_i target_i l_i`` of targets under the softmax of each group,
    ``l = s - log sum exp s``, and its gradient ``exp(l_i) T - target_i`` with T the group's sum of targets.

    A target is 1 for a chosen row, or any share that is not negative; groups without one contribute nothing.
    A row with the score -inf has the probability 0 (a target on it makes the loss infinite).  ``reduction``:
    ``"sum"``, or ``"mean"`` over the groups."""
    target = _per_row(target, "target", groups)
    struct = _choice_struct(groups, target, reduction)
    return _evaluate(struct, groups, _check_scores(scores, groups))


def policy_loss(scores: torch.Tensor, groups: RowGroups, advantage: torch.Tensor, old_log_probs: torch.Tensor, *,
                reference_log_probs: torch.Tensor | None = None, clip: tuple[float, float] = (0.2, 0.2),
                kl_coef: float = 0.0, reduction: str = "sum") -> PolicyLoss:
    """Clipped policy loss of the softmax over each group, with the divergence from a reference policy.

    Rows with an advantage that is not 0 are the ones an earlier policy took.  With l the log-probability of a
    row and ``q = exp(l - old)``, such a row costs ``-min(q A, clamp(q, 1 - low, 1 + high) A)``; its gradient
    is cut off where the clamped ratio is the smaller of the two.  A group costs ``kl_coef`` times
    ``sum_i exp(l_i) (l_i - reference_i)``, over all its rows.

    A row with the score -inf is masked: its probability is 0, its gradient is 0, and whatever else is given
    for it is not looked at; neither is the old log-probability of a row that was not taken.  A ratio that
    float32 does not hold (``l - old`` above 88.7, where it is not cut off) is infinite, and with it the loss
    and the gradients of the group's rows.  ``reduction``: ``"sum"``, or ``"mean"`` over the groups."""
    advantage = _per_row(advantage, "advantage", groups)
    old = _per_row(old_log_probs, "old_log_probs", groups)
    reference = None if reference_log_probs is None else _per_row(reference_log_probs, "reference_log_probs", groups)
    struct = _policy_struct(groups, advantage, old, reference, clip, kl_coef, reduction)
    return _evaluate(struct, groups, _check_scores(scores, groups), policy=True)


def group_log_probs(scores: torch.Tensor, groups: RowGroups) -> torch.Tensor:
    """``s - log sum exp s`` over each row's group, in the scores' type; -inf where the score is."""
    scores = _check_scores(scores, groups)
    if _device_now() != groups.device.index:
        with torch.cuda.device(groups.device):
            return group_log_probs(scores, groups)
    lib, stream = B.lib(), groups._used_now()
    out = torch.empty_like(scores)
    if groups._log_probs_bytes is None:
        groups._log_probs_bytes = int(lib.pb_group_log_probs_bytes(groups._struct))
    nbytes = groups._log_probs_bytes
    # (held until the launches are enqueued: given back before, it could be another thread's by then)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=groups.device) if nbytes else None
    B.check(lib.pb_group_log_probs(groups._struct, scores.data_ptr(), _SCORE_TYPES[scores.dtype], out.data_ptr(),
                                   scratch.data_ptr() if nbytes else None, nbytes, stream))
    return out


# ---- what a fit learns from --------------------------------------------------------------------------


class _FitObjective:
    """An objective on the rows of a fit, in the order in which the trainer holds them."""

    def __init__(self, struct: B.Objective, layout: _Layout, kept: tuple) -> None:
        self.struct, self.layout, self._kept = struct, layout, kept
        self.workspace = torch.zeros(layout._scratch_bytes, dtype=torch.uint8, device=layout.device)

    def loss(self, preds: torch.Tensor) -> float:
        return float(_evaluate(self.struct, self.layout, preds).loss)


def _trainer_groups(group, n_rows: int, era_offsets: np.ndarray, order, device) -> RowGroups:
    """Groups of a fit: the given ones, or the eras."""
    if group is None:
        n = len(era_offsets) - 1
        return RowGroups(np.repeat(np.arange(n), np.diff(era_offsets)), n, device=device)
    group, n_groups = _check_groups(group, None)
    if group.shape[0] != n_rows:
        raise ValueError("group must align with X rows")
    return RowGroups(group if order is None else group[torch.from_numpy(order).to(group.device)], n_groups, device=device)


def _trainer_rows(values, name: str, n_rows: int, order, device, where: torch.Tensor | None = None) -> torch.Tensor:
    """A row's number of a fit, in the trainer's order; finite (``where`` it is looked at: no score of a fit is masked)."""
    values = _numbers(values, name, n_rows, device).to(torch.float32).contiguous()
    if order is not None:
        values = values[torch.from_numpy(order).to(device)]
    if not bool((torch.isfinite(values) if where is None else torch.isfinite(values) | ~where).all()):
        raise ValueError(f"{name} must be finite")
    return values


class PreferenceObjective:
    """``fit(..., objective=...)``: :func:`preference_loss` of the rows of X, whose numbers the pairs hold.  A ``"mean"`` makes
    leaves smaller by the sum of the weights (hessians are 1): the learning rate has to make up for it."""

    def __init__(self, chosen, rejected, *, weight=None, reference=None, beta: float = 1.0, label_smoothing: float = 0.0,
                 kind: str = "logistic", reduction: str = "sum") -> None:
        self.chosen, self.rejected, self.weight, self.reference = chosen, rejected, weight, reference
        self.options = (beta, label_smoothing, kind, reduction)

    def _bind(self, n_rows: int, era_offsets, order, device) -> _FitObjective:
        chosen, rejected = _check_pairs(self.chosen, self.rejected, n_rows)
        reference = self.reference
        if order is not None:
            place = torch.empty(n_rows, dtype=torch.int64)
            place[torch.from_numpy(order)] = torch.arange(n_rows)
            place = place.to(chosen.device)
            chosen, rejected = place[chosen], place[rejected]
            if reference is not None:
                reference = _numbers(reference, "reference", n_rows, device)[torch.from_numpy(order).to(device)]
        pairs = RowPairs(chosen, rejected, n_rows, weight=self.weight, reference=reference, device=device)
        return _FitObjective(_preference_struct(pairs, *self.options), pairs, ())


class ChoiceObjective:
    """``fit(..., objective=...)``: :func:`choice_loss` of the rows of X; ``group=None`` takes the eras.  (A mean: as above.)"""

    def __init__(self, target, *, group=None, reduction: str = "sum") -> None:
        self.target, self.group, self.reduction = target, group, reduction

    def _bind(self, n_rows: int, era_offsets, order, device) -> _FitObjective:
        groups = _trainer_groups(self.group, n_rows, era_offsets, order, device)
        target = _trainer_rows(self.target, "target", n_rows, order, device)
        if bool((target < 0).any()):
            raise ValueError("targets must not be negative")
        return _FitObjective(_choice_struct(groups, target, self.reduction), groups, (target,))


class PolicyObjective:
    """``fit(..., objective=...)``: :func:`policy_loss` of the rows of X; ``group=None`` takes the eras.  (A mean: as above.)"""

    def __init__(self, advantage, old_log_probs, *, group=None, reference_log_probs=None,
                 clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0, reduction: str = "sum") -> None:
        self.advantage, self.old_log_probs, self.reference_log_probs = advantage, old_log_probs, reference_log_probs
        self.group, self.options = group, (clip, kl_coef, reduction)

    def _bind(self, n_rows: int, era_offsets, order, device) -> _FitObjective:
        groups = _trainer_groups(self.group, n_rows, era_offsets, order, device)
        advantage = _trainer_rows(self.advantage, "advantage", n_rows, order, device)
        old = _trainer_rows(self.old_log_probs, "old_log_probs", n_rows, order, device, advantage != 0)
        reference = self.reference_log_probs
        if reference is not None:
            reference = _trainer_rows(reference, "reference_log_probs", n_rows, order, device)
        rows = (advantage, old, reference)
        return _FitObjective(_policy_struct(groups, *rows, *self.options), groups, rows)
