"""Plain forms in 64 bits of the operators built on the k largest of a row, for the tests."""
import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative
NONE = np.uint64(2**64 - 1)


def topk(x, k):
    """Descending, NaN first, equal values (zeros of either sign) by column."""
    key = np.where(np.isnan(x), np.inf, x).astype(np.float64)
    at = np.empty((x.shape[0], k), np.uint64)
    for r in range(x.shape[0]):
        order = sorted(range(x.shape[1]), key=lambda c: (not np.isnan(x[r, c]), -key[r, c], c)) if np.isnan(x[r]).any() \
            else np.argsort(-key[r], kind="stable")
        at[r] = order[:k]
    return np.take_along_axis(x, at.astype(np.int64), axis=1), at


def topk_bwd(indices, y_g, x_g):
    out = x_g.astype(np.float64).copy()
    for r in range(indices.shape[0]):
        for j, c in enumerate(indices[r]):
            if c < out.shape[1]:
                out[r, int(c)] += float(y_g[r, j])
    return out


def distill(x, teacher, indices, temp, weights=None):
    """-> dict of stats, row_loss, loss, grad and of bounds on the rounding of an fp32 evaluation (see `distill_bounds`)."""
    rows, cols = x.shape
    x, t = x.astype(np.float64), teacher.astype(np.float64)
    w = np.full(rows, 1.0 / rows) if weights is None else weights.astype(np.float64)
    out = {"stats": np.zeros((rows, 2)), "row_loss": np.zeros(rows), "grad": np.zeros((rows, cols)), "p": np.zeros((rows, cols)),
           "q": np.zeros((rows, cols)), "reach": np.zeros(rows)}
    with np.errstate(all="ignore"):
        for r in range(rows):
            if w[r] == 0:
                continue
            top = x[r].max()
            if top == -np.inf:
                out["stats"][r] = -np.inf, 0
                continue
            y = (x[r] - top) / temp
            ls = np.log(np.exp(y).sum())
            out["stats"][r] = top, ls
            held = indices[r] < cols
            if not held.any() or t[r][held].max() == -np.inf:
                continue
            at, v = indices[r][held].astype(np.int64), t[r][held] / temp
            v = v - v.max()
            q = np.exp(v) / np.exp(v).sum()
            log_q = v - np.log(np.exp(v).sum())
            some = q > 0
            out["row_loss"][r] = temp**2 * (q[some] * (log_q[some] - (y[at][some] - ls))).sum()
            np.add.at(out["q"][r], at, q)
            out["p"][r] = np.exp(y - ls)
            out["grad"][r] = w[r] * temp * (out["p"][r] - out["q"][r])
            low = np.where(np.isfinite(y[at][some]), y[at][some], 0.0)
            out["reach"][r] = np.abs(low).max(initial=0) + ls + np.abs(v[np.isfinite(v)]).max() + np.log(len(at) + 1.0)
        seen = w != 0
        out["loss"] = (w[seen] * out["row_loss"][seen]).sum()
    return out


def distill_bounds(ref, x, temp, w):
    """How far fp32 may be off: a scaled difference y = (x - max) / T comes with three roundings and goes through an exponential
    whose argument is multiplied by log2(e) once more, so exp(y) is off by (5 |y| + 4) halves of a step at most, as long as
    the exponential itself is good to two; a sum of `cols` positive terms adds cols / 64 + 16 (no lane adds more than a 64th of
    a row one after the other), its logarithm as much again in absolute terms."""
    rows, cols = x.shape
    with np.errstate(all="ignore"):
        y = np.abs((x.astype(np.float64) - x.max(axis=1, keepdims=True)) / temp)
    there = np.isfinite(y)
    y = np.where(there, y, 0.0)
    # terms of the sum count by their size: those far below the maximum add nothing to its error
    size = np.where(there, np.exp(-y), 0.0)
    mass = (size * (5 * y + 4)).sum(axis=1) / np.maximum(size.sum(axis=1), 1e-300)
    s = (mass + cols / 64 + 16) * EPS                       # of log sum
    p = ref["p"] * ((5 * y + 8) * EPS + s[:, None])
    q = ref["q"] * (5 * ref["reach"][:, None] + 64) * EPS   # the teacher's sum has at most 512 terms
    grad = np.abs(w)[:, None] * temp * (p + q + 2 * EPS * (ref["p"] + ref["q"])) + 2 * EPS * np.abs(ref["grad"])
    row = temp**2 * ((12 * ref["reach"] + 96) * EPS + s) + 8 * EPS * np.abs(ref["row_loss"])
    return {"ls": s + 2 * EPS * np.abs(ref["stats"][:, 1]), "grad": grad, "row_loss": row}


def expert_sort(experts, n_experts):
    held = experts < n_experts
    order = np.argsort(np.where(held, experts, n_experts), kind="stable")
    slots = np.empty(len(experts), np.uint64)
    slots[order] = np.arange(len(experts), dtype=np.uint64)
    slots[~held] = NONE
    counts = np.bincount(experts[held].astype(np.int64), minlength=n_experts)[:n_experts]
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.uint64), slots


def spread(x, slots, k, base, weights=None):
    out = base.astype(np.float64).copy()
    for i, s in enumerate(slots):
        if s < len(out):
            out[int(s)] = x[i // k].astype(np.float64) * (1.0 if weights is None else float(weights.reshape(-1)[i]))
    return out


def gather(y, slots, tokens, k, weights=None):
    """The sum per token, and the sum of the terms' magnitudes (what the rounding of the sum is relative to)."""
    out, size = np.zeros((tokens, y.shape[1])), np.zeros((tokens, y.shape[1]))
    for i, s in enumerate(slots):
        if s < len(y):
            v = y[int(s)].astype(np.float64) * (1.0 if weights is None else float(weights.reshape(-1)[i]))
            out[i // k] += v
            size[i // k] += np.abs(v)
    return out, size
