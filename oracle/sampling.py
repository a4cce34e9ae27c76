"""64-bit numpy form of the token sampler (tests only)."""
import numpy as np


def sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row of logits; the parameters as the f32 numbers that the call takes."""
    t, top_p, min_p = (float(np.float32(a)) for a in (temperature, top_p, min_p))
    z = np.asarray(z, np.float64)
    ids = np.flatnonzero(z > -np.inf)        # (NaN compares false)
    if ids.size == 0:
        return -1, 0.0
    order = ids[np.argsort(-z[ids], kind="stable")]
    if t == 0:
        return int(order[0]), 1.0
    if 0 < top_k < order.size:
        order = order[:top_k]
    top = z[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(z[order] == top, 1.0, np.exp((z[order] - top) / t))
    if top_p <= 0:
        order, w = order[:1], w[:1]
    elif top_p < 1:
        n = int(np.count_nonzero(np.concatenate(([0.0], np.cumsum(w)[:-1])) < top_p * w.sum()))
        order, w = order[:n], w[:n]
    keep = w >= min(min_p, 1.0)
    order, w = order[keep], w[keep]
    w = np.where(w >= 2.0 ** -44, w, 0.0)    # a weight is a whole number of units of 2^-44, rounded down
    by = np.argsort(order)
    order, w = order[by], w[by]
    run = np.cumsum(w)
    goal = min(max(float(np.float32(u)), 0.0), 1.0) * run[-1]
    i = int(np.searchsorted(run, goal, side="right"))
    if i >= w.size:
        i = int(np.flatnonzero(w > 0)[-1])
    return int(order[i]), float(w[i] / run[-1])
