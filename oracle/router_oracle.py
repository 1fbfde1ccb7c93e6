"""Expert routing in 64 bits: the choice, the weights and the gradient of the
logits from their definitions, and the gradient of the weighted combine."""
import numpy as np


def scores(z, score):
    z = z.astype(np.float64)
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-z))
    with np.errstate(invalid="ignore"):
        top = z.max(1, keepdims=True)
        e = np.exp(z - np.where(np.isneginf(top), 0.0, top))
        s = e.sum(1, keepdims=True)
        return np.where(s == 0, 0.0, e / np.where(s == 0, 1.0, s))


def router(z, k, score="softmax", bias=None, groups=1, topk_groups=None, group_score="max", renormalize=True,
           scale=1.0):
    """(weights, ids): order of s + bias (of z without a bias), ties to the
    lowest index, NaN as -inf."""
    n, E = z.shape
    s = scores(z, score)
    choice = z.astype(np.float64) if bias is None else s + bias.astype(np.float64)
    by = choice if bias is not None or group_score == "max" else s
    low = lambda v: np.where(np.isnan(v), -np.inf, v)
    choice, by = low(choice), low(by)
    allowed = np.ones((n, E), bool)
    if groups > 1 and (topk_groups or groups) < groups:
        best = -np.sort(-by.reshape(n, groups, E // groups), axis=2)
        total = best[:, :, 0] if group_score == "max" else best[:, :, :2].sum(2)
        rank = np.argsort(np.argsort(-total, axis=1, kind="stable"), axis=1, kind="stable")
        allowed = np.repeat(rank < topk_groups, E // groups, axis=1)
    place = np.broadcast_to(np.arange(E), (n, E))
    ids = np.lexsort((place, -choice, ~allowed), axis=1)[:, :k]
    w = np.take_along_axis(s, ids, 1)
    if renormalize:
        if score == "softmax":
            bad = np.isnan(s).any(1)
            zi = np.take_along_axis(z.astype(np.float64), ids, 1)
            w = scores(zi, "softmax")
            w[bad] = np.nan
        else:
            # shares through logs, so that scores which vanish still have one
            zi = np.take_along_axis(z.astype(np.float64), ids, 1)
            with np.errstate(invalid="ignore"):
                w = scores(-np.logaddexp(0.0, -zi), "softmax")
    return w * scale, ids.astype(np.int32)


def router_bwd(z, ids, dw, score="softmax", renormalize=True, scale=1.0):
    """dz through the scores: w = scale * s / (sum of the chosen s, or 1)."""
    s = scores(z, score)
    dw = dw.astype(np.float64) * scale
    chosen = np.take_along_axis(s, ids.astype(np.int64), 1)
    if renormalize:
        total = chosen.sum(1, keepdims=True)
        with np.errstate(invalid="ignore", divide="ignore"):
            ds_c = np.where(total == 0, 0.0, dw / total - (dw * chosen).sum(1, keepdims=True) / total ** 2)
    else:
        ds_c = dw
    ds = np.zeros(z.shape)
    for t in range(z.shape[0]):
        np.add.at(ds[t], ids[t].astype(np.int64), ds_c[t])
    if score == "sigmoid":
        return ds * s * (1.0 - s)
    return s * (ds - (s * ds).sum(1, keepdims=True))


def combine_bwd(dout, rows, slot_pos, weights):
    """(drows, dweights) of out[t] = sum_j w[t, j] rows[slot_pos[t, j]]."""
    n, k = slot_pos.shape
    drows, dw = np.zeros(rows.shape), np.zeros((n, k))
    for t in range(n):
        for j in range(k):
            p = slot_pos[t, j]
            if 0 <= p < rows.shape[0]:
                drows[p] = (1.0 if weights is None else np.float64(weights[t, j])) * dout[t].astype(np.float64)
                dw[t, j] = np.dot(dout[t].astype(np.float64), rows[p].astype(np.float64))
    return drows, dw
