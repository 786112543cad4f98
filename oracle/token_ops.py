"""The token model's operators from their definitions, in 64 bits, on NumPy arrays.

TEST INFRASTRUCTURE ONLY."""
import numpy as np


def embedding_fwd(ids, W, scale=1.0, padding_idx=-1):
    ids, W = np.asarray(ids), np.asarray(W, np.float64)
    y = np.zeros(ids.shape + W.shape[1:])
    found = (ids != padding_idx) & (ids >= 0) & (ids < W.shape[0])
    y[found] = W[ids[found]] * scale
    return y


def embedding_bwd(dy, ids, shape, scale=1.0, padding_idx=-1, add=None):
    ids = np.asarray(ids).ravel()
    dy = np.asarray(dy, np.float64).reshape(ids.size, shape[1])
    found = (ids != padding_idx) & (ids >= 0) & (ids < shape[0])
    dW = np.zeros(shape)
    np.add.at(dW, ids[found], dy[found])
    dW *= scale
    return dW if add is None else dW + np.asarray(add, np.float64)


def distill(x, top=None, teacher=None, labels=None, weights=None, temperature=1.0, soft=1.0, hard=0.0, scale=1.0):
    """(loss [n], stats [n, 3], dx [n, v])"""
    x = np.asarray(x, np.float64)
    n, v = x.shape
    loss, stats, dx = np.zeros(n), np.zeros((n, 3)), np.zeros((n, v))
    for i in range(n):
        w = 1.0 if weights is None else float(np.ravel(weights)[i])
        if w == 0:
            continue
        entries = []
        if top is not None and soft:
            entries = [(int(j), float(a)) for j, a in zip(top[i], teacher[i]) if 0 <= j < v and a != -np.inf]
        label = -1 if labels is None or not hard else int(np.ravel(labels)[i])
        if not 0 <= label < v:
            label = -1
        if not entries and label < 0:
            continue
        m = x[i].max()
        stats[i, 0] = m
        with np.errstate(all="ignore"):
            d = x[i] - m
            if entries:
                a = np.array([e[1] for e in entries]) - max(e[1] for e in entries)
                p = np.exp(a / temperature)
                log_p = a / temperature - np.log(p.sum())
                p = p / p.sum()
                e = np.exp(d / temperature)
                stats[i, 1] = e.sum()
                dx[i] += soft * temperature * e / e.sum()
                for (j, _), pk, lp in zip(entries, p, log_p):
                    if pk != 0:
                        loss[i] += soft * temperature ** 2 * pk * (lp - (d[j] / temperature - np.log(e.sum())))
                    dx[i, j] -= soft * temperature * pk
            if label >= 0:
                e = np.exp(d)
                stats[i, 2] = e.sum()
                loss[i] += hard * (np.log(e.sum()) - d[label])
                dx[i] += hard * e / e.sum()
                dx[i, label] -= hard
            loss[i] *= w
            dx[i] *= w * scale
    return loss, stats, dx
