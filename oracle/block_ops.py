"""Attention with a learned position bias and the norms around a block from their definitions, in 64 bits, on NumPy arrays.

TEST INFRASTRUCTURE ONLY."""
import numpy as np


class Attn(object):
    """Mask, scale and buckets of an attention."""

    def __init__(self, causal=False, scale=None, buckets=0, max_distance=128, bidirectional=True):
        self.causal, self.scale, self.buckets, self.max_distance, self.bidirectional = causal, scale, buckets, max_distance, bidirectional

    def bucket(self, distance):
        """The bucket of a key `distance` behind its query, by whole numbers."""
        n = self.buckets // 2 if self.bidirectional else self.buckets
        e, m = n // 2, abs(distance) if self.bidirectional else max(0, -distance)
        m, side = min(m, self.max_distance), n if self.bidirectional and distance > 0 else 0
        if m < e:
            return side + m
        t = max(t for t in range(n - e) if m ** (n - e) * e ** t >= self.max_distance ** t * e ** (n - e))
        return side + e + t


def seen(a, q_len, k_len, nq, nk, start):
    """[q_len, k_len]: which keys each query sees."""
    i, j = np.arange(q_len)[:, None], np.arange(k_len)[None, :]
    s = (i < nq) & (j < nk)
    return s & (j <= i + start) if a.causal else s


def _each(a, q, k, table, q_lengths, k_lengths, q_starts):
    """(sequence, head, head of keys, scores with -inf where nothing is seen, mask, buckets) one after the other."""
    b, sq, h, d = q.shape
    sk, g = k.shape[1:3]
    scale = d ** -0.5 if a.scale is None else a.scale
    for i in range(b):
        nq = sq if q_lengths is None else min(max(int(q_lengths[i]), 0), sq)
        nk = sk if k_lengths is None else min(max(int(k_lengths[i]), 0), sk)
        start = sk - sq if q_starts is None else int(q_starts[i])
        mask = seen(a, sq, sk, nq, nk, start)
        which = None
        if a.buckets:
            of = {m: a.bucket(m) for m in range(-start - sq + 1, sk - start)}
            which = np.array([[of[j - x - start] for j in range(sk)] for x in range(sq)]).reshape(sq, sk)
        for head in range(h):
            rows, keys = np.where(mask.any(1))[0], np.where(mask.any(0))[0]   # (what is seen by nobody may be anything)
            s = np.full((sq, sk), -np.inf)
            s[np.ix_(rows, keys)] = scale * (q[i, rows, head] @ k[i, keys, head * g // h].T)
            if which is not None:
                s = s + table[which, head]
            s[~mask] = -np.inf
            yield i, head, head * g // h, s, mask, which


def _rows(t, keep):
    return np.where(keep[:, None], t, 0.0)


def attention(a, q, k, v, table=None, q_lengths=None, k_lengths=None, q_starts=None):
    """(o, lse)"""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    o, lse = np.zeros(q.shape), np.full((q.shape[0], q.shape[2], q.shape[1]), -np.inf)
    for i, head, kv, s, mask, _ in _each(a, q, k, table, q_lengths, k_lengths, q_starts):
        some = np.isfinite(s).any(1)
        top = np.where(some, s.max(1, initial=-np.inf), 0.0)
        p = np.exp(s - top[:, None])
        total = p.sum(1)
        with np.errstate(divide="ignore"):
            lse[i, head] = np.where(some, top + np.log(total), -np.inf)
        o[i, :, head] = (p / np.where(some, total, 1.0)[:, None]) @ _rows(v[i, :, kv], mask.any(0))
    return o, lse


def attention_bwd(a, do, q, k, v, o, lse, table=None, q_lengths=None, k_lengths=None, q_starts=None):
    """(dq, dk, dv, dtable) from the o and lse that are given"""
    do, q, k, v, o = (np.asarray(t, np.float64) for t in (do, q, k, v, o))
    scale = q.shape[3] ** -0.5 if a.scale is None else a.scale
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    dtable = None if table is None else np.zeros(np.shape(table))
    for i, head, kv, s, mask, which in _each(a, q, k, table, q_lengths, k_lengths, q_starts):
        row, key = mask.any(1), mask.any(0)
        p = np.exp(s - np.where(np.isfinite(lse[i, head]), lse[i, head], 0.0)[:, None])
        d, x = _rows(do[i, :, head], row), _rows(o[i, :, head], row)
        ds = p * (d @ _rows(v[i, :, kv], key).T - (d * x).sum(1)[:, None])
        dv[i, :, kv] += p.T @ d
        dq[i, :, head] = scale * ds @ _rows(k[i, :, kv], key)
        dk[i, :, kv] += scale * ds.T @ _rows(q[i, :, head], row)
        if which is not None:
            np.add.at(dtable[:, head], which[mask], ds[mask])
    return dq, dk, dv, dtable


def residual_norm(x, h=None, post=None, gate=None, scale=1.0, pre=None, eps=1e-5):
    """(y, n, stats)"""
    y = np.asarray(x, np.float64)
    stats = np.zeros((y.shape[0], 2))
    if h is not None:
        u = np.asarray(h, np.float64)
        if post is not None:
            stats[:, 0] = 1 / np.sqrt((u * u).mean(1) + eps)
            u = u * stats[:, :1] * post
        y = y + scale * u * (1.0 if gate is None else np.repeat(gate, len(y) // max(len(gate), 1), 0))
    if pre is None:
        return y, None, stats
    stats[:, 1] = 1 / np.sqrt((y * y).mean(1) + eps)
    return y, y * stats[:, 1:] * pre, stats


def residual_norm_bwd(dy, dn, y, stats, h=None, post=None, gate=None, scale=1.0, pre=None):
    """(dx, dh, dpost, dgate, dpre) from the y and stats that are given"""
    rows, dim = y.shape
    t, dh, dpost, dgate, dpre = np.zeros((rows, dim)) if dy is None else np.asarray(dy, np.float64), None, None, None, None
    if pre is not None:
        r = stats[:, 1:]
        a = dn * pre
        t = t + r * a - y * r ** 3 * (a * y).mean(1, keepdims=True)
        dpre = (dn * y * r).sum(0)
    if h is None:
        return t, dh, dpost, dgate, dpre
    each = 1.0 if gate is None else np.repeat(gate, rows // len(gate), 0)
    r = stats[:, :1] if post is not None else 1.0
    if gate is not None:
        dgate = (scale * t * h * r * (1.0 if post is None else post)).reshape(len(gate), -1, dim).sum(1)
    dh = scale * each * t
    if post is not None:
        dpost = (dh * h * r).sum(0)
        b = dh * post
        dh = r * b - h * r ** 3 * (b * h).mean(1, keepdims=True)
    return t, dh, dpost, dgate, dpre
