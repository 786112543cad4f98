"""Attention and its gradients on the GPU against their definitions in 64 bits (oracle/block_ops.py), at the sizes, types, head layouts and masks
where they can go wrong.

Tolerances, first order, u = 2^-24 half a step of fp32 and h half a step of the tensors' type.  A score is a product of D terms and two sums: off
by (D + 4) u sum |scale q k| + 4 u (|score| + |bias| + |lse|), and the power of two is good to 2 u; that, E, is a probability's relative error.
In 16-bit tensors p and ds are rounded once more before the products over them (h; binary16 is scaled so that what is below its range is
at most 2^-31 of a row's largest), sums of n terms are off by n u of their sizes, and results by h."""
import numpy as np
import pytest

from oracle import block_ops as O
from test_gpu_token_model import HALF, TINY, TYPES, U, close, ints, shifted, stored, upload

pytestmark = pytest.mark.gpu


def handle(singa, q, k, a):
    return singa.AttentionHandle(q, k, causal=a.causal, scale=a.scale, buckets=a.buckets, max_distance=a.max_distance, bidirectional=a.bidirectional)


def bounds(t, a, do, q, k, v, o, table, q_lengths, k_lengths, q_starts):
    """(of o, lse, dq, dk, dv, dtable), terms as in the module's description."""
    b, sq, h, d = q.shape
    sk = k.shape[1]
    half = 0.0 if t == "f32" else HALF[t]
    scale = d ** -0.5 if a.scale is None else a.scale
    n = sk + 64
    eo, el = np.zeros(q.shape), np.zeros((b, h, sq))
    eq, ek, ev, et = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape), None if table is None else np.zeros(table.shape)
    group = h // k.shape[2]
    for i, head, kv, s, mask, which in O._each(a, q, k, table, q_lengths, k_lengths, q_starts):
        row, key = mask.any(1), mask.any(0)
        some = np.isfinite(s).any(1)
        top = np.where(some, s.max(1, initial=-np.inf), 0.0)
        lse = np.where(some, top + np.log(np.where(some, np.exp(s - top[:, None]).sum(1), 1.0)), 0.0)
        p = np.exp(s - lse[:, None])
        Q, K, V = (np.abs(O._rows(x, keep)) for x, keep in ((q[i, :, head], row), (k[i, :, kv], key), (v[i, :, kv], key)))
        size = np.where(mask & np.isfinite(s), np.abs(s), 0.0)
        extra = 0.0 if which is None else np.abs(np.where(np.isfinite(table[:, head]), table[:, head], 0.0))[which]
        E = (d + 4) * U * abs(scale) * (Q @ K.T) + 4 * U * (size + extra + np.abs(lse)[:, None]) + 4 * U
        Er = np.where(mask, E, 0.0).max(1, initial=0.0)[:, None]
        el[i, head] = Er[:, 0] + n * U + 2 * U * np.abs(lse)
        eo[i, :, head] = (2 * Er + half + n * U) * (p @ V) + 2.0 ** -31 * V.sum(0)
        if do is None:
            continue
        dd, x = O._rows(do[i, :, head], row), O._rows(o[i, :, head], row)
        D, X = np.abs(dd), np.abs(x)
        gap = dd @ O._rows(v[i, :, kv], key).T - (dd * x).sum(1)[:, None]
        Ep = E + 2 * U * np.abs(lse)[:, None]
        Es = p * (np.abs(gap) * (Ep + 2 * U) + (d + 4) * U * (D @ V.T + (D * X).sum(1)[:, None]))
        ds = np.abs(p * gap)
        lost = 2.0 ** -33
        eq[i, :, head] = abs(scale) * ((Es + (half + n * U) * ds + lost * ds.max(1, initial=0.0)[:, None]) @ K)
        ek[i, :, kv] += abs(scale) * ((Es + (half + (group * sq + 64) * U) * ds + lost * ds.max(0, initial=0.0)[None]).T @ Q)
        ev[i, :, kv] += (p * (Ep + half + (group * sq + 64) * U) + 2.0 ** -38).T @ D
        if which is not None:
            np.add.at(et[:, head], which[mask], (Es + (b * sq * sk / 16 + 400) * U * ds)[mask])
    return eo, el, eq, ek, ev, et


def check(singa, dev, t, a, b, sq, sk, h, g, d, lengths=(None, None, None), seed=0, shift=0, sharp=1.5, grads=True, case=None):
    r = np.random.default_rng(seed + sq + 7 * sk + 31 * h + d)
    if case is None:
        q, k, v, do = (stored(t, s * r.standard_normal(shape)) for s, shape in ((sharp, (b, sq, h, d)), (1, (b, sk, g, d)), (1, (b, sk, g, d)), (1, (b, sq, h, d))))
        table = stored("f32", r.standard_normal((a.buckets, h))) if a.buckets else None
    else:
        q, k, v, do, table = case
    put = (lambda x: shifted(singa, dev, t, x, shift)) if shift else (lambda x: upload(singa, dev, t, x))
    dq_, dk_, dv_, ddo = (put(x) for x in (q, k, v, do))
    dt = None if table is None else upload(singa, dev, "f32", table)
    dl = dict(zip(("q_lengths", "k_lengths", "q_starts"), (None if x is None else ints(singa, dev, x) for x in lengths)))
    H = handle(singa, dq_, dk_, a)
    go, gl = singa.AttentionForward(H, dq_, dk_, dv_, dt, **dl)
    wo, wl = O.attention(a, q, k, v, table, *lengths)
    o = go.to_numpy().astype(np.float64)
    eo, el, eq, ek, ev, et = bounds(t, a, do if grads else None, q, k, v, o, table, *lengths)

    def rounded(bound, want):
        return bound * 1.01 + HALF[t] * np.abs(want) * 1.01 + TINY[t]

    close(o, wo, rounded(eo, wo), "o")
    close(gl.to_numpy(), wl, el * 1.01, "lse")
    if not grads:
        return go, gl
    got = singa.AttentionBackward(H, ddo, dq_, dk_, dv_, go, gl, dt, **dl)
    want = O.attention_bwd(a, do, q, k, v, o, gl.to_numpy().astype(np.float64), table, *lengths)
    for name, x, w, e in zip(("dq", "dk", "dv"), got, want, (eq, ek, ev)):
        close(x.to_numpy(), w, rounded(e, w), name)
    if table is not None:
        close(got[3].to_numpy(), want[3], et * 1.01 + U * np.abs(want[3]), "dtable")
    else:
        assert got[3] is None
    again = singa.AttentionBackward(H, ddo, dq_, dk_, dv_, go, gl, dt, **dl)
    for x, y in zip(got, again):
        assert x is y is None or np.array_equal(x.to_numpy(), y.to_numpy(), equal_nan=True)   # the same bits every time
    return go, gl


# (batch, queries, keys, heads, heads of keys, dim): one of everything, tiles that are not full, one more than full, long ones, groups
SIZES = [(1, 1, 1, 1, 1, 1), (2, 3, 5, 2, 2, 8), (1, 33, 31, 3, 1, 16), (2, 64, 64, 2, 2, 32), (1, 65, 129, 4, 2, 33), (3, 128, 128, 1, 1, 64),
         (1, 129, 257, 2, 1, 63), (2, 37, 37, 4, 4, 40), (1, 300, 300, 2, 2, 96), (1, 200, 333, 3, 3, 100), (1, 257, 130, 4, 1, 128),
         (1, 5, 700, 8, 1, 65), (1, 1, 1500, 6, 2, 64), (2, 2, 900, 4, 4, 127), (1, 700, 40, 2, 2, 24), (1, 515, 515, 1, 1, 72)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_attention(dev, t, causal, size):
    from singa_amd import singa_wrap as singa
    check(singa, dev, t, O.Attn(causal), *size)


# few buckets, a band that ends inside a tile, one that reaches over all distances, no gap between the buckets' borders
BIAS = [(4, 3, True), (8, 20, True), (32, 128, True), (2, 5, False), (16, 64, False), (32, 100, False), (128, 1024, True)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("buckets,distance,both", BIAS)
@pytest.mark.parametrize("causal,size", [(False, (2, 70, 70, 2, 2, 16)), (True, (1, 200, 200, 4, 2, 40)), (False, (1, 150, 301, 2, 1, 64)),
                                         (True, (1, 1, 600, 8, 2, 32)), (False, (1, 400, 17, 3, 3, 128))])
def test_attention_with_a_position_bias(dev, t, buckets, distance, both, causal, size):
    from singa_amd import singa_wrap as singa
    check(singa, dev, t, O.Attn(causal, buckets=buckets, max_distance=distance, bidirectional=both), *size)


# lengths of zero, one and all; more than there is and less than none; queries in front of every key, and behind
LENGTHS = [((0, 1, 90, 64), (0, 1, 90, 64), None), (None, (90, 0, 33, 1), None), ((90, 500, -3, 64), (1000, 90, 90, -1), None),
           (None, None, (0, 60, -40, -200)), ((5, 90, 90, 90), (90, 70, 90, 0), (-(1 << 30), 1 << 30, 17, 0))]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal,buckets", [(False, 0), (True, 0), (True, 16), (False, 16)])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_padded_batches(dev, t, causal, buckets, lengths):
    """Rows behind a sequence hold NaN and infinities: they reach nothing, and their results are 0."""
    from singa_amd import singa_wrap as singa
    if buckets and lengths[2] is not None:
        lengths = (lengths[0], lengths[1], tuple(max(-300, min(300, x)) for x in lengths[2]))   # (the oracle lists the distances)
    r = np.random.default_rng(5)
    b, sq, sk, h, g, d = 4, 90, 90, 4, 2, 24
    case = [stored(t, r.standard_normal(s)) for s in ((b, sq, h, d), (b, sk, g, d), (b, sk, g, d), (b, sq, h, d))]
    for i in range(b):
        for which, n in ((0, lengths[0]), (3, lengths[0]), (1, lengths[1]), (2, lengths[1])):
            if n is not None:
                rest = case[which][i, max(0, n[i]):]
                rest[...] = np.resize([np.nan, np.inf, -np.inf], rest.shape)
    case.append(stored("f32", r.standard_normal((buckets, h))) if buckets else None)
    check(singa, dev, t, O.Attn(causal, buckets=buckets, max_distance=40), b, sq, sk, h, g, d, lengths=lengths, case=case)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("sq,buckets", [(1, 0), (1, 16), (9, 0), (50, 0), (200, 16)])
def test_the_unused_part_of_a_cache(dev, t, sq, buckets):
    """Keys behind the last query of a causal sequence hold NaN and infinities, and no lengths of the keys are given."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(8)
    b, sk, h, g, d, starts = 3, 700, 4, 2, 40, (0, 290, 61)
    q, do, k, v = (stored(t, r.standard_normal(s)) for s in ((b, sq, h, d), (b, sq, h, d), (b, sk, g, d), (b, sk, g, d)))
    table = stored("f32", r.standard_normal((buckets, h))) if buckets else None
    for x in (k, v):
        for i in range(b):
            rest = x[i, starts[i] + sq:]
            rest[...] = np.resize([np.nan, np.inf, -np.inf], rest.shape)
    seen = tuple(s + sq for s in starts)
    a = O.Attn(True, buckets=buckets, max_distance=40)
    H = handle(singa, upload(singa, dev, t, q), upload(singa, dev, t, k), a)
    results = []
    for k_lengths in (None, seen):
        args = [upload(singa, dev, t, x) for x in (q, k, v)]
        dt = upload(singa, dev, "f32", table) if buckets else None
        how = dict(k_lengths=None if k_lengths is None else ints(singa, dev, k_lengths), q_starts=ints(singa, dev, starts))
        o, lse = singa.AttentionForward(H, *args, dt, **how)
        grads = singa.AttentionBackward(H, upload(singa, dev, t, do), *args, o, lse, dt, **how)
        results.append([x.to_numpy() for x in (o, lse) + tuple(grads) if x is not None])
    for x, y in zip(*results):
        assert np.isfinite(x).all() and np.array_equal(x, y)
    for i in range(b):
        assert not results[0][3][i, seen[i]:].any() and not results[0][4][i, seen[i]:].any()
    check(singa, dev, t, a, b, sq, sk, h, g, d, lengths=(None, seen, starts), case=[q, k, v, do, table])


@pytest.mark.parametrize("t", TYPES)
def test_one_new_token_over_caches_of_different_lengths(dev, t):
    from singa_amd import singa_wrap as singa
    keys = (1, 3000, 64, 1999, 0)
    starts = tuple(n - 1 for n in keys)
    for buckets, (h, g) in ((0, (8, 2)), (32, (8, 2)), (32, (3, 3))):
        check(singa, dev, t, O.Attn(True, buckets=buckets, bidirectional=False), 5, 1, 3000, h, g, 48, lengths=(None, keys, starts))


# one row to 32 and one more, the rounds of four wavefronts (128 keys) full, not full and one more, parts of the keys that do not come out even
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [20, 64, 70, 128])
@pytest.mark.parametrize("sq,sk,h,g", [(1, 65, 1, 1), (1, 128, 32, 1), (3, 129, 10, 2), (8, 511, 4, 1), (16, 513, 4, 2), (7, 1070, 2, 2), (11, 1300, 3, 1), (1, 9001, 6, 2)])
def test_few_queries(dev, t, d, sq, sk, h, g):
    from singa_amd import singa_wrap as singa
    for causal, buckets, scale in ((True, 0, None), (False, 32, -0.3), (True, 16, 0.0)):
        a = O.Attn(causal, scale, buckets=buckets, max_distance=200)
        check(singa, dev, t, a, 3, sq, sk, h, g, d, lengths=((sq, max(0, sq - 2), 0), (sk, sk - 33, sk // 2), (sk - sq, sk - 50, -1)), grads=False)
        check(singa, dev, t, a, 1, sq, sk, h, g, d, shift=1, grads=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [1, 7, 8, 64, 70])
def test_tensors_at_any_element(dev, t, d):
    from singa_amd import singa_wrap as singa
    for shift in (1, 2, 8):
        check(singa, dev, t, O.Attn(True, buckets=8, max_distance=30), 2, 70, 100, 2, 1, d, shift=shift)


@pytest.mark.parametrize("t", TYPES)
def test_no_queries_no_keys_no_sequences(dev, t):
    from singa_amd import singa_wrap as singa
    for a in (O.Attn(), O.Attn(True, buckets=4, max_distance=9)):
        for size in ((2, 0, 5, 2, 1, 16), (2, 5, 0, 2, 1, 16), (0, 5, 5, 2, 1, 16)):
            b, sq, sk, h, g, d = size
            q, k = singa.Tensor((b, sq, h, d), dev, upload(singa, dev, t, [0.0]).data_type()), singa.Tensor((b, sk, g, d), dev, upload(singa, dev, t, [0.0]).data_type())
            table = upload(singa, dev, "f32", np.ones((a.buckets, h))) if a.buckets else None
            if q.Size():
                q.SetFloatValue(1.0)
            if k.Size():
                k.SetFloatValue(1.0)
            H = handle(singa, q, k, a)
            o, lse = singa.AttentionForward(H, q, k, k, table)
            dq, dk, dv, dtable = singa.AttentionBackward(H, q, q, k, k, o, lse, table)
            for x in (o, dq, dk, dv) + ((dtable,) if table is not None else ()):
                assert not x.to_numpy().any()
            assert (lse.to_numpy() == -np.inf).all()


@pytest.mark.parametrize("t", TYPES)
def test_peaked_and_flat_rows(dev, t):
    """Scores far apart (one key takes all), equal ones, and a bias of -inf for some buckets (those keys take nothing)."""
    from singa_amd import singa_wrap as singa
    check(singa, dev, t, O.Attn(), 1, 130, 260, 2, 2, 64, sharp=12.0)
    check(singa, dev, t, O.Attn(True, scale=0.0), 1, 130, 260, 2, 2, 64)
    check(singa, dev, t, O.Attn(scale=-0.3), 1, 40, 50, 2, 2, 20)
    r = np.random.default_rng(1)
    a = O.Attn(buckets=8, max_distance=16)
    case = [stored(t, r.standard_normal(s)) for s in ((1, 90, 2, 16),) * 4] + [stored("f32", r.standard_normal((8, 2)))]
    case[4][0, 0] = case[4][3, 1] = case[4][6, 1] = -np.inf
    check(singa, dev, t, a, 1, 90, 90, 2, 2, 16, case=case, grads=False)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-6, 1.0, 3e3])
def test_gradients_of_any_size(dev, t, size):
    """The products over the probabilities' gradients keep their bits whatever the size of the result's gradient: halves' small ones as well.  The
    bound on what leaves the type is the type's own (half of its smallest step), on top of the usual one."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(3)
    q, k, v = (stored(t, 0.5 * r.standard_normal((1, 300, 2, 64))) for _ in range(3))
    do = stored(t, size * r.standard_normal((1, 300, 2, 64)))
    do[:, ::3] *= 0.125
    do = stored(t, do)   # (what the device holds: the small ones lose bits)
    check(singa, dev, t, O.Attn(True), 1, 300, 300, 2, 2, 64, case=(q, k, v, do, None))


def test_gradients_against_differences(dev):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(2)
    a = O.Attn(True, buckets=6, max_distance=11)
    q, k, v, do = (stored("f32", r.standard_normal(s)) for s in ((2, 40, 4, 16), (2, 45, 2, 16), (2, 45, 2, 16), (2, 40, 4, 16)))
    table = stored("f32", r.standard_normal((6, 4)))
    lengths = ((40, 31), (45, 37), None)
    dl = dict(q_lengths=ints(singa, dev, lengths[0]), k_lengths=ints(singa, dev, lengths[1]))
    dq, dk, dv, ddo, dt = (upload(singa, dev, "f32", x) for x in (q, k, v, do, table))
    H = handle(singa, dq, dk, a)
    o, lse = singa.AttentionForward(H, dq, dk, dv, dt, **dl)
    grads = singa.AttentionBackward(H, ddo, dq, dk, dv, o, lse, dt, **dl)
    args, step = [q, k, v, table], 1e-4
    for i, g in enumerate(grads):
        along = r.standard_normal(args[i].shape)
        along /= np.linalg.norm(along)
        ends = []
        for sign in (1, -1):
            moved = [x + sign * step * along if j == i else x for j, x in enumerate(args)]
            ends.append((O.attention(a, *moved, *lengths)[0] * do).sum())
        got = (g.to_numpy().astype(np.float64) * along).sum()
        # the third derivative over step^2 / 6 is below 1e3 * 1e-8 / 6 of |do| |v|; fp32 gradients of up to 45 terms: 1e-5
        assert abs(got - (ends[0] - ends[1]) / (2 * step)) < 1e-4 * max(1.0, np.linalg.norm(g.to_numpy())), i


@pytest.mark.parametrize("t", TYPES)
def test_recorded_calls_replay(dev, t):
    """A forward and a backward pass of two sizes in one recording, replayed on other values with the program's own calls in between."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(4)
    a = O.Attn(True, buckets=16, max_distance=50, bidirectional=False)
    sizes = [(2, 150, 150, 4, 2, 32), (1, 1, 1300, 8, 2, 64), (1, 20, 900, 2, 2, 40)]
    made = []
    for b, sq, sk, h, g, d in sizes:
        ts = [upload(singa, dev, t, r.standard_normal(s)) for s in ((b, sq, h, d), (b, sk, g, d), (b, sk, g, d), (b, sq, h, d))]
        made.append((handle(singa, ts[0], ts[1], a), ts, upload(singa, dev, "f32", r.standard_normal((16, h)))))

    def run():
        out = []
        for H, (q, k, v, do), table in made:
            o, lse = singa.AttentionForward(H, q, k, v, table)
            out += [o, lse, *singa.AttentionBackward(H, do, q, k, v, o, lse, table)]
        return out

    run()
    dev.Sync()
    dev.EnableGraph(True)
    kept = run()
    dev.EnableGraph(False)
    try:
        for turn in range(4):
            for _, ts, table in made:
                for x in ts:
                    fresh = stored(t, r.standard_normal(x.shape()))
                    if t == "f32":
                        x.CopyFloatDataFromHostPtr(fresh)
                    else:
                        x.CopyHalfDataFromHostPtr(fresh.astype(np.float16) if t == "f16" else singa.float_to_bf16_bits(fresh))
            dev.RunGraph()
            want = run()
            dev.Sync()
            for x, y in zip(kept, want):
                x, y = x.to_numpy(), y.to_numpy()
                assert np.isfinite(y).all() and np.array_equal(x, y), turn
    finally:
        dev.ResetGraph()


@pytest.mark.parametrize("t", TYPES)
def test_one_recording_for_a_cache_that_grows(dev, t):
    """The lengths and positions are read on the device: one recording of a token's step serves every length, whatever the cache's rest holds."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(12)
    b, sk, h, g, d = 3, 1500, 8, 2, 64
    q, k, v = (stored(t, r.standard_normal(s)) for s in ((b, 1, h, d), (b, sk, g, d), (b, sk, g, d)))
    for x in (k, v):
        x[:, 1400:] = np.nan
    dq_, dk_, dv_ = (upload(singa, dev, t, x) for x in (q, k, v))
    table = stored("f32", r.standard_normal((16, h)))
    dt, dl, ds = upload(singa, dev, "f32", table), ints(singa, dev, (1, 1, 1)), ints(singa, dev, (0, 0, 0))
    a = O.Attn(True, buckets=16, max_distance=50, bidirectional=False)
    H = handle(singa, dq_, dk_, a)
    run = lambda: singa.AttentionForward(H, dq_, dk_, dv_, dt, k_lengths=dl, q_starts=ds)
    run()
    dev.Sync()
    dev.EnableGraph(True)
    o, lse = run()
    dev.EnableGraph(False)
    try:
        for n in ((1, 2, 3), (64, 1400, 0), (1400, 513, 700), (5, 128, 129), (1, 1, 1)):
            dl.CopyIntDataFromHostPtr(np.asarray(n, np.int32))
            ds.CopyIntDataFromHostPtr(np.asarray(n, np.int32) - 1)
            dev.RunGraph()
            eo, el = run()
            dev.Sync()
            assert np.array_equal(o.to_numpy(), eo.to_numpy()) and np.array_equal(lse.to_numpy(), el.to_numpy()), n
            wo, wl = O.attention(a, q, k, v, table, None, n, tuple(x - 1 for x in n))
            bo, bl = bounds(t, a, None, q, k, v, o.to_numpy().astype(np.float64), table, None, n, tuple(x - 1 for x in n))[:2]
            close(o.to_numpy(), wo, bo * 1.01 + HALF[t] * np.abs(wo) * 1.01 + TINY[t], "o")
            close(lse.to_numpy(), wl, bl * 1.01, "lse")
    finally:
        dev.ResetGraph()


def test_two_streams_at_once(dev):
    """Calls on the auxiliary stream beside others on the main one: each has its own workspace."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(6)
    q, k, do = (upload(singa, dev, "bf16", r.standard_normal(s)) for s in ((1, 300, 4, 64), (1, 700, 2, 64), (1, 300, 4, 64)))
    H = singa.AttentionHandle(q, k, causal=True)
    o, lse = singa.AttentionForward(H, q, k, k)
    want = [o, lse, *singa.AttentionBackward(H, do, q, k, k, o, lse)[:3]]
    want = [x.to_numpy() for x in want]

    class _Beside(object):
        def __init__(self, stream):
            self.__dict__.update(dev.__dict__)
            self.stream = stream

    for _ in range(3):
        aux = dev.Fork()
        held, out = [], []
        main = dev.stream
        for turn in range(4):
            dev.stream = aux if turn % 2 else main
            try:
                o, lse = singa.AttentionForward(H, q, k, k)
                out.append([o, lse, *singa.AttentionBackward(H, do, q, k, k, o, lse)[:3]])
            finally:
                dev.stream = main
            held.append(out[-1])
            if turn % 2:
                dev.UsedOn(aux, q, k, do, *out[-1])
            dev.Join() if turn == 3 else None
        dev.Sync()
        for each in out:
            for x, w in zip(each, want):
                assert np.array_equal(x.to_numpy(), w)


def test_a_long_cache_with_offsets_beyond_32_bits(dev):
    """Keys of more than 2^32 bytes in all and for one sequence: the last sequence's and the last rows' are the ones that count."""
    from singa_amd import singa_wrap as singa
    sk, g, d = 1 << 20, 16, 128          # 4 GB of bfloat16 for a sequence
    b = 2
    k = singa.Tensor((b, sk, g, d), dev, singa.kBFloat16)
    k.SetFloatValue(0.0)
    r = np.random.default_rng(8)
    rows = 300
    tail = stored("bf16", r.standard_normal((rows, g, d)))
    bits = singa.float_to_bf16_bits(tail)
    at = k.ptr + (k.Size() - tail.size) * 2
    view = singa.from_device_pointer(at, tail.shape, dev, singa.kBFloat16, keepalive=k)
    view.CopyHalfDataFromHostPtr(bits)
    q = stored("bf16", r.standard_normal((b, 1, g, d)))
    dq = upload(singa, dev, "bf16", q)
    H = singa.AttentionHandle(dq, k)
    o, lse = singa.AttentionForward(H, dq, k, k)
    s = np.einsum("hd,rhd->hr", q[1, 0], tail) * d ** -0.5
    e = np.exp(s)
    total = e.sum(1) + (sk - rows)       # keys of zeros have a score of 0
    want = np.einsum("hr,rhd->hd", e, tail) / total[:, None]
    got = o.to_numpy().astype(np.float64)
    assert not got[0].any()
    # the sums of up to 2^20 equal terms in chains of at most 2^14: 2^-10; a probability's and the result's rounding
    size = np.einsum("hr,rhd->hd", e, np.abs(tail)) / total[:, None]
    assert (np.abs(got[1, 0] - want) <= 3 * 2.0 ** -8 * size).all()
    np.testing.assert_allclose(lse.to_numpy()[:, :, 0], np.stack([np.full(g, np.log(sk)), np.log(total)]), rtol=0, atol=2.0 ** -10)


# queries on both sides of a tile of 32 or 64, shared and own heads of keys, every form of the kernels' rows
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bias", [12.0, 30.0, 100.0])
@pytest.mark.parametrize("causal,sq,sk,h,g,d", [(False, 37, 37, 2, 2, 16), (True, 31, 31, 4, 2, 40), (False, 65, 50, 2, 1, 64), (True, 63, 63, 2, 2, 100), (False, 33, 129, 3, 3, 128),
                                                (True, 64, 64, 1, 1, 24), (False, 300, 200, 4, 1, 64)])
def test_a_large_position_bias(dev, monkeypatch, t, bias, causal, sq, sk, h, g, d):
    """What softmax cannot see, a number added to the whole table, and large values of some buckets: the rows behind the last query, which a tile of
    queries holds as zeros, have no probabilities.

    Beside the usual bounds stands that of numbers below fp32's least normal one, 2^-126, which are zeros on the device (e^-100 is 2^-144): a
    result has fewer than 3 * 300 * 200 < 2^18 terms, each a probability times |do (v - o)| |scale k| < 2^8 or less: 2^-100."""
    from singa_amd import singa_wrap as singa
    usual = close
    monkeypatch.setitem(globals(), "close", lambda got, want, bound, what: usual(got, want, bound + 2.0 ** -100, what))
    r = np.random.default_rng(17)
    a = O.Attn(causal, buckets=8, max_distance=20)
    for some in (False, True):
        q, do, k, v = (stored(t, r.standard_normal((3, n, c, d))) for n, c in ((sq, h), (sq, h), (sk, g), (sk, g)))
        table = r.standard_normal((8, h))
        table[[1, 2, 6] if some else slice(None)] += bias
        case = (q, k, v, do, stored("f32", table))
        check(singa, dev, t, a, 3, sq, sk, h, g, d, case=case)
        check(singa, dev, t, a, 3, sq, sk, h, g, d, case=case, lengths=((sq - 2, sq, 1), (sk, sk - 5, sk), None))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("buckets", [0, 8])
def test_no_queries_over_a_cache(dev, t, buckets):
    """More keys than the backward pass has in one part: their gradients and the table's are zeros."""
    from singa_amd import singa_wrap as singa
    a = O.Attn(True, buckets=buckets, max_distance=20)
    kind = upload(singa, dev, t, [0.0]).data_type()
    q, k = singa.Tensor((2, 0, 4, 24), dev, kind), upload(singa, dev, t, np.ones((2, 700, 2, 24)))
    table = upload(singa, dev, "f32", np.ones((buckets, 4))) if buckets else None
    H = handle(singa, q, k, a)
    o, lse = singa.AttentionForward(H, q, k, k, table)
    dq, dk, dv, dtable = singa.AttentionBackward(H, q, q, k, k, o, lse, table)
    assert o.shape() == dq.shape() == [2, 0, 4, 24] and lse.shape() == [2, 4, 0]
    for x in (dk, dv) + ((dtable,) if buckets else ()):
        assert not x.to_numpy().any()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float32).min, -2.5e38, -2.2e38])
def test_a_bias_that_hides_keys(dev, t, low):
    """Buckets of -inf, and of values from fp32's lowest on up to -2.1e38 (-3e38 in units of log2), which hide keys alike: both passes, with queries
    that see nothing else.  Their results and gradients are 0."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(1)
    for causal, (sq, sk, h, g, d) in ((False, (90, 90, 2, 2, 16)), (True, (70, 70, 4, 2, 64)), (True, (33, 33, 2, 1, 128))):
        a = O.Attn(causal, buckets=8, max_distance=16)
        q, do, k, v = (stored(t, r.standard_normal((2, n, c, d))) for n, c in ((sq, h), (sq, h), (sk, g), (sk, g)))
        table = stored("f32", r.standard_normal((8, h)))
        table[0, 0] = table[3, 1] = table[6, 1] = -np.inf   # (a causal first query sees the first key only, of bucket 0)
        lengths = ((sq, sq - 3), (sk, 1), None)
        device = np.where(np.isinf(table), np.float32(low), table.astype(np.float32))
        dq_, dk_, dv_, ddo, dt = (upload(singa, dev, kind, x) for kind, x in ((t, q), (t, k), (t, v), (t, do), ("f32", device)))
        dl = dict(q_lengths=ints(singa, dev, lengths[0]), k_lengths=ints(singa, dev, lengths[1]))
        H = handle(singa, dq_, dk_, a)
        o, lse = singa.AttentionForward(H, dq_, dk_, dv_, dt, **dl)
        grads = [x.to_numpy() for x in singa.AttentionBackward(H, ddo, dq_, dk_, dv_, o, lse, dt, **dl)]
        assert all(np.isfinite(x).all() for x in grads)
        if causal:   # the first query of head 0 has no key left
            assert (lse.to_numpy()[:, 0, 0] == -np.inf).all() and not o.to_numpy()[:, 0, 0].any() and not grads[0][:, 0, 0].any()
        assert not grads[3][np.isinf(table)].any()
        check(singa, dev, t, a, 2, sq, sk, h, g, d, case=(q, k, v, do, table), lengths=lengths)
        hidden = upload(singa, dev, "f32", table)   # the same bits as of -inf
        again = singa.AttentionForward(H, dq_, dk_, dv_, hidden, **dl)
        for x, y in zip((o, lse), again):
            assert np.array_equal(x.to_numpy(), y.to_numpy())
        for x, y in zip(grads, singa.AttentionBackward(H, ddo, dq_, dk_, dv_, *again, hidden, **dl)):
            assert np.array_equal(x, y.to_numpy())


@pytest.mark.parametrize("t", TYPES)
def test_few_queries_and_hidden_keys(dev, t):
    """The form for few queries, its keys in parts: a bias of fp32's lowest value for all keys but those of one bucket, and for all."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(2)
    a = O.Attn(True, buckets=8, max_distance=16, bidirectional=False)
    q, k, v = (stored(t, r.standard_normal(s)) for s in ((2, 1, 4, 64), (2, 1500, 2, 64), (2, 1500, 2, 64)))
    for some in (True, False):
        table = np.full((8, 4), np.finfo(np.float32).min, np.float32)
        if some:
            table[2] = 0.5   # the key two places back
        dq_, dk_, dv_, dt = upload(singa, dev, t, q), upload(singa, dev, t, k), upload(singa, dev, t, v), upload(singa, dev, "f32", table)
        o, lse = singa.AttentionForward(handle(singa, dq_, dk_, a), dq_, dk_, dv_, dt)
        if some:
            want = np.repeat(v[:, 1497:1498], 2, 2)
            close(o.to_numpy(), want, (HALF[t] * 2 + 4 * U) * np.abs(want) + TINY[t], "o")   # (p is 1, o and p v are rounded)
        else:
            assert not o.to_numpy().any() and (lse.to_numpy() == -np.inf).all()


def _part(singa, dev, t, at, shape):
    """`shape` elements of a bfloat16 tensor from the element `at` on, as a view over its memory."""
    return singa.from_device_pointer(t.ptr + at * 2, shape, dev, singa.kBFloat16, keepalive=t)


def _zeros(singa, dev, shape):
    t = singa.Tensor(shape, dev, singa.kBFloat16)
    t.SetFloatValue(0.0)
    return t


def test_gradients_of_a_long_cache_with_offsets_beyond_32_bits(dev):
    """Keys of 2^32 bytes for a sequence: the last sequence's last rows are not zeros, nor are the gradients there."""
    from singa_amd import singa_wrap as singa
    b, sk, g, d, rows, scale = 2, 1 << 20, 16, 128, 300, 128 ** -0.5
    r = np.random.default_rng(9)
    k = _zeros(singa, dev, (b, sk, g, d))
    tail = stored("bf16", r.standard_normal((rows, g, d)))
    _part(singa, dev, k, k.Size() - tail.size, tail.shape).CopyHalfDataFromHostPtr(singa.float_to_bf16_bits(tail))
    q, do = (stored("bf16", r.standard_normal((b, 1, g, d))) for _ in range(2))
    dq_, ddo = upload(singa, dev, "bf16", q), upload(singa, dev, "bf16", do)
    H = singa.AttentionHandle(dq_, k)
    o, lse = singa.AttentionForward(H, dq_, k, k)
    dq, dk, dv, _ = singa.AttentionBackward(H, ddo, dq_, k, k, o, lse)
    o, lse = o.to_numpy().astype(np.float64), lse.to_numpy().astype(np.float64)[:, :, 0]
    read = lambda t, at, shape: _part(singa, dev, t, at, shape).to_numpy().astype(np.float64)
    row, half = g * d, HALF["bf16"]
    # a probability is off by the product's (d + 4) u, 4 u of the logarithm (14) and of the score (below 30): E; then as in the module's description
    E = (d + 4 + 4 * 44 + 8) * U
    gap_size = (np.abs(do[1, 0]) * np.abs(o[1, 0])).sum(1)
    s = np.einsum("hd,rhd->rh", q[1, 0], tail) * scale
    size = np.einsum("hd,rhd->rh", np.abs(q[1, 0]), np.abs(tail)) * scale
    p = np.exp(s - lse[1])
    gap = np.einsum("hd,rhd->rh", do[1, 0], tail) - (do[1, 0] * o[1, 0]).sum(1)
    off = p * (np.abs(gap) * E * (1 + size) + (d + 4) * U * (np.einsum("hd,rhd->rh", np.abs(do[1, 0]), np.abs(tail)) + gap_size))
    want = p[:, :, None] * do[1, 0]
    close(read(dv, dv.Size() - tail.size, tail.shape), want, (2 * half + E * (1 + size[:, :, None])) * np.abs(want) * 1.01, "dv")
    want = scale * (p * gap)[:, :, None] * q[1, 0]
    close(read(dk, dk.Size() - tail.size, tail.shape), want, (2 * half * np.abs(want) + scale * off[:, :, None] * np.abs(q[1, 0])) * 1.01, "dk")
    want = scale * np.einsum("rh,rhd->hd", p * gap, tail)
    room = scale * np.einsum("rh,rhd->hd", off + (half + 400 * U) * np.abs(p * gap), np.abs(tail)) + half * np.abs(want)
    close(dq.to_numpy()[1, 0], want, room * 1.01, "dq")
    # keys of zeros on both sides of where a sequence ends: a probability of e^-lse, do . v of 0
    for i, at in ((0, 0), (0, (sk - 5) * row), (1, sk * row), (1, (2 * sk - rows - 5) * row)):
        each = np.exp(-lse[i])[:, None]
        want = np.broadcast_to(each * do[i, 0], (5, g, d))
        close(read(dv, at, (5, g, d)), want, (2 * half + E) * np.abs(want) * 1.01, "dv of zeros")
        want = np.broadcast_to(-scale * each * (do[i, 0] * o[i, 0]).sum(1)[:, None] * q[i, 0], (5, g, d))
        room = 2 * half * np.abs(want) + scale * each * (E + (d + 4) * U) * (np.abs(do[i, 0]) * np.abs(o[i, 0])).sum(1)[:, None] * np.abs(q[i, 0])
        close(read(dk, at, (5, g, d)), want, room * 1.01, "dk of zeros")
    assert not dq.to_numpy()[0].any()


def test_gradients_of_long_sequences_with_offsets_beyond_32_bits(dev):
    """Queries of 2^32 bytes for a sequence: only the last sequence's last rows are not zeros."""
    from singa_amd import singa_wrap as singa
    b, sq, sk, h, d, rows = 2, 1 << 20, 40, 16, 128, 300
    r = np.random.default_rng(10)
    q, do = (stored("bf16", r.standard_normal((1, rows, h, d))) for _ in range(2))
    k, v = (stored("bf16", r.standard_normal((b, sk, h, d))) for _ in range(2))
    dq_, ddo = _zeros(singa, dev, (b, sq, h, d)), _zeros(singa, dev, (b, sq, h, d))
    for t, x in ((dq_, q), (ddo, do)):
        _part(singa, dev, t, t.Size() - x.size, x.shape).CopyHalfDataFromHostPtr(singa.float_to_bf16_bits(x))
    dk_, dv_ = upload(singa, dev, "bf16", k), upload(singa, dev, "bf16", v)
    H = singa.AttentionHandle(dq_, dk_)
    o, lse = singa.AttentionForward(H, dq_, dk_, dv_)
    dq, dk, dv, _ = singa.AttentionBackward(H, ddo, dq_, dk_, dv_, o, lse)
    read = lambda t, at, shape: _part(singa, dev, t, at, shape).to_numpy().astype(np.float64)
    tail_o = read(o, o.Size() - q.size, q.shape)
    a, K, V = O.Attn(), k[1:], v[1:]
    wo, wl = O.attention(a, q, K, V)
    eo, el, eq, ek, ev, _ = bounds("bf16", a, do, q, K, V, tail_o, None, None, None, None)
    rounded = lambda bound, want: bound * 1.01 + HALF["bf16"] * np.abs(want) * 1.01
    close(tail_o, wo, rounded(eo, wo), "o")
    tail_lse = lse.to_numpy()[1:, :, sq - rows:]
    close(tail_lse, wl, el * 1.01, "lse")
    want = O.attention_bwd(a, do, q, K, V, tail_o, tail_lse.astype(np.float64))
    close(read(dq, dq.Size() - q.size, q.shape), want[0], rounded(eq, want[0]), "dq")
    for name, x, w, e in (("dk", dk, want[1], ek), ("dv", dv, want[2], ev)):   # (rows without a gradient add zeros)
        x = x.to_numpy()
        close(x[1:], w, rounded(e, w), name)
        assert not x[0].any(), name
    for at in (0, (sq - 3) * h * d, sq * h * d, (2 * sq - rows - 3) * h * d):
        assert not read(dq, at, (3, h, d)).any()
        i = at // (sq * h * d)
        mean = np.broadcast_to(v[i].mean(0), (3, h, d))   # a query of zeros sees all keys alike
        close(read(o, at, (3, h, d)), mean, (2 * HALF["bf16"] + 200 * U) * np.abs(v[i]).mean(0) * 1.01, "o of zeros")
