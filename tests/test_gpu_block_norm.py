"""The norms around a block on the GPU against their definitions in 64 bits (oracle/block_ops.py).

Tolerances, first order, u = 2^-24 half a step of fp32 and h of the tensors' type.  A root is off by (n / 2 + 4) u of itself for a row of n; every
further operation by one u of its result's size."""
import numpy as np
import pytest

from oracle import block_ops as O
from test_gpu_token_model import HALF, TINY, TYPES, U, close, shifted, stored, upload

pytestmark = pytest.mark.gpu
# one value, less than a vector, a vector and one more, every team's last row and the next longer one
DIMS = [1, 3, 7, 8, 9, 63, 64, 65, 250, 257, 512, 513, 1001, 1025, 2049, 4097, 8192, 8193, 16384]
# (a block's result, a norm behind it, a norm before the next)
FORMS = [(False, False, True), (True, False, False), (True, False, True), (True, True, False), (True, True, True)]


def check(singa, dev, t, rows, dim, form, gates, scale=0.75, shift=0, no_dy=False, eps=1e-5):
    r = np.random.default_rng(rows + dim + gates)
    block, after, before = form
    x, dy, dn = (stored(t, r.standard_normal((rows, dim))) for _ in range(3))
    h = stored(t, r.standard_normal((rows, dim))) if block else None
    post = stored("f32", 1 + 0.2 * r.standard_normal(dim)) if after else None
    pre = stored("f32", 1 + 0.2 * r.standard_normal(dim)) if before else None
    gate = stored(t, r.standard_normal((gates, dim))) if gates else None
    if not before:
        dn = None
    put = lambda a, k=t: None if a is None else shifted(singa, dev, k, a, shift) if shift else upload(singa, dev, k, a)
    given = dict(post=put(post, "f32"), gate=put(gate), scale=scale, pre=put(pre, "f32"))
    dx_, dh_ = put(x), put(h)
    y, n, stats = singa.ResidualNormForward(dx_, dh_, eps=eps, **given)
    wy, wn, ws = O.residual_norm(x, h, post, gate, scale, pre, eps)
    root = (dim / 2 + 8) * U
    size = np.abs(wy) * 0
    if block:
        g = 1.0 if gate is None else np.repeat(np.abs(gate), rows // gates, 0)
        size = scale * g * np.abs(h) * (1.0 if post is None else ws[:, :1] * np.abs(post))
        ey = (root + 6 * U) * size + U * np.abs(wy)
        close(y.to_numpy(), wy, ey * 1.01 + HALF[t] * np.abs(wy) * 1.01 + TINY[t], "y")
    else:
        assert y is dx_
        ey = np.zeros_like(wy)
    rel = (ey * np.abs(wy)).mean(1) * ws[:, 1] ** 2 + root   # of the second root
    close(stats.to_numpy(), ws, np.stack([root * ws[:, 0], rel * ws[:, 1]], 1) * 1.01, "stats")
    if before:
        en = ws[:, 1:] * np.abs(pre) * ey + (rel[:, None] + 3 * U) * np.abs(wn)
        close(n.to_numpy(), wn, en * 1.01 + HALF[t] * np.abs(wn) * 1.01 + TINY[t], "n")
    else:
        assert n is None

    ddy, ddn = None if no_dy else put(dy), put(dn)
    got = singa.ResidualNormBackward(ddy, ddn, y, stats, dh_, **given)
    y64, s64 = y.to_numpy().astype(np.float64), stats.to_numpy().astype(np.float64)
    want = O.residual_norm_bwd(None if no_dy else dy, dn, y64, s64, h, post, gate, scale, pre)
    et = np.zeros((rows, dim))
    if before:
        s = s64[:, 1:]
        w = np.abs(dn * pre)
        et = (dim + 8) * U * (s * w + np.abs(y64) * s ** 3 * (w * np.abs(y64)).mean(1, keepdims=True))
        sums = np.abs(dn * y64 * s).sum(0)
        close(got[4].to_numpy(), want[4], (rows + 4) * U * sums * 1.01, "dpre")
    et = et + 2 * U * np.abs(want[0])
    close(got[0].to_numpy(), want[0], et * 1.01 + HALF[t] * np.abs(want[0]) * 1.01 + TINY[t], "dx")
    if block:
        g = np.ones((rows, 1)) if gate is None else np.repeat(np.abs(gate), rows // gates, 0)
        T, A, s, p = np.abs(want[0]), np.abs(h), s64[:, :1] if after else 1.0, np.abs(post) if after else 1.0
        eb, b = scale * g * p * (et + 6 * U * T), scale * g * p * T
        eh = eb
        if after:
            eh = s * eb + A * s ** 3 * (eb * A).mean(1, keepdims=True) + (dim + 8) * U * (s * b + A * s ** 3 * (b * A).mean(1, keepdims=True))
            close(got[2].to_numpy(), want[2], ((scale * g * A * s * (et + 8 * U * T)).sum(0) + (rows + 4) * U * (scale * g * A * s * T).sum(0)) * 1.01, "dpost")
        close(got[1].to_numpy(), want[1], eh * 1.01 + HALF[t] * np.abs(want[1]) * 1.01 + TINY[t], "dh")
        if gates:
            each = (scale * A * s * p * (et + 8 * U * T)).reshape(gates, -1, dim).sum(1)
            each += (rows // gates + 4) * U * (scale * A * s * p * T).reshape(gates, -1, dim).sum(1)
            close(got[3].to_numpy(), want[3], each * 1.01 + HALF[t] * np.abs(want[3]) * 1.01 + TINY[t], "dgate")
    for i, there in enumerate((True, block, after, gates, before)):
        assert (got[i] is not None) == bool(there)
    again = singa.ResidualNormBackward(ddy, ddn, y, stats, dh_, **given)
    assert all(a is b is None or np.array_equal(a.to_numpy(), b.to_numpy()) for a, b in zip(got, again))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", DIMS)
def test_rows_of_every_length(dev, t, form, dim):
    from singa_amd import singa_wrap as singa
    for gates in (0, 1, 3, 6) if form[0] else (0,):
        check(singa, dev, t, 6, dim, form, gates)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim,gates", [(1, 40, 1), (2, 1025, 2), (5000, 8, 10), (4999, 64, 4999), (9000, 100, 3000), (7000, 200, 7), (3003, 513, 3),
                                            (2600, 1030, 2), (2048, 2049, 128), (1100, 5000, 1), (700, 9001, 350), (601, 16384, 1), (30000, 33, 0),
                                            (40000, 16, 40000)])
def test_rows_of_every_count(dev, t, rows, dim, gates):
    """Several rows to a team, parts of a gate's rows, whole gates, more gates than teams; teams without a row."""
    from singa_amd import singa_wrap as singa
    check(singa, dev, t, rows, dim, (True, True, True), gates)
    check(singa, dev, t, rows, dim, (True, False, True), gates)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [5, 64, 1001, 8193])
def test_rows_at_any_element(dev, t, dim):
    from singa_amd import singa_wrap as singa
    for shift in (1, 3):
        check(singa, dev, t, 50, dim, (True, True, True), 5, shift=shift)
    check(singa, dev, t, 50, dim, (True, True, True), 5, no_dy=True)
    check(singa, dev, t, 50, dim, (False, False, True), 0, scale=1.0, no_dy=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [64, 4096, 10000])
def test_rows_of_zeros_and_of_nan(dev, t, dim):
    """A row of zeros has a root of eps^-0.5 and finite gradients; a row with a NaN is NaN, and its neighbours are not."""
    from singa_amd import singa_wrap as singa
    rows = 9
    x, h = np.ones((rows, dim), np.float32), np.ones((rows, dim), np.float32)
    x[3] = h[3] = 0
    x[5, dim - 1] = np.nan
    ones = upload(singa, dev, "f32", np.ones(dim))
    put = lambda a: upload(singa, dev, t, a)
    y, n, stats = singa.ResidualNormForward(put(x), put(h), post=ones, pre=ones)
    s, z = stats.to_numpy(), n.to_numpy()
    np.testing.assert_allclose(s[3], 1e-5 ** -0.5, rtol=4e-7)
    assert not z[3].any() and np.isnan(z[5]).all() and np.isfinite(np.delete(z, 5, 0)).all()
    one = put(np.ones((rows, dim)))
    dx, dh, dpost, _, dpre = singa.ResidualNormBackward(one, one, y, stats, put(h), post=ones, pre=ones)
    for a in (dx, dh):
        a = a.to_numpy()
        assert np.isnan(a[5]).any() and np.isfinite(np.delete(a, (3, 5), 0)).all()
    # in front of a row of zeros the gradient grows by both roots: 1 + 316, times 316 is 1e5, more than binary16 has
    np.testing.assert_allclose(dx.to_numpy()[3], float(stored(t, [1 + 1e-5 ** -0.5])[0]), rtol=2 * HALF[t])
    want = np.inf if t == "f16" else (1 + 1e-5 ** -0.5) * 1e-5 ** -0.5
    np.testing.assert_allclose(dh.to_numpy()[3], want, rtol=2 * HALF[t])
    assert np.isnan(dpre.to_numpy()).any()


def test_no_rows(dev):
    from singa_amd import singa_wrap as singa
    x, w = singa.Tensor((0, 12), dev), upload(singa, dev, "f32", np.ones(12))
    y, n, stats = singa.ResidualNormForward(x, x, post=w, pre=w)
    got = singa.ResidualNormBackward(x, x, y, stats, x, post=w, pre=w)
    assert n.shape() == [0, 12] and not got[2].to_numpy().any() and not got[4].to_numpy().any()


def test_gradients_against_differences(dev):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(3)
    rows, dim, gates, scale = 12, 70, 4, 0.6
    x, h, dy, dn = (stored("f32", r.standard_normal((rows, dim))) for _ in range(4))
    post, pre, gate = (stored("f32", 1 + 0.3 * r.standard_normal(s)) for s in ((dim,), (dim,), (gates, dim)))
    put = lambda a: upload(singa, dev, "f32", a)
    given = dict(post=put(post), gate=put(gate), scale=scale, pre=put(pre))
    y, _, stats = singa.ResidualNormForward(put(x), put(h), **given)
    got = singa.ResidualNormBackward(put(dy), put(dn), y, stats, put(h), **given)

    def value(x, h, post, gate, pre):
        y, n, _ = O.residual_norm(x, h, post, gate, scale, pre)
        return (y * dy).sum() + (n * dn).sum()

    args, step = [x, h, post, gate, pre], 1e-5
    for i, g in enumerate(got):
        along = r.standard_normal(args[i].shape)
        ends = [value(*[a + s * step * along if j == i else a for j, a in enumerate(args)]) for s in (1, -1)]
        want = (ends[0] - ends[1]) / (2 * step)
        # (fp32 gradients: 1e-6 of their sizes; differences in 64 bits of values of up to 1e4: 1e-12 / 1e-5)
        assert abs((g.to_numpy() * along).sum() - want) < 2e-5 * np.abs(g.to_numpy() * along).sum() + 1e-5, i


@pytest.mark.parametrize("t", TYPES)
def test_recorded_calls_replay(dev, t):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(4)
    made = []
    for rows, dim, gates in ((700, 96, 7), (40, 9000, 40), (3000, 257, 1)):
        made.append(([upload(singa, dev, t, r.standard_normal((rows, dim))) for _ in range(4)], upload(singa, dev, t, r.standard_normal((gates, dim))),
                     upload(singa, dev, "f32", 1 + 0.1 * r.standard_normal(dim))))

    def run():
        out = []
        for (x, h, dy, dn), gate, w in made:
            y, n, stats = singa.ResidualNormForward(x, h, w, gate, 0.5, w)
            out += [y, n, stats, *singa.ResidualNormBackward(dy, dn, y, stats, h, w, gate, 0.5, w)]
        return out

    run()
    dev.Sync()
    dev.EnableGraph(True)
    kept = run()
    dev.EnableGraph(False)
    try:
        for turn in range(4):
            for ts, _, _ in made:
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
@pytest.mark.parametrize("gates", [0, 1, 5])
def test_no_rows_and_a_gate(dev, t, gates):
    from singa_amd import singa_wrap as singa
    w = upload(singa, dev, "f32", np.ones(12))
    kind = upload(singa, dev, t, [0.0]).data_type()
    x, gate = singa.Tensor((0, 12), dev, kind), singa.Tensor((0, 12), dev, kind) if gates == 0 else upload(singa, dev, t, np.ones((gates, 12)))
    y, n, stats = singa.ResidualNormForward(x, x, w, gate, 0.5, w)
    dx, dh, dpost, dgate, dpre = singa.ResidualNormBackward(x, x, y, stats, x, w, gate, 0.5, w)
    assert y.shape() == n.shape() == dx.shape() == dh.shape() == [0, 12] and stats.shape() == [0, 2] and dgate.shape() == [gates, 12]
    for g in (dpost, dgate, dpre):
        assert not g.to_numpy().any()


@pytest.mark.parametrize("dim,gates", [(16384, 1), (4096, 2), (1000, 0)])
def test_tensors_of_more_than_32_bits(dev, dim, gates):
    """More than 2^32 values, zeros but for the last row: the same bits as of that row alone, zeros where a shorter offset would have put them."""
    from singa_amd import singa_wrap as singa
    rows = ((1 << 32) // dim + 300) // 4 * 4
    r = np.random.default_rng(dim)
    f = lambda t, row, n=1: singa.from_device_pointer(t.ptr + row * dim * 2, (n, dim), dev, singa.kBFloat16, keepalive=t)
    kept = [stored("bf16", r.standard_normal((1, dim))) for _ in range(4)]
    large = []
    for x in kept:
        t = singa.Tensor((rows, dim), dev, singa.kBFloat16)
        t.SetFloatValue(0.0)
        f(t, rows - 1).CopyHalfDataFromHostPtr(singa.float_to_bf16_bits(x))
        large.append(t)
    post, pre = (upload(singa, dev, "f32", 1 + 0.2 * r.standard_normal(dim)) for _ in range(2))
    gate = stored("bf16", r.standard_normal((max(gates, 1), dim)))

    def run(tensors, gate):
        x, h, dy, dn = tensors
        given = dict(post=post, gate=None if gate is None else upload(singa, dev, "bf16", gate), scale=0.5, pre=pre)
        y, n, stats = singa.ResidualNormForward(x, h, **given)
        return [y, n, stats, *singa.ResidualNormBackward(dy, dn, y, stats, h, **given)]

    got = run(large, gate if gates else None)
    want = run([upload(singa, dev, "bf16", x) for x in kept], gate[-1:] if gates else None)
    for name, x, w in zip(("y", "n", "stats", "dx", "dh", "dpost", "dgate", "dpre"), got, want):
        if name in ("y", "n", "dx", "dh"):
            assert np.array_equal(f(x, rows - 1).to_numpy(), w.to_numpy()), name
            for row in (0, rows - 2, rows - 1 - (1 << 31) // dim, rows - 2 - (1 << 31) // dim, rows - 1 - (1 << 32) // dim, rows - 2 - (1 << 32) // dim):
                assert not f(x, row).to_numpy().any(), (name, row)
        elif name == "stats":
            x = x.to_numpy()
            assert np.array_equal(x[-1], w.to_numpy()[0]) and (x[:-1] == x[0]).all()
        elif w is not None:   # (a sum of one row's and zeros)
            assert np.array_equal(x.to_numpy()[-1:] if name == "dgate" else x.to_numpy(), w.to_numpy()), name
            assert name != "dgate" or not x.to_numpy()[:-1].any()
