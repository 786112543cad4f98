"""The token model's operators on the GPU against their definitions in 64 bits (oracle/token_ops.py): token vectors and their gradient,
the distillation loss and its gradient, at the sizes, types and masks where they can go wrong.

Tolerances.  u = 2^-24 is half a step of fp32, `half(t)` half a step of the storage type.  A sum of n fp32 terms in any order is off by at
most n u sum |terms| (first order; n + 2 covers the products around it).  exp of d / tau: the difference d = x - m is rounded once, multiplied
by a rounded constant, and the instruction is good to one step, so its relative error is at most (4 |d| / tau + 4) u."""
import numpy as np
import pytest

from oracle import token_ops as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}   # half of the smallest subnormal
TYPES = ["f32", "f16", "bf16"]


def kind(singa, t):
    return {"f32": singa.kFloat32, "f16": singa.kFloat16, "bf16": singa.kBFloat16}[t]


def stored(t, a):
    """The values of `a` as the type holds them, as float64."""
    from singa_amd.singa_wrap import bf16_bits_to_float, float_to_bf16_bits
    a = np.asarray(a, np.float32)
    if t == "f16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16).astype(np.float64)
    return (bf16_bits_to_float(float_to_bf16_bits(a)) if t == "bf16" else a).astype(np.float64)


def upload(singa, dev, t, a):
    from singa_amd.singa_wrap import float_to_bf16_bits
    a = np.asarray(a, np.float32)
    out = singa.Tensor(a.shape, dev, kind(singa, t))
    if t == "f32":
        out.CopyFloatDataFromHostPtr(a)
    else:
        with np.errstate(over="ignore"):
            out.CopyHalfDataFromHostPtr(a.astype(np.float16) if t == "f16" else float_to_bf16_bits(a))
    return out


def shifted(singa, dev, t, a, by):
    """`a` on the device, `by` elements behind the start of its memory."""
    a = np.asarray(a, np.float32)
    flat = upload(singa, dev, t, np.concatenate([np.full(by, 7.0, np.float32), a.ravel(), np.full(8, 7.0, np.float32)]))
    size = 4 if t == "f32" else 2
    return singa.from_device_pointer(flat.ptr + by * size, a.shape, dev, kind(singa, t), keepalive=flat)


def ints(singa, dev, a):
    return singa.from_numpy(np.asarray(a, np.int32), dev)


def close(got, want, bound, what):
    got, want, bound = (np.asarray(v, np.float64) for v in (got, want, bound))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound) & ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), "%s: %d of %d, first at %s: %r for %r, %r allowed" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0].tolist(), got[bad][0], want[bad][0], np.broadcast_to(bound, got.shape)[bad][0])


# ------------------------------------------------------------------------------------ token vectors

# (tokens, vocab, dim): one value, less than a vector of either type, a vector, one more, a wavefront's worth and more, odd ones
FWD = [(1, 1, 1), (3, 5, 3), (7, 5, 4), (9, 11, 7), (5, 3, 8), (2, 10, 9), (64, 100, 16), (33, 50, 33), (1000, 37, 201), (5, 1000, 1000),
       (3, 4, 2047), (2, 10, 4097), (300, 2, 513)]


def some_ids(r, tokens, vocab, pad):
    ids = r.integers(0, vocab, tokens)
    ids[r.random(tokens) < 0.2] = pad
    return ids


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim", FWD)
def test_embedding_forward(dev, t, tokens, vocab, dim):
    """One rounding of one fp32 product: the bits are known."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(tokens + dim)
    W = stored(t, r.standard_normal((vocab, dim)))
    pad = vocab // 2
    ids = some_ids(r, tokens, vocab, pad)
    scale = float(np.float32(np.sqrt(dim)))
    want = stored(t, O.embedding_fwd(ids, W.astype(np.float32) * np.float32(scale), 1.0, pad))
    for W_ in (upload(singa, dev, t, W), shifted(singa, dev, t, W, 1)):
        y = singa.EmbeddingForward(ints(singa, dev, ids), W_, scale=scale, padding_idx=pad)
        assert y.shape() == [tokens, dim]
        assert np.array_equal(y.to_numpy().astype(np.float64), want)
    assert singa.IndexErrors(dev) == 0


def test_embedding_ids_outside_the_table_are_zeros_and_counted(dev):
    from singa_amd import singa_wrap as singa
    W = np.ones((6, 200), np.float32)
    ids = np.array([[0, 6, -1], [5, -7, 2147483647]])
    singa.IndexErrors(dev)
    d_ids, d_W = ints(singa, dev, ids), upload(singa, dev, "f32", W)
    y = singa.EmbeddingForward(d_ids, d_W, scale=2.0)
    assert y.shape() == [2, 3, 200] and np.array_equal(y.to_numpy(), O.embedding_fwd(ids, W, 2.0))
    assert singa.IndexErrors(dev) == 3 and singa.IndexErrors(dev) == 0   # (-1 is padding here)
    dW = singa.EmbeddingBackwardW(y, d_ids, d_W, scale=2.0)
    assert singa.IndexErrors(dev) == 3
    assert np.array_equal(dW.to_numpy(), O.embedding_bwd(y.to_numpy(), ids, (6, 200), 2.0))
    many = np.tile(ids.ravel(), 400)   # (behind the sort)
    dW = singa.EmbeddingBackwardW(upload(singa, dev, "f32", np.ones((2400, 200))), ints(singa, dev, many), d_W)
    assert singa.IndexErrors(dev) == 1200
    assert np.array_equal(dW.to_numpy()[[0, 5]], np.full((2, 200), 400.0)) and not dW.to_numpy()[1:5].any()


# few tokens (looked through), then sorted ones: one pass of digits, two, three; more than one stretch; whole tiles of one row
BWD = [(0, 5, 3), (1, 1, 1), (3, 5, 3), (7, 5, 4), (9, 300, 7), (5, 3, 8), (64, 100, 16), (500, 1000, 201), (1024, 37, 100), (1000, 700, 513), (512, 37, 100), (513, 37, 100), (512, 3, 600), (700, 2, 2100),
       (1025, 3, 5), (1500, 300, 33), (3000, 10000, 64), (5000, 600, 129), (4097, 300000, 3), (9000, 77, 520), (20000, 1, 9), (12289, 5000, 40),
       (8192, 900, 20), (8193, 511, 33), (17001, 512, 64), (70000, 3000, 24), (18000, 262144, 2)]


def bwd_bound(t, want, terms, counts, scale):
    """`terms`: sum of |dy| (times scale) in every place, plus |add|"""
    return (counts[:, None] + 3) * U * terms + HALF[t] * np.abs(want) * 1.01 + TINY[t]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim", BWD)
def test_embedding_gradient(dev, t, tokens, vocab, dim):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(tokens + dim)
    pad, scale = vocab // 3, 1.5
    ids = np.minimum((vocab + 1.0) ** r.random(tokens) - 1, vocab - 1).astype(np.int64)   # few ids often, many seldom
    ids[r.random(tokens) < 0.1] = pad if vocab > 1 else -1
    pad = pad if vocab > 1 else -1
    dy, add = stored(t, r.standard_normal((tokens, dim))), stored(t, r.standard_normal((vocab, dim)))
    counts = np.bincount(ids[ids != pad], minlength=vocab)
    size = O.embedding_bwd(np.abs(dy), ids, (vocab, dim), scale, pad)
    d_ids, d_dy, d_W = ints(singa, dev, ids), upload(singa, dev, t, dy), upload(singa, dev, t, add)
    want = O.embedding_bwd(dy, ids, (vocab, dim), scale, pad)
    got = singa.EmbeddingBackwardW(d_dy, d_ids, d_W, scale=scale, padding_idx=pad)
    close(got.to_numpy(), want, bwd_bound(t, want, size, counts, scale), "dW")
    again = singa.EmbeddingBackwardW(d_dy, d_ids, d_W, scale=scale, padding_idx=pad)
    assert np.array_equal(again.to_numpy(), got.to_numpy())
    # onto another gradient, into a new tensor and in place; rows without a token keep its bits
    both = want + add
    bound = bwd_bound(t, both, size + np.abs(add), counts, scale)
    out = singa.EmbeddingBackwardW(d_dy, d_ids, d_W, scale=scale, padding_idx=pad, add=d_W)
    close(out.to_numpy(), both, bound, "dW + add")
    assert np.array_equal(d_W.to_numpy().astype(np.float64), add)
    place = shifted(singa, dev, t, add, 3)
    assert singa.EmbeddingBackwardW(shifted(singa, dev, t, dy, 1), d_ids, d_W, scale=scale, padding_idx=pad, add=place, out=place) is place
    assert np.array_equal(place.to_numpy(), out.to_numpy())
    assert np.array_equal(place.to_numpy()[counts == 0].astype(np.float64), add[counts == 0])
    edges = place._block.keepalive.to_numpy()
    assert (edges[:3] == 7).all() and (edges[-8:] == 7).all()
    assert singa.IndexErrors(dev) == 0


@pytest.mark.parametrize("tokens", [1000, 6000])
def test_embedding_gradient_against_differences(dev, tokens):
    """sum(c * forward(W)) is linear in W: its difference along a direction is <dW, direction>."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(4)
    vocab, dim = 500, 24
    ids = r.integers(0, vocab, tokens)
    W, along, c = (r.standard_normal(s).astype(np.float32) for s in ((vocab, dim), (vocab, dim), (tokens, dim)))
    d_ids = ints(singa, dev, ids)

    def f(w):
        y = singa.EmbeddingForward(d_ids, upload(singa, dev, "f32", w), scale=3.0, padding_idx=7).to_numpy()
        return float((y.astype(np.float64) * c).sum())

    dW = singa.EmbeddingBackwardW(upload(singa, dev, "f32", c), d_ids, upload(singa, dev, "f32", W), scale=3.0, padding_idx=7).to_numpy()
    size = np.abs(c).sum() * 3.0 * (np.abs(W).max() + np.abs(along).max())
    got, want = f(W + along) - f(W), float((dW.astype(np.float64) * along).sum())
    # (W + along rounds once, y once in each pass; the sums of dW are of tokens / vocab terms)
    assert abs(got - want) <= 8 * U * size * 3


def test_embedding_gradient_of_one_row_with_all_tokens(dev):
    """Whole tiles of one row, their joining, and the ends of the row's tokens."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(5)
    for tokens, other in ((64, 0), (130, 65), (512, 0), (513, 0), (1000, 400), (4096, 0), (4097, 1), (70001, 63)):
        ids = np.full(tokens, 2)
        ids[:other] = 0
        dy = r.integers(-8, 9, (tokens, 12)).astype(np.float32)   # (sums of whole numbers: exact in any order)
        W = upload(singa, dev, "f32", np.zeros((4, 12)))
        dW = singa.EmbeddingBackwardW(upload(singa, dev, "f32", dy), ints(singa, dev, ids), W)
        assert np.array_equal(dW.to_numpy(), O.embedding_bwd(dy, ids, (4, 12)))


@pytest.mark.parametrize("tokens,dim", [(1025, 256), (8192, 256), (700, 400), (5001, 400), (9000, 400)])
def test_embedding_gradient_beside_a_large_table(dev, tokens, dim):
    """Rows without a token of more than 64 and 96 MB beside the sort; sums of whole numbers are exact."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(8)
    vocab = 66001
    ids = np.where(r.random(tokens) < 0.3, r.integers(0, 5, tokens), r.integers(-2, vocab + 2, tokens))
    dy = r.integers(-8, 9, (tokens, dim)).astype(np.float32)
    want = np.zeros((vocab, dim), np.float32)
    known = (ids >= 0) & (ids < vocab)
    np.add.at(want, ids[known], dy[known])
    singa.IndexErrors(dev)
    out = singa.Tensor((vocab, dim), dev)
    out.SetFloatValue(9.0)
    assert singa.EmbeddingBackwardW(upload(singa, dev, "f32", dy), ints(singa, dev, ids), out, out=out) is out
    assert np.array_equal(out.to_numpy(), want)
    assert singa.IndexErrors(dev) == int((~known & (ids != -1)).sum())


@pytest.mark.parametrize("dim", [400, 403])
def test_embedding_forward_of_more_than_the_caches(dev, dim):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(9)
    W, ids = r.standard_normal((900, dim)).astype(np.float32), r.integers(0, 900, 70000)
    y = singa.EmbeddingForward(ints(singa, dev, ids), upload(singa, dev, "f32", W), scale=0.5)
    assert np.array_equal(y.to_numpy(), (0.5 * W)[ids])


def test_embedding_gradient_of_rows_that_end_with_a_tile(dev):
    """Rows of whole tiles side by side, of whole tiles and some, and of less than a tile, in memory that held large numbers."""
    from singa_amd import singa_wrap as singa
    from singa_amd._lib import lib
    r = np.random.default_rng(6)
    for unit in (16, 32, 64, 128, 1024):
        for runs in ([2, 2, 2, 40], [1, 3, 0.5, 0.5, 2, 30, 1], [40, 1, 0.25, 1.75, 1], [0.5, 35, 0.5, 1, 1, 1, 1.5, 2.5]):
            ids = r.permutation(np.repeat(np.arange(len(runs)), [int(n * unit) for n in runs]))
            if ids.size <= 1024:
                ids = np.concatenate([ids, np.full(1025 - ids.size, len(runs))])
            vocab, dim = len(runs) + 1, 20
            dy = r.integers(-8, 9, (ids.size, dim)).astype(np.float32)
            need = lib().sgh_embedding_bwd_workspace_bytes(ids.size, vocab, dim)
            assert need
            dirty = singa.from_numpy(np.full(need // 4, 0x7f7f7f7f, np.int32), dev)
            del dirty    # (the pool hands this block to the call)
            dW = singa.EmbeddingBackwardW(upload(singa, dev, "f32", dy), ints(singa, dev, ids), upload(singa, dev, "f32", np.zeros((vocab, dim))))
            assert np.array_equal(dW.to_numpy(), O.embedding_bwd(dy, ids, (vocab, dim)))


@pytest.mark.parametrize("t,tokens,dim", [("f16", 70000, 800), ("bf16", 70000, 807), ("f32", 8400001, 3)])
def test_embedding_forward_past_the_caches(dev, t, tokens, dim):
    """16-bit results of more than 96 MB, and rows of less than a vector."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(10)
    W = r.integers(-100, 101, (900, dim)).astype(np.float32)   # (whole numbers of at most 8 bits: every type holds them and their halves)
    ids = r.integers(-1, 900, tokens)
    y = singa.EmbeddingForward(ints(singa, dev, ids), upload(singa, dev, t, W), scale=0.5).to_numpy()
    want = np.concatenate([0.5 * W, np.zeros((1, dim), np.float32)])
    for at in range(0, tokens, 1 << 20):
        assert np.array_equal(y[at:at + (1 << 20)], want[ids[at:at + (1 << 20)]])


def whole_gradient(singa, dev, t, r, tokens, vocab, dim, ids, add=False):
    """Whole numbers of at most 3 bits: their sums are exact in fp32 in any order, the result one rounding of these."""
    dy = r.integers(-4, 5, (tokens, dim), dtype=np.int8).astype(np.float32)
    want = r.integers(-4, 5, (vocab, dim), dtype=np.int8).astype(np.float32) if add else np.zeros((vocab, dim), np.float32)
    W = upload(singa, dev, t, want) if add else singa.Tensor((vocab, dim), dev, kind(singa, t))
    known = (ids >= 0) & (ids < vocab)
    order = np.argsort(ids[known], kind="stable")
    rows, first = np.unique(ids[known][order], return_index=True)
    want[rows] += np.add.reduceat(dy[known][order], first, axis=0)
    singa.IndexErrors(dev)
    got = singa.EmbeddingBackwardW(upload(singa, dev, t, dy), ints(singa, dev, ids), W, add=W if add else None)
    assert np.array_equal(got.to_numpy().astype(np.float64), stored(t, want))
    assert singa.IndexErrors(dev) == int((~known & (ids != -1)).sum())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim", [(300, 300000, 8), (300, 300001, 16), (512, 140000, 3), (411, 262144, 1), (77, 600000, 5)])
def test_embedding_gradient_of_few_tokens_in_a_long_table(dev, t, tokens, vocab, dim):
    """Several groups of rows to a workgroup, tokens in more than one of them, more rows than a wavefront has lanes."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(41)
    near = r.integers(0, 300, tokens) + 1000 * r.integers(0, 3, tokens)        # (many in the same workgroups, some more than once)
    ids = np.where(r.random(tokens) < 0.7, near, r.integers(-3, vocab + 3, tokens))
    for add in (False, True):
        whole_gradient(singa, dev, t, r, tokens, vocab, dim, ids, add)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim", [(140000, 77, 8), (140001, 5000, 3), (270000, 5000, 7), (270001, 77, 4), (270000, 300000, 2)])
def test_embedding_gradient_of_long_stretches(dev, t, tokens, vocab, dim):
    """More tokens than 64 workgroups hold at once: each goes through its own in several turns."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(42)
    ids = np.where(r.random(tokens) < 0.1, r.integers(0, 3, tokens), r.integers(-2, vocab + 2, tokens))
    whole_gradient(singa, dev, t, r, tokens, vocab, dim, ids)


# (fp32; 16 bits: dim is twice as long) of more than 96 MB: dy alone, in jobs of eight and of four; dy and the result; the result alone, and with few tokens
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim", [(97001, 3000, 260), (9601, 700, 2653), (9001, 12001, 2800), (7000, 70001, 400), (400, 72001, 1056)])
def test_embedding_gradient_past_the_caches(dev, t, tokens, vocab, dim):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(43)
    dim *= 1 if t == "f32" else 2
    ids = np.where(r.random(tokens) < 0.2, r.integers(0, 5, tokens), r.integers(-2, vocab + 2, tokens))
    whole_gradient(singa, dev, t, r, tokens, vocab, dim, ids, add=tokens == 9601)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens", [300, 3000, 20000])   # (looked through, counted, sorted in passes)
def test_embedding_of_nan_and_infinities_where_nothing_reads(dev, t, tokens):
    """Rows of the table that are padding or that no id names, and gradients of tokens that take part in nothing."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(44)
    vocab, dim, pad = 700, 24, 5
    ids = r.integers(0, vocab // 2, tokens)
    ids[::7], ids[3::11] = pad, vocab + 1
    W = r.integers(-100, 101, (vocab, dim)).astype(np.float32)
    W[pad], W[vocab // 2:] = np.nan, np.inf
    d_ids, d_W = ints(singa, dev, ids), upload(singa, dev, t, W)
    y = singa.EmbeddingForward(d_ids, d_W, scale=0.5, padding_idx=pad).to_numpy()
    assert np.array_equal(y, O.embedding_fwd(ids, W, 0.5, pad)) and not y[::7].any()
    dy = r.integers(-4, 5, (tokens, dim)).astype(np.float32)
    out = (ids == pad) | (ids >= vocab)
    dy[out] = np.where(r.random((out.sum(), 1)) < 0.5, np.nan, np.inf)
    dy[np.flatnonzero(~out)[0]] = np.nan            # one that counts: its row alone
    got = singa.EmbeddingBackwardW(upload(singa, dev, t, dy), d_ids, d_W, padding_idx=pad).to_numpy()
    want = stored(t, O.embedding_bwd(np.where(out[:, None], 0, dy), ids, (vocab, dim), 1.0, pad))
    assert np.isnan(want).any(1).sum() == 1 and np.array_equal(got, want, equal_nan=True)
    singa.IndexErrors(dev)


@pytest.mark.parametrize("tokens,vocab", [(9000, 300), (20000, 3000), (40000, 300000), (300, 100000)])
def test_recorded_gradients_of_other_ids(dev, tokens, vocab):
    """Recorded once, replayed on other ids and gradients each time, beside eager calls of the same sizes."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(45)
    dim = 20
    ids, dy, W = ints(singa, dev, np.zeros(tokens)), upload(singa, dev, "f32", np.zeros((tokens, dim))), singa.Tensor((vocab, dim), dev)
    singa.EmbeddingBackwardW(dy, ids, W)
    dev.Sync()
    dev.EnableGraph(True)
    out = singa.EmbeddingBackwardW(dy, ids, W)
    dev.EnableGraph(False)
    try:
        for _ in range(4):
            new_ids = np.where(r.random(tokens) < 0.3, r.integers(0, 4), r.integers(0, vocab, tokens)).astype(np.int32)
            ids.CopyIntDataFromHostPtr(new_ids)
            dy.CopyFloatDataFromHostPtr(r.standard_normal((tokens, dim)).astype(np.float32))
            out.SetFloatValue(-77.0)
            eager = singa.EmbeddingBackwardW(dy, ids, W).to_numpy()
            dev.RunGraph()
            assert np.array_equal(out.to_numpy(), eager)
            counts = np.bincount(new_ids, minlength=vocab)
            assert not eager[counts == 0].any() and eager[counts > 0].any(1).all()
    finally:
        dev.ResetGraph()


def row_of(singa, dev, t, tensor, row):
    """One row of a matrix, as a tensor over its memory."""
    dim = tensor.shape()[1]
    return singa.from_device_pointer(tensor.ptr + row * dim * (4 if t == "f32" else 2), (1, dim), dev, kind(singa, t), keepalive=tensor)


def put_row(singa, dev, t, tensor, row, values):
    from singa_amd.singa_wrap import float_to_bf16_bits
    assert t == "bf16"
    row_of(singa, dev, t, tensor, row).CopyHalfDataFromHostPtr(float_to_bf16_bits(np.asarray(values, np.float32)))


def test_embedding_of_more_than_32_bits_of_elements(dev):
    """A table, a result and a gradient of 4.48e9 elements: rows on both sides of 2^31 and 2^32."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(46)
    many, dim = 70000001, 64
    far = np.array([0, 1, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, many - 1])
    values = r.integers(-100, 101, (far.size, dim)).astype(np.float32)
    big = singa.Tensor((many, dim), dev, singa.kBFloat16)
    big.SetFloatValue(2.0)
    for row, v in zip(far, values):
        put_row(singa, dev, "bf16", big, row, v)
    ids = np.concatenate([far, far + 5, far - 3, [many, -1]])
    want = np.full((ids.size, dim), 2.0, np.float32)
    want[:far.size] = values
    want[(ids < 0) | (ids >= many)] = 0
    got = singa.EmbeddingForward(ints(singa, dev, ids), big).to_numpy()
    assert np.array_equal(got, want)
    assert singa.IndexErrors(dev) == int((ids >= many).sum() + (ids < -1).sum())
    # its gradient: looked through, counted and sorted
    for tokens in (300, 3000, 9000):
        ids = far[r.integers(0, far.size, tokens)]
        dy = r.integers(-4, 5, (tokens, dim)).astype(np.float32)
        big.SetFloatValue(9.0)
        assert singa.EmbeddingBackwardW(upload(singa, dev, "bf16", dy), ints(singa, dev, ids), big, out=big) is big
        want = stored("bf16", np.stack([dy[ids == f].sum(0) for f in far]))
        for f, w in zip(far, want):
            assert np.array_equal(row_of(singa, dev, "bf16", big, f).to_numpy()[0].astype(np.float64), w)
            for near in (f - 2, f + 2):
                if 0 <= near < many:
                    assert not row_of(singa, dev, "bf16", big, near).to_numpy().any()
    # and as many tokens: each row of a small table is the sum of 70000 and more (whole numbers, exact in fp32)
    vocab = 997
    ids = (np.arange(many) * 31 % vocab).astype(np.int32)
    d_ids = ints(singa, dev, ids)
    big.SetFloatValue(1.0)
    for row, v in zip(far, values):
        put_row(singa, dev, "bf16", big, row, v)
    want = np.repeat(np.bincount(ids, minlength=vocab).astype(np.float32)[:, None], dim, 1)
    np.add.at(want, ids[far], values - 1)
    table = upload(singa, dev, "bf16", values[:1].repeat(vocab, 0) + np.arange(vocab)[:, None] % 100)
    dW = singa.EmbeddingBackwardW(big, d_ids, table)
    assert np.array_equal(dW.to_numpy().astype(np.float64), stored("bf16", want))
    del big
    y = singa.EmbeddingForward(d_ids, table)
    rows = table.to_numpy()
    for f in far:
        assert np.array_equal(row_of(singa, dev, "bf16", y, f).to_numpy()[0], rows[ids[f]])
    assert singa.IndexErrors(dev) == 0


# ------------------------------------------------------------------------------------ distillation

def make_case(r, t, n, v, k, masked=True):
    x = stored(t, r.standard_normal((n, v)) * 3)
    top = np.stack([r.permutation(max(v, k))[:k] % v for _ in range(n)]) if k else None
    teacher = (r.standard_normal((n, k)) * 2).astype(np.float32) if k else None
    labels, weights = r.integers(0, v, n), np.abs(r.standard_normal(n)).astype(np.float32) + 0.1
    if masked:
        labels[r.random(n) < 0.3] = -1
        weights[r.random(n) < 0.2] = 0
        if k:
            top[r.random((n, k)) < 0.2] = -1
            top[r.random(n) < 0.2] = -1           # rows whose list is empty
            if k > 1:
                top[0, 0] = top[0, -1] = 0        # a column twice
                teacher[n // 2, 0] = -np.inf
    return x, top, teacher, labels, weights


def run_all(singa, dev, t, x, top, teacher, labels, weights, scale=1.0, shift=0, **how):
    """(loss, stats, dx of the three entry points) as arrays; dx in place for one of them"""
    put = (lambda: shifted(singa, dev, t, x, shift)) if shift else (lambda: upload(singa, dev, t, x))
    d_top = ints(singa, dev, top) if top is not None else None
    d_teacher = singa.from_numpy(np.asarray(teacher, np.float32), dev) if teacher is not None else None
    rest = dict(labels=None if labels is None else ints(singa, dev, labels),
                weights=None if weights is None else singa.from_numpy(np.asarray(weights, np.float32), dev), **how)
    d_x = put()
    loss, stats = singa.DistillationFwd(d_x, d_top, d_teacher, **rest)
    dx = singa.DistillationBwd(d_x, stats, d_top, d_teacher, scale=scale, **rest)
    both_loss, both_dx = singa.DistillationFwdBwd(d_x, d_top, d_teacher, scale=scale, **rest)
    assert np.array_equal(d_x.to_numpy().astype(np.float64), np.asarray(x, np.float64), equal_nan=True)
    place = put()
    assert singa.DistillationBwd(place, stats, d_top, d_teacher, scale=scale, out=place, **rest) is place
    assert np.array_equal(place.to_numpy(), dx.to_numpy(), equal_nan=True)
    again = put()
    place_loss, _ = singa.DistillationFwdBwd(again, d_top, d_teacher, scale=scale, out=again, **rest)
    assert np.array_equal(again.to_numpy(), both_dx.to_numpy(), equal_nan=True)
    assert np.array_equal(place_loss.to_numpy(), both_loss.to_numpy(), equal_nan=True)
    if shift:
        for p in (place, again):
            edges = p._block.keepalive.to_numpy()
            assert (edges[:shift] == 7).all() and (edges[-8:] == 7).all()
    return loss.to_numpy(), stats.to_numpy(), dx.to_numpy(), both_loss.to_numpy(), both_dx.to_numpy()


def bounds(t, x, top, teacher, labels, weights, scale, temperature, soft, hard):
    """Allowed errors of (loss, stats, dx), from the magnitudes of what is added up."""
    n, v = x.shape
    k = 0 if top is None else top.shape[1]
    w = np.ones(n) if weights is None else np.asarray(weights, np.float64)
    spread = np.array([np.ptp(row[np.isfinite(row)]) if np.isfinite(row).any() else 0.0 for row in x])
    spread_t = 0.0 if not k else float(np.ptp(teacher[np.isfinite(teacher)])) if np.isfinite(teacher).any() else 0.0
    sums = v / 64 + 40                                   # a lane's terms one behind the other, then pairwise
    rel_t, rel_1 = (4 * spread / temperature + 8 + sums) * U, (4 * spread + 8 + sums) * U
    rel_p = (4 * spread_t / temperature + 8 + k / 64 + 40) * U
    logs = 4 * (np.log(v) + spread / temperature + spread_t / temperature + 1) * U
    loss = w * (soft * temperature ** 2 * (rel_t + rel_p * (4 + np.log(v) + spread / temperature + spread_t / temperature) + logs * (k / 64 + 8))
                + hard * (rel_1 + 4 * (np.log(v) + spread + 1) * U * 4)) if k or labels is not None else np.zeros(n)
    one = [O.distill(x, top, teacher, labels, weights, temperature, s, h, scale)[2] for s, h in ((soft, 0.0), (0.0, hard))]
    # both parts of a term: the probability, and the share that is taken off (at most 1 in all)
    share = w[:, None] * abs(scale)
    dx = share * (soft * temperature * (rel_t[:, None] + rel_p) + hard * (rel_1[:, None] + 2 * U)) * at_least(x, top, labels)
    dx = dx + (np.abs(one[0]) + np.abs(one[1])) * (rel_t + rel_1)[:, None] * 2 + HALF[t] * 1.01 * np.abs(one[0] + one[1]) + TINY[t] + 1e-37
    return loss + 1e-37, np.stack([0 * rel_t, rel_t, rel_1], 1), dx


def at_least(x, top, labels):
    """1 where a list entry or a label is taken off, 0 elsewhere (there the error is relative to the probability)"""
    out = np.zeros(x.shape)
    for i in range(x.shape[0]):
        for j in ([] if top is None else top[i]):
            if 0 <= j < x.shape[1]:
                out[i, j] = 1
        if labels is not None and 0 <= labels[i] < x.shape[1]:
            out[i, labels[i]] = 1
    return out


def check_case(singa, dev, t, case, scale=1.0, shift=0, temperature=1.0, soft=1.0, hard=0.0):
    x, top, teacher, labels, weights = case
    how = dict(temperature=temperature, soft=soft, hard=hard)
    want = O.distill(x, top, teacher, labels, weights, scale=scale, **how)
    loss, stats, dx, loss2, dx2 = run_all(singa, dev, t, x, top, teacher, labels, weights, scale, shift, **how)
    b_loss, b_stats, b_dx = bounds(t, x, top, teacher, labels, weights, scale, temperature, soft, hard)
    close(loss, want[0], b_loss, "loss")
    close(loss2, want[0], b_loss, "loss of the two in one")
    close(stats, want[1], b_stats * np.abs(want[1]), "stats")
    close(dx, want[2], b_dx, "dx")
    close(dx2, want[2], b_dx, "dx of the two in one")
    none = (want[1][:, 0] == 0) & (want[0] == 0) & ~want[2].any(1)
    assert not loss[none].any() and not dx[none].any() and not dx2[none].any()
    return loss, stats, dx, loss2, dx2


# (rows, columns, list): one column, less than a vector, odd ones, on both sides of every way to share a row out
SIZES = [(1, 1, 1), (3, 2, 1), (5, 7, 3), (9, 64, 5), (2, 513, 40), (6, 1000, 5), (3, 2048, 16), (4, 2049, 64), (3, 4100, 7), (2, 10007, 8),
         (3, 16385, 100), (1, 33000, 20), (2, 70001, 65), (128, 35001, 3), (1500, 520, 3), (700, 5003, 20), (2100, 1300, 70), (300, 19001, 2)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,v,k", SIZES)
def test_distillation(dev, t, n, v, k):
    from singa_amd import singa_wrap as singa
    case = make_case(np.random.default_rng(n * v + k), t, n, v, k)
    check_case(singa, dev, t, case, temperature=2.0, soft=0.7, hard=0.3, scale=0.5)
    check_case(singa, dev, t, case, temperature=1.0, soft=1.0, hard=0.0, shift=3)
    assert singa.IndexErrors(dev) == 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("temperature,soft,hard", [(1.0, 0.5, 0.5), (1.0, 0.0, 1.0), (0.5, 1.0, 0.25), (8.0, 2.0, 0.0), (3.0, 0.0, 0.0)])
@pytest.mark.parametrize("n,v,k", [(5, 1003, 12), (4, 5001, 33)])
def test_distillation_terms(dev, t, temperature, soft, hard, n, v, k):
    from singa_amd import singa_wrap as singa
    case = make_case(np.random.default_rng(7), t, n, v, k)
    check_case(singa, dev, t, case, temperature=temperature, soft=soft, hard=hard, scale=1.0 / n)
    x, top, teacher, labels, weights = case
    check_case(singa, dev, t, (x, None, None, labels, None), temperature=temperature, soft=soft, hard=hard)   # labels alone
    check_case(singa, dev, t, (x, top, teacher, None, None), temperature=temperature, soft=soft, hard=hard)   # the list alone
    check_case(singa, dev, t, (x, None, None, None, weights), temperature=temperature, soft=soft, hard=hard)  # nothing


def test_distillation_longest_list_and_one_longer(dev):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(11)
    for v in (1500, 3000):
        case = make_case(r, "f32", 2, v, 1024)
        check_case(singa, dev, "f32", case, temperature=1.5, soft=1.0, hard=0.5)
    x = upload(singa, dev, "f32", np.zeros((2, 3000)))
    with pytest.raises(singa.SingaHipError):
        singa.DistillationFwd(x, ints(singa, dev, np.zeros((2, 1025))), singa.from_numpy(np.zeros((2, 1025), np.float32), dev))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [300, 9001, 40003])
def test_distillation_masked_columns_and_odd_values(dev, t, v):
    """Columns at -inf and at the type's lowest value, rows of nothing but the lowest value, NaN and infinities in rows that do not count."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(v)
    n, k = 8, 6
    x, top, teacher, labels, _ = make_case(r, t, n, v, k, masked=False)
    weights = np.ones(n, np.float32)
    lowest = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}[t]
    keep = np.zeros(v, bool)
    keep[::7] = True
    top = np.where(np.ones((n, k), bool), (np.arange(k) * 7)[None, :] + 7 * np.arange(n)[:, None], 0)
    labels[:] = 14
    x[0][~keep] = -np.inf
    x[1][~keep] = lowest
    x[2][:] = lowest                 # a uniform distribution
    x[3][~keep], x[3, 5] = -np.inf, lowest
    x[4][:], weights[4] = np.nan, 0
    x[5][:], top[5], labels[5] = np.inf, -1, -1
    x[6][:], weights[6] = -np.inf, 0
    top[7], labels[7], x[7, 3] = -1, -1, np.nan
    case = (x, top, teacher, labels, weights)
    for temperature in (1.0, 2.0):
        loss, stats, dx, loss2, dx2 = check_case(singa, dev, t, case, temperature=temperature, soft=0.5, hard=0.5)
        assert not loss[4:].any() and not dx[4:].any() and np.isfinite(loss).all() and np.isfinite(dx).all() and np.isfinite(dx2).all()
        if t != "f16":
            assert not dx[1][~keep].any() and not dx[0][~keep].any()


@pytest.mark.parametrize("t", TYPES)
def test_distillation_of_rows_without_a_softmax_is_nan(dev, t):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(3)
    for v in (100, 5000, 50000):
        x, top, teacher, labels, _ = make_case(r, t, 4, v, 4, masked=False)
        x[0][:] = -np.inf
        x[1, v // 2] = np.nan
        x[2, v - 1] = np.inf
        loss, stats, dx, loss2, dx2 = run_all(singa, dev, t, x, top, teacher, labels, None, soft=0.5, hard=0.5, temperature=2.0)
        for l, d in ((loss, dx), (loss2, dx2)):
            assert np.isnan(l[:3]).all() and np.isfinite(l[3]) and np.isfinite(d[3]).all()
            assert np.isnan(d[0]).all() and np.isnan(d[1]).all() and np.isnan(d[2, v - 1])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [300, 4000, 50000])
def test_distillation_towards_columns_without_a_probability(dev, t, v):
    """The teacher wants columns that the student masks: the loss is infinite, the gradient is not."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(13)
    x, top, teacher, _, weights = make_case(r, t, 4, v, 5, masked=False)
    top = np.tile(np.arange(5) * 11, (4, 1))
    x[0, 11] = -np.inf                # one of the entries
    x[1, top[1]] = -np.inf            # all of them
    x[2, :], x[2, 200:] = -np.inf, 1  # and all else
    teacher[3, :4] = -np.inf          # entries without a share may be anything
    x[3, :44] = -np.inf
    want = O.distill(x, top, teacher, None, weights, temperature=2.0)
    loss, stats, dx, loss2, dx2 = run_all(singa, dev, t, x, top, teacher, None, weights, temperature=2.0)
    b_loss, _, b_dx = bounds(t, x, top, teacher, None, weights, 1.0, 2.0, 1.0, 0.0)
    for l, d in ((loss, dx), (loss2, dx2)):
        assert (l[:3] == np.inf).all()
        close(l[3:], want[0][3:], b_loss[3:], "loss")
        close(d, want[2], b_dx, "dx")


@pytest.mark.parametrize("n,v", [(110000, 500), (2700, 20001), (1300, 45000), (1000, 54000), (900, 66003)])
def test_distillation_of_more_than_the_caches(dev, n, v):
    """Logits of more than 96 MB and more rows than the chip holds: some of the rows, by each entry point, and in a smaller batch.  (Not the same bits
    there: a row of an odd length begins elsewhere in its 16 bytes, and a thread's sum has other terms.)"""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(17)
    k = 4
    x = (r.standard_normal((n, v), dtype=np.float32) * 2).astype(np.float16)
    top, labels = r.integers(0, v, (n, k)), r.integers(-1, v, n)
    teacher = r.standard_normal((n, k)).astype(np.float32)
    weights = np.where(r.random(n) < 0.3, 0, 1).astype(np.float32)
    how = dict(temperature=2.0, soft=0.7, hard=0.3)

    def run(rows):
        d_x, d_top, d_teacher = upload(singa, dev, "f16", x[rows]), ints(singa, dev, top[rows]), singa.from_numpy(teacher[rows], dev)
        rest = dict(labels=ints(singa, dev, labels[rows]), weights=singa.from_numpy(weights[rows], dev), **how)
        loss, stats = singa.DistillationFwd(d_x, d_top, d_teacher, **rest)
        dx = singa.DistillationBwd(d_x, stats, d_top, d_teacher, **rest)
        return [t.to_numpy() for t in (loss, dx) + singa.DistillationFwdBwd(d_x, d_top, d_teacher, **rest)]

    whole = run(slice(0, n))
    rows = np.unique(np.concatenate([[0, 1, 255, 256, 257, 511, 512, n - 2, n - 1], r.integers(0, n, 20)]))
    part = run(rows)
    x64 = x[rows].astype(np.float64)
    want = O.distill(x64, top[rows], teacher[rows], labels[rows], weights[rows], **how)
    b = bounds("f16", x64, top[rows], teacher[rows], labels[rows], weights[rows], 1.0, 2.0, 0.7, 0.3)
    for got in ([a[rows] for a in whole], part):
        for i in (0, 2):
            close(got[i], want[0], b[0], "loss")
            close(got[i + 1], want[2], b[2], "dx")


# (fp32; 16 bits: twice the columns) a wavefront to a row, few and many vectors of a thread held, and rows that are read twice; of more than 96 MB and of less
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,v", [(110000, 240), (2700, 10001), (1700, 15001), (1100, 24001), (900, 30001), (700, 40003),
                                 (1000, 15001), (600, 24001), (500, 30001), (300, 70001)])
def test_distillation_of_many_long_rows(dev, t, n, v):
    """Each way to share the rows out, in each type: some of the rows, by each entry point, in place too."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(19)
    k, v = 4, v * (1 if t == "f32" else 2)
    x = np.resize((r.standard_normal(1000003, dtype=np.float32) * 2).astype(np.float16), (n, v))
    if t == "bf16":   # values that the type holds
        x = (x.view(np.uint16) & 0xfff8).view(np.float16)
    top, labels = r.integers(0, v, (n, k)), r.integers(-1, v, n)
    teacher = r.standard_normal((n, k)).astype(np.float32)
    weights = np.where(r.random(n) < 0.3, 0, 1).astype(np.float32)
    how = dict(temperature=2.0, soft=0.7, hard=0.3)
    d_x, d_top, d_teacher = upload(singa, dev, t, x), ints(singa, dev, top), singa.from_numpy(teacher, dev)
    rest = dict(labels=ints(singa, dev, labels), weights=singa.from_numpy(weights, dev), **how)
    loss, stats = singa.DistillationFwd(d_x, d_top, d_teacher, **rest)
    got = [a.to_numpy() for a in (loss, singa.DistillationBwd(d_x, stats, d_top, d_teacher, **rest)) + singa.DistillationFwdBwd(d_x, d_top, d_teacher, **rest)]
    in_place = singa.DistillationFwdBwd(d_x, d_top, d_teacher, out=d_x, **rest)
    for a, b in zip(in_place, got[2:]):
        assert np.array_equal(a.to_numpy(), b)
    none = (weights == 0)
    assert not got[0][none].any() and not got[1][none].any() and not got[3][none].any()
    rows = np.unique(np.concatenate([[0, 1, 255, 256, 257, 299, n - 2, n - 1], r.integers(0, n, 12)]))
    x64 = x[rows].astype(np.float64)
    want = O.distill(x64, top[rows], teacher[rows], labels[rows], weights[rows], **how)
    b = bounds(t, x64, top[rows], teacher[rows], labels[rows], weights[rows], 1.0, 2.0, 0.7, 0.3)
    for i in (0, 2):
        close(got[i][rows], want[0], b[0], "loss")
        close(got[i + 1][rows], want[2], b[2], "dx")


def test_distillation_of_more_than_32_bits_of_elements(dev):
    """4.59e9 logits: rows on both sides of 2^31 and 2^32 elements, by each entry point and in place."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(24)
    n, v, k = 70001, 65537, 3
    rows = np.array([0, 32766, 32767, 32768, 65534, 65535, 65536, 70000])
    top, labels = r.integers(0, v, (n, k)), r.integers(-1, v, n)
    teacher = r.standard_normal((n, k)).astype(np.float32)
    x64 = stored("bf16", r.standard_normal((rows.size, v)) * 3)
    x64[3] = 0.5
    x = singa.Tensor((n, v), dev, singa.kBFloat16)
    x.SetFloatValue(0.5)
    for row, a in zip(rows, x64):
        put_row(singa, dev, "bf16", x, row, a)
    how = dict(temperature=2.0, soft=0.7, hard=0.3)
    d_top, d_teacher, d_labels = ints(singa, dev, top), singa.from_numpy(teacher, dev), ints(singa, dev, labels)
    want = O.distill(x64, top[rows], teacher[rows], labels[rows], None, **how)
    b = bounds("bf16", x64, top[rows], teacher[rows], labels[rows], None, 1.0, 2.0, 0.7, 0.3)

    def look(loss, dx):
        if loss is not None:
            close(loss.to_numpy()[rows], want[0], b[0], "loss")
        close(np.concatenate([row_of(singa, dev, "bf16", dx, i).to_numpy() for i in rows]), want[2], b[2], "dx")

    loss, stats = singa.DistillationFwd(x, d_top, d_teacher, d_labels, **how)
    look(loss, singa.DistillationBwd(x, stats, d_top, d_teacher, d_labels, **how))
    look(*singa.DistillationFwdBwd(x, d_top, d_teacher, d_labels, **how))
    look(None, singa.DistillationBwd(x, stats, d_top, d_teacher, d_labels, out=x, **how))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,v,k", [(9, 500, 1024), (9, 300, 700), (1030, 90, 65)])
def test_distillation_of_long_lists_over_few_columns(dev, t, n, v, k):
    """Lists longer than the row, every column there several times, a wavefront to a row."""
    from singa_amd import singa_wrap as singa
    case = make_case(np.random.default_rng(v), t, n, v, k)
    check_case(singa, dev, t, case, temperature=2.0, soft=0.7, hard=0.3, scale=0.5)
    check_case(singa, dev, t, case, shift=1)


def record_of(dev, call):
    """Milliseconds of the one profiling record that `call` leaves."""
    import ctypes as C
    from singa_amd._lib import check, lib
    L, n, buf, ms, work = lib(), C.c_int(), C.create_string_buffer(64), C.c_float(), C.c_double()
    dev.Sync()
    check(L.sgh_prof_enable(1), "sgh_prof_enable")
    try:
        call()
        dev.Sync()
        check(L.sgh_prof_count(C.byref(n)), "sgh_prof_count")
        assert n.value == 1
        check(L.sgh_prof_get(0, buf, 64, C.byref(ms), C.byref(work)), "sgh_prof_get")
    finally:
        L.sgh_prof_enable(0)
        L.sgh_prof_clear()
    return ms.value


def test_distillation_of_more_rows_than_a_launch_takes(dev):
    """Both in one call for 3 * 2^20 rows and some: rows on both sides of every launch, and one profiling record around all of them."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(23)
    one, n, v, k = 1 << 20, (3 << 20) + 5, 20, 2
    x = np.resize(r.standard_normal(1000003, dtype=np.float32), (n, v))
    top, labels, weights = r.integers(0, v, (n, k)), r.integers(-1, v, n), (r.random(n) < 0.8).astype(np.float32)
    teacher = np.resize(r.standard_normal(999983, dtype=np.float32), (n, k))
    how = dict(temperature=2.0, soft=0.7, hard=0.3)
    d = [upload(singa, dev, "f32", x), ints(singa, dev, top), singa.from_numpy(teacher, dev), ints(singa, dev, labels), singa.from_numpy(weights, dev)]
    part = [upload(singa, dev, "f32", x[:one]), ints(singa, dev, top[:one]), singa.from_numpy(teacher[:one], dev), ints(singa, dev, labels[:one]),
            singa.from_numpy(weights[:one], dev)]
    loss, dx = (a.to_numpy() for a in singa.DistillationFwdBwd(*d, **how))
    singa.DistillationFwdBwd(*part, **how)
    rows = np.unique(np.concatenate([[0, n - 1], *[[i * one - 1, i * one, i * one + 1] for i in (1, 2, 3)], r.integers(0, n, 30)]))
    x64 = x[rows].astype(np.float64)
    want = O.distill(x64, top[rows], teacher[rows], labels[rows], weights[rows], **how)
    b = bounds("f32", x64, top[rows], teacher[rows], labels[rows], weights[rows], 1.0, 2.0, 0.7, 0.3)
    close(loss[rows], want[0], b[0], "loss")
    close(dx[rows], want[2], b[2], "dx")
    times = [record_of(dev, lambda: singa.DistillationFwdBwd(*a, **how)) for a in (part, d)]
    assert times[1] > 2 * times[0], times   # (three times the rows and more)


def test_distillation_entries_out_of_range_are_left_out_and_counted(dev):
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(9)
    for v in (50, 5000, 50000):
        x, top, teacher, labels, weights = make_case(r, "f32", 3, v, 5, masked=False)
        top[0, 1], top[1, 2], top[2, 0] = v, -2, 2147483647
        labels[1], labels[2] = v, -5
        singa.IndexErrors(dev)
        want = O.distill(x, top, teacher, labels, weights, soft=1.0, hard=1.0)
        d_x, d_top, d_teacher = upload(singa, dev, "f32", x), ints(singa, dev, top), singa.from_numpy(teacher, dev)
        rest = dict(labels=ints(singa, dev, labels), weights=singa.from_numpy(weights, dev), hard=1.0)
        loss, stats = singa.DistillationFwd(d_x, d_top, d_teacher, **rest)
        assert singa.IndexErrors(dev) == 5
        singa.DistillationBwd(d_x, stats, d_top, d_teacher, **rest)
        assert singa.IndexErrors(dev) == 0
        _, dx = singa.DistillationFwdBwd(d_x, d_top, d_teacher, **rest)
        assert singa.IndexErrors(dev) == 5
        b = bounds("f32", x, top, teacher, labels, weights, 1.0, 1.0, 1.0, 1.0)
        close(loss.to_numpy(), want[0], b[0], "loss")
        close(dx.to_numpy(), want[2], b[2], "dx")


@pytest.mark.parametrize("v", [200, 6000, 20000])
def test_distillation_gradient_against_differences(dev, v):
    """Central differences of the loss along a direction of at most 1 in every place.  The third derivative of the logarithm of a sum of
    exponentials of y / tau along such a direction is a third central moment of a variable in [-1, 1], at most 1 by size, over tau^3."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(21)
    n, k, tau, h = 6, 9, 2.0, 2.0 ** -5
    x, top, teacher, labels, weights = make_case(r, "f32", n, v, k)
    along = r.uniform(-1, 1, (n, v))
    d_top, d_teacher = ints(singa, dev, top), singa.from_numpy(teacher, dev)
    rest = dict(labels=ints(singa, dev, labels), weights=singa.from_numpy(weights, dev), temperature=tau, soft=0.8, hard=0.4)
    f = lambda y: singa.DistillationFwd(upload(singa, dev, "f32", y), d_top, d_teacher, **rest)[0].to_numpy().astype(np.float64)
    _, dx = singa.DistillationFwdBwd(upload(singa, dev, "f32", x), d_top, d_teacher, **rest)
    got = (f(x + h * along) - f(x - h * along)) / (2 * h)
    want = (dx.to_numpy().astype(np.float64) * along).sum(1)
    b_loss = bounds("f32", x, top, teacher, labels, weights, 1.0, tau, 0.8, 0.4)[0]
    moved = U * np.abs(x).max() / h * 2 * (0.8 * tau + 0.4)       # the logits' own rounding
    assert (np.abs(got - want) <= weights * (h * h / 6 * (0.8 / tau + 0.4) + moved) + 2 * b_loss / (2 * h) + 1e-6).all()


# ------------------------------------------------------------------------------------ recorded, and on another stream

def test_recorded_calls_replay(dev):
    """Both gradients and the loss in one recording, replayed beside eager calls of other sizes: each replay stores the eager bits."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(31)
    vocab, dim, n, k = 3000, 40, 1500, 4
    ids, table = ints(singa, dev, r.integers(0, vocab, n)), upload(singa, dev, "f32", r.standard_normal((vocab, dim)))
    few = ints(singa, dev, r.integers(0, vocab, 90))
    long = upload(singa, dev, "bf16", r.standard_normal((3, 50000)))
    x = upload(singa, dev, "f32", r.standard_normal((n, vocab)))
    top, teacher = ints(singa, dev, r.integers(0, vocab, (n, k))), singa.from_numpy(r.standard_normal((n, k)).astype(np.float32), dev)
    long_top, long_teacher = ints(singa, dev, r.integers(0, 50000, (3, k))), singa.from_numpy(r.standard_normal((3, k)).astype(np.float32), dev)

    def calls():
        y = singa.EmbeddingForward(ids, table)
        loss, stats = singa.DistillationFwd(x, top, teacher)
        dx = singa.DistillationBwd(x, stats, top, teacher, scale=1.0 / n)
        loss2, dx2 = singa.DistillationFwdBwd(x, top, teacher, scale=1.0 / n)
        few_rows = [t for f in (singa.DistillationFwd, singa.DistillationFwdBwd) for t in f(long, long_top, long_teacher)]
        return few_rows + [y, loss, stats, dx, loss2, dx2, singa.EmbeddingBackwardW(y, ids, table),
                singa.EmbeddingBackwardW(singa.EmbeddingForward(few, table), few, table)]

    want = [t.to_numpy() for t in calls()]
    dev.Sync()
    dev.EnableGraph(True)
    outs = calls()
    dev.EnableGraph(False)
    try:
        for _ in range(4):
            for t in outs:
                t.SetFloatValue(-77.0)
            dev.RunGraph()
            calls()
            for t, w in zip(outs, want):
                assert np.array_equal(t.to_numpy(), w)
    finally:
        dev.ResetGraph()


def test_entry_points_on_the_auxiliary_stream(dev):
    from singa_amd import singa_wrap as singa
    from singa_amd._lib import check, lib
    r = np.random.default_rng(32)
    vocab, dim, n = 900, 30, 2000
    ids, table = ints(singa, dev, r.integers(0, vocab, n)), upload(singa, dev, "f32", r.standard_normal((vocab, dim)))
    dy = upload(singa, dev, "f32", r.standard_normal((n, dim)))
    want = singa.EmbeddingBackwardW(dy, ids, table).to_numpy()
    out = singa.Tensor((vocab, dim), dev)
    need = lib().sgh_embedding_bwd_workspace_bytes(n, vocab, dim)
    ws = singa.Tensor((need // 4,), dev)
    aux = dev.Fork()
    check(lib().sgh_embedding_bwd_f32(ids.ptr, dy.ptr, None, out.ptr, n, vocab, dim, 1.0, -1, ws.ptr, need, aux), "embedding_bwd")
    dev.Join()
    assert np.array_equal(out.to_numpy(), want)


def test_two_streams_at_once(dev):
    """Few long rows (in parts, a workspace each) and a sorted gradient on both streams at the same time."""
    from singa_amd import singa_wrap as singa
    from singa_amd._lib import check, lib
    r = np.random.default_rng(33)
    n, v, k, tokens, vocab, dim = 5, 60000, 6, 3000, 700, 40
    L = lib()
    x = [upload(singa, dev, "f32", r.standard_normal((n, v))) for _ in range(2)]
    top, teacher = ints(singa, dev, r.integers(0, v, (n, k))), singa.from_numpy(r.standard_normal((n, k)).astype(np.float32), dev)
    ids = [ints(singa, dev, r.integers(0, vocab, tokens)) for _ in range(2)]
    dy, table = upload(singa, dev, "f32", r.standard_normal((tokens, dim))), singa.Tensor((vocab, dim), dev)
    want = [[t.to_numpy() for t in singa.DistillationFwdBwd(x[i], top, teacher, temperature=2.0) + (singa.EmbeddingBackwardW(dy, ids[i], table),)]
            for i in range(2)]
    need, sort = L.sgh_distill_workspace_bytes(n, v, 4, 1), L.sgh_embedding_bwd_workspace_bytes(tokens, vocab, dim)
    assert need and sort
    out = [[singa.Tensor(s, dev) for s in ((n,), (n, v), (vocab, dim), (need // 4,), (sort // 4,))] for _ in range(2)]
    aux = dev.Fork()
    for _ in range(3):
        for i, stream in enumerate((dev.stream, aux)):
            loss, dx, dW, ws, ws_sort = out[i]
            check(L.sgh_distill_fwd_bwd_f32(x[i].ptr, top.ptr, teacher.ptr, None, None, n, v, k, 2.0, 1.0, 0.0, 1.0, loss.ptr, dx.ptr, ws.ptr, need,
                                            stream), "distill_fwd_bwd")
            check(L.sgh_embedding_bwd_f32(ids[i].ptr, dy.ptr, None, dW.ptr, tokens, vocab, dim, 1.0, -1, ws_sort.ptr, sort, stream), "embedding_bwd")
    dev.Join()
    for i in range(2):
        for t, w in zip(out[i], want[i]):
            assert np.array_equal(t.to_numpy(), w)


def test_index_errors_of_two_streams(dev):
    """Counted on the auxiliary stream while the main one reads the count: each once."""
    from singa_amd import singa_wrap as singa
    from singa_amd._lib import check, lib
    L, tokens, vocab, dim, calls = lib(), 200, 50, 40, 400
    ids, table = ints(singa, dev, np.where(np.arange(tokens) % 4 == 0, vocab + 1, 3)), upload(singa, dev, "f32", np.ones((vocab, dim)))
    x, top = upload(singa, dev, "f32", np.zeros((3, vocab))), ints(singa, dev, np.full((3, 2), -5))
    y, loss, stats = (singa.Tensor(s, dev) for s in ((tokens, dim), (3,), (3, 3)))
    teacher = singa.from_numpy(np.zeros((3, 2), np.float32), dev)
    dev.Sync()
    singa.IndexErrors(dev)
    aux, met = dev.Fork(), 0
    for i in range(calls):
        check(L.sgh_embedding_fwd_f32(ids.ptr, table.ptr, y.ptr, tokens, vocab, dim, 1.0, -1, aux), "embedding_fwd")
        check(L.sgh_distill_fwd_f32(x.ptr, top.ptr, teacher.ptr, None, None, 3, vocab, 2, 1.0, 1.0, 0.0, loss.ptr, stats.ptr, None, 0, aux), "distill_fwd")
        if i % 5 == 4:
            met += singa.IndexErrors(dev)
    dev.Join()
    assert met + singa.IndexErrors(dev) == calls * (tokens // 4 + 6)
    assert singa.IndexErrors(dev) == 0
