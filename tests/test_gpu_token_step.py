"""The token model's operators together on the GPU, as a training program runs them: whole steps of the tape against the oracle's, recorded
steps, and a model whose table is its output matrix as well."""
import numpy as np
import pytest

from oracle import token_ops as O
from oracle.ops import OracleOps
from singa_amd import workloads as wl

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("name,batch,steps", [("token_mlp_small", None, 3), ("token_mlp_small", 1, 1), ("token_mlp", None, 1),
                                              ("token_mlp", 400, 1)])   # (400 rows of 4: more tokens than one launch takes)
def test_steps_match_the_oracle(dev, fused, name, batch, steps):
    hip = wl.HipOps(dev)
    hip.set_fusion(fused)
    res = wl.run_parity_case(name, dev, OracleOps(), batch=batch, steps=steps, share_activations=not fused, hip_ops=hip)
    errors = res["errors"]
    assert any(k.endswith("grad.embedding.W") for k in errors) and not any(k.endswith("grad.input") for k in errors)
    # fp32 products of up to 10000 terms with errors of either sign; own forward passes differ where a ReLU's argument is next to 0
    worst = max(errors, key=errors.get)
    assert errors[worst] < 1e-3, (worst, errors[worst])


def test_step_among_a_half_precision_models_operations(dev):
    """The operations of a 16-bit tape leave a token model in fp32: the same step."""
    from singa_amd import singa_wrap as singa
    res = wl.run_parity_case("token_mlp_small", dev, OracleOps(), hip_ops=wl.HalfHipOps(dev, singa.kFloat16))
    assert max(res["errors"].values()) < 1e-3


def test_fused_and_separate_losses_train_alike(dev):
    """The gradient formed with the loss and the one formed from its statistics are the same formula: parameters after three steps differ by
    roundings alone."""
    ids, targets = wl.make_inputs("token_mlp_small")
    out = []
    for fused in (False, True):
        hip = wl.HipOps(dev)
        hip.fuse_distill = fused
        net = wl.build("token_mlp_small", hip)
        for _ in range(3):
            net.forward(*net.inputs(ids, targets))
            net.backward_and_update(fused_update=True)
        out.append([hip.to_numpy(p) for _, p in net.params()])
    for a, b in zip(*out):
        assert np.linalg.norm(a - b) <= 1e-5 * np.linalg.norm(b)


@pytest.mark.parametrize("name,batch", [("token_mlp_small", 24), ("token_mlp", 300)])
def test_recorded_training_step(dev, name, batch):
    """Forward, loss, backward and update in one recording, replayed on another batch each time (its ids, lists and labels are copied into
    the recorded tensors), beside a network that runs the same steps eagerly: the same bits."""
    hip = wl.HipOps(dev)
    ids, targets = wl.make_inputs(name, batch)
    nets = [wl.build(name, hip) for _ in range(2)]
    inputs = [net.inputs(ids, targets) for net in nets]
    eager, replayed = nets

    def step(i):
        nets[i].forward(*inputs[i])
        nets[i].backward_and_update(fused_update=True)

    for _ in range(2):
        step(0), step(1)
    dev.Sync()
    dev.EnableGraph(True)
    step(1)
    dev.EnableGraph(False)
    try:
        for i in range(4):
            turn = 5 * i + 1
            for x, t in inputs:
                x.CopyIntDataFromHostPtr(np.roll(ids, turn, axis=0))
                t.top.CopyIntDataFromHostPtr(np.roll(targets.top, turn, axis=0))
                t.labels.CopyIntDataFromHostPtr(np.roll(targets.labels, 2 * turn))
            step(0)
            dev.RunGraph()
            for (k, a), (_, b) in zip(eager.params(), replayed.params()):
                a, b = hip.to_numpy(a), hip.to_numpy(b)
                assert np.isfinite(a).all() and np.array_equal(a, b), (i, k)
    finally:
        dev.ResetGraph()


@pytest.mark.parametrize("tokens", [60, 1500])
def test_table_that_is_the_output_matrix_too(dev, tokens):
    """logits = vectors x table^T: the table's gradient from the output side is what the lookup's gradient is added to, in place."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(7)
    vocab, dim, k, scale = 333, 24, 8, 1.5
    table = (r.standard_normal((vocab, dim)) / 4).astype(np.float32)
    ids = r.integers(0, vocab, tokens).astype(np.int32)
    top, labels = r.integers(0, vocab, (tokens, k)).astype(np.int32), r.integers(-1, vocab, tokens).astype(np.int32)
    teacher = r.standard_normal((tokens, k)).astype(np.float32)
    weights = np.where(r.random(tokens) < 0.2, 0, 1).astype(np.float32)   # a padded batch
    ids[weights == 0] = 0                                                # id 0 is the padding
    W = singa.from_numpy(table, dev)
    ti, tt, tl = (singa.from_numpy(a, dev) for a in (ids, top, labels))
    te, tw = singa.from_numpy(teacher, dev), singa.from_numpy(weights, dev)
    how = dict(temperature=2.0, soft=0.8, hard=0.2)
    y = singa.EmbeddingForward(ti, W, scale, 0)
    x = singa.Mult(y, W.T())
    loss, dx = singa.DistillationFwdBwd(x, tt, te, tl, tw, scale=1.0 / tokens, out=x, **how)
    dW = singa.Mult(dx.T(), y)
    dy = singa.Mult(dx, W)
    got = singa.EmbeddingBackwardW(dy, ti, W, scale, 0, add=dW, out=dW)
    assert got is dW

    E = table.astype(np.float64)
    y64 = O.embedding_fwd(ids, E, scale, 0)
    l64, _, dx64 = O.distill(y64 @ E.T, top, teacher.astype(np.float64), labels, weights.astype(np.float64), scale=1.0 / tokens, **how)
    want = dx64.T @ y64 + O.embedding_bwd(dx64 @ E, ids, E.shape, scale, 0)
    # logits: sums of `dim` products, off by (dim + 2) u of the sum of their sizes; that moves a probability by that much of itself (twice, with
    # the row's sum), plus the operator's own (4 |d| / tau + 6 + sums) u with d up to the logits' range
    size = np.abs(y64) @ np.abs(E).T
    off = ((dim + 2) * U * size).max()
    span = np.ptp(y64 @ E.T, axis=1).max()
    rel = 2 * off + (4 * span + vocab / 8 + 60) * U
    np.testing.assert_allclose(loss.to_numpy(), l64, rtol=0, atol=4 * rel * (1 + span))
    # |dx| of a row sums to at most 2 (soft tau + hard) / tokens, all of it off by `rel`
    row = 2 * (0.8 * 2 + 0.2) / tokens
    g_dx = rel * row
    bound = tokens * g_dx * np.abs(y64).max() + scale * np.abs(E).max() * g_dx * np.bincount(ids, minlength=vocab).max()
    bound += (tokens + vocab + 8) * U * (row * tokens * np.abs(y64).max() + scale * row * np.abs(E).max() * np.bincount(ids, minlength=vocab).max())
    assert np.abs(got.to_numpy() - want).max() <= bound
    assert np.linalg.norm(got.to_numpy() - want) <= 1e-5 * np.linalg.norm(want)   # (errors of either sign: far below the bound)
