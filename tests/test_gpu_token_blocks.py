"""Attention and the norms around blocks together with the token model's ends and dense layers, as a training program runs them."""
import numpy as np
import pytest

from oracle import block_ops as O
from oracle.ops import OracleOps
from singa_amd import workloads as wl
from test_gpu_token_model import ints, stored, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("name,batch,steps", [("token_attention_small", None, 3), ("token_attention_small", 1, 1), ("token_attention", 4, 1)])
def test_steps_match_the_oracle(dev, fused, name, batch, steps):
    hip = wl.HipOps(dev)
    hip.set_fusion(fused)
    errors = wl.run_parity_case(name, dev, OracleOps(), batch=batch, steps=steps, share_activations=False, hip_ops=hip)["errors"]
    assert any(k.endswith("attention.table") for k in errors) and any(k.endswith("norm1.gate") for k in errors)
    # (moving all keys of a row by one vector moves all its scores alike: the gradient of the keys' bias is nothing but roundings)
    errors = {k: e for k, e in errors.items() if not (".k.b" in k and ("grad." in k or "param." in k))}
    # fp32 products of up to 10000 terms with errors of either sign; own forward passes differ where a ReLU's argument is next to 0
    worst = max(errors, key=errors.get)
    assert errors[worst] < 1e-3, (worst, errors[worst])


def test_recorded_training_step(dev):
    """Forward, loss, backward and update in one recording, replayed on another batch each time beside a network that runs the same steps
    eagerly: the same bits."""
    hip = wl.HipOps(dev)
    ids, targets = wl.make_inputs("token_attention_small")
    nets = [wl.build("token_attention_small", hip) for _ in range(2)]
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
            for x, t in inputs:
                x.CopyIntDataFromHostPtr(np.roll(ids, i + 1, axis=0))
                t.top.CopyIntDataFromHostPtr(np.roll(targets.top, 5 * i + 1, axis=0))
                t.labels.CopyIntDataFromHostPtr(np.roll(targets.labels, 3 * i + 2))
            step(0)
            dev.RunGraph()
            for (k, a), (_, b) in zip(eager.params(), replayed.params()):
                a, b = hip.to_numpy(a), hip.to_numpy(b)
                assert np.isfinite(a).all() and np.array_equal(a, b), (i, k)
    finally:
        dev.ResetGraph()


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_a_padded_16_bit_block(dev, t):
    """One attention block on 16-bit tensors of a padded batch: vectors by id, norm, products, attention with a bias, product, norm with a gate for
    each sequence, gate and sum, and back; every tensor against the same chain in 64 bits on what the device stored in between."""
    from singa_amd import singa_wrap as singa
    r = np.random.default_rng(11)
    b, s, h, g, d, vocab = 5, 70, 4, 2, 16, 50
    dim, rows = h * d, b * s
    lengths = (70, 1, 33, 0, 64)
    half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[t]
    put = lambda a, k=t: upload(singa, dev, k, a)
    ids, E = r.integers(0, vocab, (b, s)), stored(t, r.standard_normal((vocab, dim)))
    W = [stored(t, r.standard_normal((dim, n)) / 8) for n in (dim, g * d, g * d, dim)]
    pre, post, last = (stored("f32", 1 + 0.2 * r.standard_normal(dim)) for _ in range(3))
    gate, table, dn = stored(t, r.standard_normal((b, dim))), stored("f32", r.standard_normal((8, h))), stored(t, r.standard_normal((rows, dim)))
    dn.reshape(b, s, dim)[[np.arange(s) >= n for n in lengths]] = 0   # (the loss has no weight behind a sequence)
    dW = [put(w) for w in W]
    dp, dpo, dl, dg, dtab, dlen = put(pre, "f32"), put(post, "f32"), put(last, "f32"), put(gate), put(table, "f32"), ints(singa, dev, lengths)

    x = singa.EmbeddingForward(ints(singa, dev, ids), put(E), 2.0).Reshape((rows, dim))
    _, n, st0 = singa.ResidualNormForward(x, pre=dp)
    q, k, v = (singa.Mult(n, w).Reshape((b, s, c, d)) for w, c in zip(dW[:3], (h, g, g)))
    H = singa.AttentionHandle(q, k, causal=True, buckets=8, max_distance=32, bidirectional=False)
    o, lse = singa.AttentionForward(H, q, k, v, dtab, dlen, dlen)
    out = singa.Mult(o.Reshape((rows, dim)), dW[3])
    y, m, st1 = singa.ResidualNormForward(x, out, dpo, dg, 0.5, dl)
    dx, dout, gpost, ggate, glast = singa.ResidualNormBackward(None, put(dn), y, st1, out, dpo, dg, 0.5, dl)
    do = singa.Mult(dout, dW[3].T()).Reshape((b, s, h, d))
    gq, gk, gv, gtable = singa.AttentionBackward(H, do, q, k, v, o, lse, dtab, dlen, dlen)
    got = {"n": n, "o": o, "y": y, "m": m, "dx": dx, "dout": dout, "gate": ggate, "post": gpost, "last": glast, "dq": gq, "dk": gk, "dv": gv, "table": gtable}
    f = lambda a: a.to_numpy().astype(np.float64)
    a = O.Attn(True, buckets=8, max_distance=32, bidirectional=False)
    want = {"n": O.residual_norm(f(x), pre=pre)[1], "o": O.attention(a, f(q), f(k), f(v), table, lengths, lengths)[0]}
    want["y"], want["m"], _ = O.residual_norm(f(x), f(out), post, gate, 0.5, last)
    want["dx"], want["dout"], want["post"], want["gate"], want["last"] = O.residual_norm_bwd(None, dn, f(y), f(st1), f(out), post, gate, 0.5, last)
    want["dq"], want["dk"], want["dv"], want["table"] = O.attention_bwd(a, f(do), f(q), f(k), f(v), f(o), f(lse), table, lengths, lengths)
    for name, w in want.items():
        # one rounding of the result and at most one of the terms of a product over 70 others, as a share of the largest value; fp32 sums 1e-5
        room = (2.5 * half if got[name].data_type() != singa.kFloat32 else 1e-5) * np.abs(w).max()
        assert np.abs(f(got[name]) - w).max() <= room, (name, np.abs(f(got[name]) - w).max(), room)
    for name in ("o", "dq", "dk", "dv"):
        for i, count in enumerate(lengths):
            assert not f(got[name])[i, count:].any(), (name, i)
