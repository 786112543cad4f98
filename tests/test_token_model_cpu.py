"""The token model's operators without a GPU: the definitions against differences, the whole tape against a NumPy restatement, refusals of
the C ABI and of the Python mirror, and what the entry points launch (a stand-in for the HIP runtime, hip_recorder.py)."""
import numpy as np
import pytest

from hip_recorder import recorded
from oracle import token_ops as O
from oracle.ops import OracleOps
from singa_amd import workloads as wl

EINVAL, EWORKSPACE, ELIMIT = -1, -2, -6


# ------------------------------------------------------------------------------------ definitions

@pytest.mark.parametrize("temperature,soft,hard", [(1.0, 1.0, 0.0), (2.0, 0.7, 0.3), (0.5, 0.0, 1.0)])
def test_distillation_gradient_is_the_difference_of_the_loss(temperature, soft, hard):
    r = np.random.default_rng(1)
    n, v, k = 6, 30, 5
    x, teacher = r.standard_normal((n, v)), r.standard_normal((n, k))
    top, labels, w = r.integers(0, v, (n, k)), r.integers(0, v, n), r.random(n)
    top[0], labels[0] = -1, -1          # nothing to learn here
    top[1] = top[1, 0]                  # one column five times
    top[2, 1:], w[3] = -1, 0
    teacher[4, 2] = -np.inf
    how = dict(temperature=temperature, soft=soft, hard=hard)
    loss, _, dx = O.distill(x, top, teacher, labels, w, scale=0.5, **how)
    h = 1e-5
    for along in (r.standard_normal((n, v)), np.eye(n, v, 3)):
        got = (O.distill(x + h * along, top, teacher, labels, w, **how)[0] - O.distill(x - h * along, top, teacher, labels, w, **how)[0]) / (2 * h)
        # (h^2 / 6 of a third derivative of at most 4^3 along a direction of at most 4, and the loss's rounding over h)
        np.testing.assert_allclose(0.5 * got, (dx * along).sum(1), rtol=0, atol=2e-9 + 1e-14 / h * 20)
    assert loss[0] == 0 and not dx[0].any() and loss[3] == 0 and not dx[3].any()
    assert abs(dx.sum(1)).max() < 1e-14   # a gradient of logits sums to nothing


def test_distillation_from_the_students_own_logits_is_nothing():
    r = np.random.default_rng(2)
    x = r.standard_normal((4, 9))
    order = np.argsort(-x, axis=1)
    loss, _, dx = O.distill(x, order, np.take_along_axis(x, order, 1), temperature=3.0)
    assert np.abs(loss).max() < 1e-13 and np.abs(dx).max() < 1e-14


def test_embedding_gradient_is_the_transpose_of_the_lookup():
    r = np.random.default_rng(3)
    ids = r.integers(-1, 12, (7, 5))    # below and behind the table as well
    W, dy = r.standard_normal((10, 6)), r.standard_normal((7, 5, 6))
    y = O.embedding_fwd(ids, W, 1.5, 3)
    assert not y[(ids == 3) | (ids < 0) | (ids >= 10)].any()
    assert abs((y * dy).sum() - (O.embedding_bwd(dy, ids, W.shape, 1.5, 3) * W).sum()) < 1e-10


def test_token_model_step_matches_a_numpy_restatement():
    ops = OracleOps()
    net = wl.build("token_mlp_small", ops, lr=0.05, momentum=0.0)
    ids, targets = wl.make_inputs("token_mlp_small")
    E, W0, B0, W1, B1 = (np.array(p, np.float64) for _, p in net.params())
    net.forward(*net.inputs(ids, targets))
    net.backward_and_update(keep_grads=True)
    n, dim = ids.shape[0], E.shape[1]
    x0 = (E[ids] * np.sqrt(dim)).reshape(n, -1)
    z = x0 @ W0 + B0
    h = np.maximum(z, 0)
    loss, _, dl = O.distill(h @ W1 + B1, targets.top, targets.teacher, targets.labels, None, targets.temperature, targets.soft, targets.hard, 1.0 / n)
    dz = (dl @ W1.T) * (z > 0)
    dE = np.zeros_like(E)
    np.add.at(dE, ids.ravel(), np.sqrt(dim) * (dz @ W0.T).reshape(-1, dim))
    want = {"embedding.W": (E, dE), "linear1.W": (W0, x0.T @ dz), "linear1.b": (B0, dz.sum(0)), "linear2.W": (W1, h.T @ dl), "linear2.b": (B1, dl.sum(0))}
    for name, p in net.params():
        before, grad = want[name]
        # fp32 products of up to 1003 terms
        np.testing.assert_allclose(net.grad_log[name], grad, rtol=0, atol=1003 * 2.0 ** -24 * np.abs(grad).max() * 4, err_msg=name)
        np.testing.assert_allclose(p, before - 0.05 * grad, rtol=2e-6, atol=0.05 * 1003 * 2.0 ** -24 * np.abs(grad).max() * 4, err_msg=name)


def test_the_other_configurations_inputs_are_what_they_were():
    x, labels = wl.make_inputs("mlp", 3)
    assert x.shape == (3, 784) and labels.shape == (3,)
    ids, targets = wl.make_inputs("token_mlp_small", 5)
    more, more_targets = wl.make_inputs("token_mlp_small", 9)
    assert ids.dtype.kind == "i" and 0 <= ids.min() and ids.max() < 1003
    assert np.array_equal(more[:5], ids) and np.array_equal(more_targets.top[:5], targets.top)   # a smaller batch is a prefix


# ------------------------------------------------------------------------------------ refusals

def test_embedding_refusals():
    ok, refused, short, nothing = recorded("""
S = SPACE
T, V, D = 3000, 500, 40
need = lib.sgh_embedding_bwd_workspace_bytes(T, V, D)
def fwd(ids=S, W=2 * S, y=3 * S, t=T, v=V, d=D, fn=lib.sgh_embedding_fwd_f32):
    return fn(ids, W, y, t, v, d, 1.0, -1, None), len(kernels())
def bwd(ids=S, dy=2 * S, add=None, dW=3 * S, t=T, v=V, d=D, ws=4 * S, n=need, fn=lib.sgh_embedding_bwd_f32):
    return fn(ids, dy, add, dW, t, v, d, 1.0, -1, ws, n, None), len(kernels())
table, rows = V * D * 4, T * D * 4
ok = [fwd(), fwd(y=2 * S + table), fwd(W=3 * S + rows), bwd(), bwd(add=5 * S), bwd(add=3 * S), bwd(add=3 * S + table), bwd(dW=2 * S + rows)]
refused = [fwd(ids=None), fwd(W=None), fwd(y=None), fwd(t=1 << 31), fwd(v=1 << 31), fwd(d=(1 << 21) + 1), fwd(y=2 * S), fwd(y=2 * S + table - 4),
           fwd(y=2 * S - rows + 4), fwd(y=S), fwd(y=S + T * 4 - 4),
           bwd(ids=None), bwd(dy=None), bwd(dW=None), bwd(t=1 << 31), bwd(v=1 << 31), bwd(d=(1 << 21) + 1), bwd(dW=2 * S), bwd(dW=2 * S - table + 4),
           bwd(dW=2 * S + rows - 4), bwd(dW=S), bwd(add=3 * S + 4), bwd(add=3 * S - table + 4), bwd(ws=4 * S + 4)]
short = [bwd(ws=None), bwd(n=need - 1), bwd(n=0), bwd(fn=lib.sgh_embedding_bwd_f16, ws=None), bwd(fn=lib.sgh_embedding_bwd_bf16, n=need - 1)]
nothing = [fwd(t=0, ids=None, W=None, y=None), fwd(d=0, y=None), bwd(v=0, dW=None), bwd(d=0, dy=None)]
answer([ok, refused, short, nothing])
""")
    assert all(rc == 0 and n > 0 for rc, n in ok), ok
    assert all(r == [EINVAL, 0] for r in refused), [(i, r) for i, r in enumerate(refused) if r != [EINVAL, 0]]
    assert all(r == [EWORKSPACE, 0] for r in short), short
    assert all(r == [0, 0] for r in nothing), nothing


def test_distillation_refusals():
    ok, short, refused, limit = recorded("""
S = SPACE
N, V, K = 6, 700, 9
inf, nan = float("inf"), float("nan")
def fwd(x=S, top=2 * S, teacher=3 * S, labels=4 * S, w=5 * S, n=N, v=V, k=K, tau=2.0, loss=6 * S, stats=7 * S, sfx="f32", ws=9 * S, wn=1 << 20):
    return getattr(lib, "sgh_distill_fwd_" + sfx)(x, top, teacher, labels, w, n, v, k, tau, 1.0, 1.0, loss, stats, ws, wn, None), len(kernels())
def bwd(x=S, stats=7 * S, top=2 * S, teacher=3 * S, labels=4 * S, w=5 * S, n=N, v=V, k=K, tau=2.0, dx=8 * S, sfx="f32"):
    return getattr(lib, "sgh_distill_bwd_" + sfx)(x, stats, top, teacher, labels, w, n, v, k, tau, 1.0, 1.0, 1.0, dx, None), len(kernels())
def both(x=S, top=2 * S, teacher=3 * S, labels=4 * S, w=5 * S, n=N, v=V, k=K, tau=2.0, loss=6 * S, dx=8 * S, sfx="f32", ws=9 * S, wn=1 << 20):
    return getattr(lib, "sgh_distill_fwd_bwd_" + sfx)(x, top, teacher, labels, w, n, v, k, tau, 1.0, 1.0, 1.0, loss, dx, ws, wn, None), len(kernels())
size = N * V * 4
ok = [f(**how) for f in (fwd, bwd, both) for how in ({}, {"k": 0, "top": None, "teacher": None}, {"labels": None, "w": None}, {"v": 1}, {"k": 1024},
                                                     {"v": 200000}, {"sfx": "f16"}, {"sfx": "bf16", "v": 50000})]
ok += [f(dx=S) for f in (bwd, both)] + [f(dx=S + size) for f in (bwd, both)] + [f(dx=S - size) for f in (bwd, both)]
refused = [f(**how) for f in (fwd, bwd, both) for how in ({"x": None}, {"top": None}, {"teacher": None}, {"v": 0}, {"n": 1 << 31}, {"v": (1 << 28) + 1},
                                                          {"tau": 0.0}, {"tau": -1.0}, {"tau": inf}, {"tau": nan}, {"tau": 1e-40}, {"tau": 1e30})]
refused += [fwd(loss=None), both(loss=None), fwd(stats=None), bwd(stats=None)]
for f in (bwd, both):
    refused += [f(dx=d) for d in (None, S + 4, S - size + 4, S + size - 4, 2 * S, 2 * S + N * K * 4 - 4, 3 * S, 4 * S, 5 * S)]
refused += [bwd(dx=7 * S), fwd(loss=S + size - 4), fwd(loss=2 * S), fwd(loss=7 * S + N * 12 - 4), fwd(loss=4 * S), fwd(stats=S), fwd(stats=3 * S + 4),
            fwd(stats=6 * S - N * 12 + 4), both(loss=8 * S + size - 4), both(loss=S), both(loss=5 * S)]
limit = [f(k=1025) for f in (fwd, bwd, both)]
empty = [f(n=0) for f in (fwd, bwd, both)]
ok += [(rc, 1 - n) for rc, n in empty]      # nothing to do, nothing launched
ok += [f(ws=None, wn=0) for f in (fwd, both)]
need = lib.sgh_distill_workspace_bytes(N, 200000, 4, 0)
assert need == lib.sgh_distill_workspace_bytes(N, 200000, 4, 1)
ok += [f(v=200000, wn=need) for f in (fwd, both)]
short = [f(v=200000, **how) for f in (fwd, both) for how in ({"wn": need - 1}, {"ws": None}, {"sfx": "bf16", "wn": 0})]
refused += [f(v=200000, ws=9 * S + 8) for f in (fwd, both)]
answer([ok, short, refused, limit])
""")
    assert all(rc == 0 and n in (1, 2) for rc, n in ok), ok
    assert all(r == [EWORKSPACE, 0] for r in short), short
    assert all(r == [EINVAL, 0] for r in refused), [(i, r) for i, r in enumerate(refused) if r != [EINVAL, 0]]
    assert all(r == [ELIMIT, 0] for r in limit), limit


def test_mirror_refusals():
    """Types, shapes and devices are looked at before anything is allocated: needs no GPU."""
    from singa_amd import singa_wrap as singa

    class _NoDevice(object):
        stream = None

    dev, other = _NoDevice(), _NoDevice()
    make = lambda shape, t=singa.kFloat32, d=dev: singa.from_device_pointer(0x1000, shape, d, t)
    ids, W, dy = make((3, 4), singa.kInt), make((10, 8)), make((3, 4, 8))
    for call in (lambda: singa.EmbeddingForward(make((3, 4)), W), lambda: singa.EmbeddingForward(ids, make((10, 8, 1))),
                 lambda: singa.EmbeddingForward(ids, W.T()), lambda: singa.EmbeddingForward(ids, make((10, 8), d=other)),
                 lambda: singa.EmbeddingForward(ids, make((10, 8), singa.kInt)),
                 lambda: singa.EmbeddingBackwardW(make((12, 8)), ids, W), lambda: singa.EmbeddingBackwardW(make((3, 4, 8), singa.kFloat16), ids, W),
                 lambda: singa.EmbeddingBackwardW(dy, ids, W, add=make((8, 10))), lambda: singa.EmbeddingBackwardW(dy, ids, W, out=make((10, 8), singa.kFloat16)),
                 lambda: singa.EmbeddingBackwardW(dy, ids, W, add=make((10, 8), d=other))):
        with pytest.raises(singa.SingaHipError):
            call()
    x, top, teacher, labels, stats = make((5, 20)), make((5, 3), singa.kInt), make((5, 3)), make((5,), singa.kInt), make((5, 3))
    for call in (lambda: singa.DistillationFwd(make((100,)), top, teacher), lambda: singa.DistillationFwd(x.T(), top, teacher),
                 lambda: singa.DistillationFwd(x, top, None), lambda: singa.DistillationFwd(x, None, teacher),
                 lambda: singa.DistillationFwd(x, make((5, 3)), teacher), lambda: singa.DistillationFwd(x, top, make((5, 3), singa.kFloat16)),
                 lambda: singa.DistillationFwd(x, top, make((5, 4))), lambda: singa.DistillationFwd(x, make((4, 3), singa.kInt), make((4, 3))),
                 lambda: singa.DistillationFwd(x, top, teacher, labels=make((5,))), lambda: singa.DistillationFwd(x, top, teacher, labels=make((4,), singa.kInt)),
                 lambda: singa.DistillationFwd(x, top, teacher, weights=make((5,), singa.kInt)), lambda: singa.DistillationFwd(x, top, make((5, 3), d=other)),
                 lambda: singa.DistillationFwd(make((5, 20), singa.kInt), top, teacher),
                 lambda: singa.DistillationBwd(x, make((5, 2)), top, teacher), lambda: singa.DistillationBwd(x, stats, top, teacher, out=make((5, 21))),
                 lambda: singa.DistillationFwdBwd(x, top, teacher, labels=labels, out=make((5, 20), singa.kFloat16))):
        with pytest.raises(singa.SingaHipError):
            call()


# ------------------------------------------------------------------------------------ launches

def test_what_the_embedding_launches():
    """Few tokens in one launch without a workspace, up to 8192 sorted by one more, others by two launches for each 9 bits of the ids;
    grids of the largest sizes stay within a launch."""
    few, one, two, three, largest = recorded("""
S = SPACE
def run(t, v, d, add=None, fn=lib.sgh_embedding_bwd_bf16):
    need = lib.sgh_embedding_bwd_workspace_bytes(t, v, d)
    rc = fn(S, 2 * S, add, 3 * S, t, v, d, 1.0, -1, 4 * S if need else None, need, None)
    return rc, need, [n[n.index("k_embed"):][:12] for n, _, _ in launched()]
most = (1 << 31) - 1
largest = [lib.sgh_embedding_fwd_f32(S, 1 << 50, 1 << 55, most, most, 4, 1.0, -1, None), lib.sgh_embedding_fwd_f32(S, 1 << 50, 1 << 55, 5, 7, 1 << 21, 1.0, -1, None)]
S2 = 1 << 50
for t, v, d in ((5, most, 4), (most, 9, 4), (9000, 7, 1 << 21), (17000, 7, 1 << 21), (most, most, 1)):
    need = lib.sgh_embedding_bwd_workspace_bytes(t, v, d)
    largest.append(lib.sgh_embedding_bwd_f32(S2, 2 * S2, None, 3 * S2, t, v, d, 1.0, -1, 4 * S2, need, None))
launched()
answer([run(512, 5000, 64), run(8192, 5000, 64), run(8193, 131071, 64), run(8193, 1 << 18, 64), largest])
""")
    assert few[:2] == [0, 0] and [k[:11] for k in few[2]] == ["k_embed_row"], few
    assert one[0] == 0 and one[1] > 0 and [k[:11] for k in one[2]] == ["k_embed_ran", "k_embed_til", "k_embed_joi"], one
    pair = ["k_embed_cou", "k_embed_mov"]
    assert [k[:11] for k in two[2]] == 2 * pair + ["k_embed_til", "k_embed_joi"], two
    assert [k[:11] for k in three[2]] == 3 * pair + ["k_embed_til", "k_embed_joi"], three
    assert all(rc == 0 for rc in largest), largest


def test_what_the_distillation_launches():
    """One launch; two for the loss of few long rows, which are cut in parts, and a workspace then."""
    got = recorded("""
S = 1 << 50
out = []
for n, v, k in ((1, 1, 0), (3, 1000, 5), (1 << 20, 32, 64), ((1 << 31) - 1, 1, 0), (5000, 131072, 64), (300, 300000, 3), (7, 1 << 28, 1024), (1, 131072, 16)):
    for sfx, e in (("f32", 4), ("f16", 2), ("bf16", 2)):
        need = lib.sgh_distill_workspace_bytes(n, v, e, 1)
        a = (S, 2 * S, 3 * S, 4 * S, 5 * S, n, v, k, 1.5, 1.0, 1.0)
        ws = (9 * S if need else None, need, None)
        rcs = [getattr(lib, "sgh_distill_fwd_" + sfx)(*a, 6 * S, 7 * S, *ws), len(kernels()), getattr(lib, "sgh_distill_fwd_bwd_" + sfx)(*a, 1.0, 6 * S, 8 * S, *ws),
               len(kernels()), getattr(lib, "sgh_distill_bwd_" + sfx)(S, 7 * S, *a[1:], 1.0, 8 * S, None), len(kernels())]
        out.append((n <= 7 and v > 100000, need, rcs))
answer(out)
""")
    for parts, need, rcs in got:
        if rcs[3] == 2048:   # (2^31 rows of one: 2^20 of them a launch)
            rcs[3] = 1
        assert (need > 0) == parts and rcs == ([0, 2, 0, 2, 0, 1] if parts else [0, 1, 0, 1, 0, 1]), got


# ------------------------------------------------------------------------------------ counts of what is out of range

# A counter in memory, to which an operator on another stream adds 2 right behind each time that it is read
COUNTER = r"""
static int counter = 3;
extern "C" {
int hipStreamSynchronize(void *) { return 0; }
int hipGetSymbolAddress(void **p, const void *) { *p = &counter; return 0; }
static int copy(void *to, const void *from, size_t n) { memcpy(to, from, n); if (from == &counter) counter += 2; return 0; }
int hipMemcpyAsync(void *to, const void *from, size_t n, int, void *) { return copy(to, from, n); }
int hipMemcpy(void *to, const void *from, size_t n, int) { return copy(to, from, n); }
int hipMemcpyFromSymbol(void *to, const void *, size_t n, size_t, int) { return copy(to, &counter, n); }
int hipMemcpyToSymbol(const void *, const void *from, size_t n, size_t, int) { return copy(&counter, from, n); }
int recorder_left() { return counter; }
}
// the one kernel that is run here: (counter, what is taken off)
static int subtracting(const void *f, void **args) {
  if (names()[f].find("k_subtract") != std::string::npos) **static_cast<int **>(args[0]) -= *static_cast<int *>(args[1]);
  return 0;
}
"""


@pytest.mark.parametrize("entry", ["sgh_embedding_index_errors", "sgh_distill_index_errors", "sgh_softmax_ce_label_errors"])
def test_index_errors_met_while_they_are_read_are_counted_next_time(monkeypatch, entry):
    import hip_recorder
    launch = "int hipLaunchKernel(const void *f, Dim g, Dim b, void **, size_t, void *) { return launch(f, g, b); }"
    assert launch in hip_recorder.SOURCE
    source = hip_recorder.SOURCE.replace(launch, launch.replace("void **,", "void **args,").replace("{ ", "{ subtracting(f, args); "))
    monkeypatch.setattr(hip_recorder, "SOURCE", source.replace('extern "C" {', COUNTER + 'extern "C" {', 1))
    got = recorded("""
n = C.c_int()
out = []
for _ in range(3):
    assert lib.%s(None, C.byref(n)) == 0
    out.append(n.value)
answer([out, recorder.recorder_left(), lib.%s(None, None)])
""" % (entry, entry))
    assert got == [[3, 2, 2], 2, EINVAL]   # nothing is lost, nothing counted twice


# ------------------------------------------------------------------------------------ kernels

def test_every_kernel_of_the_token_model_is_reached(monkeypatch):
    """Each form that is built is what some call launches (256 compute units)."""
    import hip_recorder
    monkeypatch.setattr(hip_recorder, "SOURCE", hip_recorder.SOURCE + r"""
extern "C" const char *recorder_built() {
  static std::string out;
  for (auto &n : names()) out += n.second + "\n";
  return out.c_str();
}
""")
    built, run = recorded("""
S, out = 1 << 50, set()
def note():
    out.update(n for n, _, _ in launched())
for sfx, e in (("f32", 4), ("f16", 2), ("bf16", 2)):
    for n in (1, 16, 100, 200, 400, 1000, 3000, 20000, 300000):
        for v in (2, 200, 1000, 3000, 7000, 15000, 20000, 30000, 40000, 60000, 120000, 300000):
            for sizes in ((n, v, 0), (n, v, 100)):
                need = [lib.sgh_distill_workspace_bytes(n, v, e, g) for g in (0, 1)]
                a = (S, 2 * S, 3 * S, 4 * S, 5 * S) + sizes + (1.5, 1.0, 1.0)
                assert getattr(lib, "sgh_distill_fwd_" + sfx)(*a, 6 * S, 7 * S, 9 * S, need[0], None) == 0
                assert getattr(lib, "sgh_distill_fwd_bwd_" + sfx)(*a, 1.0, 6 * S, 8 * S, 9 * S, need[1], None) == 0
                assert getattr(lib, "sgh_distill_bwd_" + sfx)(S, 7 * S, *a[1:], 1.0, 8 * S, None) == 0
            note()
    for t in (1, 300, 3000, 8193, 100000, 40000000):
        for v, d in ((1000, 1), (1000, 100), (40000, 3), (40000, 1024), (300000, 100), (300000, 8), (300000, 1024), (1000, 8192)):
            need = lib.sgh_embedding_bwd_workspace_bytes(t, v, d)
            assert getattr(lib, "sgh_embedding_fwd_" + sfx)(S, 2 * S, 3 * S, t, v, d, 1.0, -1, None) == 0
            assert getattr(lib, "sgh_embedding_bwd_" + sfx)(S, 2 * S, None, 3 * S, t, v, d, 1.0, -1, 4 * S, need, None) == 0
        note()
recorder.recorder_built.restype = C.c_char_p
answer([recorder.recorder_built().decode().split(), sorted(out)])
""")
    ours = {n for n in built if "k_embed_" in n or "k_distill_" in n}
    assert len(ours) > 100 and set(run) <= ours
    left = sorted(ours - set(run))
    assert not left, "\n" + "\n".join(left)
