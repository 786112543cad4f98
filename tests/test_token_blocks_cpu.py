"""Attention and the norms around blocks without a GPU: the definitions against differences, the borders of the position buckets, refusals of the C
ABI and of the Python mirror, and what the entry points launch (a stand-in for the HIP runtime, hip_recorder.py)."""
import ctypes as C

import numpy as np
import pytest

from hip_recorder import recorded
from oracle import block_ops as O
from oracle.ops import OracleOps
from singa_amd import _lib
from singa_amd import workloads as wl

EINVAL, EWORKSPACE, ELIMIT = -1, -2, -6


def test_attention_gradients_are_the_differences():
    r = np.random.default_rng(1)
    a = O.Attn(True, buckets=6, max_distance=5)
    args = [r.standard_normal(s) for s in ((2, 7, 4, 3), (2, 9, 2, 3), (2, 9, 2, 3), (6, 4))]
    lengths, do = ((7, 4), (9, 5), (1, 0)), r.standard_normal((2, 7, 4, 3))
    o, lse = O.attention(a, *args, *lengths)
    grads = O.attention_bwd(a, do, *args[:3], o, lse, args[3], *lengths)
    for i, g in enumerate(grads):
        along = r.standard_normal(args[i].shape)
        ends = [(O.attention(a, *[x + h * along if j == i else x for j, x in enumerate(args)], *lengths)[0] * do).sum() for h in (1e-5, -1e-5)]
        assert abs((ends[0] - ends[1]) / 2e-5 - (g * along).sum()) < 1e-7
    assert not o[1, 4:].any() and (lse[1, :, 4:] == -np.inf).all() and not grads[1][1, 5:].any()


@pytest.mark.parametrize("buckets,distance,both", [(32, 128, True), (32, 128, False), (8, 300, True), (5, 7, False), (64, 1024, True), (64, 33, False),
                                                   (128, 1024, True), (2, 2, False), (4, 1024, True), (6, 16, False)])
def test_borders_of_the_buckets(buckets, distance, both):
    """Powers land on borders (16 is the first of its bucket with 8 single ones and 128 at the end of 8 more): whole numbers decide."""
    g = _lib.AttnGeom()
    assert _lib.lib().sgh_attn_geom_init(C.byref(g), 1, 4, 4, 2, 1, 8, 0, 1.0, buckets, distance, int(both)) == 0
    a = O.Attn(buckets=buckets, max_distance=distance, bidirectional=both)
    n = buckets // 2 if both else buckets
    assert g.bounds == n - 1
    borders = list(g.bound[:g.bounds])
    for m in range(distance + 3):
        assert sum(b <= m for b in borders) == a.bucket(-m), m
        assert a.bucket(m) == (a.bucket(-m) + n if both and m else 0)


def test_sequence_step_matches_differences():
    """The whole tape of a token model with blocks: parameters' gradients against differences of the loss (the oracle's, in 64 bits between
    fp32 roundings)."""
    ops = OracleOps()
    ids, targets = wl.make_inputs("token_attention_small", 2)
    net = wl.build("token_attention_small", ops, lr=0.0, momentum=0.0)

    def loss():
        return np.asarray(net.forward(*net.inputs(ids, targets)), np.float64).sum() / (2 * 11)

    loss()
    net.backward_and_update(keep_grads=True)
    grads = {k: v.astype(np.float64) for k, v in net.grad_log.items()}
    r = np.random.default_rng(2)
    params = dict(net.params())
    for name in ("blocks.0.attention.table", "blocks.0.attention.q.W", "blocks.0.attention.v.W", "blocks.0.norm0.gate", "blocks.0.norm0.post",
                 "blocks.0.norm1.pre", "blocks.norm.pre", "embedding.W"):
        p = params[name]
        along = r.standard_normal(p.shape).astype(np.float32)
        kept, step, ends = p.copy(), 2e-3, []
        for sign in (1, -1):
            p[...] = kept + sign * np.float32(step) * along
            ends.append(loss())
        p[...] = kept
        got, want = (ends[0] - ends[1]) / (2 * step), (grads[name] * along).sum()
        # fp32 losses of about 12: 12 * 2^-23 / 4e-3 = 4e-4 and as much from the chain in front of them; second differences over the step
        assert abs(got - want) < 4e-3 + 0.03 * np.sqrt((grads[name] ** 2).sum()), (name, got, want)


# ------------------------------------------------------------------------------------ refusals

def test_geometry_refusals():
    g, lib = _lib.AttnGeom(), _lib.lib()
    good = dict(batch=2, q_len=5, k_len=7, heads=4, kv_heads=2, dim=16, causal=0, scale=0.5, buckets=0, max_distance=0, both=0)
    run = lambda **how: lib.sgh_attn_geom_init(C.byref(g), *dict(good, **how).values())
    nan, inf = float("nan"), float("inf")
    for how in (dict(), dict(batch=0), dict(q_len=0), dict(k_len=0), dict(dim=128), dict(heads=1, kv_heads=1), dict(scale=0.0), dict(scale=-3.0),
                dict(buckets=2, max_distance=2), dict(buckets=4, max_distance=2, both=1), dict(buckets=64, max_distance=1024), dict(buckets=128, max_distance=1024, both=1),
                dict(batch=65536, heads=32, kv_heads=1), dict(heads=8192, kv_heads=8192, dim=128)):
        assert run(**how) == 0, how
    for how in (dict(batch=-1), dict(q_len=-1), dict(k_len=-1), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(scale=nan), dict(scale=inf),
                dict(buckets=1, max_distance=9), dict(buckets=-4, max_distance=9), dict(buckets=2, max_distance=9, both=1), dict(buckets=7, max_distance=9, both=1),
                dict(buckets=8, max_distance=4), dict(buckets=8, max_distance=-1)):
        assert run(**how) == EINVAL, how
    for how in (dict(dim=129), dict(q_len=(1 << 28) + 1), dict(heads=16384, kv_heads=1, dim=128), dict(batch=1 << 20, heads=8, kv_heads=1),
                dict(k_len=1 << 28, batch=2), dict(buckets=65, max_distance=1000), dict(buckets=130, max_distance=1000, both=1), dict(buckets=8, max_distance=1025)):
        assert run(**how) == ELIMIT, how
    assert lib.sgh_attn_geom_init(None, *good.values()) == EINVAL
    assert lib.sgh_attn_fwd_workspace_bytes(None) == 0 and lib.sgh_attn_bwd_workspace_bytes(None) == 0
    run(buckets=8, max_distance=20)
    g.bounds = 64    # a structure that was not filled in
    assert lib.sgh_attn_fwd_f32(C.byref(g), *[1 << 40] * 10, 1 << 40, None) == EINVAL


def test_attention_refusals():
    ok, refused, short = recorded("""
S = SPACE
g, gb = _lib.AttnGeom(), _lib.AttnGeom()
B, SQ, SK, H, G, D = 2, 50, 600, 4, 2, 24
assert lib.sgh_attn_geom_init(C.byref(g), B, SQ, SK, H, G, D, 1, 0.2, 0, 0, 0) == 0
assert lib.sgh_attn_geom_init(C.byref(gb), B, SQ, SK, H, G, D, 1, 0.2, 8, 20, 1) == 0
nf, nb = lib.sgh_attn_fwd_workspace_bytes(C.byref(g)), lib.sgh_attn_bwd_workspace_bytes(C.byref(gb))
assert nf and nb
def fwd(geom=g, q=S, k=2 * S, v=3 * S, table=None, ql=None, kl=None, st=None, o=5 * S, lse=6 * S, ws=7 * S, n=nf, sfx="f32"):
    return getattr(lib, "sgh_attn_fwd_" + sfx)(C.byref(geom), q, k, v, table, ql, kl, st, o, lse, ws, n, None), len(kernels())
def bwd(geom=gb, do=8 * S, q=S, k=2 * S, v=3 * S, o=5 * S, lse=6 * S, table=4 * S, ql=None, kl=None, st=None, dq=9 * S, dk=10 * S, dv=11 * S,
        dt=12 * S, ws=7 * S, n=nb, sfx="f32"):
    return getattr(lib, "sgh_attn_bwd_" + sfx)(C.byref(geom), do, q, k, v, o, lse, table, ql, kl, st, dq, dk, dv, dt, ws, n, None), len(kernels())
qn, kn, ln, tn = B * SQ * H * D * 4, B * SK * G * D * 4, B * SQ * H * 4, 8 * H * 4
lengths = dict(ql=13 * S, kl=14 * S, st=15 * S)
ok = [fwd(), fwd(**lengths), fwd(geom=gb, table=4 * S, n=1 << 30), fwd(o=S + qn), fwd(lse=5 * S + qn), fwd(sfx="f16"), fwd(sfx="bf16", q=S + 2), bwd(), bwd(**lengths),
      bwd(sfx="f16"), bwd(sfx="bf16"), bwd(dk=9 * S + qn, dv=9 * S + qn + kn), fwd(k=2 * S, v=2 * S), bwd(k=2 * S, v=2 * S)]
refused = [fwd(q=None), fwd(k=None), fwd(v=None), fwd(o=None), fwd(lse=None), fwd(geom=gb, n=1 << 30), fwd(o=S), fwd(o=2 * S - qn + 4), fwd(o=3 * S + kn - 4),
           fwd(lse=5 * S + qn - 4), fwd(lse=2 * S), fwd(ws=7 * S + 4), fwd(ws=5 * S), fwd(ws=S), fwd(o=13 * S, ql=13 * S + 4), fwd(lse=14 * S, kl=14 * S),
           fwd(geom=gb, table=4 * S, o=4 * S + 16, n=1 << 30), fwd(st=5 * S)]
refused += [bwd(**{n: None}) for n in ("do", "q", "k", "v", "o", "lse", "table", "dq", "dk", "dv", "dt")]
refused += [bwd(dq=8 * S), bwd(dq=S), bwd(dk=2 * S + kn - 4), bwd(dv=3 * S), bwd(dt=4 * S), bwd(dt=12 * S, dq=12 * S + tn - 4), bwd(dv=10 * S + 4), bwd(dq=5 * S),
            bwd(dq=6 * S), bwd(ws=7 * S + 8), bwd(ws=9 * S), bwd(ws=8 * S), bwd(dk=13 * S, kl=13 * S)]
short = [fwd(ws=None), fwd(n=nf - 1), fwd(n=0), bwd(ws=None), bwd(n=nb - 1), bwd(sfx="bf16", n=0)]
answer([ok, refused, short])
""")
    assert all(rc == 0 and n > 0 for rc, n in ok), ok
    assert all(r == [EINVAL, 0] for r in refused), [(i, r) for i, r in enumerate(refused) if r != [EINVAL, 0]]
    assert all(r == [EWORKSPACE, 0] for r in short), short


def test_residual_norm_refusals():
    ok, refused, limit, short, nothing = recorded("""
S = SPACE
R, D, G = 60, 200, 4
inf, nan = float("inf"), float("nan")
need = lib.sgh_residual_norm_bwd_workspace_bytes(R, D, G, 4)
assert need and lib.sgh_residual_norm_bwd_workspace_bytes(0, D, 0, 4) == 0 and lib.sgh_residual_norm_bwd_workspace_bytes(R, D, 7, 4) == 0
def fwd(x=S, h=2 * S, post=3 * S, gate=4 * S, pre=5 * S, r=R, d=D, g=G, eps=1e-5, y=6 * S, n=7 * S, stats=8 * S, sfx="f32"):
    return getattr(lib, "sgh_residual_norm_fwd_" + sfx)(x, h, post, gate, pre, r, d, g, 0.5, eps, y, n, stats, None), len(kernels())
def bwd(dy=9 * S, dn=10 * S, y=6 * S, stats=8 * S, h=2 * S, post=3 * S, gate=4 * S, pre=5 * S, r=R, d=D, g=G, dx=11 * S, dh=12 * S, dpost=13 * S, dgate=14 * S,
        dpre=15 * S, ws=16 * S, n=need, sfx="f32"):
    return getattr(lib, "sgh_residual_norm_bwd_" + sfx)(dy, dn, y, stats, h, post, gate, pre, r, d, g, 0.5, dx, dh, dpost, dgate, dpre, ws, n, None), len(kernels())
size = R * D * 4
no_gate, first = dict(gate=None, g=0), dict(h=None, post=None, gate=None)
ok = [fwd(), fwd(**no_gate), fwd(post=None), fwd(pre=None, n=None), fwd(y=None, **first), fwd(y=S + size), fwd(eps=0.0), fwd(sfx="f16", x=S + 2), fwd(sfx="bf16"), fwd(d=16384),
      fwd(x=S, h=S), bwd(), bwd(**no_gate), bwd(dgate=None, **no_gate), bwd(dy=None), bwd(post=None, dpost=None), bwd(pre=None, dn=None, y=None, dpre=None), bwd(dh=None, dpost=None, dgate=None, **first),
      bwd(sfx="f16"), bwd(sfx="bf16", n=1 << 30), bwd(dx=9 * S + size), bwd(dy=10 * S), bwd(d=16384, n=1 << 40)]
refused = [fwd(x=None), fwd(y=None), fwd(n=None), fwd(stats=None), fwd(h=None), fwd(h=None, post=None), fwd(h=None, gate=None), fwd(pre=None, y=None, **first), fwd(g=0), fwd(g=7), fwd(g=61),
           fwd(r=1 << 31), fwd(eps=-1.0), fwd(eps=nan), fwd(eps=inf), fwd(y=S), fwd(y=2 * S + size - 4), fwd(y=7 * S - size + 4), fwd(n=S), fwd(n=3 * S + 4), fwd(n=5 * S), fwd(n=4 * S),
           fwd(stats=6 * S + size - 4), fwd(stats=S)]
refused += [bwd(**{n: None}) for n in ("dn", "y", "stats", "h", "dx", "dh", "dpost", "dgate", "dpre")]
refused += [bwd(dy=None, dn=None, pre=None, dpre=None), bwd(g=0), bwd(g=7), bwd(r=1 << 31), bwd(dx=9 * S), bwd(dx=10 * S), bwd(dx=6 * S), bwd(dx=12 * S + 4), bwd(dh=2 * S), bwd(dh=10 * S),
            bwd(dpost=3 * S), bwd(dpost=13 * S, dpre=13 * S + D * 4 - 4), bwd(dgate=4 * S), bwd(dpre=5 * S), bwd(dpre=8 * S), bwd(ws=16 * S + 8), bwd(ws=9 * S), bwd(ws=11 * S + 16)]
limit = [fwd(d=16385), bwd(d=16385)]
short = [bwd(ws=None), bwd(n=need - 1), bwd(n=0, sfx="f16")]
nothing = [fwd(r=0, x=None), fwd(d=0), bwd(d=0)]
answer([ok, refused, limit, short, nothing])
""")
    assert all(rc == 0 and n > 0 for rc, n in ok), ok
    assert all(r == [EINVAL, 0] for r in refused), [(i, r) for i, r in enumerate(refused) if r != [EINVAL, 0]]
    assert all(r == [ELIMIT, 0] for r in limit) and all(r == [EWORKSPACE, 0] for r in short) and all(r == [0, 0] for r in nothing), (limit, short, nothing)


def test_mirror_refusals():
    """Types, shapes and devices are looked at before anything is allocated: needs no GPU."""
    from singa_amd import singa_wrap as singa

    class _NoDevice(object):
        stream = None

    dev, other = _NoDevice(), _NoDevice()
    make = lambda shape, t=singa.kFloat32, d=dev: singa.from_device_pointer(0x1000, shape, d, t)
    q, k, lse, ints = make((2, 5, 4, 8)), make((2, 7, 2, 8)), make((2, 4, 5)), make((2,), singa.kInt)
    table = make((8, 4))
    plain, biased = singa.AttentionHandle(q, k), singa.AttentionHandle(q, k, buckets=8, max_distance=20)
    A, half = singa.AttentionHandle, make((2, 5, 4, 8), singa.kFloat16)
    fwd = lambda h=plain, q=q, k=k, v=k, **how: (lambda: singa.AttentionForward(h, q, k, v, **how))
    bwd = lambda h=plain, do=q, q=q, k=k, v=k, o=q, lse=lse, **how: (lambda: singa.AttentionBackward(h, do, q, k, v, o, lse, **how))
    for call in (lambda: A(make((2, 5, 32)), k), lambda: A(q, make((3, 7, 2, 8))), lambda: A(q, make((2, 7, 2, 9))), lambda: A(q, make((2, 7, 3, 8))), lambda: A(half, k),
                 lambda: A(ints.Reshape((2, 1, 1, 1)), ints.Reshape((2, 1, 1, 1))), lambda: A(make((2, 5, 4, 200)), make((2, 5, 4, 200))), lambda: A(q, k, buckets=7),
                 lambda: A(q, k, buckets=8, max_distance=2), lambda: A(q, k, scale=float("nan")),
                 fwd(q=half), fwd(q=make((2, 6, 4, 8))), fwd(k=make((2, 7, 4, 8))), fwd(v=make((2, 7, 2, 8), singa.kFloat16)), fwd(v=make((2, 7, 2, 8), d=other)), fwd(table=table),
                 fwd(h=biased), fwd(h=biased, table=make((4, 8))), fwd(h=biased, table=make((8, 4), singa.kFloat16)), fwd(h=biased, table=make((4, 8)).T()), fwd(k_lengths=make((2,))),
                 fwd(q_lengths=make((3,), singa.kInt)), fwd(q_starts=make((2,), singa.kInt, other)), bwd(do=half), bwd(o=make((2, 5, 4, 9))), bwd(lse=make((2, 5, 4))),
                 bwd(lse=make((2, 4, 5), singa.kFloat16)), bwd(lse=make((2, 4, 5), d=other)), bwd(h=biased)):
        with pytest.raises(singa.SingaHipError):
            call()
    x, w, gate, stats = make((3, 4, 6)), make((6,)), make((4, 6)), make((12, 2))
    F, B = singa.ResidualNormForward, singa.ResidualNormBackward
    for call in (lambda: F(x), lambda: F(x, post=w, pre=w), lambda: F(x, gate=gate, pre=w), lambda: F(make(())), lambda: F(x, make((12, 6))), lambda: F(x, make((3, 4, 6), singa.kFloat16)),
                 lambda: F(x, x, post=make((4,))), lambda: F(x, x, pre=make((6,), singa.kFloat16)), lambda: F(x, x, gate=make((5, 6))), lambda: F(x, x, gate=make((6,))),
                 lambda: F(x, x, gate=make((4, 6), singa.kFloat16)), lambda: F(x, x, gate=make((0, 6))), lambda: F(x, x, pre=make((6,), d=other)), lambda: F(ints, ints, pre=w),
                 lambda: B(x, None, x, stats, pre=w), lambda: B(x, x, x, stats, x), lambda: B(None, None, x, stats, x), lambda: B(x, x, x, make((12, 3)), pre=w),
                 lambda: B(make((12, 6)), x, x, stats, pre=w), lambda: B(x, x, x, make((12, 2), d=other), pre=w), lambda: B(x, x, make((3, 4, 6), d=other), stats, pre=w)):
        with pytest.raises(singa.SingaHipError):
            call()


# ------------------------------------------------------------------------------------ launches

def test_largest_sizes_stay_within_a_launch_and_every_kernel_is_reached(monkeypatch):
    """Each form that is built is what some call launches (256 compute units); grids of the largest sizes stay within a launch."""
    import hip_recorder
    monkeypatch.setattr(hip_recorder, "SOURCE", hip_recorder.SOURCE + r"""
extern "C" const char *recorder_built() {
  static std::string out;
  for (auto &n : names()) out += n.second + "\n";
  return out.c_str();
}
""")
    built, run, largest = recorded("""
S, out, largest = 1 << 50, set(), []
def note():
    out.update(n for n, _, _ in launched())
def attention(sfx, *how):
    g = _lib.AttnGeom()
    assert lib.sgh_attn_geom_init(C.byref(g), *how) == 0, how
    t = S * 4 if how[8] else None
    f, b = lib.sgh_attn_fwd_workspace_bytes(C.byref(g)), lib.sgh_attn_bwd_workspace_bytes(C.byref(g))
    rcs = [getattr(lib, "sgh_attn_fwd_" + sfx)(C.byref(g), S, 2 * S, 3 * S, t, None, None, None, 5 * S, 6 * S, 7 * S, f, None),
           getattr(lib, "sgh_attn_bwd_" + sfx)(C.byref(g), 8 * S, S, 2 * S, 3 * S, 5 * S, 6 * S, t, None, None, None, 9 * S, 10 * S, 11 * S, 12 * S if t else None, 7 * S, b, None)]
    note()
    return rcs
for sfx in ("f32", "f16", "bf16"):
    for d in (16, 33, 80, 128):
        for buckets in (0, 32):
            for sizes in ((1, 1, 5000, 8, 2), (1, 60, 60, 2, 2), (8, 2000, 2000, 16, 16), (2, 100, 9000, 4, 1), (2, 9000, 100, 4, 1)):
                assert attention(sfx, *sizes, d, 0, 0.1, buckets, 100, 1) == [0, 0]
    largest += attention(sfx, 1, 1 << 26, 1, 1, 1, 128, 0, 0.1, 0, 0, 0) + attention(sfx, 1, 1, 1 << 26, 1, 1, 128, 0, 0.1, 32, 1024, 1) + attention(sfx, 1 << 21, 1, 1, 2, 1, 8, 0, 0.1, 0, 0, 0)
    largest += attention(sfx, 65536, 7, 3, 64, 64, 128, 0, 0.1, 128, 1024, 1)
    e = 4 if sfx == "f32" else 2
    for d in (1, 30, 200, 500, 1000, 2000, 4000, 8000, 16000):
        for rows, gates in ((1, 1), (7000, 0), (70000, 7), (70000, 70000), ((1 << 31) - 1, 1 if d < 100 else 0)):
            n = lib.sgh_residual_norm_bwd_workspace_bytes(rows, d, gates, e)
            g = 4 * S if gates else None
            largest.append(getattr(lib, "sgh_residual_norm_fwd_" + sfx)(S, 2 * S, 3 * S, g, 5 * S, rows, d, gates, 0.5, 1e-5, 6 * S, 7 * S, 8 * S, None))
            largest.append(getattr(lib, "sgh_residual_norm_bwd_" + sfx)(9 * S, 10 * S, 6 * S, 8 * S, 2 * S, 3 * S, g, 5 * S, rows, d, gates, 0.5, 11 * S, 12 * S, 13 * S, 14 * S, 15 * S,
                                                                         16 * S, n, None))
            note()
recorder.recorder_built.restype = C.c_char_p
answer([recorder.recorder_built().decode().split(), sorted(out), largest])
""")
    assert all(rc == 0 for rc in largest), largest
    ours = {n for n in built if "k_attn_" in n or "k_norm_" in n}
    assert len(ours) > 100 and not {n for n in run if "k_attn" in n or "k_norm" in n} - ours
    left = sorted(ours - set(run))
    assert not left, "\n" + "\n".join(left)


@pytest.mark.parametrize("q_len,k_len", [(0, 256), (0, 257), (0, 5000), (0, 1 << 24), (5000, 0), (1 << 20, 0), (0, 0), (1, 1 << 24)])
def test_geometries_without_queries_or_keys(q_len, k_len):
    """What a handle asks for of an empty batch of queries over a cache, and of queries over an empty one; in a process of its own."""
    asked, runs = recorded("""
S, runs, asked = 1 << 50, [], []
for buckets in (0, 8):
    g = _lib.AttnGeom()
    assert lib.sgh_attn_geom_init(C.byref(g), 2, %d, %d, 4, 2, 24, 0, 0.2, buckets, 20, 1) == 0
    f, b = lib.sgh_attn_fwd_workspace_bytes(C.byref(g)), lib.sgh_attn_bwd_workspace_bytes(C.byref(g))
    asked.append([f, b])
    t, d = (4 * S, 12 * S) if buckets else (None, None)
    for sfx in ("f32", "f16", "bf16"):
        runs.append(getattr(lib, "sgh_attn_fwd_" + sfx)(C.byref(g), S, 2 * S, 3 * S, t, None, None, None, 5 * S, 6 * S, 7 * S, f, None))
        runs.append(getattr(lib, "sgh_attn_bwd_" + sfx)(C.byref(g), 8 * S, S, 2 * S, 3 * S, 5 * S, 6 * S, t, None, None, None, 9 * S, 10 * S, 11 * S, d, 7 * S, b, None))
answer([asked, runs])
""" % (q_len, k_len))
    assert runs == [0] * len(runs)
    if q_len == 0:
        assert all(f == 0 for f, _ in asked)


def test_copied_attention_handles_pass_their_own_geometry(monkeypatch):
    """Both passes of a handle that was copied, unpickled or given another geometry call with the structure that it holds."""
    import copy
    import pickle

    from singa_amd import singa_wrap as singa

    class Device(object):
        stream = None

    passed, dev = [], Device()
    make = lambda shape: singa.from_device_pointer(4096, shape, dev, singa.kFloat32)
    q, k, lse = make((2, 5, 4, 8)), make((2, 7, 2, 8)), make((2, 4, 5))
    monkeypatch.setattr(singa, "_fn", lambda name, t: (lambda geom, *rest: passed.append(geom) or 0, name))
    monkeypatch.setattr(singa, "_empty", lambda *a: q)
    monkeypatch.setattr(singa, "_like", lambda t: t)
    h = singa.AttentionHandle(q, k)
    other, loaded = copy.deepcopy(h), pickle.loads(pickle.dumps(h))
    for handle in (h, other, loaded):
        singa.AttentionForward(handle, q, k, k)
        singa.AttentionBackward(handle, q, q, k, k, q, lse)
    assert passed == [C.addressof(x.geom) for x in (h, other, loaded) for _ in range(2)] and len(set(passed)) == 3
    for x in (other, loaded):
        assert bytes(x.geom) == bytes(h.geom) and vars(x).keys() == vars(h).keys()
    h.geom = other.geom
    singa.AttentionForward(h, q, k, k)
    assert passed[-1] == C.addressof(other.geom)


def test_most_heads_with_a_position_bias():
    """Every head has a sum for every bucket: heads of one value, as many as a row may have, stay within a launch."""
    runs, seen = recorded("""
S, runs, seen = 1 << 50, [], []
for heads, buckets, both in ((1 << 20, 128, 1), (1 << 20, 2, 0), (1 << 19, 64, 0)):
    g = _lib.AttnGeom()
    assert lib.sgh_attn_geom_init(C.byref(g), 1, 5, 5, heads, 1, 1, 0, 1.0, buckets, 128, both) == 0
    f, b = lib.sgh_attn_fwd_workspace_bytes(C.byref(g)), lib.sgh_attn_bwd_workspace_bytes(C.byref(g))
    for sfx in ("f32", "f16", "bf16"):
        runs.append(getattr(lib, "sgh_attn_fwd_" + sfx)(C.byref(g), S, 2 * S, 3 * S, 4 * S, None, None, None, 5 * S, 6 * S, 7 * S, f, None))
        launched()
        runs.append(getattr(lib, "sgh_attn_bwd_" + sfx)(C.byref(g), 8 * S, S, 2 * S, 3 * S, 5 * S, 6 * S, 4 * S, None, None, None, 9 * S, 10 * S, 11 * S, 12 * S, 7 * S, b, None))
        seen += [[heads * buckets, x * y * z, t] for n, (x, y, z), t in launched() if "k_attn_dtable" in n]
answer([runs, seen])
""")
    assert runs == [0] * 18
    assert len(seen) == 9 and all(want == blocks and threads == 256 for want, blocks, threads in seen), seen


@pytest.mark.parametrize("how", [dict(batch=1 << 21, q_len=(1 << 28) - 32, heads=1 << 20), dict(batch=1 << 30, q_len=(1 << 28) - 32, heads=1 << 11),
                                 dict(batch=1 << 21, k_len=(1 << 28) - 32, heads=1 << 20, kv_heads=1 << 20), dict(batch=(1 << 31) - 1, q_len=1 << 28, heads=1 << 20)])
def test_counts_of_blocks_beyond_64_bits_are_refused(how):
    """Products of sizes that are 0 modulo 2^64 (2^21 * 2^20 * 2^23) are as large as they are."""
    g = _lib.AttnGeom()
    sizes = dict(dict(batch=1, q_len=5, k_len=5, heads=1, kv_heads=1), **how)
    assert _lib.lib().sgh_attn_geom_init(C.byref(g), *sizes.values(), 1, 0, 1.0, 0, 0, 0) == ELIMIT


def test_norms_of_no_rows_with_a_gate():
    """Any number of gates divides no rows: the forward pass has nothing to do, the backward pass leaves zeros for the weights and the gate."""
    runs, refused = recorded("""
S, runs, refused = 1 << 50, [], []
for sfx in ("f32", "f16", "bf16"):
    for g in (0, 1, 4):
        n = lib.sgh_residual_norm_bwd_workspace_bytes(0, 24, g, 4 if sfx == "f32" else 2)
        fwd = getattr(lib, "sgh_residual_norm_fwd_" + sfx)(None, None, 3 * S, 4 * S, 5 * S, 0, 24, g, 0.5, 1e-5, None, None, None, None), kernels()
        bwd = getattr(lib, "sgh_residual_norm_bwd_" + sfx)(9 * S, 10 * S, 6 * S, 8 * S, 2 * S, 3 * S, 4 * S, 5 * S, 0, 24, g, 0.5, 11 * S, 12 * S, 13 * S, 14 * S, 15 * S, None, n, None), launched()
        runs.append([g, n, fwd[0], len(fwd[1]), bwd[0], len(bwd[1])])
    refused.append(getattr(lib, "sgh_residual_norm_bwd_" + sfx)(9 * S, 10 * S, 6 * S, 8 * S, 2 * S, 3 * S, 4 * S, 5 * S, 0, 24, 2, 0.5, 11 * S, 12 * S, 13 * S, None, 15 * S, None, 0, None))
answer([runs, refused])
""")
    assert runs == [[g, 0, 0, 0, 0, 3 if g else 2] for _ in range(3) for g in (0, 1, 4)], runs
    assert refused == [EINVAL] * 3


def test_assembly_names_the_register_that_it_writes():
    """What the compiler is not told of it may keep a value in."""
    import os
    import re

    where = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "singa_amd", "csrc")
    found = 0
    for name in sorted(os.listdir(where)):
        with open(os.path.join(where, name)) as f:
            for statement in re.findall(r"\basm\b[^;]*;", f.read()):
                if re.search(r"\bs_mov_b32 m0\b", statement):
                    found += 1
                    assert '"m0"' in statement.rsplit(":", 1)[1], (name, statement)
    assert found


def test_a_geometry_of_other_sizes_is_refused(monkeypatch):
    """A handle's tensors are held to its sizes; a structure put in place of its own that has others would read beyond them."""
    from singa_amd import singa_wrap as singa

    class Device(object):
        stream = None

    passed, dev = [], Device()
    make = lambda shape: singa.from_device_pointer(4096, shape, dev, singa.kFloat32)
    q, k, lse = make((2, 5, 4, 8)), make((2, 7, 2, 8)), make((2, 4, 5))
    monkeypatch.setattr(singa, "_fn", lambda name, t: (lambda geom, *rest: passed.append(geom) or 0, name))
    monkeypatch.setattr(singa, "_empty", lambda *a: q)
    monkeypatch.setattr(singa, "_like", lambda t: t)
    h = singa.AttentionHandle(q, k)
    own = h.geom
    for shape in ((2, 6, 4, 8), (2, 5, 2, 8)):
        h.geom = singa.AttentionHandle(make(shape), k).geom
        for call in (lambda: singa.AttentionForward(h, q, k, k), lambda: singa.AttentionBackward(h, q, q, k, k, q, lse)):
            with pytest.raises(singa.SingaHipError):
                call()
    h.geom = singa.AttentionHandle(q, make((2, 9, 2, 8))).geom
    with pytest.raises(singa.SingaHipError):
        singa.AttentionForward(h, q, k, k)
    assert not passed
    h.geom = own
    singa.AttentionForward(h, q, k, k)
    h.geom = singa.AttentionHandle(q, k, causal=True).geom
    singa.AttentionForward(h, q, k, k)
    assert passed == [C.addressof(own), C.addressof(h.geom)]
