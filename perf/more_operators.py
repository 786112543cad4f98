"""The middle of a token model, as cases to be measured: attention with a learned position bias, and the norms around a block.

Four operators, through ``singa_amd.singa_wrap``:

* ``attn_fwd`` -- ``AttentionForward``: softmax(scale q k^T + bias) v of every head, with the logarithm of every row's sum.  `buckets`: the
  bias is learned, one value for each head and bucket of distances.
* ``attn_bwd`` -- ``AttentionBackward``: the gradients of q, k, v and of the bias, the probabilities computed anew.
* ``norm_fwd`` -- ``ResidualNormForward``: a block's result normalised, gated, scaled and added to the stream that passes by the block, and
  the stream normalised for the next block.
* ``norm_bwd`` -- ``ResidualNormBackward``: the gradients of the stream, the block's result, the gate and both weights.

Sequences of a padded batch have lengths between half and all of its rows.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # a few short sentences with a learned bias in full precision: a call of a few microseconds
        {"name": "attn_fwd_f32_s37_bias", "op": "attn_fwd", "type": "f32", "batch": 3, "q_len": 37, "k_len": 37, "heads": 4, "kv_heads": 4,
         "dim": 16, "causal": False, "padded": True, "buckets": 32, "distance": 128},
        # the forward pass of a training batch, four heads to a head of keys, sequences of different lengths
        {"name": "attn_fwd_bf16_s4096_groups", "op": "attn_fwd", "type": "bf16", "batch": 4, "q_len": 4096, "k_len": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True, "padded": True, "buckets": 0, "distance": 0},
        # one new token for each of 16 sequences over long caches, with the bias
        {"name": "attn_fwd_f16_one_token", "op": "attn_fwd", "type": "f16", "batch": 16, "q_len": 1, "k_len": 16384, "heads": 16,
         "kv_heads": 4, "dim": 64, "causal": True, "padded": True, "buckets": 32, "distance": 128},
        # sentences of an odd length, heads of an odd size, in half precision, with the bias's gradient
        {"name": "attn_bwd_f16_s333_bias", "op": "attn_bwd", "type": "f16", "batch": 8, "q_len": 333, "k_len": 333, "heads": 6, "kv_heads": 2,
         "dim": 40, "causal": False, "padded": True, "buckets": 32, "distance": 128},
        # an ordinary batch in full precision
        {"name": "attn_bwd_f32_s512", "op": "attn_bwd", "type": "f32", "batch": 8, "q_len": 512, "k_len": 512, "heads": 8, "kv_heads": 8,
         "dim": 64, "causal": True, "padded": False, "buckets": 0, "distance": 0},
        # a bidirectional model's batch with the bias's gradient
        {"name": "attn_bwd_bf16_s1024_bias", "op": "attn_bwd", "type": "bf16", "batch": 8, "q_len": 1024, "k_len": 1024, "heads": 12,
         "kv_heads": 12, "dim": 64, "causal": False, "padded": False, "buckets": 32, "distance": 128},
        # long sequences: the largest
        {"name": "attn_bwd_bf16_s8192", "op": "attn_bwd", "type": "bf16", "batch": 2, "q_len": 8192, "k_len": 8192, "heads": 16, "kv_heads": 16,
         "dim": 128, "causal": True, "padded": False, "buckets": 0, "distance": 0},
        # one step's tokens between two blocks, a learned gate for each channel
        {"name": "norm_fwd_f32_r16", "op": "norm_fwd", "type": "f32", "rows": 16, "dim": 1000, "block": True, "after": True, "gates": 1,
         "before": True},
        # a large training batch between two blocks, a gate for each sequence
        {"name": "norm_fwd_bf16_r32768", "op": "norm_fwd", "type": "bf16", "rows": 32768, "dim": 4096, "block": True, "after": True, "gates": 16,
         "before": True},
        # rows of an odd length, a gate for each token, no norm behind the block
        {"name": "norm_bwd_f16_r2047_token_gate", "op": "norm_bwd", "type": "f16", "rows": 2047, "dim": 1001, "block": True, "after": False,
         "gates": 2047, "before": True},
        # the first block's norm in full precision: no block in front of it
        {"name": "norm_bwd_f32_r8192_first", "op": "norm_bwd", "type": "f32", "rows": 8192, "dim": 768, "block": False, "after": False,
         "gates": 0, "before": True},
        # a large training batch between two blocks, all gradients
        {"name": "norm_bwd_bf16_r32768", "op": "norm_bwd", "type": "bf16", "rows": 32768, "dim": 4096, "block": True, "after": True, "gates": 16,
         "before": True},
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _draw_attention(rng, op):
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
    group = rng.choice([1, 1, 1, 2, 4, 8])
    shape = rng.choice(["own", "own", "own", "other", "one"] if op == "attn_fwd" else ["own", "own", "own", "other"])
    q_len = 1 if shape == "one" else _log_int(rng, 2, 16384)
    k_len = q_len if shape == "own" else _log_int(rng, 1, 65536 if shape == "one" else 16384)
    buckets = rng.choice([0, 0, 8, 32, 64])
    return {"op": op, "type": rng.choice(["f32", "f16", "bf16", "bf16"]), "batch": _log_int(rng, 1, 64), "q_len": q_len, "k_len": k_len,
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([64, 128, _log_int(rng, 8, 128)]),
            "causal": shape == "one" or shape == "own" and rng.random() < 0.6, "padded": rng.random() < 0.5, "buckets": buckets,
            "distance": rng.choice([64, 128, 300]) if buckets else 0}


def _draw_norm(rng, op):
    block = rng.random() < 0.8
    rows = _log_int(rng, 1, 65536)
    return {"op": op, "type": rng.choice(["f32", "f16", "bf16", "bf16"]), "rows": rows, "dim": _log_int(rng, 16, 16384), "block": block,
            "after": block and rng.random() < 0.6, "gates": rng.choice([0, 1, _some_divisor(rng, rows), rows]) if block else 0,
            "before": not block or rng.random() < 0.8}


def _some_divisor(rng, n):
    return rng.choice([d for d in range(1, int(math.isqrt(n)) + 1) if n % d == 0])


def draw(rng):
    op = rng.choice(["attn_fwd", "attn_fwd", "attn_bwd", "attn_bwd", "norm_fwd", "norm_bwd"])
    while True:
        if op.startswith("attn"):
            case = _draw_attention(rng, op)
            per_pair = case["dim"] * (4 if case["type"] == "f32" else 1) * (1.0 if op == "attn_bwd" else 0.4)
            values = case["batch"] * (case["q_len"] * case["heads"] + case["k_len"] * case["kv_heads"]) * case["dim"]
            pairs = case["batch"] * case["heads"] * case["q_len"] * case["k_len"]
            if pairs * per_pair < 1.4e11 and pairs < 2.1e9 and values < 1.4e8:
                return case
        else:
            case = _draw_norm(rng, op)
            if case["rows"] * case["dim"] < 1.3e8:
                return case


# ------------------------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, shape, kind="f32", std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(TYPES[kind])


def _lengths(count, longest, spread=0.5):
    """The same lengths for every seed, so that a case is the same work: between `spread` and all of `longest`."""
    return [max(1, int(round(longest * (spread + (1 - spread) * ((0.37 + 0.618034 * i) % 1.0))))) for i in range(count)]


def _case_lengths(case):
    """(queries, keys, position of the first query) of every sequence as lists, None where all rows of the tensors count."""
    b, sq, sk = case["batch"], case["q_len"], case["k_len"]
    if not case["padded"]:
        return None, None, None
    keys = _lengths(b, sk)
    if sq == 1:
        return None, keys, [n - 1 for n in keys]       # the new token is the last of its sequence
    if sq == sk:
        return keys, keys, None
    return _lengths(b, sq), keys, None


def _int32(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def _attn_inputs(case, seed):
    gen = _generator(seed)
    b, sq, sk, h, g, d, kind = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim", "type"))
    ql, kl, starts = _case_lengths(case)
    state = {"case": case, "q": _randn(gen, (b, sq, h, d), kind, 1.5), "k": _randn(gen, (b, sk, g, d), kind), "v": _randn(gen, (b, sk, g, d), kind),
             "q_lengths": _int32(ql), "k_lengths": _int32(kl), "q_starts": _int32(starts), "table": None}
    if case["buckets"]:
        state["table"] = _randn(gen, (case["buckets"], h))
    if case["op"] == "attn_bwd":   # what the forward pass left
        state["do"] = _randn(gen, (b, sq, h, d), kind, 1e-2)
        state["o"], state["lse"] = _plain_attn_fwd(state)
    return state


def _norm_inputs(case, seed):
    gen = _generator(seed)
    r, d, kind = case["rows"], case["dim"], case["type"]
    state = {"case": case, "scale": 0.7 if case["block"] else 1.0, "h": None, "post": None, "gate": None, "pre": None}
    state["x"] = _randn(gen, (r, d), kind, 3.0)
    if case["block"]:
        state["h"] = _randn(gen, (r, d), kind, 0.5)
    if case["after"]:
        state["post"] = 1 + _randn(gen, (d,), std=0.1)
    if case["gates"]:
        state["gate"] = _randn(gen, (case["gates"], d), kind, 0.5)
    if case["before"]:
        state["pre"] = 1 + _randn(gen, (d,), std=0.1)
    if case["op"] == "norm_bwd":   # what the forward pass left
        out = _plain_norm_fwd(state)
        state["y"], state["stats"] = out.get("y", state["x"]), out["stats"]
        del state["x"]
        state["dy"] = _randn(gen, (r, d), kind, 1e-2)
        state["dn"] = _randn(gen, (r, d), kind, 1e-2) if case["before"] else None
    return state


def _library(state):
    """The same inputs as the library's tensors over the same memory, with its device, and the plan of the attention."""
    from singa_amd import singa_wrap as singa
    kinds = {torch.float32: singa.kFloat32, torch.float16: singa.kFloat16, torch.bfloat16: singa.kBFloat16, torch.int32: singa.kInt}
    dev = singa.create_hip_gpu_on(0)
    held = {k: singa.from_device_pointer(t.data_ptr(), t.shape, dev, kinds[t.dtype], keepalive=t)
            for k, t in state.items() if isinstance(t, torch.Tensor)}
    case, handle = state["case"], None
    if case["op"].startswith("attn"):
        handle = singa.AttentionHandle(held["q"], held["k"], causal=case["causal"], buckets=case["buckets"], max_distance=case["distance"],
                                       bidirectional=not case["causal"])
    return {"singa": singa, "held": held, "views": {}, "handle": handle}


def prepare(case, seed):
    state = _attn_inputs(case, seed) if case["op"].startswith("attn") else _norm_inputs(case, seed)
    torch.cuda.synchronize()
    if own:
        state["library"] = _library(state)
    return state


# ------------------------------------------------------------------------------------ one pass

class _DeviceArray(object):
    def __init__(self, ptr, shape, typestr):
        self.__cuda_array_interface__ = {"data": (int(ptr), False), "shape": tuple(shape), "typestr": typestr, "version": 3}


def _as_torch(lib, t):
    """A library tensor as a torch tensor over the same memory (a view for each address is kept: the pool hands the same few out)."""
    key = (t.ptr, tuple(t.shape()), t.data_type())
    v = lib["views"].get(key)
    if v is None:
        s = lib["singa"]
        typestr, as_type = {s.kFloat32: ("<f4", None), s.kFloat16: ("<f2", None), s.kBFloat16: ("<i2", torch.bfloat16)}[t.data_type()]
        v = torch.as_tensor(_DeviceArray(*key[:2], typestr), device="cuda")
        lib["views"][key] = v = v if as_type is None else v.view(as_type)
    return v


def _own(state):
    lib = state["library"]
    singa, held, op = lib["singa"], lib["held"], state["case"]["op"]
    if op.startswith("attn"):
        given = dict(table=held.get("table"), q_lengths=held.get("q_lengths"), k_lengths=held.get("k_lengths"),
                     q_starts=held.get("q_starts"))
        if op == "attn_fwd":
            names, out = ("o", "lse"), singa.AttentionForward(lib["handle"], held["q"], held["k"], held["v"], **given)
        else:
            names = ("dq", "dk", "dv", "dtable")
            out = singa.AttentionBackward(lib["handle"], held["do"], held["q"], held["k"], held["v"], held["o"], held["lse"], **given)
    else:
        given = dict(post=held.get("post"), gate=held.get("gate"), scale=state["scale"], pre=held.get("pre"))
        if op == "norm_fwd":
            names, out = ("y", "n", "stats"), singa.ResidualNormForward(held["x"], held.get("h"), eps=EPS, **given)
        else:
            names = ("dx", "dh", "dpost", "dgate", "dpre")
            out = singa.ResidualNormBackward(held["dy"], held.get("dn"), held["y"], held["stats"], held.get("h"), **given)
    lib["out"] = out   # the memory behind the views
    out = {k: _as_torch(lib, v) for k, v in zip(names, out) if v is not None}
    if op == "norm_fwd" and state["h"] is None:
        del out["y"]   # the stream itself
    return out


def _bucket_of(distance, buckets, longest, bidirectional):
    """The bucket of a key that is `distance` behind its query, in whole numbers (a tensor of int64)."""
    n = buckets // 2 if bidirectional else buckets
    exact = n // 2
    a = distance.abs() if bidirectional else (-distance).clamp(min=0)
    bounds = list(range(1, exact + 1))   # where the next bucket begins
    for t in range(1, n - exact):
        m = bounds[-1]
        while m ** (n - exact) * exact ** t < longest ** t * exact ** (n - exact):
            m += 1
        bounds.append(m)
    b = torch.searchsorted(torch.tensor(bounds, device=distance.device), a.clamp(max=longest), right=True)
    return b + n * (distance > 0) if bidirectional else b


def _plain_distance(state, i):
    """Key position minus query position of sequence i."""
    case = state["case"]
    start = case["k_len"] - case["q_len"] if state["q_starts"] is None else state["q_starts"][i].long()
    return (torch.arange(case["k_len"], device="cuda")[None, :] - start - torch.arange(case["q_len"], device="cuda")[:, None])


def _plain_mask(state, i, distance):
    case = state["case"]
    seen = torch.ones((case["q_len"], case["k_len"]), dtype=torch.bool, device="cuda")
    if case["causal"]:
        seen &= distance <= 0
    if state["q_lengths"] is not None:
        seen &= (torch.arange(case["q_len"], device="cuda") < state["q_lengths"][i])[:, None]
    if state["k_lengths"] is not None:
        seen &= (torch.arange(case["k_len"], device="cuda") < state["k_lengths"][i])[None, :]
    return seen


def _parts(state):
    """(sequence, first and last head of keys of a stretch) so that the scores of a stretch fit 2 GB."""
    case = state["case"]
    group = case["heads"] // case["kv_heads"]
    step = max(1, (1 << 29) // (case["q_len"] * case["k_len"] * group))
    for i in range(case["batch"]):
        for g in range(0, case["kv_heads"], step):
            yield i, g, min(case["kv_heads"], g + step), group


def _heads(t, i, a, b):
    """[heads, rows, dim] of sequence i in 32 bits."""
    return t[i, :, a:b].float().transpose(0, 1).contiguous()


def _plain_scores(state, i, g, e, group):
    """Scores [kv heads, group, q_len, k_len] of a stretch with -inf where the mask is, and the buckets of all pairs."""
    case = state["case"]
    q, k = _heads(state["q"], i, g * group, e * group), _heads(state["k"], i, g, e)
    s = torch.matmul(q.reshape(e - g, group * case["q_len"], case["dim"]), k.transpose(1, 2))
    s = s.mul_(1 / math.sqrt(case["dim"])).view(e - g, group, case["q_len"], case["k_len"])
    distance = _plain_distance(state, i)
    buckets = None
    if state["table"] is not None:
        buckets = _bucket_of(distance, case["buckets"], case["distance"], not case["causal"])
        for head in range(g * group, e * group):
            s[head // group - g, head % group] += state["table"][:, head][buckets]
    return q, k, s.masked_fill_(~_plain_mask(state, i, distance), -torch.inf), buckets


def _plain_attn_fwd(state):
    case = state["case"]
    o = torch.empty_like(state["q"])
    lse = torch.empty((case["batch"], case["heads"], case["q_len"]), device="cuda")
    for i, g, e, group in _parts(state):
        _, _, s, _ = _plain_scores(state, i, g, e, group)
        top = s.max(3, keepdim=True).values
        p = s.sub_(top.clamp(min=-3e38)).exp_()
        total = p.sum(3, keepdim=True)
        r = torch.matmul(p.view(e - g, group * case["q_len"], case["k_len"]), _heads(state["v"], i, g, e))
        r = r.view(e - g, group, case["q_len"], case["dim"]) / torch.where(total > 0, total, 1.0)
        o[i, :, g * group:e * group] = r.reshape((e - g) * group, case["q_len"], case["dim"]).transpose(0, 1).to(o.dtype)
        lse[i, g * group:e * group] = (top + total.log()).reshape((e - g) * group, case["q_len"])
    return o, lse


def _plain_attn_bwd(state):
    case = state["case"]
    sq, sk, d = case["q_len"], case["k_len"], case["dim"]
    dq, dk, dv = torch.empty_like(state["q"]), torch.empty_like(state["k"]), torch.empty_like(state["v"])
    dtable = torch.zeros_like(state["table"]) if state["table"] is not None else None
    for i, g, e, group in _parts(state):
        q, k, s, buckets = _plain_scores(state, i, g, e, group)
        lse = state["lse"][i, g * group:e * group].view(e - g, group, sq, 1)
        p = s.sub_(lse.clamp(min=-3e38)).exp_().view(e - g, group * sq, sk)
        do, o, v = (_heads(state[n], i, g * f, e * f) for n, f in (("do", group), ("o", group), ("v", 1)))
        delta = (do * o).sum(2).view(e - g, group * sq, 1)
        q, do = q.reshape(e - g, group * sq, d), do.reshape(e - g, group * sq, d)
        dv[i, :, g:e] = torch.matmul(p.transpose(1, 2), do).transpose(0, 1).to(dv.dtype)
        ds = torch.matmul(do, v.transpose(1, 2)).sub_(delta)
        ds = torch.where(p > 0, ds, 0.0).mul_(p)
        if dtable is not None:
            # the sums of the diagonals, then of the diagonals of a bucket: rows from the last to the first, each moved one further
            each = torch.nn.functional.pad(ds.view((e - g) * group, sq, sk).flip(1), (0, sq)).flatten(1)
            each = each[:, :sq * (sk + sq - 1)].view(-1, sq, sk + sq - 1).sum(1)
            dtable[:, g * group:e * group].index_add_(0, torch.cat([buckets[1:, 0].flip(0), buckets[0]]), each.T)
        r = torch.matmul(ds, k).mul_(1 / math.sqrt(d)).view((e - g) * group, sq, d)
        dq[i, :, g * group:e * group] = r.transpose(0, 1).to(dq.dtype)
        dk[i, :, g:e] = torch.matmul(ds.transpose(1, 2), q).mul_(1 / math.sqrt(d)).transpose(0, 1).to(dk.dtype)
    out = {"dq": dq, "dk": dk, "dv": dv}
    if dtable is not None:
        out["dtable"] = dtable
    return out


def _each_gate(state):
    """The gate of every row in 32 bits, or 1."""
    if state["gate"] is None:
        return 1.0
    return state["gate"].float().repeat_interleave(state["case"]["rows"] // state["case"]["gates"], 0)


def _plain_norm_fwd(state):
    case = state["case"]
    y = state["x"].float()
    stats = torch.zeros((case["rows"], 2), device="cuda")
    out = {}
    if state["h"] is not None:
        u = state["h"].float()
        if state["post"] is not None:
            stats[:, 0] = torch.rsqrt((u * u).mean(1) + EPS)
            u = u * stats[:, :1] * state["post"]
        y = y + state["scale"] * _each_gate(state) * u
        out["y"] = y.to(state["x"].dtype)
    if state["pre"] is not None:
        stats[:, 1] = torch.rsqrt((y * y).mean(1) + EPS)
        out["n"] = (y * stats[:, 1:] * state["pre"]).to(state["x"].dtype)
    out["stats"] = stats
    return out


def _plain_norm_bwd(state):
    case, out = state["case"], {}
    kind = state["y"].dtype
    r, d = case["rows"], case["dim"]
    dx = state["dy"].float()
    if state["pre"] is not None:
        y, dn, s = state["y"].float(), state["dn"].float(), state["stats"][:, 1:]
        a = dn * state["pre"]
        dx = dx + s * a - y * (s * s * s * (a * y).sum(1, keepdim=True) / d)
        out["dpre"] = (dn * y * s).sum(0)
    out["dx"] = dx.to(kind)
    if state["h"] is None:
        return out
    h, s, gate = state["h"].float(), state["stats"][:, :1], _each_gate(state)
    u = h if state["post"] is None else h * s * state["post"]
    if state["gate"] is not None:
        out["dgate"] = (dx * u * state["scale"]).view(case["gates"], r // case["gates"], d).sum(1).to(kind)
    du = dx * gate * state["scale"]
    if state["post"] is not None:
        out["dpost"] = (du * h * s).sum(0)
        a = du * state["post"]
        du = s * a - h * (s * s * s * (a * h).sum(1, keepdim=True) / d)
    out["dh"] = du.to(kind)
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "attn_fwd":
        return dict(zip(("o", "lse"), _plain_attn_fwd(state)))
    return {"attn_bwd": _plain_attn_bwd, "norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd}[op](state)


# ------------------------------------------------------------------------------------ what a pass cannot do without

def _pairs(case):
    """(pairs of a query and a key that it sees, for one head; queries; keys) over all sequences."""
    ql, kl, starts = _case_lengths(case)
    pairs = queries = keys = 0
    for i in range(case["batch"]):
        nq, nk = ql[i] if ql else case["q_len"], kl[i] if kl else case["k_len"]
        start = starts[i] if starts else case["k_len"] - case["q_len"]
        queries, keys = queries + nq, keys + nk
        if not case["causal"]:
            pairs += nq * nk
        else:   # query j sees the keys up to start + j
            first = max(0, -start)
            full = max(first, min(nq, nk - start))   # queries from here on see all keys
            pairs += sum(start + j + 1 for j in (first, full - 1)) * (full - first) // 2 if full > first else 0
            pairs += (nq - full) * nk
    return pairs, queries, keys


def work(case):
    e = SIZE[case["type"]]
    if case["op"].startswith("attn"):
        pairs, queries, keys = _pairs(case)
        h, g, d = case["heads"], case["kv_heads"], case["dim"]
        rows = case["batch"] * case["q_len"]
        small = 4 * case["buckets"] * h + 4 * queries * h
        if case["op"] == "attn_fwd":
            return {"bytes": (queries + rows) * h * d * e + 2 * keys * g * d * e + small, "flops": 4 * pairs * h * d}
        return {"bytes": (3 * queries + rows) * h * d * e + (2 * keys + 2 * case["batch"] * case["k_len"]) * g * d * e + 2 * small,
                "flops": 10 * pairs * h * d}
    n = case["rows"] * case["dim"]
    gate, weights = case["gates"] * case["dim"] * e, 4 * case["dim"] * (case["after"] + case["before"])
    if case["op"] == "norm_fwd":   # x, h, y, n
        return {"bytes": n * e * ((3 if case["block"] else 1) + case["before"]) + gate + weights + 8 * case["rows"],
                "flops": n * (4 * case["block"] + 3 * case["after"] + 4 * case["before"])}
    # dy, dx; dn, y; h, dh
    return {"bytes": n * e * (2 + 2 * case["before"] + 2 * case["block"]) + 2 * gate + 2 * weights + 8 * case["rows"],
            "flops": n * (4 * case["block"] + 8 * case["after"] + 9 * case["before"])}


# ------------------------------------------------------------------------------------ the definition, in 64 bits

def _exact_bias(state, i, head):
    """The bias of every pair of sequence i: bucket by bucket, a distance at a time."""
    case, table = state["case"], state["table"][:, head].double()
    n = case["buckets"] if case["causal"] else case["buckets"] // 2
    exact, longest = n // 2, case["distance"]

    def bucket(m):
        if m < exact:
            return m
        t = 0
        while t < n - exact - 1 and m ** (n - exact) * exact ** (t + 1) >= longest ** (t + 1) * exact ** (n - exact):
            t += 1
        return exact + t

    near = [bucket(m) for m in range(longest + 1)]
    start = case["k_len"] - case["q_len"] if state["q_starts"] is None else int(state["q_starts"][i])
    index = []
    for distance in range(-(start + case["q_len"] - 1), case["k_len"] - start):
        if case["causal"]:
            index.append(near[min(longest, max(0, -distance))])
        else:
            index.append(near[min(longest, abs(distance))] + (n if distance > 0 else 0))
    index = torch.tensor(index, device="cuda")
    rows = torch.arange(case["q_len"] - 1, -1, -1, device="cuda")[:, None] + torch.arange(case["k_len"], device="cuda")[None, :]
    return index[rows], table


def _exact_attn(state):
    case = state["case"]
    sq, sk, h, d = case["q_len"], case["k_len"], case["heads"], case["dim"]
    group = h // case["kv_heads"]
    backward = case["op"] == "attn_bwd"
    out = {k: torch.zeros(state[k[1:] if backward else "q"].shape, dtype=torch.float64, device="cuda")
           for k in (("dq", "dk", "dv") if backward else ("o",))}
    out.update({"dtable": torch.zeros_like(state["table"], dtype=torch.float64)} if backward and state["table"] is not None else {})
    if not backward:
        out["lse"] = torch.full((case["batch"], h, sq), -torch.inf, dtype=torch.float64, device="cuda")
    lists = [None if state[k] is None else state[k].tolist() for k in ("q_lengths", "k_lengths", "q_starts")]
    for i in range(case["batch"]):
        nq, nk = (n if given is None else given[i] for n, given in ((sq, lists[0]), (sk, lists[1])))
        start = sk - sq if lists[2] is None else lists[2][i]
        first = max(0, -start) if case["causal"] else 0    # queries in front of it see no key
        if nq <= first or nk == 0:
            continue
        hide = None
        if case["causal"]:
            hide = torch.arange(nk, device="cuda")[None, :] > (start + torch.arange(first, nq, device="cuda"))[:, None]
        which = None
        for head in range(h):
            q, k, v = (state[n][i, a:b, x].double() for n, a, b, x in (("q", first, nq, head), ("k", 0, nk, head // group),
                                                                      ("v", 0, nk, head // group)))
            s = q @ k.T / math.sqrt(d)
            if state["table"] is not None:
                if which is None:
                    which = _exact_bias(state, i, head)[0][first:nq, :nk]
                s += state["table"][:, head].double()[which]
            if hide is not None:
                s[hide] = -torch.inf
            if not backward:
                lse = torch.logsumexp(s, 1)
                out["lse"][i, head, first:nq] = lse
                out["o"][i, first:nq, head] = torch.exp(s - lse[:, None]) @ v
                continue
            # (the result and the logarithms are arguments: what the forward pass stored)
            p = torch.exp(s - state["lse"][i, head, first:nq, None].double())
            do = state["do"][i, first:nq, head].double()
            ds = p * (do @ v.T - (do * state["o"][i, first:nq, head].double()).sum(1, keepdim=True))
            out["dv"][i, :nk, head // group] += p.T @ do
            out["dq"][i, first:nq, head] = ds @ k / math.sqrt(d)
            out["dk"][i, :nk, head // group] += ds.T @ q / math.sqrt(d)
            if state["table"] is not None:
                out["dtable"][:, head] += torch.bincount(which.reshape(-1), ds.reshape(-1), case["buckets"])
    return out


def _exact_norm(state):
    """The formulas of both directions, a stretch of rows of one gate at a time."""
    case, f64 = state["case"], torch.float64
    r, d, scale = case["rows"], case["dim"], state["scale"]
    backward = case["op"] == "norm_bwd"
    per = r // case["gates"] if case["gates"] else r
    out = {}

    def put(name, shape, at, value):
        out.setdefault(name, torch.zeros(shape, dtype=f64, device="cuda"))[at] += value

    post, pre = (None if state[n] is None else state[n].to(f64) for n in ("post", "pre"))
    stretch = max(1, (1 << 23) // d)
    a = 0
    while a < r:
        z = min(r, a + stretch, (a // per + 1) * per if per > 1 else r)
        rows, gate = slice(a, z), 1.0
        gate_at = slice(a // per, a // per + 1) if per > 1 else rows
        if state["gate"] is not None:
            gate = state["gate"][gate_at].to(f64)
        h = state["h"][rows].to(f64) if case["block"] else None
        if not backward:
            y = state["x"][rows].to(f64)
            if case["block"]:
                if case["after"]:
                    root = 1 / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / d + EPS)
                    put("stats", (r, 2), (rows, slice(0, 1)), root)
                    h = h * root * post
                y = torch.addcmul(y, h, scale * gate * torch.ones_like(h))
                put("y", (r, d), rows, y)
            if case["before"]:
                root = 1 / torch.sqrt(torch.linalg.vector_norm(y, dim=1, keepdim=True) ** 2 / d + EPS)
                put("stats", (r, 2), (rows, slice(1, 2)), root)
                put("n", (r, d), rows, y * root * pre)
        else:   # (the stream and both roots are arguments: what the forward pass stored)
            roots = state["stats"][rows].to(f64)
            stream = state["dy"][rows].to(f64)
            if case["before"]:
                unit, dn = state["y"][rows].to(f64) * roots[:, 1:], state["dn"][rows].to(f64)
                put("dpre", (d,), slice(None), torch.linalg.vecdot(dn, unit, dim=0))
                dn = dn * pre
                stream = stream + roots[:, 1:] * (dn - unit * torch.linalg.vecdot(dn, unit, dim=1)[:, None] / d)
            put("dx", (r, d), rows, stream)
            if case["block"]:
                unit = h * roots[:, :1] if case["after"] else h
                each = scale * stream * unit
                if case["gates"]:
                    each_gate = each if post is None else each * post
                    put("dgate", (case["gates"], d), gate_at, each_gate if per == 1 else each_gate.sum(0, keepdim=True))
                dh = scale * stream * gate
                if case["after"]:
                    put("dpost", (d,), slice(None), (each * gate).sum(0))
                    dh = dh * post
                    dh = roots[:, :1] * (dh - unit * torch.linalg.vecdot(dh, unit, dim=1)[:, None] / d)
                put("dh", (r, d), rows, dh)
        a = z
    if not backward and "stats" not in out:
        out["stats"] = torch.zeros((r, 2), dtype=f64, device="cuda")
    return out


def exact(case, seed):
    if case["op"].startswith("attn"):
        return _exact_attn(_attn_inputs(case, seed))
    return _exact_norm(_norm_inputs(case, seed))
