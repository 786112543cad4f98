"""The two ends of a token model, as cases to be measured: the table of token vectors and the loss over the vocabulary.

Five operators, through ``singa_amd.singa_wrap``:

* ``embed_fwd``   -- ``EmbeddingForward``: rows of a table by token id, times a scale.
* ``embed_bwd``   -- ``EmbeddingBackwardW``: the table's gradient, the gradients of a token's places summed (with ``tied``: on top of
  the gradient that the same matrix got as the output layer).
* ``distill_fwd`` -- ``DistillationFwd``: loss against a teacher's top logits and labels.
* ``distill_bwd`` -- ``DistillationBwd``: the gradient of the logits from the statistics that the forward pass kept.
* ``distill``     -- ``DistillationFwdBwd``: both in one call.

Token ids follow the distribution of text (the id with rank r about 1 / r), a share of them is padding; the teacher's lists have different
lengths, some places have no label and some no weight.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAD = 0            # the id that fills up short sequences
PAD_SHARE = 0.06   # of the tokens
NO_WEIGHT, NO_LABEL = 1.0 / 16, 1.0 / 8   # shares of the rows: fill-up, and places whose next token is not to be learnt


def listed():
    return [
        # one new token for each of 32 sequences: a call of a few microseconds
        {"name": "embed_fwd_f32_t32", "op": "embed_fwd", "type": "f32", "tokens": 32, "vocab": 10000, "dim": 1000},
        # a training batch's tokens out of a large table
        {"name": "embed_fwd_bf16_t16384", "op": "embed_fwd", "type": "bf16", "tokens": 16384, "vocab": 131072, "dim": 4096},
        # a batch of 128 with four tokens of context each, rows of an odd number of 2-byte values
        {"name": "embed_bwd_f16_t512_ragged", "op": "embed_bwd", "type": "f16", "tokens": 512, "vocab": 10007, "dim": 201, "tied": False},
        # an ordinary batch, full-precision table
        {"name": "embed_bwd_f32_t8192", "op": "embed_bwd", "type": "f32", "tokens": 8192, "vocab": 32000, "dim": 1024, "tied": False},
        # a large batch onto the gradient that the table got as the output layer's weights
        {"name": "embed_bwd_bf16_t65536_tied", "op": "embed_bwd", "type": "bf16", "tokens": 65536, "vocab": 131072, "dim": 2048, "tied": True},
        # the loss of a few sequences' last tokens, labels beside a short list
        {"name": "distill_fwd_f32_n16", "op": "distill_fwd", "type": "f32", "rows": 16, "vocab": 10007, "top": 8, "temperature": 2.0,
         "soft": 0.5, "hard": 0.5},
        # an ordinary batch in half precision, rows of an odd length
        {"name": "distill_fwd_f16_n4096", "op": "distill_fwd", "type": "f16", "rows": 4096, "vocab": 50001, "top": 64, "temperature": 1.0,
         "soft": 1.0, "hard": 0.0},
        # a small batch's gradient, labels and lists at two temperatures
        {"name": "distill_bwd_f32_n64", "op": "distill_bwd", "type": "f32", "rows": 64, "vocab": 32000, "top": 16, "temperature": 4.0,
         "soft": 0.7, "hard": 0.3},
        # a large batch's gradient
        {"name": "distill_bwd_bf16_n8192", "op": "distill_bwd", "type": "bf16", "rows": 8192, "vocab": 65536, "top": 32, "temperature": 2.0,
         "soft": 0.9, "hard": 0.1},
        # one row at a time over a small vocabulary, both directions
        {"name": "distill_f16_n3", "op": "distill", "type": "f16", "rows": 3, "vocab": 1000, "top": 5, "temperature": 1.5, "soft": 1.0,
         "hard": 0.25},
        # the whole loss of a large batch: the largest
        {"name": "distill_bf16_n8192", "op": "distill", "type": "bf16", "rows": 8192, "vocab": 131072, "top": 64, "temperature": 2.0,
         "soft": 0.9, "hard": 0.1},
        # labels alone: the cross entropy of an odd vocabulary
        {"name": "distill_bf16_n2048_labels", "op": "distill", "type": "bf16", "rows": 2048, "vocab": 65001, "top": 0, "temperature": 1.0,
         "soft": 0.0, "hard": 1.0},
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_bwd", "embed_bwd", "distill_fwd", "distill_bwd", "distill", "distill"])
    case = {"op": op, "type": rng.choice(["f32", "f16", "bf16"])}
    while True:
        if op.startswith("embed"):
            case.update(tokens=_log_int(rng, 1, 131072), vocab=_log_int(rng, 100, 262144), dim=_log_int(rng, 16, 8192))
            if op == "embed_bwd":
                case["tied"] = rng.random() < 0.3
            values = case["tokens"] * case["dim"] + case["vocab"] * case["dim"] * (1 if op == "embed_bwd" else 0.25)
            if values < 4e8:
                return case
        else:
            vocab = _log_int(rng, 500, 262144)
            top = rng.choice([0, _log_int(rng, 1, 256), _log_int(rng, 1, 256), _log_int(rng, 1, 256)])
            case.update(rows=_log_int(rng, 1, 16384), vocab=vocab, top=min(top, vocab // 2),
                        temperature=rng.choice([1.0, round(rng.uniform(0.5, 8.0), 2)]),
                        soft=round(rng.uniform(0.1, 1.0), 2) if top else 0.0,
                        hard=round(rng.uniform(0.1, 1.0), 2) if not top or rng.random() < 0.6 else 0.0)
            if case["rows"] * vocab < 5e8:
                return case


# ------------------------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64)


def _randn(gen, shape, kind="f32", std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(TYPES[kind])


def _text(gen, count, vocab):
    """Ids of text: rank r with a share of log((r + 2) / (r + 1)) / log(vocab + 1), ranks from 0."""
    return (torch.exp(_rand(gen, count) * math.log(vocab + 1)).long() - 1).clamp(0, vocab - 1)


def _embed_inputs(case, seed):
    gen = _generator(seed)
    t, v, d, kind = case["tokens"], case["vocab"], case["dim"], case["type"]
    ids = _text(gen, t, v)
    ids = torch.where(_rand(gen, t) < PAD_SHARE, PAD, ids).int()
    state = {"op": case["op"], "ids": ids, "scale": math.sqrt(d)}
    if case["op"] == "embed_fwd":
        state["W"] = _randn(gen, (v, d), kind, 1.0 / math.sqrt(d))
    else:
        state.update(dy=_randn(gen, (t, d), kind, 1e-2), shape=(v, d), add=_randn(gen, (v, d), kind, 1e-2) if case["tied"] else None)
        state["W"] = state["add"] if case["tied"] else torch.empty((v, d), dtype=TYPES[kind], device="cuda")
    return state


def _distill_inputs(case, seed):
    gen = _generator(seed)
    n, v, k, kind = case["rows"], case["vocab"], case["top"], case["type"]
    x = torch.randn((n, v), generator=gen, device="cuda", dtype=TYPES[kind]).mul_(2.0)
    top = teacher = None
    if k:   # different ids in a row, logits that fall; the student knows a part of it
        start, step = _text(gen, n, v)[:, None], 1 + (_rand(gen, n, 1) * (v // k)).long().clamp(max=v // k - 1)
        top = (start + step * torch.arange(k, device="cuda")) % v
        teacher = (6.0 + torch.randn((n, k), generator=gen, device="cuda")
                   - 1.5 * torch.log1p(torch.arange(k, device="cuda", dtype=torch.float32)))
        x.scatter_add_(1, top, (0.7 * teacher).to(x.dtype))
        length = 1 + (_rand(gen, n, 1).sqrt() * k).long().clamp(max=k - 1)   # lists cut where the teacher's mass is reached
        top = torch.where(torch.arange(k, device="cuda") < length, top, -1).int()
    labels = None
    if case["hard"]:
        labels = torch.where(_rand(gen, n) < NO_LABEL, -1, _text(gen, n, v)).int()
    w = torch.where(_rand(gen, n) < NO_WEIGHT, 0.0, 1.0).float()
    state = {"op": case["op"], "x": x, "top": top, "teacher": teacher, "labels": labels, "w": w, "temperature": case["temperature"],
             "soft": case["soft"], "hard": case["hard"], "scale": 1.0 / n}
    if case["op"] == "distill_bwd":   # the statistics that the forward pass left
        state["stats"] = _plain_statistics(state)
    return state


def _library(state):
    """The same inputs as the library's tensors over the same memory, with its device."""
    from singa_amd import singa_wrap as singa
    kinds = {torch.float32: singa.kFloat32, torch.float16: singa.kFloat16, torch.bfloat16: singa.kBFloat16, torch.int32: singa.kInt}
    dev = singa.create_hip_gpu_on(0)
    held = {k: singa.from_device_pointer(t.data_ptr(), t.shape, dev, kinds[t.dtype], keepalive=t)
            for k, t in state.items() if isinstance(t, torch.Tensor)}
    return {"singa": singa, "held": held, "views": {}}


def prepare(case, seed):
    state = _embed_inputs(case, seed) if case["op"].startswith("embed") else _distill_inputs(case, seed)
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
    singa, held = lib["singa"], lib["held"]
    if state["op"] == "embed_fwd":
        out = {"y": singa.EmbeddingForward(held["ids"], held["W"], scale=state["scale"], padding_idx=PAD)}
    elif state["op"] == "embed_bwd":
        out = {"dW": singa.EmbeddingBackwardW(held["dy"], held["ids"], held["W"], scale=state["scale"], padding_idx=PAD,
                                              add=held.get("add"))}
    else:
        given = dict(labels=held.get("labels"), weights=held["w"], temperature=state["temperature"], soft=state["soft"],
                     hard=state["hard"])
        top, teacher = held.get("top"), held.get("teacher")
        if state["op"] == "distill_fwd":
            loss, stats = singa.DistillationFwd(held["x"], top, teacher, **given)
            out = {"loss": loss, "stats": stats}
        elif state["op"] == "distill_bwd":
            out = {"dx": singa.DistillationBwd(held["x"], held["stats"], top, teacher, scale=state["scale"], **given)}
        else:
            loss, dx = singa.DistillationFwdBwd(held["x"], top, teacher, scale=state["scale"], **given)
            out = {"loss": loss, "dx": dx}
    lib["out"] = out   # the memory behind the views
    return {k: _as_torch(lib, v) for k, v in out.items()}


def _parts(state):
    """(rows with a soft term, rows with a hard term, present entries of the lists)."""
    used = state["w"] != 0
    present = soft = hard = torch.zeros_like(used)
    if state["top"] is not None and state["soft"]:
        present = state["top"] >= 0
        soft = used & present.any(1)
    if state["labels"] is not None and state["hard"]:
        hard = used & (state["labels"] >= 0)
    return soft, hard, present


def _plain_statistics(state):
    """For each row: its maximum m, the sums of exp((x - m) / temperature) and of exp(x - m); zero where no term asks for them."""
    soft, hard, _ = _parts(state)
    n = state["x"].shape[0]
    out = torch.zeros((n, 3), device="cuda")
    step = max(1, (1 << 29) // state["x"].shape[1])
    for a in range(0, n, step):
        x, s, h = state["x"][a:a + step].float(), soft[a:a + step], hard[a:a + step]
        m = x.max(1).values
        out[a:a + step, 0] = torch.where(s | h, m, 0.0)
        x = x - m[:, None]
        if state["soft"]:
            out[a:a + step, 1] = torch.where(s, (x / state["temperature"]).exp_().sum(1), 0.0)
        if state["hard"]:
            out[a:a + step, 2] = torch.where(h, x.exp_().sum(1), 0.0)
    return out


def _teacher_shares(state, present):
    """p of every list entry, absent ones 0."""
    t = torch.where(present, state["teacher"], -torch.inf)
    e = torch.exp((t - t.max(1, keepdim=True).values.clamp(min=-3e38)) / state["temperature"])
    return e / e.sum(1, keepdim=True).clamp(min=1e-30)


def _plain_loss(state, stats):
    soft, hard, present = _parts(state)
    loss = torch.zeros(state["x"].shape[0], device="cuda")
    if state["top"] is not None and state["soft"]:
        p = _teacher_shares(state, present)
        x = torch.gather(state["x"], 1, state["top"].clamp(min=0).long()).float()
        log_q = (x - stats[:, :1]) / state["temperature"] - torch.log(stats[:, 1:2])
        each = torch.where(p > 0, p * (torch.log(p) - log_q), 0.0)
        loss += torch.where(soft, state["soft"] * state["temperature"] ** 2 * each.sum(1), 0.0)
    if state["labels"] is not None and state["hard"]:
        x = torch.gather(state["x"], 1, state["labels"].clamp(min=0).long()[:, None]).float()[:, 0]
        loss += torch.where(hard, state["hard"] * (torch.log(stats[:, 2]) - (x - stats[:, 0])), 0.0)
    return loss * state["w"]


def _plain_gradient(state, stats):
    soft, hard, present = _parts(state)
    out = torch.empty_like(state["x"])
    tau, n = state["temperature"], out.shape[0]
    g = state["w"] * state["scale"]
    a = torch.where(soft, g * state["soft"] * tau, 0.0)
    b = torch.where(hard, g * state["hard"], 0.0)
    p = _teacher_shares(state, present) if state["top"] is not None and state["soft"] else None
    step = max(1, (1 << 29) // out.shape[1])
    for i in range(0, n, step):
        r = slice(i, i + step)
        x = state["x"][r].float() - stats[r, :1]
        d = torch.zeros_like(x)
        if p is not None:
            d += (x / tau).exp_().mul_((a[r] / stats[r, 1].clamp(min=1e-30))[:, None])
            d.scatter_add_(1, state["top"][r].clamp(min=0).long(), -a[r, None] * p[r])
        if state["labels"] is not None and state["hard"]:
            d += x.exp_().mul_((b[r] / stats[r, 2].clamp(min=1e-30))[:, None])
            d.scatter_add_(1, state["labels"][r].clamp(min=0).long()[:, None], -b[r, None])
        out[r] = torch.where((a[r] != 0)[:, None] | (b[r] != 0)[:, None], d, 0.0).to(out.dtype)
    return out


def _plain(state):
    if state["op"] == "embed_fwd":
        y = state["W"][state["ids"].long()].float() * state["scale"]
        return {"y": torch.where((state["ids"] == PAD)[:, None], 0.0, y).to(state["W"].dtype)}
    if state["op"] == "embed_bwd":
        ids = state["ids"].long()
        dy = torch.where((ids == PAD)[:, None], 0.0, state["dy"].float())
        dW = torch.zeros(state["shape"], device="cuda").index_add_(0, ids, dy).mul_(state["scale"])
        if state["add"] is not None:
            dW += state["add"].float()
        return {"dW": dW.to(state["dy"].dtype)}
    if state["op"] == "distill_bwd":
        return {"dx": _plain_gradient(state, state["stats"])}
    stats = _plain_statistics(state)
    loss = _plain_loss(state, stats)
    if state["op"] == "distill_fwd":
        return {"loss": loss, "stats": stats}
    return {"loss": loss, "dx": _plain_gradient(state, stats)}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ what a pass cannot do without

def _distinct(tokens, vocab):
    """How many different ids `tokens` tokens have, on average, padding left out."""
    r = np.arange(vocab, dtype=np.float64)
    share = (1 - PAD_SHARE) * np.log((r + 2) / (r + 1)) / math.log(vocab + 1)
    return float((1 - np.exp(tokens * np.log1p(-share)))[PAD + 1:].sum())


def work(case):
    e = SIZE[case["type"]]
    if case["op"].startswith("embed"):
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        # (the id of padding is also an ordinary rank here: its tokens are read and summed by nobody)
        real = t * (1 - PAD_SHARE) * (1 - math.log(2) / math.log(v + 1))
        if case["op"] == "embed_fwd":
            return {"bytes": 4 * t + (_distinct(t, v) + t) * d * e, "flops": real * d}
        return {"bytes": 4 * t + (real + v * (2 if case["tied"] else 1)) * d * e, "flops": real * d}
    n, v, k = case["rows"], case["vocab"], case["top"]
    soft, hard = bool(k and case["soft"]), bool(case["hard"])
    used = n * (1 - NO_WEIGHT) * (1.0 if soft else 1 - NO_LABEL)
    small = n * (4 + 8 * k + (4 if hard else 0))
    one = 1 + 2 * soft + 2 * hard   # a difference, and an exponential and a sum (or product) for each term
    if case["op"] == "distill_fwd":
        return {"bytes": used * v * e + small + 16 * n, "flops": used * v * one}
    if case["op"] == "distill_bwd":
        return {"bytes": (used + n) * v * e + small + 12 * n, "flops": used * v * one}
    return {"bytes": (used + n) * v * e + small + 4 * n, "flops": used * v * 2 * one}


# ------------------------------------------------------------------------------------ the definition, in 64 bits

def _exact_rows(s):
    """Loss, statistics and a function that gives the gradient, row by row from the definition."""
    tau, soft_weight, hard_weight = s["temperature"], s["soft"], s["hard"]
    n, v = s["x"].shape
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    stats = torch.zeros((n, 3), dtype=torch.float64, device="cuda")
    want_dx, dx = s["op"] != "distill_fwd", None
    if want_dx:
        dx = torch.zeros((n, v), dtype=torch.float32 if n * v > 1 << 28 else torch.float64, device="cuda")
    step = max(1, (1 << 27) // v)
    for i in range(0, n, step):
        r = slice(i, min(n, i + step))
        x, w = s["x"][r].double(), s["w"][r].double()
        grad = torch.zeros_like(x) if want_dx else None
        any_term = torch.zeros(x.shape[0], dtype=torch.bool, device="cuda")
        if s["top"] is not None and soft_weight:
            here = s["top"][r] >= 0
            has = here.any(1) & (w != 0)
            any_term |= has
            logits = (s["teacher"][r].double() / tau).masked_fill(~here, -1e300)
            log_p = logits - torch.logsumexp(logits, 1, keepdim=True)
            p = torch.where(here, log_p.exp(), 0.0)
            lse = torch.logsumexp(x / tau, 1, keepdim=True)
            log_q = torch.gather(x, 1, s["top"][r].long().clamp(min=0)) / tau - lse
            kl = torch.where(here & (p > 0), p * (log_p - log_q), 0.0).sum(1)
            loss[r] += torch.where(has, w * soft_weight * tau * tau * kl, 0.0)
            stats[r, 1] = torch.where(has, (lse[:, 0] - x.max(1).values / tau).exp(), 0.0)
            if want_dx:
                term = (x / tau - lse).exp_().scatter_add_(1, s["top"][r].long().clamp(min=0), -p)
                grad += term.mul_((has * w * s["scale"] * soft_weight * tau)[:, None])
                del term
        if s["labels"] is not None and hard_weight:
            label = s["labels"][r].long()
            has = (label >= 0) & (w != 0)
            any_term |= has
            lse = torch.logsumexp(x, 1, keepdim=True)
            at = label.clamp(min=0)[:, None]
            loss[r] += torch.where(has, w * hard_weight * (lse - torch.gather(x, 1, at))[:, 0], 0.0)
            stats[r, 2] = torch.where(has, (lse[:, 0] - x.max(1).values).exp(), 0.0)
            if want_dx:
                term = (x - lse).exp_().scatter_add_(1, at, torch.full_like(x[:, :1], -1.0))
                grad += term.mul_((has * w * s["scale"] * hard_weight)[:, None])
                del term
        stats[r, 0] = torch.where(any_term, x.max(1).values, 0.0)
        if want_dx:
            dx[r] = grad.to(dx.dtype)
    return loss, stats, dx


def exact(case, seed):
    s = _embed_inputs(case, seed) if case["op"].startswith("embed") else _distill_inputs(case, seed)
    if case["op"] == "embed_fwd":
        rows = torch.where((s["ids"] != PAD)[:, None], s["W"].index_select(0, s["ids"]).double(), 0.0)
        return {"y": rows * s["scale"]}
    if case["op"] == "embed_bwd":
        v, d = s["shape"]
        out = s["add"].double() if s["add"] is not None else torch.zeros((v, d), dtype=torch.float64, device="cuda")
        kept = torch.nonzero(s["ids"] != PAD)[:, 0]
        ids = s["ids"][kept].long()
        for a in range(0, d, 512):   # (a band of columns at a time: the indexes of scatter_add_ are as large as its source)
            source = s["dy"][kept, a:a + 512].double() * s["scale"]
            out[:, a:a + 512].scatter_add_(0, ids[:, None].expand(-1, source.shape[1]), source)
        return {"dW": out}
    loss, stats, dx = _exact_rows(s)
    if case["op"] == "distill_fwd":
        return {"loss": loss, "stats": stats}
    return {"dx": dx} if case["op"] == "distill_bwd" else {"loss": loss, "dx": dx}
