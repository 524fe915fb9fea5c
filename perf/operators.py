"""Timed cases of the operators on logits: log probabilities of given classes
with entropy and top alternatives (forward and backward), and distillation
from a teacher's top logits (loss and gradient).

Kinds of a case:

logprobs      rows of logits -> the given class's log probability and rank,
              the entropy, the k best classes with their log probabilities,
              and the statistics that the backward pass reads.
logprobs_bwd  the gradient of the logits from those of the log probabilities
              and (entropy = True) of the entropies.
distill       the loss of student logits against a teacher's k best classes
              (tail = True: with the probability of all other classes as one
              more entry) and, with hard > 0, against a label; and its
              gradient, as the delta that a training step propagates.

`pad` is the number of unused entries behind each row (its stride is classes +
pad), `allowed` the fraction of classes that are not masked with -inf,
`ignored` the fraction of rows without a class or a weight (padding).
"""
import math
import os
import sys

import torch

own = False  # True: run() calls the framework's operators, False: their plain form

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}  # ACH_F32, ACH_BF16, ACH_F16
MOST = 1 << 27  # entries of a drawn case


def listed():
    return [
        # one answer of a service with a large set of classes: latency decides
        logprobs("next_1x131072_bf16", 1, 131072, "bf16", k=20),
        # a batch of answers of which a grammar or a filter has masked most classes, odd size, sharpened
        logprobs("next_64x100003_f16_masked", 64, 100003, "f16", k=5, temperature=0.7, pad=29,
                 allowed=0.3),
        # the image classifier's benchmark batch, validated top 1 and top 5
        logprobs("classes_128x1000_f32", 128, 1000, "f32", k=5),
        # scoring a long text with the alternatives at every place
        logprobs("score_1024x131072_bf16", 1024, 131072, "bf16", k=20),
        # the teacher's side of a distillation: its best classes, softened
        logprobs("teacher_512x65536_f32", 512, 65536, "f32", k=64, temperature=2.0),
        # a policy update's forward: no alternatives, some padding
        logprobs("policy_4096x32768_bf16", 4096, 32768, "bf16", k=0, ignored=0.1),
        # its backward with an entropy bonus
        dict(name="policy_bwd_4096x32768_bf16", kind="logprobs_bwd", rows=4096, classes=32768,
             type="bf16", temperature=1.0, pad=0, entropy=True, ignored=0.1),
        # the gradient of a log likelihood alone, rows at odd addresses
        dict(name="nll_bwd_515x50021_f32", kind="logprobs_bwd", rows=515, classes=50021, type="f32",
             temperature=1.0, pad=2, entropy=False, ignored=0.0),
        # the image classifier's training batch from a teacher's 10 best of 1000 classes and the labels
        distill("distill_128x1000_f32", 128, 1000, "f32", 10, 4.0, False, 0.5, 0.5),
        # a few long rows: the work of a row is spread over the chip
        distill("distill_16x131072_f32_tail", 16, 131072, "f32", 64, 1.0, True, 1.0, 0.0),
        # odd sizes, two temperatures in one pass, padded rows
        distill("distill_1021x50021_f16", 1021, 50021, "f16", 17, 2.0, False, 0.7, 0.3, ignored=0.2),
        # a training batch of long sequences on a large set of classes
        distill("distill_2048x131072_bf16_tail", 2048, 131072, "bf16", 64, 1.0, True, 1.0, 0.0),
    ]


def logprobs(name, rows, classes, type, k, temperature=1.0, pad=0, allowed=1.0, ignored=0.0):
    c = dict(kind="logprobs", rows=rows, classes=classes, type=type, k=k, temperature=temperature,
             pad=pad, allowed=allowed, ignored=ignored)
    return dict(c, name=name) if name else c


def distill(name, rows, classes, type, k, temperature, tail, soft, hard, pad=0, ignored=0.0):
    c = dict(kind="distill", rows=rows, classes=classes, type=type, k=k, temperature=temperature,
             tail=tail, soft=soft, hard=hard, pad=pad, ignored=ignored)
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("logprobs", "logprobs_bwd", "distill"), (3, 2, 3))[0]
    classes = _log(rng, 10, 200000)
    if rng.random() < 0.4:  # sizes as networks have them
        classes = -(-classes // 64) * 64
    rows = _log(rng, 1, max(2, min(8192, MOST // classes)))
    type = rng.choice(("f32", "bf16", "f16"))
    temperature = rng.choice((1.0, 1.0, round(rng.uniform(0.5, 4.0), 2)))
    pad = rng.choice((0, 0, rng.randint(1, 64)))
    ignored = rng.choice((0.0, 0.2))
    k = min(classes, _log(rng, 1, 128))
    if kind == "logprobs":
        allowed = rng.choice((1.0, 1.0, 0.5)) if classes >= 4 * k + 64 else 1.0
        return logprobs(None, rows, classes, type, rng.choice((0, k, k)), temperature, pad, allowed,
                        ignored)
    if kind == "logprobs_bwd":
        return dict(kind=kind, rows=rows, classes=classes, type=type, temperature=temperature,
                    pad=pad, entropy=rng.random() < 0.5, ignored=ignored)
    hard = rng.choice((0.0, 0.5))
    return distill(None, rows, classes, type, min(k, max(1, classes // 2)), temperature,
                   rng.random() < 0.5, 1.0 - hard, hard, pad, ignored)


# ---- preparation -----------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 29)


def _logits(g, rows, classes, spread=2.5):
    """Logits as a trained classifier gives them: a bulk, and some classes far
    above it."""
    x = torch.randn(rows, classes, generator=g, device=DEV) * spread
    n = max(1, min(classes // 4, 32))
    at = torch.randint(classes, (rows, n), generator=g, device=DEV)
    lift = torch.empty(rows, n, device=DEV).exponential_(0.25, generator=g).clamp_(max=15.0)
    return x.scatter_add_(1, at, lift)


def _padded(x, pad, type):
    """x as rows of a wider buffer, in its type."""
    rows, classes = x.shape
    wide = torch.zeros(rows, classes + pad, dtype=TYPES[type], device=DEV)
    wide[:, :classes] = x.to(TYPES[type])
    return wide[:, :classes]


def _ids(x, g, ignored):
    """A class for each row, drawn from its distribution; -1 in ignored rows."""
    noise = torch.rand(x.shape, generator=g, device=DEV).clamp_(min=1e-9).log_().neg_().log_().neg_()
    ids = (x.float() + noise).argmax(1).to(torch.int32)
    ids[torch.rand(len(ids), generator=g, device=DEV) < ignored] = -1
    return ids


def prepare(case, seed):
    g = _gen(seed)
    rows, classes, kind = case["rows"], case["classes"], case["kind"]
    x = _logits(g, rows, classes)
    if case.get("allowed", 1.0) < 1.0:
        x[torch.rand(x.shape, generator=g, device=DEV) > case["allowed"]] = -math.inf
    s = dict(case=case, x=_padded(x, case["pad"], case["type"]))
    scale = 4096.0 if case["type"] == "f16" else 1.0  # fp16 gradients come with a loss scale
    if kind == "distill":
        t = (_logits(g, rows, classes) * 0.4 + x * 0.6) / (case["temperature"] if case["tail"] else 1.0)
        top = (t - t.logsumexp(1, keepdim=True)).topk(case["k"], 1)
        s["teacher_ids"] = top.indices.to(torch.int32).contiguous()
        s["teacher_values"] = top.values.contiguous()
        s["labels"] = _ids(t, g, 0.0) if case["hard"] else None
        w = torch.ones(rows, device=DEV)
        w[torch.rand(rows, generator=g, device=DEV) < case["ignored"]] = 0.0
        s["weights"] = w * (scale / rows)
        return s
    s["ids"] = _ids(s["x"], g, case["ignored"])
    if kind == "logprobs_bwd":
        xf = s["x"].double()  # what the forward pass left behind
        m = xf.amax(1, keepdim=True)
        d = (xf - m) / case["temperature"]
        e = d.exp()
        total = e.sum(1, keepdim=True)
        log_total = (total - 1).log1p()
        s["stats"] = torch.cat((m, log_total), 1).float()
        s["entropy"] = (log_total - (e * d).sum(1, keepdim=True) / total).float().view(-1)
        s["dlogprobs"] = torch.randn(rows, generator=g, device=DEV) * (scale / rows)
        s["dentropy"] = (torch.rand(rows, generator=g, device=DEV) * (-0.01 * scale / rows)
                         if case["entropy"] else None)
    return s


# ---- the plain forms ---------------------------------------------------------
def _plain_logprobs(x, ids, k, temperature):
    xf = x.float()
    m = xf.amax(1, keepdim=True)
    d = (xf - m) / temperature
    e = d.exp()
    # the best class counts 1: what the others add matters to the last bit where they are little
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = (total - 1).log1p().float()
    entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total.float()
    at = ids.long().clamp(min=0).view(-1, 1)
    given = ids.view(-1, 1) >= 0
    out = dict(logprobs=torch.where(given, d.gather(1, at) - log_total, 0.0).view(-1),
               ranks=torch.where(given, (xf > xf.gather(1, at)).sum(1, keepdim=True),
                                 -1).to(torch.int32).view(-1),
               entropy=entropy.view(-1), stats=torch.cat((m, log_total), 1))
    if k:
        bits = (xf + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32
        order |= torch.arange(x.shape[1] - 1, -1, -1, device=x.device)  # ties: the lowest index
        top = order.topk(k, 1).indices
        out["top_ids"] = top.to(torch.int32)
        out["top_logprobs"] = d.gather(1, top) - log_total
    return out


def _plain_logprobs_bwd(x, ids, temperature, stats, entropy, dlogprobs, dentropy):
    logp = (x.float() - stats[:, :1]) / temperature - stats[:, 1:]
    p = logp.exp()
    w = torch.where(ids >= 0, dlogprobs, 0.0).view(-1, 1)
    at = ids.long().clamp(min=0).view(-1, 1)
    grad = -w * p.scatter(1, at, logp.gather(1, at).expm1())  # p - 1 of the given class
    if dentropy is not None:
        grad -= dentropy.view(-1, 1) * torch.where(p > 0, p * (logp + entropy.view(-1, 1)), 0.0)
    return (grad / temperature).to(x.dtype)


def _plain_distill(x, teacher_ids, values, labels, weights, temperature, tail, soft, hard):
    xf = x.float()
    m = xf.amax(1, keepdim=True)
    z = (xf - m) / temperature
    e = z.exp()
    at = teacher_ids.long()
    # in 64 bits: 1 - sum(p) of a teacher that is nearly certain
    v = values.double() if tail else values.double() / temperature
    p = v.exp() if tail else (v - v.amax(1, keepdim=True)).exp()
    if not tail:
        p = p / p.sum(1, keepdim=True)
    rest = (1 - p.sum(1, keepdim=True)).clamp(min=0.0)
    others = e.scatter(1, at, 0.0).sum(1, keepdim=True, dtype=torch.float64)
    total = others + e.gather(1, at).sum(1, keepdim=True, dtype=torch.float64)
    logq = z.gather(1, at) - total.log()
    kd = (p * (p.log() - logq)).sum(1, keepdim=True)
    q = e / total.float()
    grad = q * (p.sum(1, keepdim=True) + (rest if tail else 0.0)).float()
    if tail:
        kd += torch.where(rest > 0, rest * (rest.log() - (others / total).log()), 0.0)
        grad -= (e * (rest / others).float()).scatter(1, at, 0.0)
    grad.scatter_add_(1, at, -p.float())
    loss = soft * temperature * temperature * kd
    grad *= soft * temperature
    if hard:
        y = labels.long().view(-1, 1)
        e1 = (xf - m).exp()
        s1 = e1.sum(1, keepdim=True, dtype=torch.float64)
        loss = loss + hard * ((s1 - 1).log1p() - (xf - m).gather(1, y))
        grad += hard * e1 / s1.float()
        grad.scatter_add_(1, y, torch.full_like(m, -hard))
    w = weights.view(-1, 1)
    loss = (w * loss).float().view(-1)
    return dict(loss=loss, delta=(-w * grad).to(x.dtype), cost=loss.sum())


# ---- the framework's calls -----------------------------------------------------
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _plan(s):
    """The descriptors, the workspace and the outputs that a program keeps."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "aet-cnn_amd"))
    import aetcnn
    c, x = s["case"], s["x"]
    rows, classes, k = c["rows"], c["classes"], c.get("k", 0)
    lib, ref = aetcnn.ops(), aetcnn.C.byref
    d = aetcnn.LogitsDesc(rows, classes, CODES[c["type"]], c["temperature"], x.stride(0))

    def new(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    out, ws_bytes = {}, 0
    if c["kind"] == "logprobs":
        ws_bytes = lib.ach_logprobs_workspace(ref(d), k)
        out = dict(logprobs=new(rows), ranks=new(rows, dtype=torch.int32), entropy=new(rows),
                   stats=new(rows, 2))
        if k:
            out.update(top_ids=new(rows, k, dtype=torch.int32), top_logprobs=new(rows, k))
    elif c["kind"] == "logprobs_bwd":
        out = new(rows, classes, dtype=x.dtype)
    else:
        t = aetcnn.DistillDesc(k, aetcnn.DISTILL_TAIL if c["tail"] else aetcnn.DISTILL_RENORM,
                               aetcnn.F32, c["soft"], c["hard"])
        ws_bytes = lib.ach_distill_workspace(ref(d), ref(t))
        out = dict(loss=new(rows), delta=new(rows, classes, dtype=x.dtype), cost=new(1).view(()))
        s["teacher"] = ref(t)
    ws = new(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    s.update(lib=lib, check=aetcnn.check, desc=ref(d), out=out, ws=ws, ws_bytes=ws_bytes)


def _own(s):
    if "lib" not in s:
        _plan(s)
    c, o, lib = s["case"], s["out"], s["lib"]
    if c["kind"] == "logprobs":
        rc = lib.ach_logprobs_fwd(s["desc"], _ptr(s["x"]), _ptr(s["ids"]), c["k"],
                                  _ptr(o["logprobs"]), _ptr(o["ranks"]), _ptr(o["entropy"]),
                                  _ptr(o["stats"]), _ptr(o.get("top_ids")),
                                  _ptr(o.get("top_logprobs")), _ptr(s["ws"]), s["ws_bytes"],
                                  _stream())
    elif c["kind"] == "logprobs_bwd":
        rc = lib.ach_logprobs_bwd(s["desc"], _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["stats"]),
                                  _ptr(s["entropy"]), _ptr(s["dlogprobs"]), _ptr(s["dentropy"]),
                                  _ptr(o), 0, _stream())
    else:
        rc = lib.ach_distill_xent(s["desc"], s["teacher"], _ptr(s["x"]), _ptr(s["teacher_ids"]),
                                  _ptr(s["teacher_values"]), _ptr(s["labels"]), _ptr(s["weights"]),
                                  _ptr(o["loss"]), _ptr(o["delta"]), 0, _ptr(o["cost"]),
                                  _ptr(s["ws"]), s["ws_bytes"], _stream())
    if rc:
        s["check"](rc, c["kind"])
    return o


def run(s):
    if own:
        return _own(s)
    c = s["case"]
    if c["kind"] == "logprobs":
        return _plain_logprobs(s["x"], s["ids"], c["k"], c["temperature"])
    if c["kind"] == "logprobs_bwd":
        return _plain_logprobs_bwd(s["x"], s["ids"], c["temperature"], s["stats"], s["entropy"],
                                   s["dlogprobs"], s["dentropy"])
    return _plain_distill(s["x"], s["teacher_ids"], s["teacher_values"], s["labels"], s["weights"],
                          c["temperature"], c["tail"], c["soft"], c["hard"])


# ---- what a pass cannot do without -----------------------------------------------
def work(case):
    rows, classes, k = case["rows"], case["classes"], case.get("k", 0)
    n = rows * classes
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "logprobs":  # the row; compare, subtract, scale, exp, two sums, compare with the given
        return {"bytes": n * size + rows * (4 + 5 * 4 + 8 * k), "flops": 8 * n}
    if case["kind"] == "logprobs_bwd":
        return {"bytes": 2 * n * size + rows * (5 if case["entropy"] else 4) * 4,
                "flops": (6 if case["entropy"] else 4) * n}
    return {"bytes": 2 * n * size + rows * (8 * k + 12),  # statistics, then the gradient
            "flops": (9 if not case["hard"] else 14) * n}


# ---- the definition in 64 bits ---------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    parts = [_exact_rows(s, case, a, min(case["rows"], a + 128))
             for a in range(0, case["rows"], 128)]
    if case["kind"] == "logprobs_bwd":
        return torch.cat(parts)
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    if case["kind"] == "distill":
        out["cost"] = out["loss"].sum()
    return out


def _exact_rows(s, case, a, b):
    t, rows = case["temperature"], b - a
    x = s["x"][a:b].double().requires_grad_(case["kind"] != "logprobs")
    every = torch.arange(rows, device=DEV)
    logp = torch.log_softmax(x / t, 1)
    if case["kind"] == "distill":
        ids, v = s["teacher_ids"][a:b].long(), s["teacher_values"][a:b].double()
        logt = v if case["tail"] else torch.log_softmax(v / t, 1)
        loss = (logt.exp() * (logt - logp.gather(1, ids))).sum(1)
        if case["tail"]:
            member = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids, True)
            logrest = logp.masked_fill(member, -math.inf).logsumexp(1)
            rest = -torch.expm1(logt.logsumexp(1))
            loss = loss + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - logrest), 0.0)
        loss = case["soft"] * t * t * loss
        if case["hard"]:
            y = s["labels"][a:b].long()
            loss = loss - case["hard"] * torch.log_softmax(x, 1)[every, y]
        loss = loss * s["weights"][a:b].double()
        grad, = torch.autograd.grad(loss.sum(), x)
        return dict(loss=loss.detach(), delta=-grad)
    ids = s["ids"][a:b].long()
    given = ids >= 0
    mine = torch.where(given, logp[every, ids.clamp(min=0)], 0.0)
    entropy = torch.special.entr(logp.exp()).sum(1)
    if case["kind"] == "logprobs_bwd":
        total = (mine * s["dlogprobs"][a:b].double()).sum()
        if s["dentropy"] is not None:
            total = total + (entropy * s["dentropy"][a:b].double()).sum()
        return torch.autograd.grad(total, x)[0]
    m = x.max(1).values
    chosen = x[every, ids.clamp(min=0)].view(-1, 1)
    ranks = torch.where(given, (x - chosen > 0).sum(1), -1)
    out = dict(logprobs=mine, ranks=ranks.to(torch.int32), entropy=entropy,
               stats=torch.stack((m, (x / t).logsumexp(1) - m / t), 1))
    if case["k"]:
        best = x.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]]
        out["top_ids"], out["top_logprobs"] = best.to(torch.int32), logp.gather(1, best)
    return out
