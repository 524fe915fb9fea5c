"""Timed cases of layer norm (forward and backward) and of activation
checkpoints in 8 bits (pack and unpack, and the backward passes that read them).

Kinds of a case:

norm        rows -> normalised rows and their statistics; checkpoint = True:
            also the normalised values in 8 bits, as the backward pass keeps
            them (returned as the values that the codes stand for).
norm_bwd    the gradients of the rows, the scales and the biases, from the
            rows (checkpoint = False) or from the checkpoint of their
            normalised values.
checkpoint  rows into 8 bits and back: what a training step does with an
            activation between its forward and its backward pass.
weights     the weight gradient of a fully connected layer whose input was
            kept as a checkpoint.

A checkpoint holds signed codes of 8 bits, in blocks of 32 along a row, each
with a power of two as its step: codes [rows][F] (F = features rounded up to
32), then a byte S per block [rows][F / 32]; a value is code * 2^(S - 133).

`pad` is the number of unused entries behind each row (its stride is features +
pad).
"""
import math
import os
import sys

import torch

own = False  # True: run() calls the framework's operators, False: their plain form

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}  # ACH_F32, ACH_BF16, ACH_F16
EPS = 1e-5
MOST = 1 << 25       # entries of a drawn case
MOST_FLOPS = 1.3e11  # of a drawn weight gradient


def listed():
    return [
        # one image, or one token, at a time: latency decides
        norm("norm_1x1024_bf16", 1, 1024, "bf16"),
        # the forward of a training step over many rows that keeps 8 bits for its backward
        norm("norm_16384x4096_bf16_checkpoint", 16384, 4096, "bf16", checkpoint=True),
        # odd sizes, rows of a wider buffer
        norm("norm_1021x5003_f16", 1021, 5003, "f16", pad=13),
        # the image classifier's feature maps, each image over all its 256x27x27 values
        norm("norm_128x186624_f32", 128, 186624, "f32"),
        # a fully connected layer's features at the classifier's batch
        norm_bwd("norm_bwd_128x4096_f32", 128, 4096, "f32"),
        # the backward of a training step over many rows
        norm_bwd("norm_bwd_16384x4096_bf16", 16384, 4096, "bf16"),
        # the same from the checkpoint, odd sizes
        norm_bwd("norm_bwd_1027x13001_f32_checkpoint", 1027, 13001, "f32", checkpoint=True),
        # the classifier's first feature maps (96x55x55 an image) between forward and backward
        checkpoint("checkpoint_128x290400_f32", 128, 290400, "f32"),
        # odd and ragged sizes
        checkpoint("checkpoint_2051x1003_bf16", 2051, 1003, "bf16", pad=5),
        # the classifier's largest fully connected layer at its batch
        weights("weights_128x9216x4096_f32", 128, 9216, 4096, "f32"),
        # a layer over many rows: the matrix units decide
        weights("weights_16384x4096x1024_bf16", 16384, 4096, 1024, "bf16"),
        # odd sizes, few tiles: the rows are shared out
        weights("weights_1531x1003x777_f16", 1531, 1003, 777, "f16", pad=3),
    ]


def _case(name, **c):
    return dict(c, name=name) if name else c


def norm(name, rows, features, type, pad=0, checkpoint=False):
    return _case(name, kind="norm", rows=rows, features=features, type=type, pad=pad,
                 checkpoint=checkpoint)


def norm_bwd(name, rows, features, type, pad=0, checkpoint=False):
    return _case(name, kind="norm_bwd", rows=rows, features=features, type=type, pad=pad,
                 checkpoint=checkpoint)


def checkpoint(name, rows, features, type, pad=0):
    return _case(name, kind="checkpoint", rows=rows, features=features, type=type, pad=pad)


def weights(name, rows, features, outputs, type, pad=0):
    return _case(name, kind="weights", rows=rows, features=features, outputs=outputs, type=type,
                 pad=pad)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """odd ones among them, and sizes as networks have them"""
    n = _log(rng, lo, hi)
    return n if n < 64 or rng.random() < 0.6 else n // 64 * 64


def draw(rng):
    kind = rng.choices(("norm", "norm_bwd", "checkpoint", "weights"), (3, 3, 2, 3))[0]
    type = rng.choice(("f32", "bf16", "f16"))
    pad = rng.choice((0, 0, rng.randint(1, 40)))
    if kind == "weights":
        features, outputs = _size(rng, 16, 9000), _size(rng, 10, 4000)
        most = MOST_FLOPS / (2.0 * features * outputs * (3 if type == "f32" else 2 if type == "f16" else 1))
        return weights(None, _size(rng, 1, max(2, min(20000, most))), features, outputs, type, pad)
    features = _size(rng, 8, 300000)
    rows = _size(rng, 1, max(2, min(40000, MOST // features)))
    if kind == "checkpoint":
        return checkpoint(None, rows, features, type, pad)
    return (norm if kind == "norm" else norm_bwd)(None, rows, features, type, pad,
                                                  rng.random() < 0.5)


# ---- preparation -----------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 6007 + 11)


def _activations(g, rows, features):
    """Activations as a network has them: each feature with a level and a
    spread of its own, a few features far above the others."""
    spread = torch.empty(features, device=DEV).exponential_(1.0, generator=g).add_(0.1)
    level = torch.randn(features, generator=g, device=DEV) * 0.3
    lift = torch.rand(features, generator=g, device=DEV) < 0.002
    spread = torch.where(lift, spread * 20, spread)
    return torch.randn(rows, features, generator=g, device=DEV) * spread + level


def _padded(x, pad, type):
    """x as rows of a wider buffer, in its type."""
    rows, n = x.shape
    if not pad:
        return x.to(TYPES[type])
    wide = torch.zeros(rows, n + pad, dtype=TYPES[type], device=DEV)
    wide[:, :n] = x.to(TYPES[type])
    return wide[:, :n]


def prepare(case, seed):
    g = _gen(seed)
    rows, features, kind = case["rows"], case["features"], case["kind"]
    s = dict(case=case)
    x = _padded(_activations(g, rows, features), case["pad"] if kind != "weights" else 0,
                case["type"])
    if kind in ("norm", "norm_bwd"):
        s["scales"] = torch.randn(features, generator=g, device=DEV) * 0.2 + 1
        s["biases"] = torch.randn(features, generator=g, device=DEV) * 0.1
    if kind in ("norm", "checkpoint"):
        s["x"] = x
        return s
    # gradients as a mean over the rows leaves them; fp16 ones come with a loss scale
    scale = (1024.0 if case["type"] == "f16" else 1.0) / rows
    width = case["outputs"] if kind == "weights" else features
    s["delta"] = _padded(torch.randn(rows, width, generator=g, device=DEV) * scale, case["pad"],
                         case["type"])
    if kind == "norm_bwd":  # what the forward pass left behind
        xf = x.double()
        mean = xf.mean(1, keepdim=True)
        rstd = (xf.var(1, unbiased=False, keepdim=True) + EPS).rsqrt()
        s["stats"] = torch.cat((mean, rstd), 1).float()
        if not case["checkpoint"]:
            s["x"] = x
            return s
        x = (x.float() - s["stats"][:, :1]) * s["stats"][:, 1:]
    s["kept"] = torch.cat([t.view(torch.uint8).view(-1) for t in _plain_pack(x.float())])
    return s


# ---- the plain forms ---------------------------------------------------------
def _plain_pack(xf):
    """Codes [rows][F] and block bytes [rows][F / 32] of finite float rows."""
    rows, n = xf.shape
    blocks = -(-n // 32)
    b = torch.nn.functional.pad(xf, (0, blocks * 32 - n)).view(rows, blocks, 32)
    # the step is the power of two that leaves the largest value at most 127.49
    top = b.abs().amax(2).view(torch.int32)
    S = ((top + 0x10000) >> 23).clamp(7, 254)
    codes = (b * _power(133 - S).unsqueeze(2)).round().clamp(-127, 127)
    return codes.to(torch.int8).view(rows, blocks * 32), S.to(torch.uint8)


def _power(e):
    """2^e as floats, e between -126 and 127"""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_unpack(codes, S, n):
    rows, blocks = S.shape
    v = codes.view(rows, blocks, 32).float() * _power(S.int() - 133).unsqueeze(2)
    return v.view(rows, blocks * 32)[:, :n]


def _kept(kept, rows, n):
    """The two parts of a checkpoint."""
    wide = -(-n // 32) * 32
    codes = kept[:rows * wide].view(torch.int8).view(rows, wide)
    return codes, kept[rows * wide:].view(rows, wide // 32)


def _plain_norm(x, scales, biases, keep):
    xf = x.float()
    mean = xf.mean(1, keepdim=True, dtype=torch.float64).float()
    d = xf - mean
    rstd = ((d * d).mean(1, keepdim=True) + EPS).rsqrt()
    x_norm = d * rstd
    out = dict(y=(x_norm * scales + biases).to(x.dtype), stats=torch.cat((mean, rstd), 1))
    if keep:
        out["x_norm"] = _plain_unpack(*_plain_pack(x_norm), x.shape[1]).bfloat16()  # exact
    return out


def _plain_norm_bwd(delta, x_norm, rstd, scales):
    n = x_norm.shape[1]
    d = delta.float()
    g = d * scales
    m1, m2 = g.sum(1, keepdim=True) / n, (g * x_norm).sum(1, keepdim=True) / n
    return dict(dx=(rstd * (g - m1 - x_norm * m2)).to(delta.dtype), scales=(d * x_norm).sum(0),
                biases=d.sum(0))


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
    c = s["case"]
    rows, n, kind = c["rows"], c["features"], c["kind"]
    lib, ref = aetcnn.ops(), aetcnn.C.byref
    type = CODES[c["type"]]

    def new(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    ws_bytes = 0
    if kind in ("norm", "norm_bwd"):
        x = s.get("x")
        d = aetcnn.LayernormDesc(rows, n, type, EPS, x.stride(0) if x is not None else 0)
        if kind == "norm":
            ws_bytes = lib.ach_layernorm_fwd_workspace(ref(d))
            out = dict(y=new(rows, n, dtype=x.dtype), stats=new(rows, 2))
            if c["checkpoint"]:
                out["x_norm"] = new(rows, n, dtype=torch.bfloat16)
                s["unpack"] = ref(aetcnn.CheckpointDesc(rows, n, aetcnn.BF16, 0))
        else:
            ws_bytes = lib.ach_layernorm_bwd_workspace(ref(d))
            out = dict(dx=new(rows, n, dtype=s["delta"].dtype), scales=new(n), biases=new(n))
    elif kind == "checkpoint":
        d = aetcnn.CheckpointDesc(rows, n, type, s["x"].stride(0))
        s["unpack"] = ref(aetcnn.CheckpointDesc(rows, n, type, 0))
        out = new(rows, n, dtype=s["x"].dtype)
    else:
        d = aetcnn.FcDesc(rows, n, c["outputs"], type, s["delta"].stride(0))
        ws_bytes = lib.ach_fc_bwd_filter_checkpoint_workspace(ref(d))
        out = new(c["outputs"], n)
    if "unpack" in s:
        s["kept"] = new(lib.ach_checkpoint_bytes(rows, n), dtype=torch.uint8)
    ws = new(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    s.update(lib=lib, check=aetcnn.check, desc=ref(d), out=out, ws=ws, ws_bytes=ws_bytes)


def _own(s):
    if "lib" not in s:
        _plan(s)
    c, o, lib, rc = s["case"], s["out"], s["lib"], 0
    if c["kind"] == "norm":
        rc = lib.ach_layernorm_fwd(s["desc"], _ptr(s["x"]), _ptr(s["scales"]), _ptr(s["biases"]),
                                   _ptr(o["y"]), 0, _ptr(o["stats"]), _ptr(s.get("kept")),
                                   _ptr(s["ws"]), s["ws_bytes"], _stream())
        if c["checkpoint"]:
            rc = rc or lib.ach_checkpoint_unpack(s["unpack"], _ptr(s["kept"]), _ptr(o["x_norm"]),
                                                 _stream())
    elif c["kind"] == "norm_bwd":
        rc = lib.ach_layernorm_bwd(s["desc"], _ptr(s["delta"]), s["delta"].stride(0),
                                   _ptr(s.get("x")), _ptr(s.get("kept")), _ptr(s["stats"]),
                                   _ptr(s["scales"]), _ptr(o["dx"]), 0, _ptr(o["scales"]),
                                   _ptr(o["biases"]), 0, _ptr(s["ws"]), s["ws_bytes"], _stream())
    elif c["kind"] == "checkpoint":
        rc = lib.ach_checkpoint_pack(s["desc"], _ptr(s["x"]), _ptr(s["kept"]), _stream())
        rc = rc or lib.ach_checkpoint_unpack(s["unpack"], _ptr(s["kept"]), _ptr(o), _stream())
    else:
        rc = lib.ach_fc_bwd_filter_checkpoint(s["desc"], _ptr(s["kept"]), _ptr(s["delta"]), _ptr(o),
                                              0, _ptr(s["ws"]), s["ws_bytes"], _stream())
    if rc:
        s["check"](rc, c["kind"])
    return o


def run(s):
    if own:
        return _own(s)
    c = s["case"]
    rows, n = c["rows"], c["features"]
    if c["kind"] == "norm":
        return _plain_norm(s["x"], s["scales"], s["biases"], c["checkpoint"])
    if c["kind"] == "norm_bwd":
        mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
        x_norm = (_plain_unpack(*_kept(s["kept"], rows, n), n) if c["checkpoint"]
                  else (s["x"].float() - mean) * rstd)
        return _plain_norm_bwd(s["delta"], x_norm, rstd, s["scales"])
    if c["kind"] == "checkpoint":
        v = _plain_unpack(*_plain_pack(s["x"].float()), n)
        most = torch.finfo(s["x"].dtype).max
        return v.clamp(-most, most).to(s["x"].dtype)
    return s["delta"].float().t() @ _plain_unpack(*_kept(s["kept"], rows, n), n)


# ---- what a pass cannot do without -----------------------------------------------
def work(case):
    rows, n, kind = case["rows"], case["features"], case["kind"]
    size = 4 if case["type"] == "f32" else 2
    e = rows * n
    kept = rows * -(-n // 32) * 33  # a checkpoint's bytes
    if kind == "norm":  # subtract, square, two sums, two products, one more sum
        # the values of the codes (2 bytes each) are returned for comparison
        return {"bytes": 2 * e * size + 8 * n + 8 * rows + (kept + 2 * e if case["checkpoint"] else 0),
                "flops": (12 if case["checkpoint"] else 8) * e}
    if kind == "norm_bwd":
        return {"bytes": 2 * e * size + (kept if case["checkpoint"] else e * size) + 12 * n + 8 * rows,
                "flops": 14 * e}
    if kind == "checkpoint":
        return {"bytes": 2 * e * size + kept, "flops": 6 * e}
    m = case["outputs"]
    return {"bytes": rows * m * size + kept + 4 * n * m, "flops": 2 * rows * n * m}


# ---- the definition in 64 bits ---------------------------------------------------
def _exact_values(kept, rows, n):
    """What a checkpoint's bytes stand for."""
    blocks = (n + 31) // 32
    c = kept[:rows * blocks * 32].view(torch.int8).double().view(rows, blocks, 32)
    S = kept[rows * blocks * 32:].double().view(rows, blocks, 1)
    return (c * torch.pow(2.0, S - 133)).flatten(1)[:, :n]


def _exact_rounded(x):
    """The values that a checkpoint of x stands for."""
    rows, n = x.shape
    b = torch.cat((x, x.new_zeros(rows, -n % 32)), 1).view(rows, -1, 32)
    top = b.abs().max(2, keepdim=True).values
    _, e = torch.frexp(top)  # top = m * 2^e, m at least 1/2
    step = ((e.long() - 7 + 1023) << 52).view(torch.float64)  # 2^(e - 7); pow may be an ulp off
    step = torch.where(top / step >= 127.5, 2 * step, step).clamp(min=2.0 ** -126)
    return (torch.round(b / step) * step).flatten(1)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    rows, n, kind = case["rows"], case["features"], case["kind"]
    if kind == "weights":
        return s["delta"].double().t() @ _exact_values(s["kept"], rows, n)
    if kind == "checkpoint":
        most = torch.finfo(s["x"].dtype).max
        return _exact_rounded(s["x"].double()).clamp(-most, most)
    if kind == "norm":
        x = s["x"].double()
        mean = x.sum(1, keepdim=True) / n
        rstd = 1 / torch.sqrt((x - mean).pow(2).sum(1, keepdim=True) / n + EPS)
        x_norm = (x - mean) * rstd
        out = dict(y=x_norm * s["scales"].double() + s["biases"].double(),
                   stats=torch.cat((mean, rstd), 1))
        if case["checkpoint"]:
            out["x_norm"] = _exact_rounded(x_norm)
        return out
    stats = s["stats"].double()
    x_norm = (_exact_values(s["kept"], rows, n) if case["checkpoint"]
              else (s["x"].double() - stats[:, :1]) * stats[:, 1:])
    d = s["delta"].double()
    g = d * s["scales"].double()
    along = (g * x_norm).sum(1, keepdim=True) / n
    return dict(dx=stats[:, 1:] * (g - g.sum(1, keepdim=True) / n - along * x_norm),
                scales=(d * x_norm).sum(0), biases=d.sum(0))
