"""What stands around the FP8 linears of a training step, as cases that can be timed and compared: the layer norm before a
linear, the activations that are kept in 8 bits between forward and backward, and the loss over the vocabulary at the end.

Each case is one pass through one of the operators, forward alone where a model is served or scored, forward and backward where it
is trained.  Widths are those of the repository's own configurations (hidden 7168, o_proj 16384, gate/up 36864) or generic ones;
`draw` gives further cases of the ranges that the listed ones stand for.

With `own` the operators are the framework's; without it their plain form, elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_IGNORED = -100
_EPS = 1e-5


def _hpfp8():
    path = os.path.join(os.getcwd(), "hyper-parallel_amd")       # imported from the repository's root
    if path not in sys.path:
        sys.path.insert(0, path)
    import hpfp8
    return hpfp8


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm of a decode step: a handful of sequences, where a launch's latency is what counts
        dict(name="norm_decode", kind="norm", rows=8, cols=7168, dtype="bf16", train=False, keep=False),
        # the norm before a linear of 4096 tokens, forward and backward with both vectors' gradients
        dict(name="norm_train", kind="norm", rows=4096, cols=7168, dtype="bf16", train=True, keep=False),
        # the same in a longer batch, its normalised input kept in 8 bits until the backward
        dict(name="norm_train_kept", kind="norm", rows=16384, cols=7168, dtype="bf16", train=True, keep=True),
        # a packed batch of variable-length sequences and a width that no vector divides, in half precision
        dict(name="norm_ragged", kind="norm", rows=1531, cols=1027, dtype="fp16", train=True, keep=False),
        # the activation between gate/up and down projection: its input is a layer's largest activation, kept in 8 bits
        dict(name="swiglu_kept", kind="act", rows=4096, cols=36864, dtype="bf16", act="swiglu"),
        # an ungated activation of a smaller model, ragged in both directions
        dict(name="gelu_kept_ragged", kind="act", rows=1531, cols=5003, dtype="fp16", act="gelu"),
        # an activation that a checkpoint keeps in 8 bits, and what the backward gets back of it
        dict(name="checkpoint", kind="checkpoint", rows=16384, cols=7168, dtype="bf16"),
        # the same for a small ragged one in single precision
        dict(name="checkpoint_small", kind="checkpoint", rows=37, cols=1000, dtype="fp32"),
        # scoring of a few tokens against a large vocabulary: the head's weight is read once
        dict(name="loss_score", kind="loss", tokens=5, hidden=7168, vocab=131072, train=False, smoothing=0.0),
        # a micro-batch of a smaller model
        dict(name="loss_train_micro", kind="loss", tokens=512, hidden=4096, vocab=32000, train=True, smoothing=0.0),
        # a packed batch against a vocabulary that is a multiple of nothing, with label smoothing
        dict(name="loss_train_ragged", kind="loss", tokens=1531, hidden=2048, vocab=50001, train=True, smoothing=0.1),
        # a micro-batch of 4096 tokens against a large vocabulary
        dict(name="loss_train", kind="loss", tokens=4096, hidden=7168, vocab=131072, train=True, smoothing=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, multiple=128):
    """A size spread over the logarithm of the range: half of the time a multiple of `multiple`, otherwise anything."""
    n = _log_int(rng, lo, hi)
    return max(multiple, n // multiple * multiple) if rng.random() < 0.5 else n


def draw(rng):
    most = _seconds(listed()[-1])
    while True:
        kind = rng.choice(["norm", "norm", "act", "checkpoint", "loss", "loss"])
        if kind == "norm":
            train = rng.random() < 0.75
            keep = train and rng.random() < 0.4
            case = dict(kind=kind, rows=_size(rng, 1, 65536), cols=_size(rng, 64, 16384),
                        dtype=rng.choice(["bf16", "bf16", "fp16"] if keep else ["bf16", "bf16", "fp16", "fp32"]), train=train, keep=keep)
        elif kind == "act":
            act = rng.choice(["swiglu", "swiglu", "silu", "gelu", "gelu_tanh"])
            case = dict(kind=kind, rows=_size(rng, 1, 32768), cols=2 * _size(rng, 64, 18432) if act == "swiglu" else _size(rng, 64, 36864),
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), act=act)
        elif kind == "checkpoint":
            case = dict(kind=kind, rows=_size(rng, 1, 65536), cols=_size(rng, 64, 36864), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        else:
            train = rng.random() < 0.6
            case = dict(kind=kind, tokens=_size(rng, 16, 4096) if train else _size(rng, 1, 2048, 64), hidden=_size(rng, 256, 7168, 128) // 8 * 8,
                        vocab=_size(rng, 1000, 131072), train=train, smoothing=rng.choice([0.0, 0.0, 0.1]))
        elements = case["rows"] * case["cols"] if kind != "loss" else 1
        if elements <= 4096 * 36864 and _seconds(case) <= most:
            return case


def _seconds(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


# ------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------
def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = dict(case)
    if kind == "loss":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        bf16 = torch.bfloat16
        weight = _normal(g, (v, h), bf16).mul_(0.02)
        target = torch.randint(v, (t,), generator=g, device="cuda")
        # hidden states of a model that has learnt something: the target's logit stands out by 0 to about 10
        lean = torch.rand((t, 1), generator=g, device="cuda") * (10.0 / (0.02 * h))
        x = (_normal(g, (t, h), torch.float32) + lean * weight[target].float() / 0.02).to(bf16)
        # the prompt's tokens and the padding carry no loss
        target = torch.where(torch.rand((t,), generator=g, device="cuda") < (0.06 if t > 16 else 0.0), _IGNORED, target)
        if case["train"]:
            x.requires_grad_()
            weight.requires_grad_()
        state.update(x=x, weight=weight, target=target, scale=torch.full((), 1.0, device="cuda"))
        return state
    rows, cols, dtype = case["rows"], case["cols"], _DTYPES[case["dtype"]]
    if kind == "norm":
        # a residual stream: features of unequal size, some of them many times the others, off zero
        size = torch.exp(torch.randn((cols,), generator=g, device="cuda") * 0.7)
        shift = torch.randn((cols,), generator=g, device="cuda") * 0.5
        x = (torch.randn((rows, cols), generator=g, device="cuda") * size + shift).to(dtype)
        weight = (1.0 + 0.1 * torch.randn((cols,), generator=g, device="cuda")).to(dtype)
        bias = (0.1 * torch.randn((cols,), generator=g, device="cuda")).to(dtype)
        if case["train"]:
            for t in (x, weight, bias):
                t.requires_grad_()
            state["grad"] = _normal(g, (rows, cols), dtype)
        state.update(x=x, weight=weight, bias=bias)
        return state
    x = _normal(g, (rows, cols), dtype)
    x[:, :: max(1, cols // 7)] *= 20.0          # a few outlier features
    if kind == "act":
        x.requires_grad_()
        state["grad"] = _normal(g, (rows, cols // 2 if case["act"] == "swiglu" else cols), dtype)
    state["x"] = x
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    hpfp8 = _hpfp8()
    kind = s["kind"]
    if kind == "norm":
        if not s["train"]:
            with torch.no_grad():
                return hpfp8.layer_norm(s["x"], (s["cols"],), s["weight"], s["bias"], _EPS)
        y = hpfp8.layer_norm(s["x"], (s["cols"],), s["weight"], s["bias"], _EPS, keep_8bit=s["keep"])
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if kind == "act":
        y = hpfp8.activation(s["x"], s["act"], keep_8bit=True)
        dx, = torch.autograd.grad(y, (s["x"],), s["grad"])
        return {"y": y.detach(), "dx": dx}
    if kind == "checkpoint":
        return hpfp8.quantize_activation(s["x"]).dequantize()
    if not s["train"]:
        with torch.no_grad():
            return hpfp8.linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=_IGNORED, reduction="none",
                                              label_smoothing=s["smoothing"])
    loss = hpfp8.linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=_IGNORED, label_smoothing=s["smoothing"])
    dx, dw = torch.autograd.grad(loss, (s["x"], s["weight"]), s["scale"])
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def _in_8bit(x):
    """The fp32 values that x[R, C] is kept as: E4M3 codes with one scale for 128 values of a row (the last group is what is left)."""
    rows, cols = x.shape
    groups = (cols + 127) // 128
    full = torch.zeros((rows, groups * 128), dtype=torch.float32, device=x.device)
    full[:, :cols] = x
    full = full.view(rows, groups, 128)
    amax = full.abs().amax(-1, keepdim=True).clamp_min(1e-12)
    most = torch.full_like(amax, 448.0)      # (two divisions of tensors: a division by or of a number is a product with a reciprocal)
    codes = (full * (most / amax)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (codes.float() * (amax / most)).view(rows, groups * 128)[:, :cols]


def _plain(s):
    kind = s["kind"]
    x = s["x"].detach()
    dtype = x.dtype
    if kind == "norm":
        w, b = s["weight"].detach().float(), s["bias"].detach().float()
        xf = x.float()
        centred = xf - xf.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
        hat = centred * rstd
        y = (hat * w + b).to(dtype)
        if not s["train"]:
            return y
        if s["keep"]:
            hat = _in_8bit(hat)
        go = s["grad"].float()
        wg = go * w
        dx = (wg - wg.mean(-1, keepdim=True) - hat * (wg * hat).mean(-1, keepdim=True)) * rstd
        return {"y": y, "dx": dx.to(dtype), "dw": (go * hat).sum(0).to(dtype), "db": go.sum(0).to(dtype)}
    if kind == "act":
        xf, go = x.float(), s["grad"].float()
        half = x.shape[1] // 2
        if s["act"] == "swiglu":
            kept = torch.cat((_in_8bit(xf[:, :half]), _in_8bit(xf[:, half:])), 1)
            gate, up = xf[:, :half], xf[:, half:]
            y = gate / (1.0 + torch.exp(-gate)) * up
            gate, up = kept[:, :half], kept[:, half:]
            sig = 1.0 / (1.0 + torch.exp(-gate))
            dx = torch.cat((go * up * sig * (1.0 + gate * (1.0 - sig)), go * gate * sig), 1)
            return {"y": y.to(dtype), "dx": dx.to(dtype)}
        kept = _in_8bit(xf)
        return {"y": _act(xf, s["act"])[0].to(dtype), "dx": (go * _act(kept, s["act"])[1]).to(dtype)}
    if kind == "checkpoint":
        return _in_8bit(x.float()).to(dtype)
    w, target = s["weight"].detach().float(), s["target"]
    xf, smoothing, vocab = x.float(), s["smoothing"], s["vocab"]
    counted = target != _IGNORED
    at = torch.where(counted, target, 0).unsqueeze(1)
    logits = torch.matmul(xf, w.t())
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    loss = lse - (1.0 - smoothing) * logits.gather(1, at)
    if smoothing:
        loss = loss - smoothing * logits.mean(-1, keepdim=True)
    loss = torch.where(counted, loss.squeeze(1), 0.0)
    if not s["train"]:
        return loss
    n = counted.sum()
    p.div_(total)
    if smoothing:
        p.sub_(smoothing / vocab)
    p.scatter_add_(1, at, torch.full_like(at, -(1.0 - smoothing), dtype=torch.float32))
    p.mul_(torch.where(counted, s["scale"] / n, 0.0).unsqueeze(1))
    return {"loss": loss.sum() / n, "dx": torch.matmul(p, w).to(dtype), "dw": torch.matmul(p.t(), xf).to(dtype)}


def _act(x, kind):
    """(value, derivative) of an ungated activation."""
    if kind == "silu":
        sig = 1.0 / (1.0 + torch.exp(-x))
        return x * sig, sig * (1.0 + x * (1.0 - sig))
    if kind == "gelu":
        phi = 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
        return x * phi, phi + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (x + 0.044715 * x * x * x))
    return 0.5 * x * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * x * x)


# ------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------
def _kept64(x):
    """x (64 bits) as E4M3 codes with scales of 128 values stand for it, by the format's definition: 3 bits behind the leading one,
    exponents from -6 on, the largest value 448, ties to even."""
    out = torch.empty_like(x)
    for i in range(0, x.shape[1], 128):
        part = x[:, i:i + 128]
        amax = part.abs().amax(1, keepdim=True).clamp_min(1e-12)
        v = part * (448.0 / amax)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
        out[:, i:i + 128] = (torch.round(v / step) * step).clamp(-448.0, 448.0) * (amax / 448.0)
    return out


class _Keep(torch.autograd.Function):
    """f(x) whose derivative is taken where x is kept."""

    @staticmethod
    def forward(ctx, x, kept, f):
        ctx.f = f
        ctx.save_for_backward(kept)
        return f(x)

    @staticmethod
    def backward(ctx, go):
        kept, = ctx.saved_tensors
        with torch.enable_grad():
            kept = kept.detach().requires_grad_()
            return torch.autograd.grad(ctx.f(kept), kept, go)[0], None, None


def exact(case, seed):
    s = prepare(case, seed)
    kind, dtype = case["kind"], torch.float64
    x = s["x"].detach().to(dtype)
    if kind == "checkpoint":
        return _kept64(x)
    if kind == "act":
        x.requires_grad_()
        half = x.shape[1] // 2
        f = {"swiglu": lambda t: torch.sigmoid(t[:, :half]) * t[:, :half] * t[:, half:],
             "silu": lambda t: torch.sigmoid(t) * t,
             "gelu": lambda t: t * torch.special.ndtr(t),
             "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
        with torch.no_grad():
            kept = torch.cat([_kept64(x[:, :half]), _kept64(x[:, half:])], 1) if case["act"] == "swiglu" else _kept64(x)
        y = _Keep.apply(x, kept, f)
        dx, = torch.autograd.grad(y, x, s["grad"].to(dtype))
        return {"y": y.detach(), "dx": dx}
    if kind == "norm":
        w, b = s["weight"].detach().to(dtype), s["bias"].detach().to(dtype)
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        std = torch.sqrt(var + _EPS)
        hat = (x - mean) / std
        y = torch.addcmul(b, hat, w)
        if not case["train"]:
            return y
        go = s["grad"].to(dtype)
        if case["keep"]:
            hat = _kept64(hat)
        # the Jacobian of the normalisation: (I - 1 1^T / C - hat hat^T / C) / std
        u = go * w
        along = torch.stack([torch.ones_like(hat), hat], 1)                        # [R, 2, C]
        parts = (along * u.unsqueeze(1)).sum(2, keepdim=True) / x.shape[1]
        dx = (u - (parts * along).sum(1)) / std
        return {"y": y, "dx": dx, "dw": torch.sum(go * hat, 0), "db": torch.sum(go, 0)}
    w = s["weight"].detach().to(dtype)
    counted = (s["target"] != _IGNORED).nonzero().squeeze(1)
    label = s["target"][counted]
    if case["train"]:
        x.requires_grad_()
        w.requires_grad_()
    logp = torch.log_softmax(x[counted] @ w.t(), 1)
    rows = -(1.0 - case["smoothing"]) * logp[torch.arange(len(label), device=label.device), label]
    if case["smoothing"]:
        rows = rows - case["smoothing"] * logp.mean(1)
    if not case["train"]:
        return torch.zeros(len(s["target"]), dtype=dtype, device=x.device).index_copy(0, counted, rows)
    loss = rows.sum() / len(label) if len(label) else rows.sum() * math.nan
    dx, dw = torch.autograd.grad(loss, (x, w), s["scale"].to(dtype))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "loss":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        if not case["train"]:
            return {"bytes": 2 * (t + v) * h + 12 * t, "flops": 2 * t * h * v}
        # x, the weight and their gradients; the logits, and the two products of the gradients
        return {"bytes": 4 * (t + v) * h + 8 * t, "flops": 6 * t * h * v}
    n, e = case["rows"] * case["cols"], _BYTES[case["dtype"]]
    code = 1 + 4 / 128                       # a value kept in 8 bits with its share of a scale
    if kind == "norm":
        forward = 2 * e * n + 2 * e * case["cols"]
        if not case["train"]:
            return {"bytes": forward, "flops": 8 * n}
        # the backward reads the gradient and x (or what is kept of it) and writes x's gradient
        return {"bytes": forward + 2 * e * n + (2 * code if case["keep"] else e) * n + 3 * e * case["cols"], "flops": 20 * n}
    if kind == "act":
        out = n // 2 if case["act"] == "swiglu" else n
        return {"bytes": e * (n + out) + 2 * code * n + e * (n + out), "flops": 30 * n}
    return {"bytes": (2 * e + 2 * code) * n, "flops": 8 * n}
