"""What a transformer block needs beside its linears, as cases that can be timed and compared: the root-mean-square norm with the
residual's addition (its output in its own type, or already in the 8 bits that the next product reads), the linear in 8-bit integers with
a scale for each token and each channel, and the global norm of a step's gradients with their clipping.

Each case is one pass through one of the operators as a program calls it: forward alone where a model is served, forward and backward
where it is trained.  Widths are those of the repository's own configurations (hidden 7168, gate/up 36864, o_proj 16384) or generic ones;
`draw` gives further cases of the ranges that the listed ones stand for.

With `own` the operators are the framework's; without it their plain form, elementary torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6


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
        # the norm of a decode step, its output in the FP8 form that the next product reads: a launch's latency is what counts
        dict(name="norm_decode_fp8", kind="norm", rows=8, cols=7168, dtype="bf16", residual=True, out="fp8"),
        # the norm of a prefill of 4096 tokens in the same form
        dict(name="norm_prefill_fp8", kind="norm", rows=4096, cols=7168, dtype="bf16", residual=True, out="fp8"),
        # the norm with the residual stream in training: 4096 tokens, gradients of the stream and of the weight
        dict(name="norm_train", kind="norm", rows=4096, cols=7168, dtype="bf16", residual=True, out="train"),
        # a packed batch of variable-length sequences and a width that no vector divides, in half precision, no residual
        dict(name="norm_train_ragged", kind="norm", rows=1531, cols=1027, dtype="fp16", residual=False, out="train"),
        # a decode step of an MLP in 8-bit integers: residual, norm and quantization, then the gate/up product of 8 tokens
        dict(name="int8_decode", kind="int8", tokens=8, inputs=7168, outputs=36864, dtype="bf16", norm=True, bias=False, train=False),
        # a small head with a bias on a few tokens in single precision
        dict(name="int8_few", kind="int8", tokens=37, inputs=1024, outputs=1024, dtype="fp32", norm=False, bias=True, train=False),
        # adapters trained through a frozen 8-bit weight: forward and the input's gradient of a packed batch in half precision
        dict(name="int8_tune_ragged", kind="int8", tokens=1531, inputs=2048, outputs=5120, dtype="fp16", norm=False, bias=True, train=True),
        # the gate/up product of a prefill of 4096 tokens
        dict(name="int8_prefill", kind="int8", tokens=4096, inputs=7168, outputs=36864, dtype="bf16", norm=True, bias=False, train=False),
        # the gradients of a small layer, clipped: latency
        dict(name="clip_small", kind="grads", tensors=12, largest=65536, dtype="bf16", power="2", clip=True, over=True),
        # many ragged gradients of several types: the norm alone, as a rank computes it for its shards
        dict(name="norm_of_many", kind="grads", tensors=300, largest=1 << 22, dtype="mixed", power="2", clip=False, over=True),
        # ragged gradients in half precision under a bound on their largest value that holds: nothing has to change
        dict(name="clip_within_bound", kind="grads", tensors=40, largest=1 << 24, dtype="fp16", power="inf", clip=True, over=False),
        # a block with hidden 7168: fp32 main gradients of the gate/up, down and o_proj weights
        dict(name="clip_block", kind="grads", tensors=3, largest=36864 * 7168, dtype="fp32", power="2", clip=True, over=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, multiple=128):
    """A size spread over the logarithm of the range: half of the time a multiple of `multiple`, otherwise anything."""
    n = _log_int(rng, lo, hi)
    return max(multiple, n // multiple * multiple) if rng.random() < 0.5 else n


def _times128(rng, lo, hi):
    return max(1, _log_int(rng, lo, hi) // 128) * 128


def draw(rng):
    most = max(_seconds(c) for c in listed())
    while True:
        kind = rng.choice(["norm", "int8", "grads"])
        if kind == "norm":
            out = rng.choice(["train", "train", "fp8"])
            case = dict(kind=kind, rows=_size(rng, 1, 32768), cols=_times128(rng, 128, 16384) if out == "fp8" else _size(rng, 64, 16384),
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), residual=rng.random() < 0.7, out=out)
            if case["rows"] * case["cols"] > 16384 * 7168:
                continue
        elif kind == "int8":
            case = dict(kind=kind, tokens=_size(rng, 1, 8192, 64), inputs=_times128(rng, 128, 16384), outputs=_times128(rng, 128, 36864),
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), norm=rng.random() < 0.4, bias=rng.random() < 0.5, train=False)
            case["train"] = not case["norm"] and rng.random() < 0.5
            if case["norm"] and case["dtype"] == "fp32":      # (what the norm rounds away moves codes: an output in 32 bits shows it)
                continue
        else:
            clip = rng.random() < 0.7
            case = dict(kind=kind, tensors=_log_int(rng, 1, 400), largest=_log_int(rng, 1000, 1 << 26),
                        dtype=rng.choice(["bf16", "fp16", "fp32", "mixed"]), power=rng.choice(["2", "2", "2", "inf", "1"]), clip=clip,
                        over=rng.random() < 0.75)
        if _seconds(case) <= most:
            return case


def _seconds(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 2e15


def _gradient_sizes(case):
    """[(type, elements)] of a case's gradients: the first as large as any, the others spread over the logarithm."""
    if case["largest"] == 36864 * 7168:
        return [("fp32", 36864 * 7168), ("fp32", 7168 * 18432), ("fp32", 7168 * 16384)]
    rng = random.Random(case["tensors"] * 1000003 + case["largest"])
    kinds = ["bf16", "fp32", "fp16"] if case["dtype"] == "mixed" else [case["dtype"]]
    sizes = [case["largest"]] + [_log_int(rng, 1, case["largest"]) for _ in range(case["tensors"] - 1)]
    return [(kinds[i % len(kinds)], n) for i, n in enumerate(sizes)]


# ------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------
def _stream_values(g, rows, cols, dtype):
    """A residual stream: features of unequal size, some of them many times the others, off zero."""
    size = torch.exp(torch.randn((cols,), generator=g, device="cuda") * 0.7)
    shift = torch.randn((cols,), generator=g, device="cuda") * 0.3
    return (torch.randn((rows, cols), generator=g, device="cuda") * size + shift).to(dtype)


def _int8_weight(g, outputs, inputs):
    """(codes [outputs, inputs], scales [outputs]) of a weight whose channels differ in size."""
    size = 0.02 * torch.exp(torch.randn((outputs, 1), generator=g, device="cuda") * 0.3)
    w = torch.randn((outputs, inputs), generator=g, device="cuda").mul_(size)
    scale_inv = w.abs().amax(1) / 127.0
    return torch.round(w / scale_inv.unsqueeze(1)).clamp_(-127, 127).to(torch.int8), scale_inv


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = dict(case)
    if kind == "grads":
        sizes = _gradient_sizes(case)
        # gradients lie one behind the other in one buffer for each type, as a sharding program keeps them; a step's gradients
        # arrive there anew (from a reduction) before they are clipped
        arrived, buffers, parts = {}, {}, []
        for name in dict.fromkeys(name for name, _ in sizes):
            total = sum(n for other, n in sizes if other == name)
            heavy = torch.randn((total,), generator=g, device="cuda")
            arrived[name] = heavy.mul_(1e-3 if name != "fp16" else 1e-2).to(_DTYPES[name])
            buffers[name] = arrived[name].clone()
        at = dict.fromkeys(arrived, 0)
        params = []
        for name, n in sizes:
            part = buffers[name][at[name]:at[name] + n]
            at[name] += n
            parts.append(part)
            if name == "fp32":                           # (an fp32 main gradient beside a 16-bit parameter)
                p = torch.nn.Parameter(torch.empty((1,), dtype=torch.bfloat16, device="cuda").expand(n))
                p.main_grad = part
            else:
                p = torch.nn.Parameter(torch.empty((1,), dtype=_DTYPES[name], device="cuda").expand(n))
                p.grad = part
            params.append(p)
        total = sum(n for _, n in sizes)
        expected = {"2": 1e-3 * math.sqrt(total), "1": 1e-3 * total, "inf": 1e-3}[case["power"]]
        state.update(arrived=arrived, buffers=buffers, parts=parts, params=params, max_norm=expected * (0.3 if case["over"] else 300.0))
        return state
    dtype = _DTYPES[case["dtype"]]
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        state["x"] = _stream_values(g, rows, cols, dtype)
        state["residual_stream"] = _stream_values(g, rows, cols, dtype) if case["residual"] else None
        state["weight"] = (1.0 + 0.1 * torch.randn((cols,), generator=g, device="cuda")).to(dtype)
        if case["out"] == "train":
            for t in (state["x"], state["residual_stream"], state["weight"]):
                if t is not None:
                    t.requires_grad_()
            state["grad"] = torch.randn((rows, cols), generator=g, device="cuda").to(dtype)
            if case["residual"]:
                state["grad_stream"] = torch.randn((rows, cols), generator=g, device="cuda").to(dtype)
        return state
    tokens, inputs, outputs = case["tokens"], case["inputs"], case["outputs"]
    state["x"] = _stream_values(g, tokens, inputs, dtype)
    if case["norm"]:
        state["residual_stream"] = _stream_values(g, tokens, inputs, dtype)
        state["weight"] = (1.0 + 0.1 * torch.randn((inputs,), generator=g, device="cuda")).to(dtype)
    codes, scale_inv = _int8_weight(g, outputs, inputs)
    state.update(codes=codes, scale_inv=scale_inv, codes_t=codes.t().contiguous() if case["train"] else None)
    state["bias_of"] = (0.1 * torch.randn((outputs,), generator=g, device="cuda")).to(dtype) if case["bias"] else None
    if case["train"]:
        state["x"].requires_grad_()
        state["grad"] = (1e-3 * torch.randn((tokens, outputs), generator=g, device="cuda")).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _arrive(s):
    for name, buffer in s["buffers"].items():
        buffer.copy_(s["arrived"][name])


def _own(s):
    hpfp8 = _hpfp8()
    kind = s["kind"]
    if kind == "grads":
        power = float(s["power"])
        if not s["clip"]:
            return hpfp8.get_total_norm(s["parts"], power)
        _arrive(s)
        norm = hpfp8.clip_grad_norm_(s["params"], s["max_norm"], power)
        return {"norm": norm, "grads": s["buffers"]}
    if kind == "norm":
        x, residual, weight = s["x"], s["residual_stream"], s["weight"]
        if s["out"] == "fp8":
            out = hpfp8.rms_norm_quantize_1x128(x, weight, _EPS, residual=residual)
            # (what the codes stand for, with the scales row by row)
            return {"y": hpfp8.dequantize_1x128(out[0], out[1].contiguous()), "sum": out[2] if s["residual"] else None}
        if not s["residual"]:
            y = hpfp8.rms_norm(x, (s["cols"],), weight, _EPS)
            dx, dw = torch.autograd.grad(y, (x, weight), s["grad"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        y, total = hpfp8.rms_norm(x, (s["cols"],), weight, _EPS, residual=residual)
        dx, dr, dw = torch.autograd.grad((y, total), (x, residual, weight), (s["grad"], s["grad_stream"]))
        return {"y": y.detach(), "sum": total.detach(), "dx": dx, "dr": dr, "dw": dw}
    w8 = hpfp8.Int8Weight(s["codes"], s["scale_inv"], s["codes_t"])
    if s["norm"]:
        codes, scale_inv, total = hpfp8.rms_norm_quantize_int8(s["x"], s["weight"], _EPS, residual=s["residual_stream"])
        return {"y": hpfp8.gemm_int8(codes, scale_inv, w8.codes, w8.scale_inv, bias=s["bias_of"], out_dtype=s["x"].dtype), "sum": total}
    y = hpfp8.int8_linear(s["x"], w8, s["bias_of"])
    if not s["train"]:
        return {"y": y}
    dx, = torch.autograd.grad(y, (s["x"],), s["grad"])
    return {"y": y.detach(), "dx": dx}


def _divided(x, amax, most):
    """(x scaled to the codes' range, what a code stands for): two divisions of tensors, not products with reciprocals."""
    amax = amax.clamp_min(1e-12)
    most = torch.full_like(amax, most)
    return x * (most / amax), amax / most


def _int8_rows(x):
    """(codes, scales) of the rows of x, in 32 bits."""
    scaled, scale_inv = _divided(x, x.abs().amax(1, keepdim=True), 127.0)
    return torch.round(scaled), scale_inv


def _normed(s):
    """(y in 32 bits, the sum of both streams, its 32-bit values, the rows' factors)"""
    x = s["x"].detach()
    total = x if s.get("residual_stream") is None else (x.float() + s["residual_stream"].detach().float()).to(x.dtype)
    tf = total.float()
    r = 1.0 / torch.sqrt((tf * tf).mean(-1, keepdim=True) + _EPS)
    return tf * r * s["weight"].detach().float(), total, tf, r


def _plain(s):
    kind = s["kind"]
    if kind == "grads":
        if s["clip"]:
            _arrive(s)
        parts = [b.float() for b in s["buffers"].values()]
        if s["power"] == "inf":
            norm = torch.stack([p.abs().amax() for p in parts]).amax()
        elif s["power"] == "1":
            norm = torch.stack([p.abs().sum(dtype=torch.float64) for p in parts]).sum().float()
        else:
            norm = torch.sqrt(torch.stack([(p * p).sum(dtype=torch.float64) for p in parts]).sum()).float()
        if not s["clip"]:
            return norm
        factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        for b, p in zip(s["buffers"].values(), parts):
            b.copy_(p * factor)
        return {"norm": norm, "grads": s["buffers"]}
    x = s["x"].detach()
    dtype = x.dtype
    if kind == "norm":
        y, total, tf, r = _normed(s)
        if s["out"] == "fp8":
            groups = y.view(s["rows"], -1, 128)
            scaled, scale_inv = _divided(groups, groups.abs().amax(-1, keepdim=True), 448.0)
            codes = scaled.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            return {"y": (codes.float() * scale_inv).view(y.shape).to(torch.bfloat16), "sum": total if s["residual"] else None}
        go = s["grad"].float()
        hat, u = tf * r, go * s["weight"].detach().float()
        dx = r * (u - hat * (u * hat).mean(-1, keepdim=True))
        dw = (go * hat).sum(0).to(dtype)
        if not s["residual"]:
            return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw}
        dx = (dx + s["grad_stream"].float()).to(dtype)
        return {"y": y.to(dtype), "sum": total, "dx": dx, "dr": dx, "dw": dw}
    w = s["codes"].float()
    out = {}
    if s["norm"]:
        values, out["sum"], _, _ = _normed(s)
    else:
        values = x.float()
    codes, scale_inv = _int8_rows(values)
    y = torch.matmul(codes, w.t()) * scale_inv * s["scale_inv"]
    if s["bias"]:
        y = y + s["bias_of"].float()
    out["y"] = y.to(dtype)
    if s["train"]:
        codes, scale_inv = _int8_rows(s["grad"].float() * s["scale_inv"])
        out["dx"] = (torch.matmul(codes, w) * scale_inv).to(dtype)
    return out


# ------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------
def _e4m3_64(x):
    """x[R, C] (64 bits) as E4M3 codes with a scale for 128 values of a row stand for it, by the format's definition: 3 bits behind the
    leading one, exponents from -6 on, the largest value 448, ties to even."""
    v = x.reshape(x.shape[0], -1, 128)
    amax = v.abs().amax(2, keepdim=True).clamp_min(1e-12)
    v = v * (448.0 / amax)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    return ((torch.round(v / step) * step).clamp(-448.0, 448.0) * (amax / 448.0)).reshape(x.shape)


def _int8_64(x):
    """The values (64 bits) that the rows of x are kept as in 8-bit integers.  A code is defined by steps that are rounded to 32 bits each,
    the row's value itself, 127 over the row's largest one, and the product of the two: the nearest integer to that."""
    def rounded(t):
        return t.float().double()
    x = rounded(x)
    largest = torch.max(x.abs(), 1, keepdim=True).values
    largest = torch.where(largest < rounded(torch.tensor(1e-12, dtype=x.dtype)), rounded(torch.tensor(1e-12, dtype=x.dtype)), largest)
    return torch.round(rounded(x * rounded(127.0 / largest))) * (largest / 127.0)


def exact(case, seed):
    s = prepare(case, seed)
    kind, double = case["kind"], torch.float64
    if kind == "grads":
        flat = {name: b.to(double) for name, b in s["arrived"].items()}
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(b, float(s["power"])) for b in flat.values()]), float(s["power"]))
        if not case["clip"]:
            return norm
        by = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": {name: b * by for name, b in flat.items()}}
    x = s["x"].detach().to(double)
    if kind == "norm" or case["norm"]:
        total = x
        if s["residual_stream"] is not None:             # (the stream is kept in its own type: the norm is that of the rounded sum)
            total = (x + s["residual_stream"].detach().to(double)).to(s["x"].dtype).to(double)
        w = s["weight"].detach().to(double)
        rms = torch.sqrt(torch.mean(torch.square(total), 1, keepdim=True) + _EPS)
    if kind == "norm":
        y = total / rms * w
        after = total if case["residual"] else None
        if case["out"] == "fp8":
            return {"y": _e4m3_64(y), "sum": after}
        # the Jacobian of the normalisation: (I - hat hat^T / C) / rms
        go = s["grad"].to(double)
        hat = total / rms
        u = go * w
        dx = (u - hat * ((u.unsqueeze(1) @ hat.unsqueeze(2)).squeeze(2) / x.shape[1])) / rms
        dw = torch.sum(go * hat, 0)
        if not case["residual"]:
            return {"y": y, "dx": dx, "dw": dw}
        dx = dx + s["grad_stream"].to(double)
        return {"y": y, "sum": after, "dx": dx, "dr": dx, "dw": dw}
    weight = s["codes"].to(double) * s["scale_inv"].to(double).unsqueeze(1)
    out = {}
    if case["norm"]:
        x, out["sum"] = total / rms * w, total
    y = _int8_64(x) @ weight.t()
    if case["bias"]:
        y += s["bias_of"].to(double)
    out["y"] = y
    if case["train"]:
        go = s["grad"].to(double) * s["scale_inv"].to(double)
        out["dx"] = _int8_64(go) @ s["codes"].to(double)
    return out


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "grads":
        sizes = _gradient_sizes(case)
        n, held = sum(k for _, k in sizes), sum(k * _BYTES[name] for name, k in sizes)
        # read for the norm; where they are clipped, the arriving gradients read and written, and if the bound is passed read and
        # written once more
        return {"bytes": held * (1 if not case["clip"] else 5 if case["over"] else 3), "flops": 2 * n}
    e = _BYTES[case["dtype"]]
    code = 1 + 4 / 128                       # a value in 8 bits with its share of a scale
    if kind == "norm":
        n = case["rows"] * case["cols"]
        streams = 3 if case["residual"] else 1           # x; with a residual that too, and the sum written
        if case["out"] == "fp8":                         # (the codes are read again, and the values that they stand for written)
            return {"bytes": (streams * e + 2 * code + 2) * n + e * case["cols"], "flops": 8 * n}
        backward = 4 if case["residual"] else 3          # both gradients, the sum, and the gradient of both streams
        return {"bytes": (streams + 1 + backward) * e * n + 3 * e * case["cols"], "flops": 16 * n}
    t, k, n = case["tokens"], case["inputs"], case["outputs"]
    w = n * k
    if case["train"]:
        return {"bytes": 2 * w + 2 * e * t * (k + n) + 8 * n, "flops": 4 * t * w}
    return {"bytes": w + e * t * ((3 if case["norm"] else 1) * k + n) + 4 * n, "flops": 2 * t * w}
