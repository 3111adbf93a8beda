"""What the layers behind the encoding cost, as measurable cases.

Four operators of ``permutohedral_encoding_amd.layers``, each in the uses that a training or rendering program makes of it:

  checkpoint     a tensor kept in 8 bits between forward and backward: written, and read back
  weight_grad    a linear layer's weight and bias gradient from its kept input
  activation     an activation, or a gated pair, and its gradient from the kept input
  residual_norm  y = s x + gate * norm(f), n = norm(y): what stands between a block and the next one, and all its gradients

A checkpoint has blocks of 32 channels of one row (the halves of a gated pair have one each).  A block's
largest magnitude a sets the exponent e, the least integer of at
least -126 with a / 2^e < 127.5; a value is kept as the integer next to x / 2^e, ties to even.  Every backward pass is
the gradient of the operator at the values that the checkpoint stands for.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32


def _case(**given):
    case = {"op": "residual_norm", "rows": 1 << 20, "channels": 64, "dtype": "fp32",
            "layout": "rows",      # "rows"; "levels": the encoding's own result, features first; "slice": the first channels of wider rows
            "outputs": 64,         # weight_grad: columns of the upstream gradient
            "kind": "rms",         # residual_norm: "rms" or "layer"; activation: "gelu", "silu" or "softplus"
            "gated": False,        # activation: act(a) * b of [a | b]
            "rows_per_gate": 0,    # residual_norm: 0: one gate for all rows, else this many consecutive rows (the samples of a ray) share one
            "params": "fp32",      # residual_norm: type of weights, biases and gate
            "train": True}
    assert set(given) <= set(case) | {"name"}
    case.update(given)
    return case


def listed():
    return [
        # the encoding of a toy batch, 16 levels of two features, as the encoding hands it out
        _case(name="checkpoint_4k", op="checkpoint", rows=4097, channels=32, layout="levels"),
        # the headline batch: 2^20 points, 24 levels
        _case(name="checkpoint_1m", op="checkpoint", rows=1 << 20, channels=48, layout="levels"),
        # hidden activations of a wide decoder
        _case(name="checkpoint_wide", op="checkpoint", rows=1 << 16, channels=1024, dtype="bf16"),
        # the first layer of a small decoder, a toy batch
        _case(name="weight_grad_4k", op="weight_grad", rows=4097, channels=32),
        # the same on the headline batch
        _case(name="weight_grad_1m", op="weight_grad", rows=1 << 20, channels=48),
        # a layer of a wide decoder or of a token mixer
        _case(name="weight_grad_wide", op="weight_grad", rows=1 << 14, channels=1024, outputs=4096, dtype="bf16"),
        # a hidden layer in rendering: no gradient, a few probes
        _case(name="activation_1k", op="activation", rows=1000, kind="softplus", train=False),
        # a gated hidden layer of a wide decoder
        _case(name="activation_gated", op="activation", rows=(1 << 15) - 3, channels=2048, kind="silu", gated=True, dtype="bf16"),
        # one row in rendering: what a call costs
        _case(name="norm_one", rows=1, channels=1024, dtype="bf16", train=False),
        # a decoder block on the headline batch
        _case(name="norm_1m"),
        # conditioned per ray: every ray has its gate; channels that no vector divides
        _case(name="norm_rays", rows=1023 * 128, channels=203, dtype="fp16", kind="layer", rows_per_gate=128),
        # a block of a wide decoder
        _case(name="norm_wide", rows=1 << 14, channels=4096, dtype="bf16", params="bf16"),
    ]


def draw(rng):
    bounds = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        op = rng.choice(["checkpoint", "weight_grad", "activation", "residual_norm", "residual_norm"])
        rows = int(2 ** rng.uniform(0, 20))
        channels = int(2 ** rng.uniform(3, 13))
        if rng.random() < 0.4:
            channels = 1 << round(math.log2(channels))
        elif rng.random() < 0.5:
            channels = max(8, channels // 8 * 8)
        case = _case(op=op, rows=rows, channels=channels, dtype=rng.choice(["fp32", "fp16", "bf16", "bf16"]))
        if op == "checkpoint":
            case["layout"] = rng.choice(["rows", "rows", "slice", "levels"])
        elif op == "weight_grad":
            case["layout"] = rng.choice(["rows", "rows", "slice"])
            case["outputs"] = int(2 ** rng.uniform(0, 12))
        elif op == "activation":
            case.update(kind=rng.choice(["gelu", "silu", "softplus"]), gated=rng.random() < 0.5, train=rng.random() < 0.8)
        else:
            case.update(kind=rng.choice(["rms", "layer"]), params=rng.choice(["fp32", case["dtype"]]), train=rng.random() < 0.8)
            if rng.random() < 0.4:
                case["rows_per_gate"] = rng.choice([1, 2, 7, 64, 128, 1000])
                case["rows"] = -(-rows // case["rows_per_gate"]) * case["rows_per_gate"]
        cost = work(case)
        if cost["bytes"] <= bounds[0] and cost["flops"] <= bounds[1]:
            return case


def _values(shape, generator):
    """Activations: channels of different sizes, and a value in a thousand far out."""
    rows, channels = shape
    kw = dict(generator=generator, device="cuda")
    x = torch.randn(shape, **kw) * torch.exp(0.5 * torch.randn((1, channels), **kw))
    x += (torch.rand(shape, **kw) < 1e-3) * 20.0 * torch.randn((rows, 1), **kw)
    return x


def _laid_out(x, case):
    x = x.to(TYPES[case["dtype"]])
    if case["layout"] == "levels":
        return torch.empty_strided(x.shape, (1, x.shape[0]), dtype=x.dtype, device=x.device).copy_(x)
    if case["layout"] == "slice":
        wide = torch.zeros((x.shape[0], x.shape[1] + 16), dtype=x.dtype, device=x.device)
        wide[:, : x.shape[1]] = x
        return wide[:, : x.shape[1]]
    return x.contiguous()


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    kw = dict(generator=generator, device="cuda")
    rows, channels, dtype = case["rows"], case["channels"], TYPES[case["dtype"]]
    state = {k: case[k] for k in ("op", "kind", "gated", "train", "rows_per_gate")}
    width = 2 * channels if case["op"] == "activation" and case["gated"] else channels
    state["x"] = _laid_out(_values((rows, width), generator), case)
    if case["op"] == "weight_grad":
        # the gradient of a loss that is a mean over the rows
        state["grad"] = (torch.randn((rows, case["outputs"]), **kw) / math.sqrt(rows)).to(dtype)
    elif case["op"] == "activation":
        state["grad"] = torch.randn((rows, channels), **kw).to(dtype)
    elif case["op"] == "residual_norm":
        params = TYPES[case["params"]]
        state["branch"] = _laid_out(_values((rows, channels), generator), case)
        groups = rows // case["rows_per_gate"] if case["rows_per_gate"] else 0
        state["gate"] = (0.3 + 0.1 * torch.randn((groups, channels) if groups else (channels,), **kw)).to(params)
        for name in ("post_weight", "pre_weight"):
            state[name] = (1.0 + 0.1 * torch.randn((channels,), **kw)).to(params)
        for name in ("post_bias", "pre_bias"):
            state[name] = (0.1 * torch.randn((channels,), **kw)).to(params) if case["kind"] == "layer" else None
        state["scale"], state["eps"] = 0.75, 1e-6
        state["grad_y"] = torch.randn((rows, channels), **kw).to(dtype)
        state["grad_n"] = torch.randn((rows, channels), **kw).to(dtype)
    if case["op"] in ("activation", "residual_norm") and case["train"]:
        for name in ("x", "branch", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"):
            if state.get(name) is not None:
                state[name].requires_grad_(True)
    return state


def run(state):
    if own:
        return _OWN[state["op"]](state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------------ the framework's calls

def _own_checkpoint(s):
    from permutohedral_encoding_amd import layers
    return {"values": layers.checkpoint(s["x"]).unpack()}


def _own_weight_grad(s):
    from permutohedral_encoding_amd import layers
    weight, bias = layers.checkpoint(s["x"]).weight_grad(s["grad"], bias=True)
    return {"weight": weight, "bias": bias}


def _own_activation(s):
    from permutohedral_encoding_amd import layers
    y = layers.activation(s["x"], s["kind"], gated=s["gated"])
    if not s["train"]:
        return {"y": y}
    dx, = torch.autograd.grad(y, s["x"], s["grad"])
    return {"y": y.detach(), "dx": dx}


def _own_residual_norm(s):
    from permutohedral_encoding_amd import layers
    gate = s["gate"]
    y, n = layers.residual_norm(s["x"], s["branch"], gate=gate, residual_scale=s["scale"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                                pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], kind=s["kind"], eps=s["eps"])
    out = {"y": y.detach(), "n": n.detach()}
    if s["train"]:
        names = [k for k in ("x", "branch", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[k] is not None]
        grads = torch.autograd.grad((y, n), [s[k] for k in names], (s["grad_y"], s["grad_n"]))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


_OWN = {"checkpoint": _own_checkpoint, "weight_grad": _own_weight_grad, "activation": _own_activation, "residual_norm": _own_residual_norm}


# ------------------------------------------------------------------------------------------ the plain forms

def _kept(x):
    """The values that the checkpoint of x stands for, in 32 bits."""
    x = x.float()
    rows, channels = x.shape
    blocks = torch.nn.functional.pad(x, (0, -channels % BLOCK)).view(rows, -1, BLOCK)
    largest = blocks.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(largest)  # largest = mantissa * 2^exponent, mantissa in [0.5, 1): 128 * mantissa has to stay under 127.5
    e = (exponent - 7 + (mantissa >= 127.5 / 128).to(exponent.dtype)).clamp(min=-126)
    step, per_step = ((e + 127) << 23).view(torch.float32), ((127 - e) << 23).view(torch.float32)  # 2^e and 2^-e
    kept = torch.round(blocks * per_step) * step
    return kept.view(rows, -1)[:, :channels]


def _plain_checkpoint(s):
    return {"values": _kept(s["x"]).to(s["x"].dtype)}


def _plain_weight_grad(s):
    dtype, grad, x = s["grad"].dtype, s["grad"].float(), _kept(s["x"])
    bias = grad.sum(0, dtype=torch.float64)
    # sums over a million rows: in 32 bits over 8192 of them, in 64 over those
    if grad.shape[0] > 8192:
        grad, x = (torch.nn.functional.pad(v, (0, 0, 0, -v.shape[0] % 8192)).view(-1, 8192, v.shape[1]) for v in (grad, x))
        weight = (grad.transpose(1, 2) @ x).sum(0, dtype=torch.float64)
    else:
        weight = grad.t() @ x
    return {"weight": weight.to(dtype), "bias": bias.to(dtype)}


def _act(x, kind):
    if kind == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    if kind == "silu":
        return x / (1.0 + torch.exp(-x))
    return x.clamp(min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _act_slope(x, kind):
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * math.sqrt(0.5 / math.pi)
    s = 1.0 / (1.0 + torch.exp(-x))
    return s * (1.0 + x * (1.0 - s)) if kind == "silu" else s


def _plain_activation(s):
    dtype, kind = s["x"].dtype, s["kind"]
    x = s["x"].float()
    half = x.shape[1] // 2
    y = _act(x[:, :half], kind) * x[:, half:] if s["gated"] else _act(x, kind)
    if not s["train"]:
        return {"y": y.to(dtype)}
    grad = s["grad"].float()
    if s["gated"]:  # (a checkpoint of its own for each half)
        a, b = _kept(s["x"][:, :half]), _kept(s["x"][:, half:])
        dx = torch.cat([grad * b * _act_slope(a, kind), grad * _act(a, kind)], 1)
    else:
        dx = grad * _act_slope(_kept(s["x"]), kind)
    return {"y": y.to(dtype), "dx": dx.to(dtype)}


def _normed(v, kind, eps):
    """The normed rows without weight, and the factor they were scaled by."""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    factor = torch.rsqrt((v * v).mean(1, keepdim=True) + eps)
    return v * factor, factor


def _norm_backward(d, normed, factor, kind):
    d = d - normed * (d * normed).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if kind == "layer" else 0.0)
    return d * factor


def _plain_residual_norm(s):
    dtype, kind, eps = s["x"].dtype, s["kind"], s["eps"]
    p = {k: s[k].float() if s[k] is not None else None for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias")}
    gate = p["gate"].repeat_interleave(s["rows_per_gate"], 0) if s["rows_per_gate"] else p["gate"]

    def streams(x, f):
        f_normed, f_factor = _normed(f, kind, eps)
        inner = f_normed * p["post_weight"] + (p["post_bias"] if p["post_bias"] is not None else 0.0)
        y = s["scale"] * x + gate * inner
        return f_normed, f_factor, inner, y, *_normed(y, kind, eps)

    *_, y, y_normed, _ = streams(s["x"].float(), s["branch"].float())
    n = y_normed * p["pre_weight"] + (p["pre_bias"] if p["pre_bias"] is not None else 0.0)
    out = {"y": y.to(dtype), "n": n.to(dtype)}
    if not s["train"]:
        return out
    f_normed, f_factor, inner, _, y_normed, y_factor = streams(_kept(s["x"]), _kept(s["branch"]))
    dn = s["grad_n"].float()
    dy = s["grad_y"].float() + _norm_backward(dn * p["pre_weight"], y_normed, y_factor, kind)
    d_inner = dy * gate
    sums = {"pre_weight": dn * y_normed, "pre_bias": dn, "post_weight": d_inner * f_normed, "post_bias": d_inner}
    out.update(dx=(s["scale"] * dy).to(dtype), dbranch=_norm_backward(d_inner * p["post_weight"], f_normed, f_factor, kind).to(dtype))
    out.update({"d" + k: v.sum(0, dtype=torch.float64).to(s[k].dtype) for k, v in sums.items() if s[k] is not None})
    d_gate = dy * inner
    if s["rows_per_gate"]:
        d_gate = d_gate.view(-1, s["rows_per_gate"], d_gate.shape[1])
        out["dgate"] = d_gate.sum(1, dtype=torch.float64).to(s["gate"].dtype)
    else:
        out["dgate"] = d_gate.sum(0, dtype=torch.float64).to(s["gate"].dtype)
    return out


_PLAIN = {"checkpoint": _plain_checkpoint, "weight_grad": _plain_weight_grad, "activation": _plain_activation, "residual_norm": _plain_residual_norm}


# ------------------------------------------------------------------------------------------ the definition in 64 bits

def _kept64(x):
    x = x.detach().double()
    out = torch.empty_like(x)
    for first in range(0, x.shape[1], BLOCK):
        block = x[:, first:first + BLOCK]
        a = block.abs().max(1, keepdim=True).values
        e = torch.floor(torch.log2(a.clamp(min=2.0 ** -140))) - 7.0  # never too large; the next two steps are the definition
        for _ in range(2):
            e = torch.where(a * torch.exp2(-e) < 127.5, e, e + 1.0)
        e = e.clamp(min=-126.0)
        out[:, first:first + BLOCK] = torch.round(block * torch.exp2(-e)) * torch.exp2(e)
    return out


def _act64(x, kind):
    if kind == "gelu":
        return x * torch.special.ndtr(x)
    return x * torch.sigmoid(x) if kind == "silu" else torch.logaddexp(x, torch.zeros_like(x))


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "checkpoint":
        return {"values": _kept64(s["x"])}
    if s["op"] == "weight_grad":
        grad = s["grad"].double()
        return {"weight": grad.t().contiguous() @ _kept64(s["x"]), "bias": grad.sum(0)}
    names = [k for k in ("x", "branch", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s.get(k) is not None]
    at = {k: s[k].detach().double() for k in names}

    def activation(x):
        a, b = x.chunk(2, 1) if s["gated"] else (x, 1.0)
        return _act64(a, s["kind"]) * b,

    def norm(v, weight, bias):
        if s["kind"] == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt(v.square().mean(1, keepdim=True) + s["eps"]) * weight
        return v if bias is None else v + bias

    def residual_norm(x, branch, gate, post_weight, pre_weight, post_bias=None, pre_bias=None):
        p = norm(branch, post_weight, post_bias)
        if s["rows_per_gate"]:
            y = s["scale"] * x + (p.view(gate.shape[0], -1, gate.shape[1]) * gate[:, None]).view(p.shape)
        else:
            y = s["scale"] * x + gate * p
        return y, norm(y, pre_weight, pre_bias)

    f = activation if s["op"] == "activation" else residual_norm
    out = dict(zip(("y", "n"), f(**at)))
    if s["train"]:
        for k in ("x", "branch"):
            if k in at:
                at[k] = torch.cat([_kept64(v) for v in s[k].chunk(2, 1)], 1) if s["gated"] else _kept64(s[k])
        at = {k: v.requires_grad_(True) for k, v in at.items()}
        upstream = [s["grad"].double()] if s["op"] == "activation" else [s["grad_y"].double(), s["grad_n"].double()]
        grads = torch.autograd.grad(f(**at), list(at.values()), upstream)
        out.update({"d" + k: g for k, g in zip(at, grads)})
    return out


def work(case):
    """Bytes: every input and result once, and what is kept in 8 bits written once and read once; operations of the products and, per value, of the rest."""
    rows, channels, t = case["rows"], case["channels"], 2 if case["dtype"] != "fp32" else 4
    if case["op"] == "checkpoint":
        kept = rows * (channels + -(-channels // BLOCK))
        return {"bytes": 2 * t * rows * channels + 2 * kept, "flops": 4 * rows * channels}
    if case["op"] == "weight_grad":
        o = case["outputs"]
        kept = rows * (channels + -(-channels // BLOCK))
        return {"bytes": t * (rows * (channels + o) + o * (channels + 1)) + 2 * kept, "flops": rows * o * (2 * channels + 1)}
    if case["op"] == "activation":
        width = 2 * channels if case["gated"] else channels
        nbytes, flops = t * rows * (width + channels), 12 * rows * channels
        if case["train"]:
            nbytes += t * rows * (width + channels) + 2 * rows * (width + -(-width // BLOCK))
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    nbytes, flops = 4 * t * rows * channels, 12 * rows * channels
    if case["train"]:
        nbytes += 4 * t * rows * channels + 4 * rows * (channels + -(-channels // BLOCK))
        flops *= 4
    if case["rows_per_gate"]:
        nbytes += (4 if case["params"] == "fp32" else 2) * rows // case["rows_per_gate"] * channels * (3 if case["train"] else 1)
    return {"bytes": nbytes, "flops": flops}
