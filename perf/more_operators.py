"""What a decoder of experts costs, and the optimiser's step on its stacked weights, as measurable cases.

Four operators, each in the uses that a training or rendering program makes of it:

  route          a point's experts: the largest of its logits, their weights, where each choice stands when choices are sorted by expert, and the gradient
  experts_sort   rows sorted by expert and brought back as weighted sums, with all gradients
  expert_linear  a linear layer of each expert on its own rows, with all gradients
  orthogonalise  the nearly orthogonal matrix that Newton-Schulz products make of an update

Choices are numbered row by row; those of one expert stand in that order, and choices without an expert (-1) behind those of all experts, where rows are zero.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5


def _case(**given):
    case = {"op": "expert_linear",
            "rows": 1 << 20,       # points; expert_linear: rows that are sorted already; orthogonalise: rows of a matrix
            "experts": 8,          # orthogonalise: matrices
            "choices": 2,          # experts of a point
            "channels": 64, "outputs": 64, "dtype": "fp32",
            "normalise": True,     # route: weights add up to one over the chosen, else they are shares of all experts
            "masked": 0.0,         # this part of the logits is -inf, and this part of the rows has no expert at all
            "train": True}
    assert set(given) <= set(case) | {"name"}
    case.update(given)
    return case


def listed():
    return [
        # a toy batch and a few experts
        _case(name="route_4k", op="route", rows=4097),
        # the headline batch: 2^20 points, one of many experts closed in places
        _case(name="route_1m", op="route", experts=64, masked=0.02),
        # one point in rendering: what the calls cost
        _case(name="sort_one", op="experts_sort", rows=1, experts=64, channels=1024, dtype="bf16", train=False),
        # hidden rows of a small decoder on the headline batch
        _case(name="sort_1m", op="experts_sort"),
        # hidden rows of a wide decoder, the batch padded
        _case(name="sort_wide", op="experts_sort", rows=(1 << 14) - 3, experts=64, channels=2048, dtype="bf16", masked=0.02),
        # a handful of points in rendering: what counts is reading the experts' weights
        _case(name="experts_few", rows=10, experts=64, channels=1024, outputs=4096, dtype="bf16", train=False),
        # a hidden layer of a small decoder on the headline batch
        _case(name="experts_1m"),
        # channels and outputs that no tile divides
        _case(name="experts_odd", rows=70001, experts=13, channels=203, outputs=130, dtype="fp16", masked=0.02),
        # a layer of a wide decoder
        _case(name="experts_wide", rows=1 << 15, experts=16, channels=1024, outputs=4096, dtype="bf16"),
        # a layer of a small decoder of 16 experts: all of it one call
        _case(name="orthogonal_small", op="orthogonalise", rows=256, experts=16, channels=64),
        # a single matrix of odd sizes
        _case(name="orthogonal_odd", op="orthogonalise", rows=1000, experts=1, channels=203, dtype="fp16"),
        # a layer of a wide decoder of 16 experts
        _case(name="orthogonal_wide", op="orthogonalise", rows=4096, experts=16, channels=1024, dtype="bf16"),
    ]


def draw(rng):
    bounds = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]

    def size(low, high):
        n = int(2 ** rng.uniform(low, high))
        if rng.random() < 0.4:
            return 1 << round(math.log2(n))
        return max(8, n // 8 * 8) if n >= 16 and rng.random() < 0.5 else n

    while True:
        case = _case(op=rng.choice(["route", "experts_sort", "expert_linear", "expert_linear", "orthogonalise", "orthogonalise"]),
                     dtype=rng.choice(["fp32", "fp16", "bf16", "bf16"]), rows=int(2 ** rng.uniform(0, 20)), experts=int(2 ** rng.uniform(1, 7)),
                     choices=rng.choice([1, 2, 2, 3, 4, 8]), train=rng.random() < 0.8, masked=rng.choice([0.0, 0.02, 0.2]))
        if case["op"] == "route":
            case.update(experts=int(2 ** rng.uniform(1, 10)), normalise=rng.random() < 0.6)
        elif case["op"] == "experts_sort":
            case["channels"] = size(2, 12)
        elif case["op"] == "expert_linear":
            case.update(channels=size(3, 12), outputs=size(0, 12))
        else:
            case.update(rows=size(2, 12), channels=size(2, 12), experts=int(2 ** rng.uniform(0, 6)), masked=0.0, train=False)
        case["choices"] = min(case["choices"], case["experts"])
        cost = work(case)
        if cost["bytes"] <= bounds[0] and cost["flops"] <= bounds[1]:
            return case


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    kw = dict(generator=generator, device="cuda")
    rows, number, choices, dtype = case["rows"], case["experts"], case["choices"], TYPES[case["dtype"]]
    state = {k: case[k] for k in ("op", "experts", "choices", "normalise", "train")}
    if case["op"] == "orthogonalise":
        # an update: its channels differ in size, and a few directions carry much of it
        rank = min(4, rows, case["channels"])
        wide = torch.randn((number, rows, case["channels"]), **kw) * torch.exp(0.5 * torch.randn((number, 1, case["channels"]), **kw))
        state["update"] = (1e-3 * (wide + torch.randn((number, rows, rank), **kw) @ torch.randn((number, rank, case["channels"]), **kw))).to(dtype)
        return state
    if case["op"] == "expert_linear":
        choices, shape = 1, (rows, 1)
    else:
        shape = (rows, choices)
    # experts in uneven demand
    logits = torch.randn((rows, number), **kw) + 0.7 * torch.randn((1, number), **kw)
    closed = torch.rand((rows, number), **kw) < case["masked"]
    logits.masked_fill_(closed | (torch.rand((rows, 1), **kw) < case["masked"]), -math.inf)
    if case["op"] == "route":
        state["logits"] = logits.to(dtype)
        state["grad_weights"] = torch.randn(shape, **kw)
        if case["train"]:
            state["logits"].requires_grad_(True)
        return state
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    chosen = torch.where(order.values[:, :choices] == -math.inf, -1, order.indices[:, :choices])
    if case["op"] == "experts_sort":
        state["chosen"] = chosen
        state["weights"] = torch.rand(shape, **kw)
        state["x"] = torch.randn((rows, case["channels"]), **kw).to(dtype)
        state["y"] = torch.randn((rows * choices, case["channels"]), **kw).to(dtype)  # what the experts made of the sorted rows
        state["grad_sorted"] = torch.randn((rows * choices, case["channels"]), **kw).to(dtype)
        state["grad_out"] = torch.randn((rows, case["channels"]), **kw).to(dtype)
    else:
        channels, outputs = case["channels"], case["outputs"]
        flat = chosen.view(-1)
        counts = torch.bincount(flat[flat >= 0], minlength=number).tolist()
        state["counts"] = counts
        x = torch.randn((rows, channels), **kw) * torch.exp(0.3 * torch.randn((1, channels), **kw))
        x[sum(counts):] = 0.0
        state["x"] = x.to(dtype)
        state["weight"] = (torch.randn((number, outputs, channels), **kw) / math.sqrt(channels)).to(dtype)
        state["bias"] = (0.1 * torch.randn((number, outputs), **kw)).to(dtype)
        # the gradient of a loss that is a mean over the rows
        state["grad"] = (torch.randn((rows, outputs), **kw) / math.sqrt(rows)).to(dtype)
        if own:
            from permutohedral_encoding_amd import layers
            state["routing"] = layers.routing(chosen, number)
    if case["train"]:
        for name in ("x", "y", "weights", "weight", "bias"):
            if name in state:
                state[name].requires_grad_(True)
    return state


def run(state):
    if own:
        return _OWN[state["op"]](state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------------ the framework's calls

def _own_route(s):
    from permutohedral_encoding_amd import layers
    weights, routing = layers.route(s["logits"], s["choices"], normalise=s["normalise"])
    out = {"weights": weights.detach(), "experts": routing.experts, "positions": routing.positions, "offsets": routing.offsets}
    if s["train"]:
        out["dlogits"], = torch.autograd.grad(weights, s["logits"], s["grad_weights"])
    return out


def _own_experts_sort(s):
    from permutohedral_encoding_amd import layers
    routing = layers.routing(s["chosen"], s["experts"])
    rows = layers.dispatch(s["x"], routing)
    y = layers.combine(s["y"], s["weights"], routing)
    out = {"sorted": rows.detach(), "out": y.detach()}
    if s["train"]:
        names = ("x", "y", "weights")
        grads = torch.autograd.grad((rows, y), [s[k] for k in names], (s["grad_sorted"], s["grad_out"]))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


def _own_expert_linear(s):
    from permutohedral_encoding_amd import layers
    y = layers.expert_linear(s["x"], s["weight"], s["bias"], s["routing"])
    out = {"y": y.detach()}
    if s["train"]:
        names = ("x", "weight", "bias")
        grads = torch.autograd.grad(y, [s[k] for k in names], s["grad"])
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


def _own_orthogonalise(s):
    from permutohedral_encoding_amd import optim
    return optim.orthogonalise(s["update"])


_OWN = {"route": _own_route, "experts_sort": _own_experts_sort, "expert_linear": _own_expert_linear, "orthogonalise": _own_orthogonalise}


# ------------------------------------------------------------------------------------------ the plain forms

def _plan(chosen, number):
    """Where each choice stands when choices are sorted by expert, and where each expert's begin."""
    flat = chosen.reshape(-1)
    flat = torch.where(flat < 0, number, flat)
    order = torch.sort(flat, stable=True).indices
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device=order.device)
    counts = (torch.zeros(number + 1, dtype=torch.int64, device=flat.device).index_add_(0, flat, torch.ones_like(flat, dtype=torch.int64)))
    offsets = torch.cat([counts.new_zeros(1), counts[:number].cumsum(0)])
    return positions.view(chosen.shape), offsets


def _plain_route(s):
    logits, number = s["logits"].float(), s["experts"]
    left, at = logits.clone(), torch.arange(number, device=logits.device)
    chosen = []
    for _ in range(s["choices"]):
        largest = left.amax(1, keepdim=True)
        first = torch.where(left == largest, at, number).amin(1, keepdim=True)
        chosen.append(torch.where(largest == -math.inf, -1, first))
        left.scatter_(1, first, -math.inf)
    chosen = torch.cat(chosen, 1)
    there = chosen >= 0
    picked = torch.where(there, logits.gather(1, chosen.clamp(min=0)), -math.inf)
    top = torch.where(there[:, :1], picked[:, :1], 0.0)
    exps = torch.exp(picked - top)
    total = exps.sum(1, keepdim=True) if s["normalise"] else torch.exp(logits - top).sum(1, keepdim=True)
    total = torch.where(there[:, :1], total, 1.0)
    weights = exps / total
    positions, offsets = _plan(chosen, number)
    out = {"weights": weights, "experts": chosen.to(torch.int32), "positions": positions.to(torch.int32), "offsets": offsets.to(torch.int32)}
    if s["train"]:
        upstream = weights * s["grad_weights"]
        mean = upstream.sum(1, keepdim=True)
        if s["normalise"]:
            d, along = torch.zeros_like(logits), upstream - weights * mean
        else:
            d, along = -torch.exp(logits - top) / total * mean, upstream
        d.scatter_add_(1, chosen.clamp(min=0), torch.where(there, along, 0.0))
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_experts_sort(s):
    dtype, chosen = s["x"].dtype, s["chosen"]
    positions, _ = _plan(chosen, s["experts"])
    there = (chosen >= 0)[:, :, None]
    rows, choices, channels = *chosen.shape, s["x"].shape[1]
    x, y, weights = s["x"], s["y"].float(), s["weights"][:, :, None]
    flat = positions.view(-1)

    def sort(values):  # (rows, choices, channels)
        out = torch.empty((rows * choices, channels), dtype=values.dtype, device=values.device)
        out[flat] = torch.where(there, values, 0).view(-1, channels)
        return out

    def unsort(values):
        return torch.where(there, values[flat].view(rows, choices, channels), 0)

    back = unsort(y)
    out = {"sorted": sort(x[:, None].expand(-1, choices, -1)), "out": (back * weights).sum(1).to(dtype)}
    if s["train"]:
        grad_out = s["grad_out"].float()[:, None]
        out["dx"] = unsort(s["grad_sorted"].float()).sum(1).to(dtype)
        out["dy"] = sort(grad_out * weights).to(dtype)
        out["dweights"] = (grad_out * back).sum(2)
    return out


def _plain_expert_linear(s):
    dtype, rows = s["x"].dtype, s["x"].shape[0]
    x, weight, bias = s["x"].float(), s["weight"].float(), s["bias"].float()
    y = torch.zeros((rows, weight.shape[1]), dtype=dtype, device=x.device)
    ends = [0]
    for n in s["counts"]:
        ends.append(ends[-1] + n)
    pieces = list(zip(ends, ends[1:]))
    for e, (first, last) in enumerate(pieces):
        y[first:last] = (x[first:last] @ weight[e].t() + bias[e]).to(dtype)
    out = {"y": y}
    if s["train"]:
        grad = s["grad"].float()
        dx, dweight, dbias = torch.zeros_like(s["x"]), torch.zeros_like(s["weight"]), torch.zeros_like(s["bias"])
        for e, (first, last) in enumerate(pieces):
            g, r = grad[first:last], x[first:last]
            dx[first:last] = (g @ weight[e]).to(dtype)
            dbias[e] = g.sum(0, dtype=torch.float64).to(dtype)
            # sums over many rows: in 32 bits over 8192 of them, in 64 over those
            total = torch.zeros(weight.shape[1:], dtype=torch.float64, device=x.device)
            for k in range(0, last - first, 8192):
                total += g[k:k + 8192].t() @ r[k:k + 8192]
            dweight[e] = total.to(dtype)
        out.update(dx=dx, dweight=dweight, dbias=dbias)
    return out


def _plain_orthogonalise(s):
    a, b, c = COEFFICIENTS
    x = s["update"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    norm = torch.sqrt(x.double().square().sum((1, 2), keepdim=True)).float()
    x = x / (norm + 1e-7)
    for _ in range(STEPS):
        square = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * square + c * (square @ square)) @ x
    if tall:
        x = x.transpose(1, 2).contiguous()
    return x.to(s["update"].dtype)


_PLAIN = {"route": _plain_route, "experts_sort": _plain_experts_sort, "expert_linear": _plain_expert_linear, "orthogonalise": _plain_orthogonalise}


# ------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    number, choices = case["experts"], case["choices"]
    if case["op"] == "orthogonalise":
        a, b, c = COEFFICIENTS
        g = s["update"].double()
        x = g / (g.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
        small = min(x.shape[1:])
        eye = torch.eye(small, dtype=x.dtype, device=x.device)
        for _ in range(STEPS):
            t = x.transpose(1, 2).contiguous()
            gram = x @ t if x.shape[1] == small else t @ x
            factor = a * eye + b * gram + c * (gram @ gram)
            x = factor @ x if x.shape[1] == small else x @ factor
        return x
    if case["op"] == "route":
        logits = s["logits"].detach().double().requires_grad_(True)
        order = torch.sort(logits.detach(), dim=1, descending=True, stable=True)
        chosen = torch.where(order.values[:, :choices] == -math.inf, -1, order.indices[:, :choices])
        open_rows = chosen[:, 0] >= 0
        shares = torch.softmax(torch.where(open_rows[:, None], logits, 0.0), 1)
        picked = torch.where(chosen >= 0, shares.gather(1, chosen.clamp(min=0)), 0.0)
        weights = picked
        if case["normalise"]:
            weights = picked / torch.where(open_rows[:, None], picked.sum(1, keepdim=True), 1.0)
        positions, offsets = _counted(chosen, number)
        out = {"weights": weights.detach(), "experts": chosen.to(torch.int32), "positions": positions, "offsets": offsets}
        if case["train"]:
            out["dlogits"], = torch.autograd.grad(weights, logits, s["grad_weights"].double())
        return out
    if case["op"] == "experts_sort":
        positions, offsets = _counted(s["chosen"], number)
        rows, channels = s["x"].shape
        total = int(offsets[-1])
        x, y, weights = (s[k].detach().double().requires_grad_(True) for k in ("x", "y", "weights"))
        item_at = torch.empty(rows * choices, dtype=torch.int64, device=x.device)
        item_at[positions.reshape(-1).long()] = torch.arange(rows * choices, device=x.device)
        routed = (torch.arange(rows * choices, device=x.device) < total)[:, None]
        ordered = x[item_at // choices] * routed
        summed = torch.zeros((rows, channels), dtype=x.dtype, device=x.device)
        summed = summed.index_add(0, item_at[:total] // choices, y[:total] * weights.reshape(-1)[item_at[:total], None])
        out = {"sorted": ordered.detach(), "out": summed.detach()}
        if case["train"]:
            grads = torch.autograd.grad((ordered, summed), (x, y, weights), (s["grad_sorted"].double(), s["grad_out"].double()))
            out.update(dx=grads[0], dy=grads[1], dweights=grads[2])
        return out
    x, weight, bias, grad = (s[k].detach().double() for k in ("x", "weight", "bias", "grad"))
    out = {"y": torch.zeros((x.shape[0], weight.shape[1]), dtype=x.dtype, device=x.device)}
    if case["train"]:
        out.update(dx=torch.zeros_like(x), dweight=torch.zeros_like(weight), dbias=torch.zeros_like(bias))
    first = 0
    for e, n in enumerate(s["counts"]):
        at = slice(first, first + n)
        out["y"][at] = torch.addmm(bias[e], x[at], weight[e].t())
        if case["train"]:
            out["dx"][at] = torch.mm(grad[at], weight[e])
            out["dweight"][e] = torch.mm(grad[at].t(), x[at])
            out["dbias"][e] = grad[at].sum(0)
        first += n
    return out


def _counted(chosen, number):
    """Positions and offsets by counting, expert by expert."""
    flat = chosen.reshape(-1)
    positions, offsets = torch.zeros_like(flat), [0]
    for e in [*range(number), -1]:
        mine = flat == e
        positions = torch.where(mine, offsets[-1] + mine.cumsum(0) - 1, positions)
        offsets.append(offsets[-1] + int(mine.sum()))
    return positions.view(chosen.shape).to(torch.int32), torch.tensor(offsets[:number + 1], dtype=torch.int32, device=flat.device)


def work(case):
    """Bytes: every input and result once, and the plan (positions, and the choice of each position) written where a call makes it and read where one needs it;
    operations of the products (the two symmetric ones by half) and, per value, of the rest."""
    rows, number, choices, t = case["rows"], case["experts"], case["choices"], 2 if case["dtype"] != "fp32" else 4
    channels, outputs = case["channels"], case["outputs"]
    train = case["train"]
    if case["op"] == "route":
        nbytes, flops = t * rows * number + 16 * rows * choices, (2 + choices) * rows * number
        if train:
            nbytes += 2 * t * rows * number + 4 * rows * choices if not case["normalise"] else t * rows * number + 12 * rows * choices
            flops += 3 * rows * number
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "experts_sort":
        items = rows * choices
        nbytes, flops = t * channels * (2 * rows + 2 * items) + 20 * items, 2 * items * channels
        if train:
            nbytes += t * channels * (2 * rows + 3 * items) + 8 * items
            flops += 4 * items * channels
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "expert_linear":
        touched = min(number, rows)
        nbytes = t * (rows * (channels + outputs) + touched * outputs * (channels + 1))
        flops = 2 * rows * channels * outputs
        if train:
            nbytes += t * (rows * (2 * channels + outputs) + (touched + number) * outputs * (channels + 1))
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    small, large = min(rows, channels), max(rows, channels)
    return {"bytes": 2 * t * number * rows * channels, "flops": number * STEPS * (3 * small * small * large + small ** 3)}
