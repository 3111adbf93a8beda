"""Rows that go to experts, on the GPU, against their definitions in 64 bits (expert_reference.py).

Tolerances: indices, positions and copied rows have to be equal.  An exponential of l - top is off by |l - top| 2^-24 for the rounded difference and two steps of
its own, a sum over a row's experts adds 16 roundings in a lane and 6 over the lanes, a quotient one: (|l - top| + 64) 2^-24 of a weight and, with a few more products
and sums over the choices, of the terms of a gradient.  A weighted sum of k rows makes 2 k roundings, a dot product of C channels at most C + 8."""
import math

import pytest
import torch

import expert_reference as ref
from permutohedral_encoding_amd import layers

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def random(shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def chosen_experts(rows, choices, number, seed=0, none=0.1, dtype=torch.int64):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    e = torch.randint(0, number, (rows, choices), generator=generator, device="cuda")
    return torch.where(torch.rand((rows, choices), generator=generator, device="cuda") < none, -1, e).to(dtype)


def assert_within(got, want, bound, what):
    assert got.shape == want.shape, what
    error = (got.detach().double() - want).abs()
    assert bool((error <= bound).all()), f"{what}: worst error/bound {float((error / bound).max()):.3g}"


# ------------------------------------------------------------------------------------------ route

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("rows,number,choices", [(1, 1, 1), (5, 2, 2), (1000, 7, 2), (257, 8, 8), (4097, 9, 3), (300, 16, 1), (300, 33, 5), (1000, 64, 2), (70, 100, 4), (129, 150, 3), (50, 200, 8), (61, 300, 4), (45, 390, 2),
                                                 (65, 256, 8), (33, 257, 2), (17, 512, 6), (9, 513, 2), (19, 1000, 8), (3, 1024, 4)])
def test_route(dtype, normalise, rows, number, choices):
    logits = random((rows, number + 3), 1, TYPES[dtype])[:, :number]
    closed = torch.rand(rows, number, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") < 0.3
    if rows > 4:
        logits = torch.where(closed, -math.inf, logits)
        logits[3] = -math.inf
    logits.requires_grad_(True)
    weights, routing = layers.route(logits, choices, normalise=normalise)
    grad = random((rows, choices), 3)
    chosen, w, d, m, far = ref.route(logits, choices, normalise, grad)
    assert weights.dtype == torch.float32 and routing.experts.dtype == torch.int32 and routing.number == number
    assert torch.equal(routing.experts.long(), chosen)
    assert_within(weights, w, (far + 64) * ref.U * w + 2.0 ** -126, "weights")
    positions, offsets = ref.plan(chosen, number)
    assert torch.equal(routing.positions.cpu(), positions) and torch.equal(routing.offsets.cpu(), offsets)
    dl, = torch.autograd.grad(weights, logits, grad)
    assert dl.dtype == logits.dtype
    assert_within(dl, d, (far + 64) * ref.U * m + ref.half_step(d, dl.dtype) + 2.0 ** -126, "dlogits")


def test_equal_logits_go_to_the_lowest_experts():
    for dtype in TYPES.values():
        for number in (5, 8, 64, 300, 1000):
            logits = torch.zeros(9, number, device="cuda", dtype=dtype)
            logits[:, ::2] = -0.0
            logits[4, number // 2:] = 1.0
            weights, routing = layers.route(logits, 4)
            assert torch.equal(routing.experts[:4].cpu(), torch.arange(4, dtype=torch.int32).expand(4, 4))
            first = number // 2
            expected = [e if e < number else e - number for e in range(first, first + 4)]
            assert routing.experts[4].tolist() == expected
            assert bool((weights[0] == 0.25).all())


def test_logits_that_are_not_finite():
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[1.0, nan, 2.0, 0.0], [inf, 1.0, 0.0, 0.0], [-inf, -inf, -inf, 3.0], [-inf] * 4, [nan, nan, 1.0, inf]], device="cuda", requires_grad=True)
    for normalise in (True, False):
        weights, routing = layers.route(logits, 2, normalise=normalise)
        assert routing.experts.tolist() == [[1, 2], [0, 1], [3, -1], [-1, -1], [0, 1]]
        assert bool(torch.isnan(weights[0]).all()) and bool(torch.isnan(weights[1]).any()) and bool(torch.isnan(weights[4]).all())
        assert weights[2].tolist() == [1.0, 0.0] and weights[3].tolist() == [0.0, 0.0]
        dl, = torch.autograd.grad(weights.sum(), logits)
        assert dl[2].tolist() == [0.0] * 4 and dl[3].tolist() == [0.0] * 4


def test_route_of_other_shapes():
    logits = random((4, 6, 10))
    weights, routing = layers.route(logits, 3)
    flat, flat_routing = layers.route(logits.view(24, 10), 3)
    assert weights.shape == routing.experts.shape == routing.positions.shape == (4, 6, 3)
    assert torch.equal(weights.view(24, 3), flat) and torch.equal(routing.positions.view(24, 3), flat_routing.positions)
    weights, routing = layers.route(logits.transpose(0, 1), 3)
    assert torch.equal(weights, flat.view(4, 6, 3).transpose(0, 1))
    weights, routing = layers.route(logits[:0], 2)
    assert weights.shape == (0, 6, 2) and routing.offsets.tolist() == [0] * 11
    weights, routing = layers.route(logits[0, 0], 2)
    assert weights.shape == (2,) and sorted(routing.positions.tolist()) == [0, 1]


@pytest.mark.parametrize("normalise", [True, False])
def test_the_gradient_of_route_against_differences(normalise):
    logits = random((6, 9), 5).requires_grad_(True)
    grad = random((6, 3), 6)
    weights, _ = layers.route(logits, 3, normalise=normalise)
    dl, = torch.autograd.grad(weights, logits, grad)
    step = 2.0 ** -8
    for e in range(9):
        moved = [logits.detach().clone() for _ in range(2)]
        for m, sign in zip(moved, (1.0, -1.0)):
            m[:, e] += sign * step
        plus, minus = (layers.route(m, 3, normalise=normalise) for m in moved)
        same = (plus[1].experts == minus[1].experts).all(1)
        assert bool(same.any())
        difference = ((plus[0] - minus[0]).double() * grad).sum(1) / (2 * step)
        # a third derivative of a share is at most 1, and each of the 2 * 3 weights is off by 64 2^-24
        bound = step ** 2 * grad.abs().sum(1) + 6 * 64 * ref.U * grad.abs().amax(1) / step
        assert bool(((dl[:, e].double() - difference).abs() <= bound)[same].all())


# ------------------------------------------------------------------------------------------ plans

@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,choices,number", [(0, 2, 5), (1, 1, 1), (1, 2, 64), (63, 1, 3), (64, 3, 7), (1000, 2, 8), (4096, 1, 1024), (4097, 1, 2), (2049, 2, 1000),
                                                 (16384, 1, 9), (16385, 1, 9), (8000, 2, 1024), (30000, 4, 63), (30000, 1, 64), (5, 1000, 17), (1 << 18, 2, 13)])
def test_plan(dtype, rows, choices, number):
    for none in (0.0, 0.2, 1.0):
        experts = chosen_experts(rows, choices, number, none=none, dtype=dtype)
        routing = layers.routing(experts, number)
        positions, offsets = ref.plan(experts, number)
        assert torch.equal(routing.positions.cpu(), positions) and torch.equal(routing.offsets.cpu(), offsets)


def test_plan_of_experts_that_are_none_and_of_one_alone():
    experts = torch.tensor([[5, -7], [1 << 40, 2], [3, 3], [2, -1]], device="cuda")
    routing = layers.routing(experts, 5)
    assert routing.positions.tolist() == [[4, 5], [6, 0], [2, 3], [1, 7]] and routing.offsets.tolist() == [0, 0, 0, 2, 4, 4]
    routing = layers.routing(torch.full((10000, 1), 3, device="cuda"), 9)
    assert torch.equal(routing.positions[:, 0].cpu(), torch.arange(10000, dtype=torch.int32)) and routing.offsets.tolist() == [0] * 4 + [10000] * 6
    strided = chosen_experts(50, 6, 4)[:, ::2]
    assert torch.equal(layers.routing(strided, 4).positions.cpu(), ref.plan(strided, 4)[0])


# ------------------------------------------------------------------------------------------ rows there and back

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,choices,channels", [(0, 2, 5), (1, 1, 1), (1, 2, 1024), (100, 2, 3), (257, 1, 8), (300, 3, 64), (65, 4, 203), (33, 5, 7), (20, 9, 130),
                                                   (4097, 2, 48), (7, 2, 4100)])
def test_rows_there_and_back(dtype, rows, choices, channels):
    dtype, number = TYPES[dtype], 7
    for none, weight_dtype in ((0.2, torch.float32), (0.0, dtype), (1.0, torch.float32)):
        experts = chosen_experts(rows, choices, number, seed=rows, none=none)
        routing = layers.routing(experts, number)
        at, there = routing.positions.long(), (experts >= 0)[:, :, None]
        x = random((rows, channels + 3), 1, dtype)[:, :channels].requires_grad_(True)
        y = random((rows * choices, channels + 1), 2, dtype)[:, :channels]
        total = int(routing.offsets[-1])
        y[total:] = math.nan  # (what stands in rows without an expert is not read)
        y.requires_grad_(True)
        weights = random((rows, choices), 3, weight_dtype).requires_grad_(True)

        rows_there = layers.dispatch(x, routing)
        want = torch.zeros((rows * choices, channels), dtype=dtype, device="cuda")
        want[at] = torch.where(there, x.detach()[:, None], 0)
        assert torch.equal(rows_there, want)

        out = layers.combine(y, weights, routing)
        back = torch.where(there, y.detach().double()[at], 0.0)
        w = weights.detach().double()[:, :, None]
        assert out.dtype == dtype and out.shape == (rows, channels)
        value, size = (back * w).sum(1), (back * w).abs().sum(1)
        assert_within(out, value, 2 * choices * ref.U * size + ref.half_step(value, dtype), "out")

        grad_there, grad_out = random((rows * choices, channels), 4, dtype), random((rows, channels + 2), 5, dtype)[:, :channels]
        grad_there[total:] = math.nan
        dx, dy, dw = torch.autograd.grad((rows_there, out), (x, y, weights), (grad_there, grad_out))
        g = torch.where(there, grad_there.double()[at], 0.0)
        assert dx.dtype == dtype and dw.dtype == weight_dtype
        assert_within(dx, g.sum(1), choices * ref.U * g.abs().sum(1) + ref.half_step(g.sum(1), dtype), "dx")
        want = torch.zeros((rows * choices, channels), dtype=torch.float64, device="cuda")
        want[at] = torch.where(there, grad_out.double()[:, None] * w, 0.0)
        assert_within(dy, want, ref.U * want.abs() + ref.half_step(want, dtype), "dy")
        terms = grad_out.double()[:, None] * back
        assert_within(dw, terms.sum(2), (channels + 8) * ref.U * terms.abs().sum(2) + ref.half_step(terms.sum(2), weight_dtype), "dweights")


def test_rows_of_other_shapes_and_partial_gradients():
    experts = chosen_experts(24, 2, 5, none=0.1).view(4, 6, 2)
    routing = layers.routing(experts, 5)
    x = random((6, 4, 40)).transpose(0, 1).requires_grad_(True)
    flat_routing = layers.routing(experts.view(24, 2), 5)
    there = layers.dispatch(x, routing)
    assert torch.equal(there, layers.dispatch(x.detach().reshape(24, 40), flat_routing))
    weights = random((4, 6, 2), 1)
    out = layers.combine(there, weights, routing)
    assert out.shape == (4, 6, 40)
    dx, = torch.autograd.grad(out, x, torch.ones(1, 1, 40, device="cuda").expand(4, 6, 40))
    assert_within(dx, torch.where(experts >= 0, weights.double(), 0.0).sum(2, keepdim=True).expand(4, 6, 40), 8 * ref.U * weights.abs().sum(2, keepdim=True).double() + 1e-30, "dx")
    # the weights alone, and y alone
    y, w = there.detach().requires_grad_(True), weights.clone().requires_grad_(True)
    both = torch.autograd.grad(layers.combine(y, w, routing).sum(), (y, w))
    assert torch.equal(torch.autograd.grad(layers.combine(y.detach(), w, routing).sum(), w)[0], both[1])
    assert torch.equal(torch.autograd.grad(layers.combine(y, w.detach(), routing).sum(), y)[0], both[0])
    # a row that goes to the same expert twice
    twice = layers.routing(torch.tensor([[1, 1], [0, 1]], device="cuda"), 2)
    rows = layers.dispatch(x.detach()[0, :2], twice)
    assert torch.equal(rows, x.detach()[0][[1, 0, 0, 1]])


def test_rows_behind_two_to_the_31_values():
    rows, channels = (1 << 20) + 3, 2080
    x = torch.zeros(rows, channels, dtype=torch.bfloat16, device="cuda")
    x[-5:] = random((5, channels), 1, torch.bfloat16)
    experts = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    experts[-5:] = 2
    experts[0] = 1
    routing = layers.routing(experts, 3)
    there = layers.dispatch(x, routing)
    assert torch.equal(there[-5:], x[-5:]) and not bool(there[:-5].any())
    assert torch.equal(layers.combine(there, torch.ones(rows, 1, device="cuda"), routing), x)


# ------------------------------------------------------------------------------------------ the experts' products
# A result is one chain of additions: of its channels, or of an expert's rows; twice 2^-24 of the terms' magnitudes for each, for additions that do not round to
# nearest.  Products of 16-bit values are exact, those of float32 round once: another 2^-24.

def products(x, weight, bias, grad, offsets):
    """{name: (value, magnitude, length of the chain)} in 64 bits."""
    x, weight, grad = x.detach().double(), weight.detach().double(), grad.double()
    number, outputs, channels = weight.shape
    out = {k: [torch.zeros(s, dtype=torch.float64, device="cuda") for _ in range(2)]
           for k, s in (("y", (x.shape[0], outputs)), ("dx", x.shape), ("dweight", weight.shape), ("dbias", (number, outputs)))}
    longest = 1
    for e in range(number):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        longest = max(longest, at.stop - at.start)
        for k, f in enumerate((lambda t: t, torch.abs)):
            a, w, g = f(x[at]), f(weight[e]), f(grad[at])
            out["y"][k][at] = a @ w.t() + (f(bias[e].detach().double()) if bias is not None else 0.0)
            out["dx"][k][at] = g @ w
            out["dweight"][k][e] = g.t() @ a
            out["dbias"][k][e] = g.sum(0)
    chain = {"y": channels + 1, "dx": outputs, "dweight": longest, "dbias": longest}
    return {k: (*v, 2 * chain[k] + 8) for k, v in out.items()}


def check_products(rows, number, channels, outputs, dtype, bias=True, none=0.1, extra=0, seed=0, empty=()):
    experts = chosen_experts(rows, 1, number, seed=seed, none=none)
    for e in empty:
        experts[experts == e] = (e + 1) % number
    routing = layers.routing(experts, number)
    total = int(routing.offsets[-1])
    x, grad = random((rows, channels + extra), 1, dtype)[:, :channels], random((rows, outputs + extra), 2, dtype)[:, :outputs]
    x[total:] = math.nan  # (what stands in rows without an expert is not read)
    grad[total:] = math.nan
    x.requires_grad_(True)
    weight = random((number, outputs, channels), 3, dtype).requires_grad_(True)
    b = random((number, outputs), 4, dtype).requires_grad_(True) if bias else None
    y = layers.expert_linear(x, weight, b, routing)
    given = [t for t in (x, weight, b) if t is not None]
    grads = dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, given, grad)))
    want = products(x, weight, b, grad, routing.offsets.tolist())
    for name, got in {"y": y, **grads}.items():
        value, magnitude, chain = want[name]
        assert got.dtype == dtype
        assert_within(got, value, chain * ref.U * magnitude + ref.half_step(value, dtype), name)
    return y, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(0, 3, 5, 7), (1, 1, 1, 1), (1, 8, 64, 64), (7, 3, 3, 2), (65, 2, 64, 64), (300, 5, 8, 24), (257, 4, 40, 72),
                                                          (300, 7, 72, 200), (1000, 3, 130, 65), (513, 2, 203, 130), (130, 70, 48, 16), (2000, 1, 128, 256),
                                                          (900, 4, 264, 136), (40, 1024, 16, 8), (5000, 2, 64, 3), (3000, 3, 512, 264), (700, 6, 100, 300)])
def test_expert_linear(dtype, rows, number, channels, outputs):
    check_products(rows, number, channels, outputs, TYPES[dtype])
    check_products(rows, number, channels, outputs, TYPES[dtype], bias=False, none=0.0, extra=8, empty=(0,) if number > 1 else ())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(1000, 3, 64, 64), (1000, 4, 8, 3), (999, 2, 16, 17), (700, 3, 128, 40), (513, 5, 32, 33), (2000, 2, 24, 64),
                                                          (5, 8, 264, 200), (40, 16, 512, 130), (16, 1, 1032, 65), (3, 300, 64, 100), (100, 9, 2048, 80)])
def test_expert_linear_of_narrow_layers_and_of_few_rows(dtype, rows, number, channels, outputs):
    for none in (0.0, 0.3, 1.0):
        check_products(rows, number, channels, outputs, TYPES[dtype], none=none, extra=8, empty=(1,) if number > 1 else ())
        check_products(rows, number, outputs, channels, TYPES[dtype], none=none, bias=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(500, 1, 1024, 64), (130, 7, 1032, 24), (500, 1, 1023, 63), (300, 2, 64, 1030), (65, 1, 136, 136), (900, 2, 3, 300), (900, 2, 300, 2)])
def test_expert_linear_of_long_rows_that_are_few(dtype, rows, number, channels, outputs):
    check_products(rows, number, channels, outputs, TYPES[dtype])
    check_products(rows, number, channels, outputs, TYPES[dtype], bias=False, none=0.4, extra=8, empty=(0,) if number > 1 else ())


@pytest.mark.parametrize("dtype", TYPES)
def test_expert_linear_of_rows_that_begin_anywhere(dtype):
    for extra in (1, 2, 3, 5):
        check_products(401, 3, 64, 136, TYPES[dtype], extra=extra)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(70001, 2, 64, 64), (50000, 1, 48, 130), (40000, 3, 128, 128), (20000, 300, 32, 64), (40000, 3, 101, 130),
                                                          (40000, 3, 101, 60), (30000, 2, 3, 200), (30000, 2, 200, 3), (30000, 2, 5, 6), (30000, 3, 200, 264)])
def test_expert_linear_of_many_rows(dtype, rows, number, channels, outputs):
    """(the rows of an expert are cut for its weights' gradient)"""
    first = check_products(rows, number, channels, outputs, TYPES[dtype])
    second = check_products(rows, number, channels, outputs, TYPES[dtype])
    assert torch.equal(first[0], second[0]) and all(torch.equal(first[1][k], second[1][k]) for k in first[1])


def test_what_is_not_finite_stays_with_its_expert():
    for dtype in TYPES.values():
        for channels in (64, 67):
            experts = torch.arange(5, device="cuda").repeat_interleave(50)[:, None]
            routing = layers.routing(experts, 5)
            x, weight, grad = random((250, channels), 1, dtype), random((5, 70, channels), 2, dtype), random((250, 70), 3, dtype)
            clean = layers.expert_linear(x.requires_grad_(True), weight.requires_grad_(True), None, routing)
            clean = [clean.detach(), *torch.autograd.grad(clean, (x, weight), grad)]
            with torch.no_grad():
                x[100:150], grad[100:150] = math.inf, math.nan
                weight[3] = math.nan
            y = layers.expert_linear(x, weight, None, routing)
            got = [y.detach(), *torch.autograd.grad(y, (x, weight), grad)]
            rows = torch.cat([torch.arange(100), torch.arange(200, 250)]).cuda()
            assert all(torch.equal(a[rows], b[rows]) for a, b in zip(got[:2], clean[:2]))
            assert torch.equal(got[2][[0, 1, 3, 4]], clean[2][[0, 1, 3, 4]])
            assert not bool(torch.isfinite(got[2][2]).any()) and not bool(torch.isfinite(got[0][150:200]).any())


def test_expert_linear_takes_what_it_says():
    routing = layers.routing(torch.zeros(6, 2, dtype=torch.int64, device="cuda"), 3)
    x, weight, bias = random((12, 8)), random((3, 5, 8), 1), random((3, 5), 2)
    want = layers.expert_linear(x, weight, bias, routing)
    assert torch.equal(layers.expert_linear(x, weight.transpose(1, 2).contiguous().transpose(1, 2), bias, routing), want)
    wide = random((12, 8), 3).repeat(1, 2)
    assert torch.equal(layers.expert_linear(wide[:, ::2], weight, bias, routing), layers.expert_linear(wide[:, ::2].contiguous(), weight, bias, routing))
    row = random((1, 8), 4)
    assert torch.equal(layers.expert_linear(row.expand(12, 8), weight, bias, routing), layers.expert_linear(row.repeat(12, 1), weight, bias, routing))
    # gradients that autograd broadcasts, and each parameter alone
    given = [t.clone().requires_grad_(True) for t in (x, weight, bias)]
    all_of_them = torch.autograd.grad(layers.expert_linear(*given, routing).sum(), given)
    for i in range(3):
        alone = [t.detach().requires_grad_(k == i) for k, t in enumerate(given)]
        assert torch.equal(torch.autograd.grad(layers.expert_linear(*alone, routing).sum(), alone[i])[0], all_of_them[i])
    assert bool((all_of_them[2][0] == 12.0).all()) and not bool(all_of_them[1][1:].any())
    for bad, message in [((x[:11], weight, bias), "choices"), ((x[:, :7], weight, bias), "channels"), ((x, weight[:2], bias), "sizes"),
                         ((x, weight, bias[:, :4]), "bias"), ((x, weight.half(), bias), "one type"), ((x.double(), weight, bias), "type"),
                         ((x, weight, bias.cpu()), "GPU memory")]:
        with pytest.raises(ValueError, match=message):
            layers.expert_linear(*bad, routing)


def test_expert_linear_behind_two_to_the_31_values():
    rows, channels = (1 << 20) + 3, 2080
    x = torch.zeros(rows, channels, dtype=torch.bfloat16, device="cuda")
    x[-3:] = random((3, channels), 1, torch.bfloat16)
    experts = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    experts[-3:] = 1
    routing = layers.routing(experts, 2)
    weight = random((2, 8, channels), 2, torch.bfloat16).requires_grad_(True)
    y = layers.expert_linear(x.requires_grad_(True), weight, None, routing)
    grad = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    grad[-1, 3] = 1.0
    dx, dw = torch.autograd.grad(y, (x, weight), grad)
    want = x.detach()[-3:].double() @ weight.detach()[1].double().t()
    size = x.detach()[-3:].double().abs() @ weight.detach()[1].double().abs().t()
    assert_within(y[-3:], want, (2 * channels + 8) * ref.U * size + ref.half_step(want, torch.bfloat16), "y")
    assert not bool(y[:-3].any()) and torch.equal(dx[-1], weight.detach()[1, 3]) and not bool(dx[:-1].any())
    assert torch.equal(dw[1, 3], x.detach()[-1]) and not bool(dw[0].any())


@pytest.mark.parametrize("dtype", TYPES)
def test_the_layers_of_experts_together(dtype):
    """A decoder of experts, forward and backward, against its formula with the experts that were chosen."""
    dtype, rows, number, choices, channels, hidden = TYPES[dtype], 700, 5, 2, 48, 64
    x = random((rows, channels), 1, dtype)
    router = random((number, channels), 2, dtype)
    up, bias, down = random((number, hidden, channels), 3, dtype) / 7, random((number, hidden), 4, dtype), random((number, 3, hidden), 5, dtype) / 8
    given = [t.requires_grad_(True) for t in (x, router, up, bias, down)]
    weights, routing = layers.route(layers.linear(x, router), choices)
    h = layers.expert_linear(layers.dispatch(x, routing), up, bias, routing)
    h = layers.activation(h, "silu", keep_8bit=False)
    out = layers.combine(layers.expert_linear(h, down, None, routing), weights, routing)
    grad = random((rows, 3), 6, dtype)
    grads = torch.autograd.grad(out, given, grad)

    at = [t.detach().double().requires_grad_(True) for t in given]
    xd, rd, ud, bd, dd = at
    w = torch.softmax((xd @ rd.t()).gather(1, routing.experts.long()), 1)
    want = 0.0
    for j in range(choices):
        e = routing.experts[:, j].long()
        hj = torch.nn.functional.silu((ud[e] @ xd[:, :, None])[:, :, 0] + bd[e])
        want = want + w[:, j:j + 1] * (dd[e] @ hj[:, :, None])[:, :, 0]
    wanted = torch.autograd.grad(want, at, grad.double())
    # Seven results are rounded to the type on the way of a value, twelve on that of a gradient, and the checkpoint of x has steps of 1/126 of a block's
    # largest value for the router's weight; relative to the whole, with a factor of four for values that cancel.
    eps = torch.finfo(dtype).eps
    assert float((out.detach().double() - want).norm()) <= 4 * (7 * eps + 2 * channels * ref.U) * float(want.detach().norm())
    for name, g, v in zip(("x", "router", "up", "bias", "down"), grads, wanted):
        bound = 4 * (12 * eps + 2 * rows * ref.U) + (0.02 if name == "router" else 0.0)
        assert float((g.double() - v).norm()) <= bound * float(v.norm()), name


# ------------------------------------------------------------------------------------------ refusals

def test_refusals():
    x, routing = random((6, 8)), layers.routing(chosen_experts(6, 2, 4), 4)
    logits = random((6, 4))
    cpu = layers.Routing(routing.experts, 4, routing.positions.cpu(), routing.offsets)
    for call, message in [(lambda: layers.route(logits, 5), "choose"), (lambda: layers.route(logits, 0), "choose"),
                          (lambda: layers.route(random((2, 100)), 9), "choose"), (lambda: layers.route(random((2, 1025)), 1), "experts"),
                          (lambda: layers.route(logits.double(), 1), "type"), (lambda: layers.routing(logits, 4), "int32 or int64"),
                          (lambda: layers.routing(routing.experts, 0), "experts"), (lambda: layers.routing(routing.experts, 1025), "experts"),
                          (lambda: layers.dispatch(x[:5], routing), "rows"), (lambda: layers.dispatch(x, cpu), "GPU memory"),
                          (lambda: layers.dispatch(x.long(), routing), "type"), (lambda: layers.combine(x, torch.ones(6, 2, device="cuda"), routing), "choices"),
                          (lambda: layers.combine(random((12, 8)), torch.ones(6, 1, device="cuda"), routing), "each choice"),
                          (lambda: layers.combine(random((12, 8), dtype=torch.bfloat16), torch.ones(6, 2, device="cuda", dtype=torch.float16), routing), "weights"),
                          (lambda: layers.dispatch(x, layers.Routing(None, 4, routing.positions.long(), routing.offsets)), "routing")]:
        with pytest.raises(ValueError, match=message):
            call()
    weights, _ = layers.route(logits.requires_grad_(True), 2)
    first, = torch.autograd.grad(weights.square().sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        first.sum().backward()


# ------------------------------------------------------------------------------------------ streams and graphs

def test_on_another_stream_and_in_a_graph():
    logits, x = random((500, 16)), random((500, 48), 1)

    def forward(logits, x):
        weights, routing = layers.route(logits, 2)
        return layers.combine(2.0 * layers.dispatch(x, routing), weights, routing), routing.positions

    want, want_at = forward(logits, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_at = forward(logits, x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_at, want_at)

    given = [logits.clone().requires_grad_(True), x.clone().requires_grad_(True)]
    grad = random((500, 48), 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = forward(*given)
        grads = torch.autograd.grad(out, given, grad)
    for seed in range(3):
        new = [random((500, 16), 10 + seed), random((500, 48), 20 + seed)]
        with torch.no_grad():
            for t, n in zip(given, new):
                t.copy_(n)
        graph.replay()
        eager = [t.clone().requires_grad_(True) for t in new]
        want, _ = forward(*eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, eager, grad)))


def decoder(x, logits, up, bias, down):
    weights, routing = layers.route(logits, 2)
    h = layers.activation(layers.expert_linear(layers.dispatch(x, routing), up, bias, routing), keep_8bit=False)
    return layers.combine(layers.expert_linear(h, down, None, routing), weights, routing)


def decoder_inputs(rows, number, seed, dtype=torch.float32):
    return [random(s, seed + i, t) / 4 for i, (s, t) in enumerate((((rows, 40), dtype), ((rows, number), torch.float32), ((number, 72, 40), dtype), ((number, 72), dtype),
                                                                   ((number, 40, 72), dtype)))]


def test_two_graphs_of_a_decoder_at_once():
    """Plans of several launches and weight gradients of several pieces have workspaces: two graphs, and eager work beside them, share none."""
    rows, number = 20000, 3
    grad = random((rows, 40), 9)
    streams = [torch.cuda.Stream() for _ in range(2)]
    given = [[t.requires_grad_(True) for t in decoder_inputs(rows, number, 100 * k)] for k in range(2)]
    graphs, results = [], []
    for g, s in zip(given, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            out = decoder(*g)
            results.append([out, *torch.autograd.grad(out, g, grad)])
    for seed in range(3):
        new = [decoder_inputs(rows, number, 1000 * seed + 50 * k) for k in range(2)]
        with torch.no_grad():
            for g, n in zip(given, new):
                for a, b in zip(g, n):
                    a.copy_(b)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        wanted = []
        for n in new:  # (on the current stream, meanwhile)
            eager = [t.clone().requires_grad_(True) for t in n]
            out = decoder(*eager)
            wanted.append([out, *torch.autograd.grad(out, eager, grad)])
        torch.cuda.synchronize()
        for got, want in zip(results, wanted):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_padded_batch():
    """Rows of padding have logits of -inf alone: nothing of what stands in them goes anywhere."""
    rows, padding, number = 300, 77, 4
    given = decoder_inputs(rows, number, 1)
    full = [torch.cat([given[0], torch.full((padding, 40), math.nan, device="cuda")]), torch.cat([given[1], torch.full((padding, number), -math.inf, device="cuda")]), *given[2:]]
    grad = random((rows, 40), 9)
    results = []
    for tensors, g in ((given, grad), (full, torch.cat([grad, torch.full((padding, 40), math.nan, device="cuda")]))):
        tensors = [t.clone().requires_grad_(True) for t in tensors]
        out = decoder(*tensors)
        results.append([out.detach(), *torch.autograd.grad(out, tensors, g)])
    (out, dx, dlogits, *dw), (all_out, all_dx, all_dlogits, *all_dw) = results
    assert torch.equal(all_out[:rows], out) and torch.equal(all_dx[:rows], dx) and torch.equal(all_dlogits[:rows], dlogits)
    assert not any(bool(t[rows:].any()) for t in (all_out, all_dx, all_dlogits))
    # (the rows of each expert are the same, in the same order)
    assert all(torch.equal(a, b) for a, b in zip(dw, all_dw))


def test_an_expert_twice_in_a_row():
    rows = 130
    experts = torch.randint(0, 3, (rows, 1), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").repeat(1, 3)
    routing = layers.routing(experts, 3)
    assert sorted(routing.positions.flatten().tolist()) == list(range(3 * rows))
    x, weights = random((rows, 24), 1).requires_grad_(True), random((rows, 3), 2).requires_grad_(True)
    out = layers.combine(layers.dispatch(x, routing), weights, routing)
    grad = random((rows, 24), 3)
    dx, dw = torch.autograd.grad(out, (x, weights), grad)
    xd, wd, gd = x.detach().double(), weights.detach().double(), grad.double()
    bound = 16 * ref.U * wd.abs().sum(1, keepdim=True)
    assert_within(out, xd * wd.sum(1, keepdim=True), bound * xd.abs(), "out")
    assert_within(dx, gd * wd.sum(1, keepdim=True), bound * gd.abs(), "dx")
    assert_within(dw, (xd * gd).sum(1, keepdim=True).expand(-1, 3), 64 * ref.U * (xd * gd).abs().sum(1, keepdim=True).expand(-1, 3), "dw")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("channels,outputs", [(384, 520), (512, 512)])
def test_expert_linear_of_wide_layers(dtype, channels, outputs):
    """Tiles of 256 x 256 in each direction, the last of them in quarters; experts of no row, of one, and of nearly all; rows without an expert; rows that are further apart, on
    16 bytes and not."""
    rows, number = 100000, 7
    generator = torch.Generator(device="cuda").manual_seed(5)
    experts = torch.randint(0, 4, (rows, 1), generator=generator, device="cuda").clamp_(max=2)  # (half of them to expert 2)
    experts[:300] = -1
    experts[1000] = 5
    experts[2000:2300] = 6
    routing = layers.routing(experts, number)
    total = int(routing.offsets[-1])
    assert total == rows - 300
    weight = random((number, outputs, channels), 3, TYPES[dtype]).requires_grad_(True)
    bias = random((number, outputs), 4, TYPES[dtype]).requires_grad_(True)
    for extra in (0, 8, 3):
        x, grad = random((rows, channels + extra), 1, TYPES[dtype])[:, :channels], random((rows, outputs + extra), 2, TYPES[dtype])[:, :outputs]
        x[total:] = math.nan
        grad[total:] = math.nan
        x.requires_grad_(True)
        y = layers.expert_linear(x, weight, bias, routing)
        grads = dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, (x, weight, bias), grad)))
        want = products(x, weight, bias, grad, routing.offsets.tolist())
        for name, got in {"y": y, **grads}.items():
            value, magnitude, chain = want[name]
            assert_within(got, value, chain * ref.U * magnitude + ref.half_step(value, TYPES[dtype]), name)


def test_without_gradients_and_under_autocast():
    given = decoder_inputs(200, 4, 1, torch.bfloat16)
    want = decoder(*given)
    for context in (torch.no_grad(), torch.inference_mode(), torch.autocast("cuda", dtype=torch.float16)):
        with context:
            assert torch.equal(decoder(*given), want)
    # a routing made in inference mode is saved like any other tensor made there: not at all
    leaf = given[0].clone().requires_grad_(True)
    with torch.inference_mode():
        _, routing = layers.route(given[1], 2)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        layers.dispatch(leaf, routing)
    # what the backward reads is not to be changed before
    weights, routing = layers.route(given[1].clone().requires_grad_(True), 2)
    total = weights.sum()
    routing.experts.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        total.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_sweep_trains_a_decoder_of_experts_with_both(dtype):
    from permutohedral_encoding_amd import perf_sweep
    rows = perf_sweep.experts(1000, 3, 1, width=40, number=5, dtype=dtype, levels=6, log2_capacity=10)
    assert [r["layers"] for r in rows] == ["torch", "layers"] and all(r["train"] > 0 for r in rows)
