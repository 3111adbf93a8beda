"""Sums of the layers of experts whose every partial sum is a whole number that float32 holds, so that any order gives the same: results have to be the sum of 64 bits, rounded once.

A row that is lost, doubled or read from next to where it is changes them, which a tolerance that grows with the rows does not see."""
import math

import pytest
import torch

from permutohedral_encoding_amd import layers
from settled_memory import settle
from test_gpu_experts import TYPES, chosen_experts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_is_settled():
    settle()
    yield
    settle()


def whole(shape, seed, dtype, most=2):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=generator, device="cuda").to(dtype)


def uneven_experts(rows, number, seed=0, none=300):
    """Half of the rows to the last expert, one row to expert 1, none to expert 0 (from three experts on), and some without an expert."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    e = torch.randint(0, number, (rows, 1), generator=generator, device="cuda")
    e = torch.where(torch.rand((rows, 1), generator=generator, device="cuda") < 0.5, number - 1, e)
    if number > 2:
        e[e < 2] = 2
        e[rows // 2] = 1
    e[torch.randperm(rows, generator=generator, device="cuda")[:min(none, rows // 10)]] = -1
    return e


def check_whole(rows, number, channels, outputs, dtype, extra=(0, 0), bias=True, seed=0):
    routing = layers.routing(uneven_experts(rows, number, seed), number)
    offsets = routing.offsets.tolist()
    x, grad = whole((rows, channels + extra[0]), seed + 1, dtype)[:, :channels], whole((rows, outputs + extra[1]), seed + 2, dtype)[:, :outputs]
    weight, b = whole((number, outputs, channels), seed + 3, dtype), whole((number, outputs), seed + 4, dtype)
    assert 4 * max(rows, channels, outputs) + 2 < 1 << 24
    xd, gd, wd, bd = (t.double() for t in (x, grad, weight, b))
    want = {"y": torch.zeros((rows, outputs), dtype=torch.float64, device="cuda"), "dx": torch.zeros((rows, channels), dtype=torch.float64, device="cuda"),
            "dweight": torch.zeros_like(wd), "dbias": torch.zeros_like(bd)}
    for e in range(number):
        at = slice(offsets[e], offsets[e + 1])
        want["y"][at] = xd[at] @ wd[e].t() + (bd[e] if bias else 0.0)
        want["dx"][at] = gd[at] @ wd[e]
        want["dweight"][e] = gd[at].t() @ xd[at]
        want["dbias"][e] = gd[at].sum(0)
    x[offsets[-1]:] = math.nan  # (what stands in rows without an expert is not read)
    grad[offsets[-1]:] = math.nan
    given = [t.requires_grad_(True) for t in ((x, weight, b) if bias else (x, weight))]
    y = layers.expert_linear(x, weight, b if bias else None, routing)
    got = {"y": y.detach(), **dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, given, grad)))}
    for name, g in got.items():
        wrong = g != want[name].to(dtype)
        assert not bool(wrong.any()), f"{name}: {int(wrong.sum())} of {wrong.numel()} values, the first at {wrong.nonzero()[0].tolist()}"
    # each gradient alone goes its own way
    for k, name in enumerate(("dx", "dweight", "dbias")[:len(given)]):
        alone = [t.detach().requires_grad_(i == k) for i, t in enumerate(given)]
        y = layers.expert_linear(alone[0], alone[1], alone[2] if bias else None, routing)
        assert torch.equal(torch.autograd.grad(y, alone[k], grad)[0], want[name].to(dtype)), name


# Rows of an expert are cut for the weights' gradient, in tiles of 64, 128 and (16-bit types) 256.  `extra`: how much further apart rows of x and of the gradient are than they are long: with 3 they
# begin anywhere.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(70001, 2, 64, 64), (40001, 5, 24, 56), (50000, 1, 48, 130), (40000, 3, 128, 128), (100000, 40, 136, 136), (30000, 3, 200, 264), (100003, 7, 512, 512),
                                                          (65537, 1, 1024, 1024)])
@pytest.mark.parametrize("extra", [(0, 0), (3, 5), (8, 3)])
def test_experts_of_many_rows(dtype, rows, number, channels, outputs, extra):
    check_whole(rows, number, channels, outputs, TYPES[dtype], extra)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(30000, 2, 3, 200), (30000, 2, 200, 3), (30000, 3, 5, 6), (30000, 2, 1, 64), (20000, 2, 130, 1), (40000, 3, 101, 130), (30011, 4, 264, 1032)])
def test_experts_of_odd_sizes(dtype, rows, number, channels, outputs):
    check_whole(rows, number, channels, outputs, TYPES[dtype])
    check_whole(rows, number, channels, outputs, TYPES[dtype], extra=(1, 2), bias=False, seed=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(1000, 3, 512, 512), (4000, 4, 512, 512), (500, 1, 4096, 64), (1257, 82, 2048, 24), (20, 6, 1024, 264), (300, 100, 64, 64), (1, 1, 65, 63), (129, 2, 129, 129),
                                                          (63, 1, 512, 200), (64, 1, 200, 512), (65, 1, 512, 512), (513, 1, 136, 200)])
def test_experts_of_few_rows(dtype, rows, number, channels, outputs):
    check_whole(rows, number, channels, outputs, TYPES[dtype])
    check_whole(rows, number, channels, outputs, TYPES[dtype], extra=(3, 1), seed=7)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,number,channels,outputs", [(140000, 2, 1024, 72), (140000, 2, 1032, 128), (140000, 1, 264, 1024), (70000, 3, 1024, 1040)])
def test_wide_tiles_of_results(dtype, rows, number, channels, outputs):
    check_whole(rows, number, channels, outputs, TYPES[dtype])


# Rows of a few bytes go in pieces of 2, 4 and 8 values; rows that are whole lines of 64 bytes, or long, go past the caches.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [1, 2, 3, 4, 5, 6, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 64, 200, 256, 500, 511, 512, 1000, 1024, 2049])
@pytest.mark.parametrize("choices", [1, 2, 3, 8])
def test_rows_there_and_back(dtype, channels, choices):
    rows, number, dtype = 1003, 6, TYPES[dtype]
    experts = chosen_experts(rows, choices, number, seed=channels)
    routing = layers.routing(experts, number)
    there, flat = experts >= 0, routing.positions.view(-1).long()
    items = rows * choices
    assert torch.equal(torch.sort(flat).values, torch.arange(items, device="cuda"))

    def sort(t):
        out = torch.empty((items, channels), dtype=t.dtype, device="cuda")
        out[flat] = torch.where(there[:, :, None], t, 0).reshape(items, channels)
        return out

    def back(t):
        return torch.where(there[:, :, None], t[flat].view(rows, choices, channels), 0)

    x, y, weights = whole((rows, channels), 1, dtype), whole((items, channels), 2, dtype), whole((rows, choices), 3, torch.float32, most=3)
    grad_sorted, grad_out = whole((items, channels), 4, dtype), whole((rows, channels), 5, dtype)
    total = int(routing.offsets[-1])
    y[total:] = math.nan
    grad_sorted[total:] = math.nan
    for t in (x, y, weights):
        t.requires_grad_(True)
    ordered, out = layers.dispatch(x, routing), layers.combine(y, weights, routing)
    got = dict(zip(("dx", "dy", "dweights"), torch.autograd.grad((ordered, out), (x, y, weights), (grad_sorted, grad_out))))
    yd, wd, gd = back(y.detach().double()), weights.detach().double()[:, :, None], grad_out.double()[:, None]
    want = {"sorted": sort(x.detach().double()[:, None].expand(-1, choices, -1)), "out": (yd * wd).sum(1), "dx": back(grad_sorted.double()).sum(1), "dy": sort(gd * wd), "dweights": (gd * yd).sum(2)}
    for name, g in dict(got, sorted=ordered.detach(), out=out.detach()).items():
        assert torch.equal(g, want[name].to(g.dtype)), name


# Sums of one sign, of values that are all alike: what is rounded away is of one sign, too.  A chain of n additions is off by n / 2 half steps, 2^-24 of the sum each, as its partial sums are half of
# it on average; 8192 products of fp32 are one chain, 65536 rows of 16-bit values 2048 additions of 32 products (which may be rounded twice).  Pieces are added in 64 bits; products of fp32 and the
# result are rounded once each.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(1 << 18, 8, 2048, 2048), (1 << 21, 1, 64, 64), (300000, 16, 1024, 1024)])
def test_long_sums_of_one_sign(dtype, rows, number, channels, outputs):
    dtype = TYPES[dtype]
    routing = layers.routing(torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), number)
    bound = (4096 + 2) * 2.0 ** -24 if dtype == torch.float32 else 2 * 1024 * 2.0 ** -24
    for a, b in ((1 / 3, 0.1), (1.0, 0.2504880859375), (0.7, 0.9)):
        a, b = (a, b) if dtype != torch.float16 else (a / 64, b / 64)
        x, grad = torch.full((1, channels), a, dtype=dtype, device="cuda").expand(rows, channels).contiguous(), torch.full((1, outputs), b, dtype=dtype, device="cuda").expand(rows, outputs).contiguous()
        weight, bias = (torch.zeros(s, dtype=dtype, device="cuda", requires_grad=True) for s in ((number, outputs, channels), (number, outputs)))
        y = layers.expert_linear(x.requires_grad_(True), weight, bias, routing)
        dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), grad)
        for name, got, want in (("dweight", dweight[0], rows * float(x[0, 0].detach()) * float(grad[0, 0])), ("dbias", dbias[0], rows * float(grad[0, 0]))):
            half = torch.finfo(dtype).eps / 2
            worst = float((got.double() - want).abs().max()) / want
            assert worst <= bound + half, f"{name}: {worst:.3g} of the sum, bound {bound + half:.3g}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,outputs", [(0, 3, 5), (1, 1, 1), (700, 5, 3), (513, 1, 16), (4000, 1000, 17), (100001, 4, 1), (70001, 13, 130), (1 << 20, 2, 65), (600000, 1, 7), (200000, 200, 33), (150001, 1024, 20)])
def test_the_gradient_of_the_biases_alone(dtype, rows, number, outputs):
    """Neither x nor the weights are needed for it, and x is not kept."""
    dtype = TYPES[dtype]
    routing = layers.routing(uneven_experts(rows, number) if rows > 3 else torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), number)
    offsets = routing.offsets.tolist()
    grad = whole((rows, outputs + 3), 2, dtype)[:, :outputs]
    want = torch.stack([grad[first:last].double().sum(0) for first, last in zip(offsets, offsets[1:])]).to(dtype)
    grad[offsets[-1]:] = math.nan
    x, weight, bias = whole((rows, 40), 1, dtype), whole((number, outputs, 40), 3, dtype), whole((number, outputs), 4, dtype).requires_grad_(True)
    y = layers.expert_linear(x, weight, bias, routing)
    with torch.no_grad():
        x += 1.0
    assert torch.equal(torch.autograd.grad(y, bias, grad, retain_graph=True)[0], want)
    # with the gradient of x, and by itself of a layer whose weights are trained too
    x.requires_grad_(True)
    y = layers.expert_linear(x, weight, bias, routing)
    both = torch.autograd.grad(y, (x, bias), grad)
    assert torch.equal(both[1], want)
    y = layers.expert_linear(x, weight.requires_grad_(True), bias, routing)
    all_of_them = torch.autograd.grad(y, (x, weight, bias), grad, retain_graph=True)
    assert torch.equal(all_of_them[0], both[0]) and torch.equal(all_of_them[2], want) and torch.equal(torch.autograd.grad(y, bias, grad)[0], want)


def test_the_gradient_of_the_biases_alone_takes_no_room_for_the_weights():
    routing = layers.routing(torch.zeros((4096, 1), dtype=torch.int32, device="cuda"), 4)
    x, weight, bias = torch.ones((4096, 1024), device="cuda"), torch.ones((4, 1024, 1024), device="cuda"), torch.zeros((4, 1024), device="cuda", requires_grad=True)
    y = layers.expert_linear(x, weight, bias, routing)
    grad = torch.ones_like(y)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    db, = torch.autograd.grad(y, bias, grad)
    assert torch.cuda.max_memory_allocated() - before <= 4 * weight.numel() // 8
    assert bool((db[0] == 4096.0).all()) and not bool(db[1:].any())


# Experts that a wave does not find in one step (more than 64 of them), of which some are cut and most are not.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(150001, 130, 64, 64), (150001, 130, 136, 72), (100000, 1024, 40, 48), (70000, 65, 203, 130), (150001, 200, 200, 264)])
def test_more_experts_than_a_wave_has_lanes(dtype, rows, number, channels, outputs):
    check_whole(rows, number, channels, outputs, TYPES[dtype])
    check_whole(rows, number, channels, outputs, TYPES[dtype], extra=(5, 3), seed=3)


# Layers whose experts' rows are one piece unless an expert has most of all, and tiles of results by how many there are.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,number,channels,outputs", [(16384, 16, 2048, 2048), (32768, 16, 1024, 1024), (30000, 5, 1001, 160), (70001, 13, 203, 190), (70001, 13, 190, 203)])
def test_layers_of_many_tiles(dtype, rows, number, channels, outputs):
    check_whole(rows, number, channels, outputs, TYPES[dtype])


def test_the_gradient_of_the_biases_alone_in_two_graphs():
    """Of rows that are cut: each graph has sums of its own."""
    rows, number, outputs = 20000, 3, 40
    routing = layers.routing(uneven_experts(rows, number), number)
    offsets = routing.offsets.tolist()
    x, weight = torch.zeros((rows, 8), device="cuda"), torch.zeros((number, outputs, 8), device="cuda")
    given, graphs, results = [], [], []
    for k in range(2):
        bias, grad = torch.zeros((number, outputs), device="cuda", requires_grad=True), whole((rows, outputs), k, torch.float32)
        stream = torch.cuda.Stream()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            results.append(torch.autograd.grad(layers.expert_linear(x, weight, bias, routing), bias, grad)[0])
        given.append((grad, stream))
    for seed in range(3):
        for k, (grad, _) in enumerate(given):
            grad.copy_(whole((rows, outputs), 10 * seed + k, torch.float32))
        torch.cuda.synchronize()
        for graph, (_, stream) in zip(graphs, given):
            with torch.cuda.stream(stream):
                graph.replay()
        wanted = [torch.stack([grad[a:b].double().sum(0) for a, b in zip(offsets, offsets[1:])]).float() for grad, _ in given]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, wanted))
