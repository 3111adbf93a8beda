"""Orthogonalised updates on the GPU: what results of few bits are off by, and the way of half as many bits.

A result of 16 bits should be its value rounded once: off by half a step at the value's own magnitude, and by what the steps leave before that.  Those are measured as in
test_gpu_orthogonal.py, by the same steps in float32: eight times their error, and 144 roundings of float32.  A single value is off by at most 16 times the mean of that."""
import math

import pytest
import torch

import expert_reference as ref
from permutohedral_encoding_amd import optim
from settled_memory import settle
from test_gpu_orthogonal import TYPES, assert_orthogonalised, norms, updates

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_is_settled():
    settle()
    yield
    settle()


def step_of(values, dtype):
    """The distance of neighbouring numbers of a type, at each value's magnitude."""
    info = torch.finfo(dtype)
    exponent = torch.frexp(values.abs().clamp(min=info.smallest_normal)).exponent - 1
    return torch.ldexp(torch.full_like(values, info.eps), exponent)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("matrices,rows,columns", [(1, 130, 130), (1, 203, 1000), (1, 1000, 203), (2, 257, 513), (1, 2100, 161), (3, 300, 700), (8, 512, 512), (33, 531, 390), (2, 2048, 1024), (16, 64, 256),
                                                   (2, 48, 1000)])
def test_results_of_16_bits_are_rounded_once(dtype, matrices, rows, columns):
    dtype = TYPES[dtype]
    update = updates(matrices, rows, columns, dtype)
    for given in (dict(), dict(steps=2), dict(coefficients=(1.875, -1.25, 0.375), steps=4)):
        want = ref.orthogonalise(update, **given)
        allowed = 8 * norms(ref.orthogonalise(update, dtype=torch.float32, **given).double() - want) + 144 * ref.U * norms(want)
        behind = ((optim.orthogonalise(update, **given).double() - want).abs() - step_of(want, dtype) / 2).clamp(min=0.0)
        worst = 16 * allowed / math.sqrt(rows * columns)
        assert bool((behind.amax((-1, -2)) <= worst).all()), f"{given}: worst error behind half a step/bound {float((behind.amax((-1, -2)) / worst).max()):.3g}"


@pytest.mark.parametrize("matrices,rows,columns", [(1, 130, 130), (1, 203, 1000), (1, 1000, 203), (40, 520, 530), (16, 64, 256), (1, 2100, 161), (1, 20, 3000)])
def test_halves(matrices, rows, columns):
    """X, S and the factor in float16, as the definition does with them; other types take no notice."""
    update = updates(matrices, rows, columns, torch.bfloat16)
    want = ref.orthogonalise(update)
    got = optim.orthogonalise(update, halves=True)
    allowed = 4 * norms(ref.orthogonalise(update, stored=ref.in_float16) - want) + norms(ref.half_step(want, torch.bfloat16))
    assert got.dtype == torch.bfloat16 and bool((norms(got.double() - want) <= allowed).all())
    assert torch.equal(optim.orthogonalise(update, halves=True), got)
    for dtype in (torch.float32, torch.float16):
        assert torch.equal(optim.orthogonalise(update.to(dtype), halves=True), optim.orthogonalise(update.to(dtype)))


def test_muon_in_halves():
    start = updates(2, 160, 200, torch.bfloat16, seed=1, scale=0.1)
    grad = updates(2, 160, 200, torch.bfloat16, seed=2)
    for halves in (False, True):
        p = torch.nn.Parameter(start.clone())
        opt = optim.Muon([p], lr=0.02, momentum=0.0, nesterov=False, weight_decay=0.0, halves=halves)
        p.grad = grad.clone()
        opt.step()
        # (the average of one step without momentum is the gradient itself)
        assert torch.equal(p.detach(), (start.float() - torch.tensor(0.02 * math.sqrt(1.0)).cuda() * optim.orthogonalise(grad, halves=halves).float()).bfloat16())
    # state that was saved without it
    saved = opt.state_dict()
    for group in saved["param_groups"]:
        del group["halves"]
    again = optim.Muon([p], lr=0.02)
    again.load_state_dict(saved)
    again.step()
    assert again.param_groups[0]["halves"] is False


@pytest.mark.parametrize("matrices,rows,columns", [(7, 300, 140), (9, 203, 131), (6, 129, 130), (70, 200, 5), (5, 64, 48)])
@pytest.mark.parametrize("dtype", TYPES)
def test_as_many_matrices_as_the_workspace_has_room_for(monkeypatch, dtype, matrices, rows, columns):
    """(131 * 203 values are odd: four matrices at a time at the least)"""
    update = updates(matrices, rows, columns, TYPES[dtype])
    for most in (0, 1 << 20, 3 << 20):
        monkeypatch.setattr(optim, "WORKSPACE_BYTES", most)
        assert_orthogonalised(optim.orthogonalise(update), update)
        assert_orthogonalised(optim.orthogonalise(update, steps=8), update, steps=8)
    monkeypatch.setattr(optim, "WORKSPACE_BYTES", -1)
    with pytest.raises(ValueError, match="negative"):
        optim.orthogonalise(update)


def test_muon_takes_the_parameters_of_a_size_in_several_parts(monkeypatch):
    start = [updates(2, 40, 30, torch.float32, seed=i, scale=0.1) for i in range(5)]
    grads = [updates(2, 40, 30, torch.float32, seed=10 + i) for i in range(5)]
    results = []
    for most in (4 << 30, 0, 2 * 2 * 2 * 40 * 30 * 4):  # all at once, each alone, two at a time
        monkeypatch.setattr(optim, "WORKSPACE_BYTES", most)
        params = [torch.nn.Parameter(s.clone()) for s in start]
        opt = optim.Muon(params, lr=0.02)
        for _ in range(2):
            for p, g in zip(params, grads):
                p.grad = g.clone()
            opt.step()
        results.append([t for p in params for t in (p.detach(), opt.state[p]["momentum_buffer"])])
    assert all(torch.equal(a, b) for other in results[1:] for a, b in zip(results[0], other))


def test_thin_matrices_take_no_more_than_their_sums():
    """2^24 values in matrices of one column: 16 GB if they went as large ones do."""
    update = updates(4096, 4096, 1, torch.float32)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = optim.orthogonalise(update)
    assert torch.cuda.max_memory_allocated() - before <= 10 * 4 * update.numel()
    assert_orthogonalised(got, update)


def test_a_refused_step_changes_nothing():
    """Whatever is refused, in whichever group: parameters, averages and their versions stay as they are, and the next step is the one that it would have been."""
    def refused_options(p, opt):
        opt.param_groups[1]["coefficients"] = (4.0, 0.0, 0.0)
        return ValueError, "coefficients"

    def refused_eps(p, opt):
        opt.param_groups[1]["eps"] = 0.0
        return ValueError, "eps"

    def refused_type(p, opt):
        p[2].data = p[2].data.double()
        p[2].grad = torch.ones_like(p[2])
        return ValueError, "type"

    def refused_gradient(p, opt):
        p[2].grad = p[2].grad.to_sparse()
        return RuntimeError, "dense"

    def refused_layout(p, opt):
        p[2].data = p[2].data.t().contiguous().t()
        return RuntimeError, "contiguous"

    for refusal in (refused_options, refused_eps, refused_type, refused_gradient, refused_layout):
        for steps_before in (0, 1):
            params = [torch.nn.Parameter(updates(1, 40, 30, torch.float32, seed=i, scale=0.1)[0]) for i in range(3)]
            opt = optim.Muon([dict(params=params[:2]), dict(params=params[2:])], lr=0.02)
            for p in params:
                p.grad = updates(1, 40, 30, torch.float32, seed=7)[0]
            for _ in range(steps_before):
                opt.step()
            kept = [p.detach().clone() for p in params[:2]]
            averages = [opt.state[p]["momentum_buffer"].clone() if steps_before else None for p in params]
            versions = [p._version for p in params[:2]]
            error, message = refusal(params, opt)
            with pytest.raises(error, match=message):
                opt.step()
            assert all(torch.equal(p, k) for p, k in zip(params, kept)) and versions == [p._version for p in params[:2]]
            assert all(torch.equal(opt.state[p]["momentum_buffer"], a) if steps_before else not opt.state.get(p) for p, a in zip(params, averages))
    # a single group, and one matrix
    p = torch.nn.Parameter(updates(1, 40, 30, torch.float32, scale=0.1)[0])
    opt = optim.Muon([p], lr=0.02)
    p.grad = torch.ones_like(p)
    opt.step()
    average = opt.state[p]["momentum_buffer"].clone()
    opt.param_groups[0]["coefficients"] = (4.0, 0.0, 0.0)
    with pytest.raises(ValueError, match="coefficients"):
        opt.step()
    assert torch.equal(opt.state[p]["momentum_buffer"], average)


@pytest.mark.parametrize("shape", [(3, 40, 60), (2, 140, 150), (2, 300, 140), (2, 500, 3)])
def test_coefficients_at_the_limits(shape):
    """2.4 times the Chebyshev polynomial of degree 5 has a factor of 15 below (at singular values of sqrt(5/8)), and 3 s is the most that is made of a singular value.  A few directions have all of the
    norm, so that there are such singular values."""
    rank = min(3, *shape[1:])
    for seed in range(3):
        kw = dict(generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        sizes = torch.tensor([0.79, 0.5, 0.35], device="cuda")[:rank]
        left, right = (torch.linalg.qr(torch.randn((shape[0], n, rank), **kw)).Q for n in shape[1:])
        update = (left * sizes) @ right.transpose(-1, -2).contiguous() + 1e-4 * torch.randn(shape, **kw) / math.sqrt(shape[1])
        for coefficients in ((11.99, -47.96, 38.368), (-11.99, 47.96, -38.368), (3.0, 0.0, 0.0), (2.0, 1.0, 0.0)):
            for dtype in TYPES.values():
                given = update.to(dtype)
                assert_orthogonalised(optim.orthogonalise(given, coefficients=coefficients, steps=1), given, coefficients=coefficients, steps=1)
                if dtype == torch.bfloat16:
                    assert_orthogonalised(optim.orthogonalise(given, coefficients=coefficients, steps=1, halves=True), given, coefficients=coefficients, steps=1)
    with pytest.raises(ValueError, match="coefficients"):
        optim.orthogonalise(update, coefficients=(12.02, -48.08, 38.464), steps=1)


def test_parts_and_halves_in_graphs(monkeypatch):
    """Stacks that go in parts, one after the other in the same workspace, captured and replayed, with the way of 11 bits beside."""
    monkeypatch.setattr(optim, "WORKSPACE_BYTES", 1 << 20)
    for shape in ((7, 200, 150), (9, 201, 131), (200, 900, 3)):
        given = updates(*shape, torch.bfloat16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, halves = optim.orthogonalise(given), optim.orthogonalise(given, halves=True)
        for seed in range(3):
            given.copy_(updates(*shape, torch.bfloat16, seed=seed + 1))
            graph.replay()
            want, want_halves = optim.orthogonalise(given), optim.orthogonalise(given, halves=True)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(halves, want_halves)
            assert_orthogonalised(want, given)


def test_in_inference_mode_and_without_gradients():
    update = updates(2, 140, 150, torch.bfloat16)
    want = optim.orthogonalise(update)
    for context in (torch.no_grad(), torch.inference_mode(), torch.autocast("cuda", dtype=torch.float16)):
        with context:
            assert torch.equal(optim.orthogonalise(update), want)
