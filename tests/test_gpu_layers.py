"""The layers behind the encoding on the GPU, against their formulas in 64 bits (layer_reference.py).

Tolerances: a value in a checkpoint has to be equal.  K * 2^-24 * magnitude for what goes through K roundings in 32 bits (the magnitudes are those of
layer_reference.py), and half a step of the result's type.  K is 256 for the norms: a statistic is a chain of at most 16 additions in a lane, 6 over the
lanes of a wave and 8 over its waves, with a few roundings around it; a gradient of the branch has five of them behind it (both norms forward, both
back, and the statistics of the way back), at most 40 roundings each.  A sum over rows adds at most a rounding for each of them."""
import math

import pytest
import torch

import layer_reference as ref
from permutohedral_encoding_amd import layers

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
K = 256


def values(rows, channels, dtype, seed=0, wide=None):
    """Rows with channels of different sizes and a few values far out, as the first channels of rows of ``wide``."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(generator=generator, device="cuda")
    x = torch.randn((rows, wide or channels), **kw) * torch.exp(0.5 * torch.randn((1, wide or channels), **kw))
    x = x + (torch.rand(x.shape, **kw) < 0.01) * 20.0 * torch.randn((rows, 1), **kw)
    return x.to(dtype)[:, :channels]


def assert_near(got, want, magnitude, roundings, what):
    assert got.shape == want.shape, what
    error = (got.detach().double() - want).abs()
    bound = roundings * ref.U * magnitude + ref.half_step(want, got.dtype)
    assert torch.isfinite(want).all() and bool((error <= bound).all()), f"{what}: worst error/bound {float((error / bound).max()):.3g}"


# ------------------------------------------------------------------------------------------ checkpoints

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 7), (257, 16), (64, 31), (5, 32), (100, 33), (4097, 48), (9, 203), (2, 1024), (3, 4100)])
def test_checkpoint_holds_the_defined_values(dtype, rows, channels):
    for layout in ("rows", "slice", "channels"):
        x = values(rows, channels, TYPES[dtype], wide=channels + 5 if layout == "slice" else None)
        if layout == "channels":
            x = torch.empty_strided(x.shape, (1, rows + 3), dtype=x.dtype, device="cuda").copy_(x)
        kept = layers.checkpoint(x)
        q, e = ref.kept_arrays(x)
        pitch = kept.values.shape[1]
        padded = torch.nn.functional.pad(q, (0, max(0, pitch - q.shape[1])))[:, :pitch]
        assert torch.equal(kept.values.double(), padded), layout
        assert torch.equal(kept.exponents.double(), e + 127), layout
        assert torch.equal(kept.unpack().double(), ref.kept(x)) and kept.unpack().dtype == x.dtype
        assert torch.equal(kept.unpack(torch.float32).double(), ref.kept(x))


@pytest.mark.parametrize("channels_first", [False, True])
def test_checkpoint_at_the_borders(channels_first):
    tiny, top = 2.0 ** -149, 3.4028234e38
    rows = [[0.0], [-0.0, 0.0], [tiny], [tiny, -3 * tiny], [2.0 ** -126], [127.0 * 2.0 ** -126, 2.0 ** -126], [top], [-top, 1e30], [127.4999, 1.0], [127.5, 0.5],
            [-127.5, 1.5], [127.50001], [63.75], [64.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5], [1.9921874], [1.9921875], [255.0], [2.0 ** 120, 2.0 ** -120]]
    x = torch.zeros(len(rows), 40, device="cuda")
    for i, r in enumerate(rows):
        x[i, : len(r)] = torch.tensor(r, device="cuda")
    x[:, 32:] = 1.0  # the block beside them is its own
    given = torch.empty_strided(x.shape, (1, x.shape[0]), device="cuda").copy_(x) if channels_first else x
    assert torch.equal(layers.checkpoint(given).unpack().double(), ref.kept(x))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_block_that_is_not_finite_comes_back_as_nan_and_no_other(bad):
    for dtype in TYPES.values():
        x = values(70, 100, dtype)
        x[3, 40] = bad
        x[69, 99] = bad
        for given in (x, torch.empty_strided(x.shape, (1, 70), dtype=dtype, device="cuda").copy_(x)):
            back, want = layers.checkpoint(given).unpack(), ref.kept(x)
            assert torch.equal(torch.isnan(back), torch.isnan(want)) and int(torch.isnan(want).sum()) == 32 + 4
            assert torch.equal(torch.nan_to_num(back).double(), torch.nan_to_num(want))


def test_unpacking_to_float16_stays_finite():
    x = torch.tensor([[65504.0, -65504.0, 65472.0]], dtype=torch.float16, device="cuda")
    assert ref.kept(x).abs().max() == 65536.0  # which float16 does not have
    assert torch.equal(layers.checkpoint(x).unpack(), torch.tensor([[65504.0, -65504.0, 65504.0]], dtype=torch.float16, device="cuda"))
    assert torch.equal(layers.checkpoint(x).unpack(torch.float32).double(), ref.kept(x))


def test_checkpoint_of_other_shapes():
    x = values(24, 40, torch.float32)
    want = ref.kept(x)
    for given in (x.view(2, 3, 4, 40), x.view(2, 12, 40)[:, ::3], x.view(4, 6, 40).transpose(0, 1), x[::2], x[:, ::2], x[3], x[:0], x.t().contiguous().t()):
        kept = layers.checkpoint(given)
        flat = given.reshape(-1, given.shape[-1])
        assert kept.unpack().shape == given.shape
        assert torch.equal(kept.unpack().reshape(flat.shape).double(), ref.kept(flat) if flat.numel() else flat.double())
    expanded = x[:1].expand(9, 40)
    assert torch.equal(layers.checkpoint(expanded).unpack().double(), want[:1].expand(9, 40))
    for refused in (torch.zeros((), device="cuda"), torch.zeros(3, 0, device="cuda"), x.double(), x.int()):
        with pytest.raises(ValueError):
            layers.checkpoint(refused)


def test_checkpoint_behind_two_to_the_31_values():
    """Offsets of 4 GB in the rows and 2 GB in the checkpoint."""
    rows, channels = (1 << 20) + 3, 2080
    x = torch.zeros(rows, channels, dtype=torch.bfloat16, device="cuda")
    tail = values(100, channels, torch.bfloat16)
    x[-100:] = tail
    kept = layers.checkpoint(x)
    assert torch.equal(kept.unpack()[-100:].double(), ref.kept(tail))
    grad = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    grad[-1, 3] = 1.0
    assert torch.equal(kept.weight_grad(grad, dtype=torch.float32)[3].double(), ref.kept(tail)[-1])
    del x, grad
    y = layers.activation(torch.ones(1, 1, dtype=torch.bfloat16, device="cuda").expand(rows, channels), "silu")
    assert bool((y[-1] == y[0, 0]).all())


# ------------------------------------------------------------------------------------------ the weight gradient

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,outputs", [(0, 5, 3), (1, 1, 1), (1, 48, 64), (31, 33, 65), (257, 48, 64), (300, 200, 130), (4097, 32, 64), (1000, 64, 3),
                                                   (513, 8, 257), (70000, 48, 16), (2049, 129, 128),
                                                   (7, 300, 300), (8, 257, 130), (9, 70, 66), (600, 300, 520), (40000, 129, 257), (20011, 72, 90)])
def test_weight_grad(dtype, rows, channels, outputs):
    x = values(rows, channels, TYPES[dtype], wide=channels + 3)
    grad = values(rows, outputs, TYPES[dtype], seed=1, wide=outputs + 1)
    kept = layers.checkpoint(x)
    weight, bias = kept.weight_grad(grad, bias=True)
    assert weight.dtype == bias.dtype == TYPES[dtype] and weight.shape == (outputs, channels) and bias.shape == (outputs,)
    back, g = ref.kept(x) if rows else x.double(), grad.double()
    # Every product is exact.  A wave adds 32 (three parts: 96) of them at a time for each of its steps, at least 64 workgroups and waves share more rows than
    # 16384, and their sums are one more chain: with a factor of two for additions that do not round to nearest, 2 (rows / 64 + 2048).
    chain = 2 * (rows / 64 + 2048)
    full = kept.weight_grad(grad, bias=True, dtype=torch.float32)
    for got in ((weight, bias), full):
        assert_near(got[0], g.t().contiguous() @ back, g.abs().t().contiguous() @ back.abs(), chain, "weight")
        assert_near(got[1], g.sum(0), g.abs().sum(0), chain, "bias")
    assert all(torch.equal(a, b) for a, b in zip(full, kept.weight_grad(grad, bias=True, dtype=torch.float32)))
    assert torch.equal(kept.weight_grad(grad), weight)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("outputs", [1, 2, 3, 4, 15, 16, 17, 18, 31, 32, 33])
@pytest.mark.parametrize("rows,channels", [(8, 1), (9, 33), (265, 64), (5000, 130)])
def test_weight_grad_of_few_outputs(dtype, outputs, rows, channels):
    x = values(rows, channels, TYPES[dtype], seed=2)
    wide = values(rows, outputs, TYPES[dtype], seed=3, wide=outputs + 2).clone()
    storage = torch.full((rows, outputs + 2), math.nan, dtype=TYPES[dtype], device="cuda")  # what is beside the gradient is not read
    storage[:, 1:-1] = wide
    grad = storage[:, 1:-1]
    weight, bias = layers.checkpoint(x).weight_grad(grad, bias=True, dtype=torch.float32)
    back, g = ref.kept(x), wide.double()
    chain = 2 * (rows / 64 + 2048)  # (as above)
    assert_near(weight, g.t().contiguous() @ back, g.abs().t().contiguous() @ back.abs(), chain, "weight")
    assert_near(bias, g.sum(0), g.abs().sum(0), chain, "bias")
    assert torch.equal(weight, layers.checkpoint(x).weight_grad(wide, dtype=torch.float32))


def test_weight_grad_takes_gradients_whole():
    """Single rows: a product has to come back as it is, whatever the bits and the magnitude of the gradient; infinities and NaN stay in their row and column."""
    for dtype in TYPES.values():
        info = torch.finfo(dtype)
        specials = [1.0, 1.0 + info.eps, 2.0 - info.eps, -1.0 / 3.0, info.smallest_normal, info.max / 64, 0.0]
        grad = torch.tensor([specials], device="cuda").to(dtype)
        x = torch.ones(1, 3, device="cuda") * torch.tensor([1.0, -1.0, 0.5], device="cuda")
        got = layers.checkpoint(x.to(dtype)).weight_grad(grad, dtype=torch.float32)
        assert torch.equal(got.double(), grad.double().t() @ x.double())
        bad = torch.tensor([[1.0, math.inf, -math.inf, math.nan, 2.0]], device="cuda").to(dtype)
        weight, bias = layers.checkpoint(x.to(dtype)).weight_grad(bad, bias=True, dtype=torch.float32)
        want = bad.double().t() * x.double()
        assert torch.equal(torch.nan_to_num(weight.double(), 7.0), torch.nan_to_num(want, 7.0)), (dtype, weight)
        assert torch.equal(torch.nan_to_num(bias.double(), 7.0), torch.nan_to_num(bad.double()[0], 7.0))
    x = torch.ones(2, 40, device="cuda")
    x[1, 3] = math.nan  # the first block of the second row
    weight = layers.checkpoint(x).weight_grad(torch.tensor([[1.0], [1.0]], device="cuda"))
    assert torch.isnan(weight[0, :32]).all() and torch.equal(weight[0, 32:], torch.full((8,), 2.0, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("products,channels,outputs", [(150001, 300, 390), (1040001, 129, 129), (280009, 208, 300), (100003, 512, 336), (2205, 2900, 2700)])
def test_weight_grad_of_large_products(dtype, products, channels, outputs):
    """The tiles of 256 x 256, from 2^34 multiplications on (a value of fp32 counts three times, of fp16 twice): columns that fill no tile, rows that fill no step,
    split over workgroups and not (the last), results of each type, with and without a bias."""
    parts = {"fp32": 3, "fp16": 2, "bf16": 1}[dtype]
    rows = -(-products // parts)
    assert parts * rows * channels * outputs >= 1 << 34
    x = values(rows, channels, TYPES[dtype], wide=channels + 3)
    grad = (values(rows, outputs + 1, TYPES[dtype], seed=1) / math.sqrt(rows))[:, :outputs]
    kept = layers.checkpoint(x)
    back, g = ref.kept(x), grad.double()
    want = g.t().contiguous() @ back, g.sum(0)
    magnitude = g.abs().t().contiguous() @ back.abs(), g.abs().sum(0)
    # A wave adds all the rows of its workgroup, a row as often as it has parts: they are dealt out in units of 256 to as many workgroups of a tile as 256 in all
    # allow, whose sums are one more chain.  A factor of two for additions that do not round to nearest.
    splits = max(1, 256 // (-(-channels // 256) * -(-outputs // 256)))
    chain = 2 * (parts * (rows // splits + 512) + splits)
    for result in TYPES.values():
        weight, bias = kept.weight_grad(grad, bias=True, dtype=result)
        for got, value, m, what in zip((weight, bias), want, magnitude, ("weight", "bias")):
            assert got.dtype == result
            assert_near(got, value, m, chain, what)
        assert torch.equal(weight, kept.weight_grad(grad, dtype=result))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,outputs", [(3, 40, 5), (300, 70, 3), (40000, 48, 20), (40000, 48, 64), (150001, 300, 390)])
def test_weight_grad_of_blocks_at_the_top_of_the_range(dtype, rows, channels, outputs):
    """The largest step there is, beside zeros and ordinary rows: values as `unpack` has them, for gradients of every type in tiles of every size.  (Gradients
    are so small that no sum overflows: 1600 rows of 3.4e38 times at most 2^-24 * 128.)"""
    x = values(rows, channels, torch.float32, seed=4)
    top = torch.zeros(channels, device="cuda")
    top[:6] = torch.tensor([3.4028234e38, -3.4028234e38, 1.7e38, 0.0, -1e30, 1.0], device="cuda")
    top[-1] = -3.4e38
    x[::97] = top
    x[-1] = top
    grad = (values(rows, outputs, torch.float32, seed=5).clamp(-128, 128) * 2.0 ** -24).to(TYPES[dtype])
    kept = layers.checkpoint(x)
    back, g = kept.unpack().double(), grad.double()
    assert torch.isfinite(back).all() and torch.equal(back, ref.kept(x))
    weight = kept.weight_grad(grad, dtype=torch.float32)
    # A wave adds at most the rows of a workgroup, rows / 64 and the rest of a unit of 256, three times over where a gradient is in three parts, and their
    # sums are one more chain of at most 256; a factor of two for additions that do not round to nearest.
    assert_near(weight, g.t().contiguous() @ back, g.abs().t().contiguous() @ back.abs(), 2 * (3 * (rows / 64 + 256) + 256), "weight")


# ------------------------------------------------------------------------------------------ activations

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["gelu", "silu", "softplus"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,channels", [(1, 1), (5, 33), (300, 64), (3, 1000)])
def test_activation(dtype, kind, gated, rows, channels):
    """32 bits: the special functions are off by at most 16 units of their result (exp, erf, log1p), the rest is a few roundings, none of them
    amplified beyond |x| + 1: 64 * 2^-24 of (|x| + 1), times the other factors."""
    width = 2 * channels if gated else channels
    x = 3.0 * values(rows, width, TYPES[dtype], wide=width + 1)
    grad = values(rows, channels, TYPES[dtype], seed=1)
    for keep_8bit in (True, False):
        given = x.clone().requires_grad_(True) if rows > 1 else x.detach().requires_grad_(True)
        y = layers.activation(given, kind, gated=gated, keep_8bit=keep_8bit)
        dx, = torch.autograd.grad(y, given, grad)
        assert y.dtype == dx.dtype == TYPES[dtype] and dx.shape == x.shape
        a, b = (x[:, :channels].double(), x[:, channels:].double()) if gated else (x.double(), torch.ones((), dtype=torch.float64, device="cuda"))
        assert_near(y, ref.act(a, kind) * b, (a.abs() + 1) * b.abs(), 64, "y")
        if keep_8bit:
            a, b = (ref.kept(x[:, :channels]), ref.kept(x[:, channels:])) if gated else (ref.kept(x), b)
        g = grad.double()
        assert_near(dx[:, :channels], g * b * ref.act_slope(a, kind), g.abs() * b.abs() * (a.abs() + 1), 64, "da")
        if gated:
            assert_near(dx[:, channels:], g * ref.act(a, kind), g.abs() * (a.abs() + 1), 64, "db")
    with torch.no_grad():
        assert torch.equal(layers.activation(x, kind, gated=gated), y)


def test_softplus_of_small_results():
    """Relative to the result, down to where it is exp(x): exp 2 units, the logarithm 1, two products and a sum of half a unit each, the reciprocal's share
    far below: 5 units of 2^-23 at most, here 8.  (Left of 88 the sum is x and less than a unit more.)"""
    x = torch.cat([torch.linspace(-85.0, 88.0, 1 << 20, device="cuda"), torch.linspace(-18.0, -14.0, 1 << 18, device="cuda"),
                   torch.linspace(-1e-3, 1e-3, 1 << 16, device="cuda")])[None]
    want = ref.act(x.double(), "softplus")
    error = (layers.activation(x, "softplus").double() - want).abs() / want
    assert float(error.max()) <= 8 * 2.0 ** -23, float(error.max() * 2 ** 23)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(7, 24), (50, 70), (41, 96), (1, 130), (33, 200), (3, 2100), (2, 2080), (5, 5000), (2, 66001)])
def test_rows_of_any_length_share_lanes(dtype, rows, channels):
    """Lanes of a row that are no power of two, and rows that take several turns of a workgroup: a row's results are those of the row alone."""
    x = values(rows, channels, TYPES[dtype], seed=4, wide=channels + 3)
    kept = layers.checkpoint(x)
    q, e = ref.kept_arrays(x)
    assert torch.equal(kept.values[:, :channels].double(), q[:, :channels]) and torch.equal(kept.exponents.double(), e + 127)
    assert not kept.values[:, channels:].any() and torch.equal(kept.unpack(torch.float32).double(), ref.kept(x))
    x = x.detach().requires_grad_(True)
    y = layers.activation(x, "gelu")
    grad = values(rows, channels, TYPES[dtype], seed=5)
    dx, = torch.autograd.grad(y, x, grad)
    back = ref.kept(x.detach())
    assert_near(y, ref.act(x.detach().double(), "gelu"), x.detach().double().abs() + 1, 64, "y")
    assert_near(dx, grad.double() * ref.act_slope(back, "gelu"), grad.double().abs() * (back.abs() + 1), 64, "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 7), (1, 8), (2047, 1), (2049, 1), (683, 3), (686, 3), (2048, 5), (29, 212), (1 << 17, 33)])
def test_dense_rows_without_a_checkpoint_are_one_after_the_other(dtype, rows, channels):
    x, grad = values(rows, channels, TYPES[dtype], seed=6).contiguous(), values(rows, channels, TYPES[dtype], seed=7).contiguous()
    apart, grad_apart = (torch.full((rows, channels + 1), math.nan, dtype=t.dtype, device="cuda")[:, :channels].copy_(t) for t in (x, grad))
    for kind in ("silu", "softplus"):
        out = []
        for a, g in ((x, grad), (apart, grad_apart), (x, grad_apart)):
            leaf = a.detach().requires_grad_(True)
            y = layers.activation(leaf, kind, keep_8bit=False)
            out.append((y, layers.activation(a, kind), *torch.autograd.grad(y, leaf, g)))
        for y, alone, dx in out:
            assert torch.equal(y, out[1][0]) and torch.equal(alone, y) and torch.equal(dx, out[1][2])
        assert_near(out[0][0], ref.act(x.double(), kind), x.double().abs() + 1, 64, "y")


def test_activations_far_out():
    x = torch.tensor([[-1e30, -200.0, -90.0, -20.0, -0.0, 0.0, 20.0, 90.0, 200.0, 1e30]], device="cuda")
    for kind, below in (("gelu", 0.0), ("silu", 0.0), ("softplus", 0.0)):
        given = x.clone().requires_grad_(True)
        y = layers.activation(given, kind, keep_8bit=False)
        dx, = torch.autograd.grad(y, given, torch.ones_like(y))
        assert torch.isfinite(y).all() and torch.isfinite(dx).all(), kind
        assert torch.equal(y[0, 7:], x[0, 7:]) and torch.equal(dx[0, 7:], torch.ones(3, device="cuda")), kind
        assert y[0, :2].abs().max() == below and dx[0, :2].abs().max() == below, kind
        assert_near(y[:, 2:8], ref.act(x.double(), kind)[:, 2:8], x.double().abs()[:, 2:8] + 1, 64, kind)
    nan = torch.tensor([math.nan], device="cuda")
    assert all(torch.isnan(layers.activation(nan, kind)).all() for kind in ("gelu", "silu", "softplus"))


# ------------------------------------------------------------------------------------------ norms

NORM_SHAPES = [(1, 1), (5, 3), (300, 7), (3, 8), (2, 9), (7, 31), (129, 64), (65, 100), (33, 203), (50, 512), (9, 1000), (5, 1024), (6, 2048), (3, 2051), (5, 4096), (4, 8192), (2, 8191)]


def norm_case(rows, channels, dtype, params, kind, gate, seed=0):
    t, p = TYPES[dtype], TYPES[params]
    s = {"x": values(rows, channels, t, seed, wide=channels + 1), "f": values(rows, channels, t, seed + 1),
         "grad_y": values(rows, channels, t, seed + 2), "grad_n": values(rows, channels, t, seed + 3)}
    generator = torch.Generator(device="cuda").manual_seed(seed + 4)
    draw = lambda *sizes: torch.randn(sizes, generator=generator, device="cuda")  # noqa: E731
    s["gate"] = None if gate is None else (0.3 + 0.1 * draw(*((gate, channels) if gate else (channels,)))).to(p)
    s["post_weight"], s["pre_weight"] = ((1.0 + 0.1 * draw(channels)).to(p) for _ in range(2))
    s["post_bias"], s["pre_bias"] = ((0.1 * draw(channels)).to(p) if kind == "layer" else None for _ in range(2))
    return s


def check_norm(s, keep_8bit=True, **options):
    names = [k for k in ("x", "f", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[k] is not None]
    given = {k: s[k].detach().requires_grad_(True) for k in names}
    kw = {k: v for k, v in given.items() if k not in ("x", "f")}
    y, n = layers.residual_norm(given["x"], given["f"], residual_scale=0.75, keep_8bit=keep_8bit, **kw, **options)
    grads = dict(zip(names, torch.autograd.grad((y, n), list(given.values()), (s["grad_y"], s["grad_n"]))))
    back = {"x_back": ref.kept(s["x"]), "f_back": ref.kept(s["f"])} if keep_8bit else {"x_back": s["x"], "f_back": s["f"]}
    want = ref.residual_norm(s["x"], s["f"], s["grad_y"], s["grad_n"], scale=0.75, **{k: s[k] for k in kw}, **options, **back)
    rows = s["x"].shape[0]
    for name, got in [("y", y), ("n", n)] + [({"f": "branch"}.get(k, k), g) for k, g in grads.items()]:
        assert got.dtype == (s["x"].dtype if name in ("y", "n", "x", "branch") else s[name].dtype)
        over_rows = name not in ("y", "n", "x", "branch")
        assert_near(got, *want[name], K + (rows if over_rows else 0), name)
    return y, n, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,channels", NORM_SHAPES)
def test_residual_norm(dtype, kind, rows, channels):
    if channels == 1 and kind == "layer":
        eps = 1e-2  # (one channel less its mean is zero: nothing but the bias is left)
    else:
        eps = 1e-6
    s = norm_case(rows, channels, dtype, "fp32" if rows % 2 else dtype, kind, gate=0)
    first = check_norm(s, kind=kind, eps=eps)
    again = check_norm(s, kind=kind, eps=eps)
    assert all(torch.equal(a, b) for a, b in zip(first[:2], again[:2])) and all(torch.equal(first[2][k], again[2][k]) for k in first[2])
    check_norm(s, kind=kind, eps=eps, keep_8bit=False)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,groups,channels", [(40, 40, 48), (40, 20, 48), (42, 6, 64), (700, 1, 32), (1280, 10, 100), (3000, 3, 203), (6, 3, 2048), (12, 2, 5000),
                                                  (90, 90, 1000), (20000, 2, 16), (4, 4, 4096)])
def test_gates_of_groups_of_rows(kind, rows, groups, channels):
    for params in ("fp32", "bf16"):
        check_norm(norm_case(rows, channels, "bf16", params, kind, gate=groups), kind=kind)


def test_many_rows():
    """More rows than the card takes at a time, in both layouts of gates."""
    for gate in (0, 1023):
        check_norm(norm_case(1023 * 41, 64, "fp32", "fp32", "rms", gate=gate))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_parts_of_a_residual_norm(kind):
    s = norm_case(37, 72, "fp32", "fp32", kind, gate=0)
    x, f, gy, gn = s["x"], s["f"], s["grad_y"], s["grad_n"]
    back = {"x_back": ref.kept(x), "f_back": ref.kept(f)}

    def leaves(*names):
        return {k: s[k].detach().requires_grad_(True) for k in names if s[k] is not None}

    # without a norm of the branch, without parameters
    t = leaves("x", "f")
    y, n = layers.residual_norm(t["x"], t["f"], post_norm=False, kind=kind)
    want = ref.residual_norm(x, f, gy, gn, post_norm=False, kind=kind, **back)
    grads = torch.autograd.grad((y, n), list(t.values()), (gy, gn))
    for name, got in zip(("y", "n", "x", "branch"), (y, n, *grads)):
        assert_near(got, *want[name], K, name)
    # without the norm before the next block
    t = leaves("x", "f", "gate", "post_weight", "post_bias")
    y = layers.residual_norm(t["x"], t["f"], gate=t["gate"], post_weight=t["post_weight"], post_bias=t.get("post_bias"), pre_norm=False, kind=kind)
    want = ref.residual_norm(x, f, gy, None, gate=s["gate"], post_weight=s["post_weight"], post_bias=s["post_bias"], pre_norm=False, kind=kind, **back)
    assert_near(y, *want["y"], K, "y")
    for (name, leaf), got in zip(t.items(), torch.autograd.grad(y, list(t.values()), gy)):
        name = {"f": "branch"}.get(name, name)
        assert_near(got, *want[name], K + 37, name)
    # a result that nothing uses, and a gradient that nothing wants
    t = leaves("x", "f", "gate", "pre_weight")
    for pick, upstream in ((0, (gy, None)), (1, (None, gn))):
        out = layers.residual_norm(t["x"], t["f"], gate=t["gate"], pre_weight=t["pre_weight"], kind=kind)[pick]
        want = ref.residual_norm(x, f, *upstream, gate=s["gate"], pre_weight=s["pre_weight"], kind=kind, **back)
        got = torch.autograd.grad(out, [t["f"], t["pre_weight"]], upstream[pick], allow_unused=True)
        assert_near(got[0], *want["branch"], K, "branch")
        if pick:
            assert_near(got[1], *want["pre_weight"], K + 37, "pre_weight")
        else:
            assert got[1] is None or float(got[1].abs().max()) == 0.0
    # the norm of a tensor alone
    t = leaves("x", "pre_weight", "pre_bias")
    n = layers.norm(t["x"], t["pre_weight"], t.get("pre_bias"), kind=kind)
    want = ref.residual_norm(x, None, None, gn, pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], kind=kind, x_back=back["x_back"])
    assert_near(n, *want["n"], K, "n")
    for (name, leaf), got in zip(t.items(), torch.autograd.grad(n, list(t.values()), gn)):
        assert_near(got, *want[name], K + 37, name)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("given", ["", "gate", "post_weight", "post_bias", "pre_weight", "post_weight pre_weight", "post_bias pre_bias", "gate post_bias",
                                   "gate post_weight post_bias pre_weight pre_bias"])
def test_parameters_that_are_not_given(dtype, kind, given):
    """They count as 1 (a bias: 0) in the row, and for nothing in the lanes behind its end; with upstream gradients whose mean is not zero."""
    for rows, channels in ((5, 3), (9, 8), (2, 9), (7, 48), (33, 64), (33, 72), (33, 203), (9, 520), (9, 1000), (5, 1024), (2, 2051), (3, 5000)):
        s = norm_case(rows, channels, dtype, "fp32", kind, gate=0)
        generator = torch.Generator(device="cuda").manual_seed(8)
        for name in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias"):
            if name not in given.split():
                s[name] = None
            elif s[name] is None:
                s[name] = 0.1 * torch.randn(channels, generator=generator, device="cuda")
        s["grad_y"], s["grad_n"] = s["grad_y"] + 0.5, s["grad_n"] + 1.0
        for keep_8bit in (True, False):
            check_norm(s, kind=kind, keep_8bit=keep_8bit)


@pytest.mark.parametrize("per_gate", [1, 4, 300])
def test_groups_of_rows_without_a_gate(per_gate):
    """Through the C ABI: rows_per_gate and no gate is a gate of ones."""
    import ctypes

    from permutohedral_encoding_amd import _native
    from test_layers import Norm, NormGrads
    lib, stream = _native.lib(), torch.cuda.current_stream().cuda_stream
    s = norm_case(600, 72, "fp32", "fp32", "layer", gate=None)
    x, f = s["x"].contiguous(), s["f"].contiguous()
    want = layers.residual_norm(x.requires_grad_(True), f.requires_grad_(True), kind="layer", keep_8bit=False)
    want += torch.autograd.grad(want, (x, f), (s["grad_y"], s["grad_n"]))
    y, n, dx, df = got = [torch.empty_like(x) for _ in range(4)]
    dy, dn = s["grad_y"].contiguous(), s["grad_n"].contiguous()
    norm = Norm(0, 0, 0, 1, 1, 1, 1.0, 1e-6, 600, 72, per_gate, x.data_ptr(), 72, f.data_ptr(), 72, 1)
    grads = NormGrads(dy.data_ptr(), 72, dn.data_ptr(), 72, dx.data_ptr(), df.data_ptr())
    nbytes = lib.penc_residual_norm_workspace_bytes(600, 72, per_gate)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    assert lib.penc_residual_norm(ctypes.byref(norm), y.data_ptr(), n.data_ptr(), stream) == 0
    assert lib.penc_residual_norm_backward(ctypes.byref(norm), ctypes.byref(grads), workspace.data_ptr(), nbytes, stream) == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_row_of_zeros_has_a_norm():
    x = torch.zeros(4, 64, device="cuda", requires_grad=True)
    f = torch.zeros(4, 64, device="cuda", requires_grad=True)
    for kind in ("rms", "layer"):
        y, n = layers.residual_norm(x, f, kind=kind)
        grads = torch.autograd.grad((y, n), (x, f), (torch.ones_like(y), torch.ones_like(n)))
        assert not y.any() and not n.any() and all(torch.isfinite(g).all() for g in grads)


def test_a_row_with_a_nan_leaves_the_others_alone():
    s = norm_case(9, 80, "bf16", "fp32", "rms", gate=9)
    s["f"][4, 3] = math.inf
    given = {k: s[k].detach().requires_grad_(True) for k in ("x", "f", "gate")}
    y, n = layers.residual_norm(given["x"], given["f"], gate=given["gate"])
    grads = torch.autograd.grad((y, n), list(given.values()), (s["grad_y"], s["grad_n"]))
    others = [0, 1, 2, 3, 5, 6, 7, 8]
    for t in (y, n, *grads):
        assert torch.isfinite(t[others]).all() and torch.isnan(t[4]).any()


def test_shapes_of_gates():
    x, f = values(60, 24, torch.float32), values(60, 24, torch.float32, seed=1)
    gate = torch.rand(5, 24, device="cuda")
    want = layers.residual_norm(x, f, gate=gate, pre_norm=False)
    wide = gate.repeat_interleave(12, 0)
    assert torch.equal(want, layers.residual_norm(x, f, gate=wide, pre_norm=False))
    x3, f3 = x.view(5, 12, 24), f.view(5, 12, 24)
    assert torch.equal(want.view(5, 12, 24), layers.residual_norm(x3, f3, gate=gate.view(5, 1, 24), pre_norm=False))
    assert torch.equal(want.view(5, 12, 24), layers.residual_norm(x3, f3, gate=wide.view(5, 12, 24), pre_norm=False))
    one = layers.residual_norm(x3, f3, gate=gate[0], pre_norm=False)
    assert torch.equal(one, layers.residual_norm(x3, f3, gate=gate[:1].view(1, 1, 24), pre_norm=False))
    assert torch.equal(one.view(60, 24), layers.residual_norm(x, f, gate=gate[0].expand(60, 24), pre_norm=False))
    for bad in (torch.rand(7, 24), torch.rand(24, 1), torch.rand(1, 12, 24), torch.rand(12, 24), torch.rand(5, 12, 1), torch.rand(()), torch.rand(5, 12, 24, 24)):
        with pytest.raises(ValueError):
            layers.residual_norm(x3, f3, gate=bad.cuda(), pre_norm=False)


def test_what_a_norm_refuses():
    x, f = values(6, 24, torch.bfloat16), values(6, 24, torch.bfloat16, seed=1)
    w = torch.ones(24, device="cuda")
    for call in (lambda: layers.residual_norm(x, f[:3]), lambda: layers.residual_norm(x, f.float()), lambda: layers.residual_norm(x, f, post_weight=w[:23]),
                 lambda: layers.residual_norm(x, f, post_weight=w.half()), lambda: layers.residual_norm(x, f, post_weight=w, pre_weight=w.bfloat16()),
                 lambda: layers.residual_norm(x, f, pre_weight=w, pre_norm=False), lambda: layers.residual_norm(x, f, post_bias=w, post_norm=False),
                 lambda: layers.residual_norm(x, f, gate=w.half()), lambda: layers.norm(x, w.view(1, 24)), lambda: layers.norm(torch.zeros(2, 8193, device="cuda")),
                 lambda: layers.norm(x, w.cpu()), lambda: layers.activation(x[:, :23], gated=True), lambda: layers.linear(x, torch.ones(3, 24, device="cuda")),
                 lambda: layers.linear(x, x[:, :23]), lambda: layers.linear(x, x, x[0, :5]), lambda: layers.checkpoint(x).weight_grad(f[:3]),
                 lambda: layers.residual_norm(x, f, residual_scale=w[0]), lambda: layers.norm(x, eps=w[0]), lambda: layers.norm(torch._neg_view(x)),
                 lambda: layers.checkpoint(x).unpack(torch.float64), lambda: layers.checkpoint(x).weight_grad(f, dtype=torch.int8)):
        with pytest.raises(ValueError):
            call()


def test_no_rows():
    x = torch.zeros(0, 40, device="cuda", requires_grad=True)
    f = torch.zeros(0, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    gate = torch.ones(0, 40, device="cuda", requires_grad=True)
    weight = torch.ones(3, 40, device="cuda", requires_grad=True)
    bias = torch.ones(3, device="cuda", requires_grad=True)
    y, n = layers.residual_norm(x, f, gate=gate, pre_weight=w)
    out = layers.linear(layers.activation(n), weight, bias)
    (out.sum() + y.sum()).backward()
    assert out.shape == (0, 3) and gate.grad.shape == (0, 40) and x.grad.shape == f.grad.shape == (0, 40)
    assert not w.grad.any() and not weight.grad.any() and not bias.grad.any()
    batch = torch.zeros(2, 0, 40, device="cuda", requires_grad=True)
    per_batch = torch.ones(2, 1, 40, device="cuda", requires_grad=True)
    layers.residual_norm(batch, torch.zeros_like(batch), gate=per_batch, pre_norm=False).sum().backward()
    assert per_batch.grad.shape == (2, 1, 40) and not per_batch.grad.any()


# ------------------------------------------------------------------------------------------ linear, and the layers together

@pytest.mark.parametrize("dtype", TYPES)
def test_linear(dtype):
    x, w, b = values(130, 48, TYPES[dtype]), values(64, 48, TYPES[dtype], seed=1), values(1, 64, TYPES[dtype], seed=2)[0]
    grad = values(130, 64, TYPES[dtype], seed=3)
    for given in (x, x.view(2, 65, 48), torch.empty_strided(x.shape, (1, 130), dtype=x.dtype, device="cuda").copy_(x)):
        leaves = [t.detach().requires_grad_(True) for t in (given, w, b)]
        y = layers.linear(*leaves)
        torch.testing.assert_close(y, torch.nn.functional.linear(given, w, b))
        dx, dw, db = torch.autograd.grad(y, leaves, grad.view(y.shape))
        torch.testing.assert_close(dx, (grad @ w).view(dx.shape))
        want = layers.checkpoint(given).weight_grad(grad.view(y.shape), bias=True)
        assert torch.equal(dw, want[0]) and torch.equal(db, want[1])
    # with a part of the gradients wanted
    for wanted in range(3):
        leaves = [t.detach().requires_grad_(i == wanted) for i, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(layers.linear(*leaves), leaves[wanted], grad)
        torch.testing.assert_close(got.reshape(-1), (dx.reshape(-1), dw.reshape(-1), db)[wanted])


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_any_strides_is_one_product_of_rows(dtype):
    """Never a batched product (of a transposed right operand in 16 bits: those have faulted the GPU), also where no weight wants a gradient."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Products(TorchDispatchMode):
        seen = ()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen += (func.overloadpacket.__name__,)
            return func(*args, **(kwargs or {}))

    w, b = values(64, 48, TYPES[dtype], seed=1), values(1, 64, TYPES[dtype], seed=2)[0]
    x = values(120, 48, TYPES[dtype])
    given = (x, x[7], x.view(2, 60, 48), x.view(4, 30, 48).transpose(0, 1), x.view(5, 24, 48)[:, ::3], x.view(2, 3, 20, 48).transpose(1, 2), x[:40].expand(3, 40, 48),
             x[:, :1].expand(120, 48).view(4, 30, 48), x.view(2, 60, 48)[:, :0], x.view(3, 40, 48).permute(1, 0, 2)[:1])
    for t in given:
        want = torch.nn.functional.linear(t.contiguous().view(-1, 48), w, b).view(*t.shape[:-1], 64)
        for bias in (b, None):
            with Products() as products:
                y = layers.linear(t, w, bias)
            assert not {"bmm", "baddbmm"} & set(products.seen) and {"mm", "addmm", "linear"} & set(products.seen), products.seen
            assert y.shape == want.shape and y.is_contiguous()
            if bias is not None:
                torch.testing.assert_close(y, want)
        leaves = [v.detach().requires_grad_(True) for v in (t, w, b)]
        y = layers.linear(*leaves)
        y.add_(0)  # (a result like any other: it may be changed in place)
        grad = values(max(1, y[..., 0].numel()), 64, TYPES[dtype], seed=3)[: y[..., 0].numel()].view(y.shape)
        dx, dw, db = torch.autograd.grad(y, leaves, grad)
        kept = layers.checkpoint(t.reshape(-1, 48))
        weight, bias = kept.weight_grad(grad.reshape(-1, 64), bias=True)
        torch.testing.assert_close(dx, (grad.reshape(-1, 64) @ w).view(t.shape))
        assert torch.equal(dw, weight) and torch.equal(db, bias)


def test_linear_keeps_its_weight_for_the_gradient_of_x_alone():
    """As torch.nn.functional.linear: where x wants no gradient, the weight may be changed before the backward, and hooks do not see it."""
    x, w, grad = values(50, 48, torch.float32), values(64, 48, torch.float32, seed=1), values(50, 64, torch.float32, seed=2)
    want, bias = layers.checkpoint(x).weight_grad(grad, bias=True)
    w, b = w.requires_grad_(True), torch.zeros(64, device="cuda", requires_grad=True)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.dtype), t)[1], lambda t: t):
        y = layers.linear(x, w, b)
    with torch.no_grad():
        w.mul_(2)
    dw, db = torch.autograd.grad(y, (w, b), grad)
    assert torch.equal(dw, want) and torch.equal(db, bias) and seen == [torch.int8]
    given = x.detach().requires_grad_(True)
    y = layers.linear(given, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, given, grad)


def decoder(points, width, samples):
    """An encoding and what stands behind it."""
    import numpy as np
    import permutohedral_encoding_amd as pe
    torch.manual_seed(0)
    enc = pe.PermutoEncoding(3, 1 << 12, 8, 2, np.geomspace(1.0, 1e-2, 8), device="cuda")
    with torch.no_grad():
        enc.lattice_values.mul_(1e4)
    generator = torch.Generator(device="cuda").manual_seed(1)
    draw = lambda *sizes: torch.randn(sizes, generator=generator, device="cuda")  # noqa: E731
    p = {"w0": draw(width, 16) / 4, "b0": 0.1 * draw(width), "w1": draw(width, width) / width ** 0.5, "b1": 0.1 * draw(width),
         "gate": 0.5 + 0.1 * draw(points // samples, width), "post": 1 + 0.1 * draw(width), "pre": 1 + 0.1 * draw(width), "w2": draw(2 * width, width) / width ** 0.5,
         "w3": draw(3, width) / width ** 0.5}
    p = {k: v.requires_grad_(True) for k, v in p.items()}
    return enc, p, torch.rand((points, 3), generator=generator, device="cuda")


def run_decoder(enc, p, positions):
    """Every tensor on the way, in order."""
    t = {"encoded": enc(positions)}
    t["h"] = layers.linear(t["encoded"], p["w0"], p["b0"])
    t["a"] = layers.activation(t["h"], "gelu")
    t["f"] = layers.linear(t["a"], p["w1"], p["b1"])
    t["y"], t["n"] = layers.residual_norm(t["h"], t["f"], gate=p["gate"], post_weight=p["post"], pre_weight=p["pre"])
    t["u"] = layers.linear(t["n"], p["w2"])
    t["s"] = layers.activation(t["u"], "silu", gated=True)
    t["out"] = layers.linear(t["s"] + t["y"], p["w3"])
    return t


def test_the_layers_together_behind_an_encoding():
    """Each layer's gradient against its formula at what it was given, from the gradient that came to it; sums where a tensor goes two ways."""
    points, width, samples = 1024, 64, 32
    enc, p, positions = decoder(points, width, samples)
    t = run_decoder(enc, p, positions)
    for v in t.values():
        v.retain_grad()
    grad = values(points, 3, torch.float32, seed=9)
    t["out"].backward(grad)
    d = {k: (v.grad if v.grad is not None else grad).double() for k, v in t.items()}
    v = {k: x.detach().double() for k, x in t.items()}
    w = {k: x.detach().double() for k, x in p.items()}
    chain = 2 * (points / 64 + 2048)

    def weight(name, x, dy):
        back = ref.kept(x.float())
        assert_near(p[name].grad, dy.t() @ back, dy.abs().t() @ back.abs(), chain, name)

    weight("w3", (t["s"] + t["y"]).detach(), d["out"])
    weight("w2", v["n"], d["u"])
    weight("w1", v["a"], d["f"])
    weight("w0", v["encoded"], d["h"])
    for name, at in (("b0", "h"), ("b1", "f")):
        assert_near(p[name].grad, d[at].sum(0), d[at].abs().sum(0), chain, name)
    half = ref.kept(t["u"].detach()[:, :width]), ref.kept(t["u"].detach()[:, width:])
    assert_near(t["u"].grad, torch.cat([d["s"] * half[1] * ref.act_slope(half[0], "silu"), d["s"] * ref.act(half[0], "silu")], 1),
                torch.cat([d["s"].abs() * half[1].abs() * (half[0].abs() + 1), d["s"].abs() * (half[0].abs() + 1)], 1), 64, "u")
    want = ref.residual_norm(t["h"], t["f"], d["y"], d["n"], gate=p["gate"], post_weight=p["post"], pre_weight=p["pre"], x_back=ref.kept(t["h"].detach()),
                             f_back=ref.kept(t["f"].detach()))
    assert_near(t["f"].grad, *want["branch"], K, "f")
    for name, key in (("gate", "gate"), ("post", "post_weight"), ("pre", "pre_weight")):
        assert_near(p[name].grad, *want[key], K + points, name)
    kept_h = ref.kept(t["h"].detach())
    through = d["a"] * ref.act_slope(kept_h, "gelu")
    assert_near(t["h"].grad, want["x"][0] + through, want["x"][1] + d["a"].abs() * (kept_h.abs() + 1), K, "h")
    assert enc.lattice_values.grad.abs().sum() > 0


def test_gradients_against_differences():
    """Where the inputs are what their checkpoint stands for, the gradient is the derivative of the formulas: a central difference in 64 bits along a direction."""
    x, f = (ref.kept(values(40, 96, torch.float32, seed)).float() for seed in (0, 1))
    s = norm_case(40, 96, "fp32", "fp32", "layer", gate=8)
    names = ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias")
    leaves = {k: t.detach().requires_grad_(True) for k, t in dict(x=x, f=f, **{k: s[k] for k in names}).items()}
    y, n = layers.residual_norm(leaves["x"], leaves["f"], kind="layer", **{k: leaves[k] for k in names})
    z = layers.activation(n, "gelu", keep_8bit=False)
    grads = torch.autograd.grad((y, z), list(leaves.values()), (s["grad_y"], s["grad_n"]))

    def loss(t):
        out = ref.residual_norm(t["x"], t["f"], None, None, kind="layer", **{k: t[k] for k in names})
        return float((out["y"][0] * s["grad_y"].double()).sum() + (ref.act(out["n"][0], "gelu") * s["grad_n"].double()).sum())

    for name, grad in zip(leaves, grads):
        at = {k: t.detach().double() for k, t in leaves.items()}
        direction = values(*grad.reshape(-1, 96).shape, torch.float32, seed=7).double().view(grad.shape)
        step, ends = 1e-5, []
        for sign in (1, -1):
            ends.append(loss({**at, name: at[name] + sign * step * direction}))
        slope = float((grad.double() * direction).sum())
        # (the difference's own error is of the order of step^2; the gradient's of 1000 roundings of its terms)
        assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 1e-6 * abs(slope) + 1000 * ref.U * float((grad.double() * direction).abs().sum()), name


# ------------------------------------------------------------------------------------------ autograd, streams, graphs

def test_gradients_cannot_be_differentiated_again():
    x = values(20, 32, torch.float32).requires_grad_(True)
    w = values(16, 32, torch.float32, seed=1).requires_grad_(True)
    for y in (layers.activation(x), layers.norm(x), layers.residual_norm(x, x * 2)[0], layers.linear(x, w)):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        assert torch.isfinite(g).all()
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            g.sum().backward()


def test_what_autograd_checks():
    x = values(20, 32, torch.float32).requires_grad_(True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = layers.norm(x, w).sum()
    y.backward()
    with pytest.raises(RuntimeError, match="backward through the graph a second time"):
        y.backward()
    y = layers.norm(x, w).sum()
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = layers.activation(x).sum()  # (a kept input may be changed: the checkpoint stays)
    with torch.no_grad():
        x.mul_(2)
    y.backward()
    y = layers.activation(x, keep_8bit=False).sum()
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # a graph that is kept gives the same gradients again; saved-tensor hooks see the checkpoints
    y = layers.norm(x, w).sum()
    first = torch.autograd.grad(y, (x, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, (x, w))))
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.dtype), t.cpu())[1], lambda t: t.cuda()):
        y = layers.norm(x, w).sum()
    assert torch.int8 in seen and all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, (x, w))))
    for back in (lambda t: t.cuda()[:-1], lambda t: t.cuda().to(torch.float64)):  # a hook that brings something else back
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), back):
            ys = layers.norm(x, w).sum(), layers.activation(x).sum(), layers.activation(x, keep_8bit=False).sum()
        for y in ys:
            with pytest.raises(RuntimeError, match="another form"):
                y.backward()
    # gradients of broadcast results
    a = torch.autograd.grad(layers.activation(x).sum(), x)[0]
    assert torch.equal(a, torch.autograd.grad(layers.activation(x), x, torch.ones(20, 32, device="cuda"))[0])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layers.activation(t).sum())(x.detach())
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        layers.activation(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()))


def test_gradients_that_are_negated_when_they_are_read():
    """What comes back through the imaginary part of a conjugated number."""
    x, w = values(20, 32, torch.float32).requires_grad_(True), values(16, 32, torch.float32, seed=1)
    for layer in (layers.activation, layers.norm, lambda t: layers.residual_norm(t, t)[0], lambda t: layers.linear(t, w)):
        out = []
        for through_complex in (True, False):
            y = layer(x)
            met = []
            y.register_hook(lambda g: met.append(g.is_neg()))
            z = (torch.complex(torch.zeros_like(y), y).conj() * (1 + 2j)).real if through_complex else 2 * y
            out.append(torch.autograd.grad(z.sum(), x)[0])
            assert met == [through_complex]
        torch.testing.assert_close(*out)


def test_a_step_on_another_stream():
    enc, p, positions = decoder(512, 32, 16)
    grad = values(512, 3, torch.float32)
    want = torch.autograd.grad(run_decoder(enc, p, positions)["out"], list(p.values()), grad)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = torch.autograd.grad(run_decoder(enc, p, positions)["out"], list(p.values()), grad)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)


def test_a_step_in_a_graph():
    """Forward and backward captured, replayed with the eager step between the replays, on new inputs each time."""
    enc, p, positions = decoder(512, 32, 16)
    rows, grad, upstream = values(512, 32, torch.float32), values(512, 32, torch.float32, seed=5), values(512, 32, torch.float32, seed=6)
    leaf = rows.clone().requires_grad_(True)
    q = {k: p[k] for k in ("w1", "b1", "gate", "post", "pre", "w2")}

    def step(x):
        f = layers.linear(layers.activation(x, "softplus"), q["w1"], q["b1"])
        y, n = layers.residual_norm(x, f, gate=q["gate"], post_weight=q["post"], pre_weight=q["pre"])
        s = layers.activation(layers.linear(n, q["w2"]), "gelu", gated=True)
        return [y, s, *torch.autograd.grad((y, s), [x, *q.values()], (grad, upstream))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaf)
    for k in range(4):
        with torch.no_grad():
            leaf.copy_(values(512, 32, torch.float32, seed=10 + k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(leaf)):
            torch.testing.assert_close(a, b)


def block(x, p):
    f = layers.linear(layers.activation(x, "silu"), p["w1"], p["b1"])
    y, n = layers.residual_norm(x, f, gate=p["gate"], post_weight=p["post"], pre_weight=p["pre"], kind="layer")
    return layers.activation(layers.linear(n, p["w2"]), "gelu", gated=True) + y


def block_step(x, p, grad, names=("w1", "b1", "gate", "post", "pre", "w2")):
    out = block(x, p)
    return [out, *torch.autograd.grad(out, [x, *(p[k] for k in names)], grad)]


def captured(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def test_two_graphs_in_turn_and_at_once():
    """Each has its own workspaces: replays of one, also while the other runs, leave the other's results as they are."""
    cases = []
    for seed, points in ((0, 256), (1, 4097)):
        p = decoder(points - points % 16, 32, 16)[1]
        p["gate"] = p["gate"][:1].detach().clone().requires_grad_(True)
        cases.append((values(points, 32, torch.float32, seed).requires_grad_(True), p, values(points, 32, torch.float32, seed + 2)))
    want = [[t.detach().clone() for t in block_step(*c)] for c in cases]
    graphs = [captured(lambda c=c: block_step(*c)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]

    def compare():
        torch.cuda.synchronize()
        for (_, out), expected in zip(graphs, want):
            for a, b in zip(out, expected):
                torch.testing.assert_close(a, b)
                a.detach().zero_()
        torch.cuda.synchronize()

    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
        compare()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        compare()


def test_two_steps_at_once_on_two_streams():
    p = decoder(2048, 64, 16)[1]
    inputs = [(values(2048, 64, torch.float32, k).requires_grad_(True), values(2048, 64, torch.float32, k + 2)) for k in range(2)]
    want = [block_step(x, p, grad) for x, grad in inputs]
    streams, got = [torch.cuda.Stream() for _ in inputs], [None, None]
    for _ in range(3):
        for k, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got[k] = block_step(inputs[k][0], p, inputs[k][1])
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for one, expected in zip(got, want):
            for a, b in zip(one, expected):
                torch.testing.assert_close(a, b)
        torch.cuda.synchronize()


def test_a_bias_alone_in_a_graph():
    x, w = values(5000, 48, torch.float32), values(64, 48, torch.float32, seed=1)
    b = torch.zeros(64, device="cuda", requires_grad=True)
    grad = values(5000, 64, torch.float32, seed=2)
    graph, out = captured(lambda: torch.autograd.grad(layers.linear(x, w, b), b, grad))
    want, magnitude = grad.double().sum(0), grad.double().abs().sum(0)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert_near(out[0], want, magnitude, 5000, "bias")
        out[0].zero_()


def test_one_tensor_in_several_places():
    """As the residual and the branch, as the weight of both norms; parameters that are views: every place adds to the same gradient."""
    x, w, s = values(40, 56, torch.float32), values(1, 112, torch.float32, seed=1)[0], torch.tensor(0.5, device="cuda")
    grad_y, grad_n = values(40, 56, torch.float32, seed=2), values(40, 56, torch.float32, seed=3)

    def run(x_of, branch_of, post_of, pre_of, gate_of):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, s)]
        out = layers.residual_norm(x_of(leaves[0]), branch_of(leaves[0]), gate=gate_of(leaves[2]), post_weight=post_of(leaves[1]), pre_weight=pre_of(leaves[1]))
        return [*out, *torch.autograd.grad(out, leaves, (grad_y, grad_n))]

    same = run(lambda t: t, lambda t: t, lambda t: t[::2], lambda t: t[::2], lambda t: t.expand(56))
    apart = run(lambda t: t.clone(), lambda t: t.clone(), lambda t: t[::2].clone(), lambda t: t[::2].clone(), lambda t: t.expand(56).clone())
    for a, b in zip(same, apart):
        assert torch.equal(a, b)


def test_inference_mode_and_autocast_change_nothing():
    p = decoder(64, 32, 16)[1]
    x, grad = values(64, 32, torch.float32).requires_grad_(True), values(64, 32, torch.float32, seed=1)
    want = block_step(x, p, grad)
    with torch.inference_mode():
        got = block(x, p)
        inside = values(64, 32, torch.float32)
    assert torch.equal(got, want[0]) and not got.requires_grad
    for t in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype=t):
            got = block_step(x, p, grad)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a tensor made in inference mode is an input like any other: what is kept of it is not the tensor
    got = torch.autograd.grad(block(inside, p), p["w1"], grad)
    assert torch.equal(got[0], want[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_sweep_trains_a_decoder_with_both(dtype):
    from permutohedral_encoding_amd import perf_sweep
    rows = perf_sweep.decoder(1000, 3, 1, width=40, blocks=1, dtype=dtype, levels=6, log2_capacity=10)
    assert [r["layers"] for r in rows] == ["torch", "layers"] and all(r["train"] > 0 for r in rows)
    assert rows[1]["peak_bytes"] < rows[0]["peak_bytes"]
