"""The layers behind the encoding in 64 bits, from their formulas, with the error that 32-bit arithmetic may make.

An operation in 32 bits is off by 2^-24 of its result, a sum of n terms by (its longest chain of additions) * 2^-24 times the sum of the terms'
magnitudes.  ``norms`` and its backward therefore carry beside each value a magnitude: the value with every term taken positively, statistics
included, so that k * 2^-24 times it bounds the error where a value has gone through k roundings."""
import torch

BLOCK = 32
U = 2.0 ** -24


def kept_arrays(x):
    """q (rows, blocks * 32) and e (rows, blocks) of a finite (rows, C) tensor, in 64 bits: the definition, by trying exponents one after the other."""
    x = x.detach().double()
    blocks = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).view(x.shape[0], -1, BLOCK)
    largest = blocks.abs().amax(-1)
    e = torch.full_like(largest, -126.0)
    for exponent in range(-125, 122):
        e = torch.where(largest < 127.5 * torch.exp2(e), e, torch.full_like(e, float(exponent)))
    q = torch.round(blocks * torch.exp2(-e)[..., None]).clamp(-127, 127)  # (from 127.5 * 2^121 on)
    return q.view(x.shape[0], -1), e


def kept(x):
    """The values that the checkpoint of a (rows, C) tensor stands for, in 64 bits; NaN in blocks that are not finite."""
    finite = torch.isfinite(x)
    q, e = kept_arrays(torch.where(finite, x, torch.zeros_like(x)))
    back = q * torch.exp2(e).repeat_interleave(BLOCK, 1)
    bad = torch.nn.functional.pad(~finite, (0, -x.shape[1] % BLOCK)).view(x.shape[0], -1, BLOCK).any(-1).repeat_interleave(BLOCK, 1)
    return torch.where(bad, torch.full_like(back, float("nan")), back)[:, : x.shape[1]]


def act(x, kind):
    if kind == "gelu":
        return x * torch.special.ndtr(x)
    return x * torch.sigmoid(x) if kind == "silu" else torch.logaddexp(x, torch.zeros_like(x))


def act_slope(x, kind):
    if kind == "gelu":
        return torch.special.ndtr(x) + x * torch.exp(-0.5 * x * x) / (2.0 * torch.pi) ** 0.5
    s = torch.sigmoid(x)
    return s * (1.0 + x * torch.sigmoid(-x)) if kind == "silu" else s


def half_step(value, dtype):
    """The most that rounding to ``dtype`` changes a value by."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


class Normed:
    """v~ and its magnitude m (see above), r, and the way back."""

    def __init__(self, v, m, kind, eps):
        self.kind = kind
        mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
        self.r = 1.0 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + eps)
        self.value = (v - mean) * self.r
        first = self.r * (m + (m.mean(1, keepdim=True) if kind == "layer" else 0.0))
        self.m = first + self.value.abs() * (1.0 + (self.value.abs() * first).mean(1, keepdim=True))

    def back(self, d, m):
        n = self.value
        out = self.r * (d - (d.mean(1, keepdim=True) if self.kind == "layer" else 0.0) - n * (d * n).mean(1, keepdim=True))
        # every factor once with its magnitude, the others with their values; the factor r has the relative error of its statistics
        of_r = 1.0 + (n.abs() * self.m).mean(1, keepdim=True)
        along = (d.abs() * n.abs()).mean(1, keepdim=True)
        terms = m + m.mean(1, keepdim=True) + n.abs() * (m * n.abs() + d.abs() * self.m).mean(1, keepdim=True) + self.m * along
        return out, self.r * of_r * terms


def residual_norm(x, f, grad_y, grad_n, scale=1.0, gate=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, post_norm=True, pre_norm=True,
                  kind="rms", eps=1e-6, x_back=None, f_back=None):
    """-> {name: (value, magnitude)} of y, n and all gradients, for (rows, C) tensors and a gate of (C,) or (groups, C); the gradients are those at
    ``x_back`` and ``f_back``.  A missing branch is None."""
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x, f, x_back, f_back, gate, grad_y, grad_n = map(d, (x, f, x_back, f_back, gate, grad_y, grad_n))
    rows, channels = x.shape
    one, zero = torch.ones(channels, dtype=x.dtype, device=x.device), torch.zeros(channels, dtype=x.dtype, device=x.device)
    pw, pb, nw, nb = (d(t) if t is not None else none for t, none in ((post_weight, one), (post_bias, zero), (pre_weight, one), (pre_bias, zero)))
    groups = gate.shape[0] if gate is not None and gate.dim() == 2 else 0
    g = one if gate is None else gate if not groups else gate.repeat_interleave(rows // groups, 0)

    def forward(x, f):
        y, ym, inner, im, fn = scale * x, (scale * x).abs(), None, None, None
        if f is not None:
            if post_norm:
                fn = Normed(f, f.abs(), kind, eps)
                inner, im = fn.value * pw + pb, fn.m * pw.abs() + pb.abs()
            else:
                inner, im = f, f.abs()
            y, ym = y + g * inner, ym + g.abs() * im
        return y, ym, inner, im, fn, Normed(y, ym, kind, eps) if pre_norm else None

    out = {}
    y, ym, _, _, _, yn = forward(x, f)
    out["y"] = (y, ym)
    if pre_norm:
        out["n"] = (yn.value * nw + nb, yn.m * nw.abs() + nb.abs())
    if grad_y is None and grad_n is None:
        return out
    y, ym, inner, im, fn, yn = forward(x_back, f_back)
    dy = torch.zeros_like(x) if grad_y is None else grad_y
    dm = dy.abs()
    sums = {}
    if pre_norm and grad_n is not None:
        sums["pre_weight"], sums["pre_bias"] = (grad_n * yn.value, grad_n.abs() * yn.m), (grad_n, grad_n.abs())
        more, mm = yn.back(grad_n * nw, (grad_n * nw).abs())
        dy, dm = dy + more, dm + mm
    out["x"] = (scale * dy, abs(scale) * dm)
    if f is not None:
        d_gate = (dy * inner, dm * inner.abs() + dy.abs() * im)
        di, dim = dy * g, dm * g.abs()
        if post_norm:
            sums["post_weight"], sums["post_bias"] = (di * fn.value, dim * fn.value.abs() + di.abs() * fn.m), (di, dim)
            out["branch"] = fn.back(di * pw, dim * pw.abs())
        else:
            out["branch"] = (di, dim)
        if groups:
            out["gate"] = tuple(v.view(groups, rows // groups, channels).sum(1) for v in d_gate)
        else:
            sums["gate"] = d_gate
    out.update({k: (v.sum(0), m.sum(0)) for k, (v, m) in sums.items()})
    return out
