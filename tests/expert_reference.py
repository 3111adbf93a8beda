"""Rows that go to experts, and orthogonalised updates, in 64 bits from their definitions."""
import math

import torch

U = 2.0 ** -24


def half_step(value, dtype):
    """The most that rounding to ``dtype`` changes a value by."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def choose(logits, choices):
    """The largest logits' indices, the lowest first among equal ones, -1 where only -inf is left (no NaN)."""
    order = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    return torch.where(order.values[..., :choices] == -math.inf, -1, order.indices[..., :choices])


def route(logits, choices, normalise, grad):
    """weights and their gradient's way back, each with a magnitude that every term enters positively, and the largest distance from the top in each row."""
    l, g = logits.detach().double(), grad.double()
    chosen = choose(l, choices)
    there = chosen >= 0
    some = there[:, :1]
    top = torch.where(some, l.amax(1, keepdim=True), 0.0)
    exps = torch.where(some, torch.exp(l - top), 0.0)
    picked = torch.where(there, exps.gather(1, chosen.clamp(min=0)), 0.0)
    total = torch.where(some, (picked if normalise else exps).sum(1, keepdim=True), 1.0)
    w = picked / total
    far = torch.where(torch.isfinite(l), (l - top).abs(), 0.0).amax(1, keepdim=True)
    along, along_m = (w * g).sum(1, keepdim=True), (w * g.abs()).sum(1, keepdim=True)
    d, m = torch.zeros_like(l), torch.zeros_like(l)
    if normalise:
        d.scatter_add_(1, chosen.clamp(min=0), torch.where(there, w * (g - along), 0.0))
        m.scatter_add_(1, chosen.clamp(min=0), torch.where(there, w * (g.abs() + along_m), 0.0))
    else:
        d, m = -exps / total * along, exps / total * along_m
        d.scatter_add_(1, chosen.clamp(min=0), torch.where(there, w * g, 0.0))
        m.scatter_add_(1, chosen.clamp(min=0), torch.where(there, w * g.abs(), 0.0))
    return chosen, w, d, m, far


def plan(chosen, number):
    """positions and offsets, by counting on the CPU."""
    flat = chosen.reshape(-1).cpu()
    flat = torch.where((flat >= 0) & (flat < number), flat, number).long()
    order = torch.argsort(flat, stable=True)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(len(order))
    counts = torch.bincount(flat, minlength=number + 1)
    offsets = torch.cat([counts.new_zeros(1), counts[:number].cumsum(0)])
    return positions.view(chosen.shape).int(), offsets.int()


COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalise(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7, stored=lambda t: t, dtype=torch.float64):
    """The steps in ``dtype``, X, S and the factor going through ``stored``."""
    a, b, c = coefficients
    g = update.to(dtype)
    tall = g.shape[-2] > g.shape[-1]
    g = g.transpose(-1, -2).contiguous() if tall else g
    norm = g.double().square().sum((-1, -2), keepdim=True).sqrt().to(dtype)
    x = stored(g / (norm + eps))
    for step in range(steps):
        s = stored(x @ x.transpose(-1, -2).contiguous())
        f = stored(b * s + c * (s @ s))
        x = a * x + f @ x
        x = stored(x) if step + 1 < steps else x
    return x.transpose(-1, -2).contiguous() if tall else x


def in_float16(t):
    """As 64-bit numbers, what float16 holds of them times 2^12."""
    return (t * 4096.0).half().double() / 4096.0
