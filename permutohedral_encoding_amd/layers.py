"""What the layers behind the encoding train with: checkpoints of activations in 8 bits and layers whose backward reads them, and layers of experts.

No counterpart in the reference, whose scripts take these layers from torch.  An encoding of 2^20 points and 24 levels is 200 MB that a linear layer
behind it keeps for its weight gradient, and each hidden layer keeps as much again, several times over.  The first functions here keep what their backward
needs in 8 bits a value (a quarter of fp32) and are one pass over memory in either direction:

    x = encoding(positions)                                            # (N, 48)
    h = layers.linear(x, w0, b0)
    f = layers.linear(layers.activation(h, "gelu"), w1, b1)
    h, n = layers.residual_norm(h, f, gate=gate, post_weight=wp, pre_weight=wn)     # h + gate * norm(f), and its norm for the next block

A decoder of experts sends each row to a few of many small layers, by a router that is trained with them.  Its rows are sorted by expert, multiplied, and brought back:

    weights, routing = layers.route(layers.linear(x, w_router), 2)                  # 2 of the experts for each row, their shares, and where each choice stands
    h = layers.expert_linear(layers.dispatch(x, routing), w_up, b_up, routing)      # (rows * 2, O): each expert's rows one after the other
    y = layers.expert_linear(layers.activation(h), w_down, None, routing)
    out = layers.combine(y, weights, routing)                                       # back in the rows' order, weighted

What the experts' functions need for the backward they keep as it is, and which rows go where stays on the device: nothing waits for it.

All of them take float32, float16 or bfloat16 tensors ``(..., C)`` in GPU memory, on the current stream of the tensor's device, of any strides (rows whose
channels are adjacent are read in place, as is the encoding's own result).  Sums and statistics are float32, results are rounded once, and
every call gives the same result for the same inputs.  Every backward is the gradient of the forward at the values that the checkpoint stands for.  Forward and
backward can be captured in a graph, under torch's own condition: no graph of autograd that was built outside of the capture on the same leaves is still alive.
Autocast does not apply to them.  There is no CPU path.

There is no second derivative either: differentiating a gradient of these layers again raises an error.  An eikonal loss, and whatever else is made of the
gradient with respect to the positions, needs torch's own layers behind the encoding, which itself can be differentiated twice.
"""
import torch

from . import _native

__all__ = ["Checkpoint", "checkpoint", "linear", "activation", "norm", "residual_norm", "Routing", "route", "routing", "dispatch", "expert_linear", "combine"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # PENC_FP32, PENC_FP16, PENC_BF16 (include/penc.h)
_ACTIVATIONS = {"gelu": 0, "silu": 1, "softplus": 2}
_NORMS = {"rms": 0, "layer": 1}


def _bridge():
    return _native._bridge or _native.bridge()


def _code(table, key, what):
    try:
        return table[key]
    except (KeyError, TypeError):
        raise ValueError(f"{what} should be one of {', '.join(str(k) for k in table)}, however it is {key}") from None


class Checkpoint:
    """A tensor ``(..., C)`` in 8 bits, made by :func:`checkpoint`.

    A value stands for ``values * 2 ** (exponents - 127)``, with one exponent for each block of 32 channels of a row.  It is off by at most half a step, and a
    step is at most 1/63 of the largest magnitude in the block; a block with an infinity or a NaN comes back as NaN.  A row takes C rounded up to 16 bytes and
    one for each block: less than the tensor from 5 channels of float32 or 9 of a 16-bit type on."""

    __slots__ = ("data", "rows", "shape", "dtype")

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, shape, dtype
        self.rows = shape.numel() // shape[-1]

    @property
    def values(self):
        """int8, rows of C rounded up to 16 (the rest zero)."""
        pitch = -(-self.shape[-1] // 16) * 16
        return self.data[: self.rows * pitch].view(self.rows, pitch)

    @property
    def exponents(self):
        """uint8, one for each block; 255 for one that is not finite."""
        blocks = -(-self.shape[-1] // 32)
        return self.data[self.data.numel() - self.rows * blocks:].view(torch.uint8).view(self.rows, blocks)

    def unpack(self, dtype=None):
        """The values that the checkpoint stands for, of the type of the tensor it was made of or of ``dtype`` (float16: at most 65504 in magnitude)."""
        rows = _bridge().layers_restore(self.data, self.rows, self.shape[-1], _code(_TYPES, self.dtype if dtype is None else dtype, "dtype"))
        return rows if len(self.shape) == 2 else rows.view(self.shape)

    def weight_grad(self, grad, bias=False, dtype=None):
        """What a linear layer with this input needs of the gradient ``(..., O)`` of its result: the gradient of its weight ``(O, C)``, the sum over the
        rows of ``grad[o] * input[c]``, and with ``bias`` that of its bias ``(O,)``, of ``grad``'s type or ``dtype``."""
        if grad.shape[:-1] != self.shape[:-1]:
            raise ValueError(f"grad should have the rows of the tensor kept, {tuple(self.shape)}, however it has sizes {tuple(grad.shape)}")
        code = _code(_TYPES, grad.dtype if dtype is None else dtype, "dtype")
        both = _bridge().layers_weight_grad(self.data, self.rows, self.shape[-1], grad, bias, code)
        return both if bias else both[0]


def checkpoint(x):
    """Keeps ``x`` in 8 bits: blocks of 32 channels of a row share a power of two as their step.  Outside of autograd: the
    functions below call it where they need it."""
    return Checkpoint(_bridge().layers_keep(x), x.shape, x.dtype)


def linear(x, weight, bias=None):
    """``torch.nn.functional.linear`` that keeps its input in 8 bits for the gradients of weight and bias.  ``x``, ``weight`` (O, C) and ``bias`` (O,) are of one type."""
    return _bridge().layers_linear(x, weight, bias)


def activation(x, kind="gelu", gated=False, keep_8bit=True):
    """``act(x)``; with ``gated`` the channels are ``[a | b]`` and the result ``act(a) * b`` has half of them.

    ``kind``: "gelu" (``x Phi(x)``), "silu" (``x / (1 + exp(-x))``) or "softplus" (``log(1 + exp(x))``).  ``keep_8bit=False`` keeps ``x`` itself for the
    backward (of a few channels that is less memory)."""
    return _bridge().layers_activation(x, _code(_ACTIVATIONS, kind, "kind"), gated, keep_8bit)


def norm(x, weight=None, bias=None, kind="rms", eps=1e-6, keep_8bit=True):
    """``x / sqrt(mean(x^2) + eps) * weight + bias`` over the channels ("rms"), or that of ``x - mean(x)`` ("layer").  At most 8192 channels; parameters
    are of the type of ``x`` or float32."""
    return _bridge().layers_residual_norm(x, None, None, None, None, weight, bias, 1.0, False, True, _code(_NORMS, kind, "kind"), eps, keep_8bit)[1]


def residual_norm(x, branch, gate=None, residual_scale=1.0, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, post_norm=True, pre_norm=True,
                  kind="rms", eps=1e-6, keep_8bit=True):
    """What stands between a block and the next one, in one pass: ``y = residual_scale * x + gate * norm(branch)`` and ``n = norm(y)``.

    ``x`` is the residual stream, ``branch`` (same sizes and type) what the block made of it, ``residual_scale`` a number; the result is ``(y, n)``, or ``y`` with ``pre_norm=False``.
    ``post_norm=False`` takes the branch as it is.  ``gate`` (None: 1) has sizes ``(C,)`` for all rows, those of ``x`` with trailing ones before the channels
    (a gate for each row, or for each ray of ``(rays, samples, C)``: ``(rays, 1, C)``), or ``(groups, C)`` for ``x`` of ``(rows, C)``, each for
    ``rows / groups`` consecutive rows.  The norms are those of :func:`norm`, ``n`` is of ``y`` before it is rounded."""
    if branch is None:
        raise ValueError("residual_norm should have a branch (layers.norm is the norm of a tensor alone)")
    y, n = _bridge().layers_residual_norm(x, branch, gate, post_weight, post_bias, pre_weight, pre_bias, residual_scale, post_norm, pre_norm,
                                                 _code(_NORMS, kind, "kind"), eps, keep_8bit)
    return (y, n) if pre_norm else y


class Routing:
    """Which experts rows go to, made by :func:`route` or :func:`routing`: ``experts`` (..., k) of ``number``, and where the k choices of each row stand when the
    choices of all rows are sorted by expert: ``positions`` (..., k) int32, those of one expert in their order, expert by expert from ``offsets`` (number + 1,) int32
    on, and those without an expert last."""

    __slots__ = ("experts", "number", "positions", "offsets")

    def __init__(self, experts, number, positions, offsets):
        self.experts, self.number, self.positions, self.offsets = experts, number, positions, offsets


def route(logits, choices=1, normalise=True):
    """The experts of rows: the ``choices`` (at most 8) largest of each row's logits ``(..., experts)``, at most 1024.  Returns ``(weights, routing)``, weights (..., choices) in
    float32: the softmax over the chosen experts or, with ``normalise=False``, their share of the softmax over all.
    (The softmax over a single choice is 1 and has no gradient: a router of one choice trains with ``normalise=False``.)

    Of equal logits the lowest expert's is first, a NaN is the largest, and -inf is never chosen: a row with nothing else has no expert (-1) and weights of zero."""
    weights, experts, positions, offsets = _bridge().layers_route(logits, choices, normalise)
    return weights, Routing(experts, logits.shape[-1], positions, offsets)


def routing(experts, number):
    """The :class:`Routing` of experts that are given, integers (..., choices); one outside of 0 to ``number - 1`` is no expert."""
    positions, offsets = _bridge().layers_plan(experts, number)
    return Routing(experts, number, positions, offsets)


def dispatch(x, routing):
    """The rows of ``x`` (..., C), one for each choice, sorted by expert: ``(rows * choices, C)``.  Choices without an expert are zeros, behind all others."""
    return _bridge().layers_dispatch(x, routing.positions, routing.offsets)


def expert_linear(x, weight, bias, routing):
    """A linear layer of each expert on its own rows: ``x`` (rows * choices, C) is sorted by expert, as :func:`dispatch` makes it, ``weight`` (experts, O, C) and ``bias``
    (experts, O) or None are of its type.  Rows without an expert are zeros in the result and in the gradient, and not read.  Its input is kept as it is for the backward."""
    return _bridge().layers_expert_linear(x, weight, bias, routing.positions, routing.offsets)


def combine(y, weights, routing):
    """What the experts made of the sorted rows, brought back: the sum over a row's choices of ``weights`` (..., choices) times the choice's row of ``y`` (rows * choices, C).
    ``weights`` are of the type of ``y`` or float32.  Choices without an expert are left out, and so is what stands in their rows."""
    return _bridge().layers_combine(y, weights, routing.positions, routing.offsets)
