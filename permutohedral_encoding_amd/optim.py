"""A fused AdamW for the encoding's table (``penc_adamw_step``), and Muon for the matrices behind it (``penc_orthogonalise``).

The reference library has no optimiser; its scripts step the table with ``torch.optim.AdamW``
(examples/performance.py:161), which walks the whole table with several elementwise kernels per
step.  ``AdamW`` here applies the same update (same formulas and order of operations, no amsgrad) in
one kernel per parameter, and can leave entries whose gradient is exactly zero untouched
(``skip_zero_gradients``), the usual way to train hash tables most of whose slots see no point in a
step.
"""
import math

import torch

from . import _native

WORKSPACE_BYTES = 4 << 30  # the most that orthogonalise and Muon take beside their updates (but for matrices that need more on their own), and that Muon takes for updates
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # a s + b s^3 + c s^5 takes small singular values up fastest (K. Jordan et al., "Muon", 2024)


def orthogonalise(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7, halves=False):
    """Nearly orthogonal matrices from those of ``update`` (..., rows, columns), float32, float16 or bfloat16 in GPU memory: ``X = G / (|G| + eps)`` with the Frobenius norm, and
    ``steps`` times ``X = a X + (b S + c S S) X`` with ``S = X X^T``, which takes each singular value s of X to ``a s + b s^3 + c s^5``.

    The products are of float16 twice (22 bits), sums in float32.  ``halves`` takes those of large bfloat16 matrices of float16 once (11 bits): a third of the time, and an error of 1.8e-3 to
    2.0e-3 of the result's norm, where its rounding alone makes 1.66e-3; for others it changes nothing.  Zeros stay zeros, a matrix with an infinity or a NaN becomes NaN.
    Coefficients that make more than 3 of a singular value, or more than 15 of the factor, are refused.  No gradient is recorded."""
    a, b, c = coefficients
    return _native.bridge().orthogonalise(update, steps, a, b, c, eps, halves, WORKSPACE_BYTES)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` semantics (decoupled weight decay, no amsgrad) for fp32 GPU parameters.

    ``skip_zero_gradients=True`` leaves an entry with a zero gradient as it is: value, both moments
    and weight decay.  With ``False`` (default) the result follows ``torch.optim.AdamW`` step by step.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, skip_zero_gradients=False):
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0 or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError("AdamW: lr, eps and weight_decay must be non-negative and the betas in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      skip_zero_gradients=bool(skip_zero_gradients)))

    def zero_grad(self, set_to_none=True):
        if not set_to_none:
            return super().zero_grad(set_to_none=False)
        for group in self.param_groups:
            for p in group["params"]:
                p.grad = None

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()):
                    raise RuntimeError("AdamW: parameters must be contiguous float32 tensors in GPU memory")
                grad = p.grad
                if grad.is_sparse or grad.dtype != torch.float32:
                    raise RuntimeError("AdamW: gradients must be dense float32 tensors")
                grad = grad.contiguous()
                state = self.state[p]
                if not state:
                    state["step"] = 0
                    state["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                state["step"] += 1
                # (records the in-place change for autograd's version checks and the half-precision copy a module keeps)
                _native.bridge().adamw_step(p, grad, state["exp_avg"], state["exp_avg_sq"], float(group["lr"]), float(beta1),
                                            float(beta2), float(group["eps"]), float(group["weight_decay"]), int(state["step"]),
                                            group["skip_zero_gradients"])
        return loss


class SparseTableAdamW(torch.optim.Optimizer):
    """AdamW on the tables of ``PermutoEncoding(..., sparse_table_grad=True)`` modules (``penc_adamw_step_sparse``).

    Takes the gradient from each module's ``table_grad`` and visits only the slot ranges its map names:
    an entry whose gradient is exactly zero keeps its value and both moments (``AdamW`` with
    ``skip_zero_gradients``), and the gradients used and the map are zeroed for the next step.  Other
    parameters (the MLP after the encoding) take any other optimizer.
    """

    def __init__(self, encodings, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        encodings = list(encodings) if isinstance(encodings, (list, tuple)) else [encodings]
        if not encodings or not all(getattr(e, "sparse_table_grad", False) for e in encodings):
            raise ValueError("SparseTableAdamW: pass PermutoEncoding modules built with sparse_table_grad=True")
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0 or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError("SparseTableAdamW: lr, eps and weight_decay must be non-negative and the betas in [0, 1)")
        self._encoding_of = {id(e.lattice_values): e for e in encodings}
        super().__init__([e.lattice_values for e in encodings], dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def zero_grad(self, set_to_none=True):
        """Zeroes what the gradient calls have touched since the last step (``step`` does so itself)."""
        for enc in self._encoding_of.values():
            if enc.table_grad is not None:
                enc.table_grad.clear()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            for p in group["params"]:
                sparse = self._encoding_of[id(p)].table_grad
                if sparse is None:
                    continue  # no gradient call yet
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous() and sparse.matches(p)):
                    raise RuntimeError("SparseTableAdamW: the table must be a contiguous float32 GPU tensor of the gradient's shape")
                state = self.state[p]
                if not state:
                    state["step"] = 0
                    state["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                state["step"] += 1
                _native.bridge().adamw_step_sparse(p, sparse.grad, state["exp_avg"], state["exp_avg_sq"], sparse.touched,
                                                   float(group["lr"]), float(beta1), float(beta2), float(group["eps"]),
                                                   float(group["weight_decay"]), int(state["step"]))
        return loss


class Muon(torch.optim.Optimizer):
    """Steps along orthogonalised momentum, for the weights of hidden layers: matrices, or stacks of them such as those of
    :func:`layers.expert_linear` (..., rows, columns), float32, float16 or bfloat16 in GPU memory.  As ``torch.optim.Muon`` ::

        m = m + (1 - momentum) (g - m);    u = g + momentum (m - g) with nesterov, else m
        p = (1 - lr weight_decay) p - lr scale orthogonalise(u)

    with ``scale`` sqrt(max(1, rows / columns)), or 0.2 sqrt(max(rows, columns)) with ``match_rms_adamw``.  The average m is float32, u of the parameter's type; parameters of one
    size go through the products together, in ``halves`` if that is set.  Tables, norms and biases take another optimiser.  (A captured step keeps the ``lr`` that it was captured with, and is not a parameter's first.)
    """

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.1, steps=5, coefficients=COEFFICIENTS, eps=1e-7, match_rms_adamw=False,
                 halves=False):
        if lr < 0.0 or weight_decay < 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError("Muon: lr and weight_decay must be non-negative and momentum in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=bool(nesterov), weight_decay=weight_decay, steps=steps, coefficients=tuple(coefficients), eps=eps,
                                      match_rms_adamw=bool(match_rms_adamw), halves=bool(halves)))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2:
                    raise ValueError(f"Muon: parameters must be matrices or stacks of them, not of sizes {tuple(p.shape)}")

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("halves", False)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (which brings floating-point state to the parameters' type: the averages stay float32)
        params = [p for group in self.param_groups for p in group["params"]]
        numbers = [n for group in state_dict["param_groups"] for n in group["params"]]
        for p, n in zip(params, numbers):
            if n in state_dict["state"]:
                self.state[p]["momentum_buffer"] = state_dict["state"][n]["momentum_buffer"].to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # (what may be refused is looked at before anything is changed)
        bridge = _native.bridge()
        for group in self.param_groups:
            bridge.orthogonal_options(group["steps"], *group["coefficients"], group["eps"], group["halves"], WORKSPACE_BYTES)
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not (p.is_cuda and p.is_contiguous()):
                    raise RuntimeError("Muon: parameters must be contiguous tensors in GPU memory")
                if p.grad.layout != torch.strided or p.grad.dtype != p.dtype:
                    raise RuntimeError("Muon: gradients must be dense and of the parameter's type")
                bridge.orthogonal_sizes(p, p.grad)
                if not self.state.get(p) and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("Muon: a step has to be taken before one is captured (a graph would begin the averages anew each time)")
        for group in self.param_groups:
            together = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                together.setdefault((tuple(p.shape), p.dtype, p.device), []).append((p, p.grad.contiguous(), state["momentum_buffer"]))
            for (shape, _, _), members in together.items():
                rows, columns = shape[-2:]
                scale = 0.2 * math.sqrt(max(rows, columns)) if group["match_rms_adamw"] else math.sqrt(max(1.0, rows / columns))
                params, grads, averages = map(list, zip(*members))
                bridge.muon_step(params, grads, averages, group["steps"], *group["coefficients"], group["eps"], group["halves"], WORKSPACE_BYTES,
                                 group["momentum"], group["nesterov"], 1.0 - group["lr"] * group["weight_decay"], group["lr"] * scale)
        return loss
