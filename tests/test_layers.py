"""The layers behind the encoding without a GPU: what they refuse, what the library asks for, and the reference of the GPU tests itself."""
import ctypes

import numpy as np
import pytest
import torch

from layer_reference import kept, kept_arrays
from permutohedral_encoding_amd import _native, layers


class Norm(ctypes.Structure):
    """penc_norm of include/penc.h."""
    _fields_ = [(n, ctypes.c_int) for n in ("type", "param_type", "gate_type", "kind", "post_norm", "pre_norm")] + \
               [("residual_scale", ctypes.c_float), ("eps", ctypes.c_float)] + \
               [(n, ctypes.c_int64) for n in ("rows", "channels", "rows_per_gate")] + \
               [("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("branch", ctypes.c_void_p), ("branch_stride", ctypes.c_int64),
                ("has_branch", ctypes.c_int)] + \
               [(n, ctypes.c_void_p) for n in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias", "x_values", "x_exponents", "branch_values",
                                               "branch_exponents")]


class NormGrads(ctypes.Structure):
    """penc_norm_grads of include/penc.h."""
    _fields_ = [("y", ctypes.c_void_p), ("y_stride", ctypes.c_int64), ("n", ctypes.c_void_p), ("n_stride", ctypes.c_int64)] + \
               [(n, ctypes.c_void_p) for n in ("x", "branch", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")]


def _memory():
    block = np.zeros(4096, np.uint8)
    return block, block.ctypes.data + (-block.ctypes.data) % 64


def test_checkpoints_have_rows_of_sixteen_bytes_and_a_byte_for_each_block():
    lib = _native.lib()
    for channels in (1, 15, 16, 17, 31, 32, 33, 48, 64, 65, 1000, 8192):
        assert lib.penc_kept_pitch(channels) == -(-channels // 16) * 16
        assert lib.penc_kept_blocks(channels) == -(-channels // 32)


def test_the_entry_points_refuse_before_they_launch():
    lib = _native.lib()
    block, p = _memory()
    z = None
    # types, sizes, strides, pointers, alignment
    assert lib.penc_keep(3, 4, 4, p, 4, 1, p, p, z) == 10
    assert lib.penc_keep(-1, 4, 4, p, 4, 1, p, p, z) == 10
    assert lib.penc_keep(0, -1, 4, p, 4, 1, p, p, z) == 12
    assert lib.penc_keep(0, 4, 0, p, 4, 1, p, p, z) == 12
    assert lib.penc_keep(0, 4, (1 << 24) + 1, p, 4, 1, p, p, z) == 12
    assert lib.penc_keep(0, 4, 4, p, 8, 2, p, p, z) == 12  # neither rows nor channels adjacent
    assert lib.penc_keep(0, 4, 4, z, 4, 1, p, p, z) == 1 and lib.penc_keep(0, 4, 4, p, 4, 1, z, p, z) == 1 and lib.penc_keep(0, 4, 4, p, 4, 1, p, z, z) == 1
    assert lib.penc_keep(0, 4, 4, p, 4, 1, p + 8, p, z) == 5  # checkpoints are aligned to 16 bytes
    assert lib.penc_keep(0, 4, 4, p + 2, 4, 1, p, p, z) == 5 and lib.penc_keep(1, 4, 4, p + 1, 4, 1, p, p, z) == 5
    assert lib.penc_keep(0, 0, 4, z, 4, 1, z, z, z) == 0  # no rows: nothing to do
    assert lib.penc_restore(0, 4, 4, z, p, p, z) == 1 and lib.penc_restore(5, 4, 4, p, p, p, z) == 10 and lib.penc_restore(0, 0, 4, z, z, z, z) == 0
    assert lib.penc_activation(0, 3, 0, 4, 4, p, 4, p, z, z, z) == 11 and lib.penc_activation(0, -1, 0, 4, 4, p, 4, p, z, z, z) == 11
    assert lib.penc_activation(0, 0, 0, 4, 4, p, 4, p, p, z, z) == 1  # values without exponents
    assert lib.penc_activation(0, 0, 0, 4, 4, p, 4, z, z, z, z) == 1 and lib.penc_activation(0, 0, 1, 0, 4, z, 4, z, z, z, z) == 0
    assert lib.penc_activation_backward(0, 0, 0, 4, 4, z, 4, z, z, p, 4, p, z) == 1  # neither the input nor its checkpoint
    assert lib.penc_activation_backward(0, 0, 0, 4, 4, p, 4, z, z, p + 1, 4, p, z) == 5
    # partial sums need their workspace
    need = lib.penc_weight_grad_workspace_bytes(100, 48, 64)
    assert need >= 4 * 49 * 64 and lib.penc_weight_grad_workspace_bytes(100, 0, 64) == 0 == lib.penc_weight_grad_workspace_bytes(100, 1 << 20, 1 << 20)
    assert lib.penc_weight_grad(0, 0, 100, 48, 64, p, p, p, 64, p, z, p, need - 1, z) == 8
    assert lib.penc_weight_grad(0, 0, 100, 48, 64, p, p, p, 64, p, z, z, need, z) == 1
    assert lib.penc_weight_grad(0, 4, 100, 48, 64, p, p, p, 64, p, z, p, need, z) == 10
    assert lib.penc_weight_grad(0, 0, 100, 48, 0, p, p, p, 64, p, z, p, need, z) == 12
    assert lib.penc_weight_grad(0, 0, 100, 48, 64, p, p, p, -64, p, z, p, need, z) == 12
    for status in (10, 11, 12):
        assert lib.penc_status_string(status) != lib.penc_status_string(99)


def test_the_products_that_the_gpu_tests_call_large_are():
    """The rows of a product of 300 channels by 390 outputs are split over 64 workgroups in tiles of 256 x 256 and over 7 in those of 64 x 64, so that the
    workspace says which of them fp32 takes from 2^34 multiplications on (three for each of its own)."""
    lib = _native.lib()
    splits = lambda rows: lib.penc_weight_grad_workspace_bytes(rows, 300, 390) // (4 * 301 * 390)  # noqa: E731
    assert splits(50001) > 40 and splits(48000) <= 7


def test_the_norms_refuse_before_they_launch():
    lib = _native.lib()
    block, p = _memory()

    def forward(y=p, n=p, **given):
        norm = Norm(0, 0, 0, 0, 1, 1, 1.0, 1e-6, 4, 8, 0, p, 8, p, 8, 1)
        for k, v in given.items():
            setattr(norm, k, v)
        return lib.penc_residual_norm(ctypes.byref(norm), y, n, None)

    def backward(workspace=p, nbytes=None, grads=None, **given):
        norm = Norm(0, 0, 0, 0, 1, 1, 1.0, 1e-6, 4, 8, 0, p, 8, p, 8, 1)
        for k, v in given.items():
            setattr(norm, k, v)
        g = NormGrads(p, 8, p, 8, p, p)
        for k, v in (grads or {}).items():
            setattr(g, k, v)
        need = lib.penc_residual_norm_workspace_bytes(norm.rows, norm.channels, norm.rows_per_gate)
        return lib.penc_residual_norm_backward(ctypes.byref(norm), ctypes.byref(g), workspace, need if nbytes is None else nbytes, None)

    for call in (forward, backward):
        assert call(type=3) == 10 and call(type=1, param_type=2) == 10 and call(gate_type=1) == 10
        assert call(kind=2) == 11
        assert call(rows=-1) == 12 and call(channels=0) == 12 and call(channels=8193) == 12 and call(rows_per_gate=3) == 12 and call(rows_per_gate=-1) == 12
        assert call(x=p + 2) == 5 and call(gate=p + 1) == 5 and call(x_values=p + 4, x_exponents=p) == 5
        assert call(x=None) == 1 and call(branch=None) == 1 and call(x_values=p) == 1
    assert forward(n=None) == 1 and forward(y=None, pre_norm=0) == 1 and forward(rows=0, x=None) == 0
    assert lib.penc_residual_norm(None, p, p, None) == 1
    assert backward(workspace=None) == 1 and backward(nbytes=16) == 8 and backward(grads={"y": p + 2}) == 5
    assert backward(has_branch=0, grads={"gate": p}) == 1
    assert backward(x_values=p, x_exponents=p) == 1  # a kept x needs a kept branch
    assert lib.penc_residual_norm_workspace_bytes(10, 8193, 0) == 0 and lib.penc_residual_norm_workspace_bytes(1 << 20, 64, 0) < 1 << 24


def test_tensors_in_host_memory_and_unknown_kinds_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    for call in (lambda: layers.checkpoint(x), lambda: layers.linear(x, w), lambda: layers.activation(x), lambda: layers.norm(x),
                 lambda: layers.residual_norm(x, x)):
        with pytest.raises(ValueError, match="GPU memory"):
            call()
    with pytest.raises(ValueError, match="gelu, silu, softplus"):
        layers.activation(x, "relu")
    with pytest.raises(ValueError, match="rms, layer"):
        layers.norm(x, kind="batch")
    with pytest.raises(ValueError, match="branch"):
        layers.residual_norm(x, None)
    with pytest.raises(ValueError, match="torch.Tensor"):
        layers.checkpoint([1.0])


def test_the_reference_of_checkpoints_is_off_by_half_a_step_at_most():
    rng = np.random.default_rng(0)
    for scale in (1e-42, 1e-38, 1e-3, 1.0, 1e30):
        x = (rng.standard_normal((50, 75)) * scale).astype(np.float32)
        q, e = kept_arrays(torch.from_numpy(x))
        assert q.abs().max() <= 127 and e.min() >= -126
        back = kept(torch.from_numpy(x)).numpy()
        step = np.repeat(2.0 ** e.numpy().astype(np.float64), 32, 1)[:, :75]
        assert np.all(np.abs(back - x.astype(np.float64)) <= step / 2)
        largest = np.abs(np.pad(x, ((0, 0), (0, 21)))).reshape(50, 3, 32).max(2).astype(np.float64)
        # the least exponent that does: one less would not hold the largest value
        assert np.all((largest < 127.5 * 2.0 ** e.numpy()) & ((largest >= 127.5 * 2.0 ** (e.numpy() - 1.0)) | (e.numpy() == -126)))
