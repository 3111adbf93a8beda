"""The workspace of the experts' weight gradients, without a GPU."""
import numpy as np
import pytest

from permutohedral_encoding_amd import _native


@pytest.mark.parametrize("type", [0, 1, 2])
@pytest.mark.parametrize("rows,experts,channels,outputs", [(1 << 15, 16, 1024, 4096), (1 << 17, 64, 512, 512), (1 << 20, 1024, 256, 256), (1 << 16, 3, 1024, 1024), (100003, 7, 512, 512)])
def test_sums_only_of_experts_with_several_pieces(type, rows, experts, channels, outputs):
    """Pieces have 512 rows at the least, and there are less than twice as many of them, of experts that have several, as whole ones fit the rows.  Of many experts a piece is twice the rows that an
    expert has on average, so that the sums are no more than all weights in float32.  (With room for the pieces that are written as they are it was 1.1 to 1.5 times as much.)"""
    need = _native.lib().penc_expert_weight_grad_workspace_bytes(type, rows, experts, channels, outputs)
    of_one = 4 * outputs * (channels + 1)
    assert need % of_one == 0 and need <= 2 * (rows // 512) * of_one
    if experts >= 16:
        assert need <= experts * of_one


@pytest.mark.parametrize("type", [0, 1, 2])
def test_rows_that_no_expert_is_cut_for_take_none(type):
    lib = _native.lib()
    assert lib.penc_expert_weight_grad_workspace_bytes(type, 512, 1, 64, 64) == 0 == lib.penc_expert_weight_grad_workspace_bytes(type, 0, 5, 1024, 1024)
    assert lib.penc_expert_weight_grad_workspace_bytes(type, 1 << 20, 1, 64, 64) > 0


def test_the_biases_gradient_refuses_before_it_launches():
    block = np.zeros(4096, np.uint8)
    p = block.ctypes.data + (-block.ctypes.data) % 64
    z, lib = None, _native.lib()
    assert lib.penc_expert_bias_grad(7, 4, 2, 8, p, 8, p, p, p, 0, z) == 10
    for bad in ((-1, 2, 8), (1 << 31, 2, 8), (4, 0, 8), (4, 1025, 8), (4, 2, 0), (4, 2, (1 << 18) + 1)):
        assert lib.penc_expert_bias_grad(0, *bad, p, 1 << 19, p, p, p, 0, z) == 12 and lib.penc_expert_bias_grad_workspace_bytes(0, *bad) == 0
    for stride in (7, -8, (1 << 20) + 1):
        assert lib.penc_expert_bias_grad(0, 4, 2, 8, p, stride, p, p, p, 0, z) == 12
    for k in range(3):  # the gradient, the offsets and the biases'
        given = [p] * 3
        given[k] = z
        assert lib.penc_expert_bias_grad(0, 4, 2, 8, given[0], 8, given[1], given[2], p, 0, z) == 1
        given[k] = p + 2
        assert lib.penc_expert_bias_grad(0, 4, 2, 8, given[0], 8, given[1], given[2], p, 0, z) == 5
    need = lib.penc_expert_bias_grad_workspace_bytes(0, 1 << 20, 2, 65)
    assert 0 < need <= 4 * 65 * 2 * 1024 and lib.penc_expert_bias_grad_workspace_bytes(0, 512, 2, 65) == 0 == lib.penc_expert_bias_grad_workspace_bytes(5, 1 << 20, 2, 65)
    assert lib.penc_expert_bias_grad(0, 1 << 20, 2, 65, p, 65, p, p, p, need - 1, z) == 8 and lib.penc_expert_bias_grad(0, 1 << 20, 2, 65, p, 65, p, p, z, need, z) == 1
