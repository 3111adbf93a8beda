"""The workspace of the experts' weight gradients, without a GPU."""
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
