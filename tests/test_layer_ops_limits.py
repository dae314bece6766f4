"""Workspace sizes and refusals of the transformer-layer operators through the C ABI beyond those of
test_layer_ops_refusals; none reaches a device."""
import pytest

import stx
from test_layer_ops_refusals import BF16, F32, GB, INVALID, L, desc, norm, ref


@pytest.mark.parametrize("ne", [[256, 1, 1, 1 << 20], [257, 1, 1, 1 << 18], [48, 4000, 1, 3], [512, 1344]])
def test_norm_forward_needs_no_room_for_the_gradients(ne):
    """The forward call's workspace holds pairs of sums and a number a group, not one a position of every slice."""
    a = desc(ne, type=BF16)
    fwd, both = L.stx_group_norm_cl_forward_workspace_size(ref(a), BF16, 2), L.stx_group_norm_cl_workspace_size(ref(a), BF16, 2)
    slices = ne[3] if len(ne) > 3 else 1
    assert 0 < fwd < both
    assert norm(a=a, type=BF16, groups=2, nbytes=fwd - 1) == INVALID and b"workspace" in L.stx_last_error()
    if slices > 1000:                    # a pair of doubles for each group in each column tile (17 at most up to 512 columns), and a double a group
        assert fwd <= slices * 2 * (17 * 16 + 8) + 512 and both >= slices * ne[0] * 16 and fwd <= both // 8


def test_norm_forward_workspace_of_bad_arguments():
    assert L.stx_group_norm_cl_forward_workspace_size(None, F32, 2) == 0
    assert L.stx_group_norm_cl_forward_workspace_size(ref(desc([32, 10])), F32, 0) == 0
