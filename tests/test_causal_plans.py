"""How the selective scan's calls are spread over workgroups, without a GPU."""
import pytest


def _workgroups(batch, length, channels, groups, states):
    """Of the gradient: each writes one partial gradient of B and C; what else is in the workspace are those of A, D and dt_bias, one for each sequence."""
    from m2_amd._lib import lib
    partials = lib.m2_selective_scan_bwd_workspace_bytes(batch, length, channels, groups, states) - 4 * batch * channels * (states + 2)
    assert partials % (8 * length * states) == 0
    return partials // (8 * length * states)


@pytest.mark.parametrize("batch,length,channels,groups,states", [(1, 16384, 1536, 1, 128), (1, 8192, 1536, 1, 128), (1, 32768, 768, 1, 64), (2, 8192, 1536, 1, 128), (2, 16384, 768, 1, 61), (1, 65536, 3584, 4, 64),
                                                                 (1, 8192, 1536, 1, 256), (1, 262144, 1536, 1, 16), (3, 16384, 1000, 8, 100)])
def test_scan_gradient_keeps_a_workgroup_for_each_compute_unit(batch, length, channels, groups, states):
    """Sets of channels that share a workgroup, and with it its partial gradients, save memory, but leave no compute unit without work that has some with one set a workgroup."""
    # the fewest lanes a channel: two states each up to 128 of them, so 32 / (states / 4) channels a workgroup at most
    lanes = max(4, 1 << (-(-states // 2) - 1).bit_length())
    most = groups * batch * -(-(channels // groups) // max(1, 64 // min(lanes, 64)))
    assert _workgroups(batch, length, channels, groups, states) >= min(256, most)
