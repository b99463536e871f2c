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


def _plan(batch, length, channels, groups, states, backward):
    import ctypes
    from m2_amd._lib import lib
    found = (ctypes.c_int * 5)()
    assert lib.m2_selective_scan_plan(batch, length, channels, groups, states, backward, found) == 0
    return list(found)


def test_scan_plans():
    """A workgroup's waves lie within a launch's limits, its lanes hold all states, and all channels have a workgroup; the gradient's workspace holds what its workgroups write."""
    for batch in (1, 3, 40, 700):
        for length in (1, 17, 100, 8192):
            for channels, groups in ((1, 1), (24, 8), (768, 1), (1536, 2), (1919, 1), (4096, 4)):
                for states in (1, 2, 3, 5, 16, 24, 61, 64, 100, 128, 200, 256):
                    if batch * length * groups * states >= 2 ** 32:      # (refused)
                        continue
                    for backward in (0, 1):
                        lanes, each, waves, workgroups, sets = _plan(batch, length, channels, groups, states, backward)
                        assert lanes & (lanes - 1) == 0 and 1 <= lanes <= 64 and each in (1, 2, 4) and lanes * each >= states and 1 <= waves <= 12 and sets >= 1
                        assert workgroups == batch * groups * -(-(channels // groups) // (64 // lanes * sets))
                    assert _workgroups(batch, length, channels, groups, states) == workgroups


def test_scan_plan_refusals():
    import ctypes
    from m2_amd._lib import lib
    found = (ctypes.c_int * 5)()
    assert lib.m2_selective_scan_plan(1, 8, 16, 1, 4, 0, None) == -1 and lib.m2_selective_scan_plan(1, 8, 16, 3, 4, 0, found) == -1
    assert lib.m2_selective_scan_plan(0, 8, 16, 1, 4, 1, found) == -1 and lib.m2_selective_scan_plan(1, 8, 16, 1, 257, 1, found) == -2
    assert lib.m2_selective_scan_plan(1 << 20, 8, 64, 1, 256, 0, found) == -1
