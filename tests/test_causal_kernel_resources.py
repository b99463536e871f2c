"""The causal mixer's kernels keep what they work on in registers: none sends any of it through scratch memory."""
import pytest

from test_kernel_resources import _kernels


@pytest.mark.parametrize("kernel,count", [("causal_conv_kernel", 32), ("causal_conv_bwd_kernel", 32), ("causal_conv_step_kernel", 4), ("selective_scan_kernel", 38), ("selective_scan_bwd_kernel", 24),
                                          ("selective_scan_step_kernel", 8), ("scan_join_kernel", 2), ("norm_rows_kernel", 54), ("norm_rows_bwd_kernel", 54), ("norm_partials_kernel", 6),
                                          ("norm_apply_kernel", 6), ("norm_bwd_partials_kernel", 6), ("norm_bwd_apply_kernel", 6), ("norm_stats_kernel", 1), ("norm_bwd_sums_kernel", 1),
                                          ("sum_partials_kernel", 1)])
def test_kernels_without_scratch(kernel, count):
    mine = {n: k[".private_segment_fixed_size"] for n, k in _kernels().items() if f"{len(kernel)}{kernel}" in n}
    assert len(mine) == count and not any(mine.values()), mine
