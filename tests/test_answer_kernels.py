"""What the kernels of Int4Linear and token_logprobs take of a compute unit: none of them goes through scratch memory."""
import pytest

from test_kernel_resources import _kernels


@pytest.mark.parametrize("kernel", ["int4_few_rows_kernel", "int4_rows_kernel", "int4_operand_kernel", "int4_many_rows_kernel", "token_scores_kernel",
                                    "token_scores_join_kernel", "token_scores_grad_kernel"])
def test_kernels_without_scratch(kernel):
    mine = {n: k for n, k in _kernels().items() if f"{len(kernel)}{kernel}" in n}
    assert mine, kernel
    assert not {n: k[".private_segment_fixed_size"] for n, k in mine.items() if k[".private_segment_fixed_size"]}
