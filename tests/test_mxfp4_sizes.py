"""Sizes at which the 4-bit products change their form or are refused, asked of the library on the CPU."""

import pytest


@pytest.mark.parametrize("rows", [1, 2, 8, 16])
def test_rows_too_long_for_shared_memory_are_not_taken_by_the_few_row_kernels(rows):
    """Also those whose bytes in shared memory pass 32 bits (16 rows of 2^27 numbers are 2^32 + 1024 bytes, 1 row of 2^31 - 256 is -448)."""
    from tandemllm_b200.kernels import mxfp4
    lib = mxfp4.lib()
    for k in [1 << b for b in range(20, 31)] + [(1 << 31) - 256, (1 << 27) + 128, (1 << 28) + 128, 3 << 27]:
        for act in (0, 1):
            assert not lib.tl_mxfp4_few_fits(rows, 4096, k, act)
        if rows <= 8:
            assert not lib.tl_mxfp4_experts_fit(rows, 4, k, 64) and not lib.tl_mxfp4_experts_fit(rows, 4, 64, k)
    if rows <= 8:
        assert lib.tl_mxfp4_few_fits(rows, 4096, 2048, 0) and lib.tl_mxfp4_experts_fit(rows, 4, 2048, 1792)


def test_products_of_more_than_8_rows_go_to_the_tensor_cores():
    """Measured on both sides: from 9 rows on the few-row kernel was slower nearly everywhere, and loses what is far below a row's largest."""
    from tandemllm_b200.kernels import mxfp4
    assert mxfp4.FEW_ROWS == 8
    for rows in range(1, 20):
        for n, k, act in ((2048, 7168, 0), (7168, 2048, 1), (1000, 600, 0)):
            assert bool(mxfp4.lib().tl_mxfp4_few_fits(rows, n, k, act)) == (rows <= 8)
