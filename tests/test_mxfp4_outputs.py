"""Outputs that a caller gives a 4-bit product."""

import pytest
import torch


@pytest.mark.parametrize("out", [torch.zeros(1, 16).expand(4, 16), torch.zeros(100).as_strided((4, 16), (15, 1)), torch.zeros(4, 32)[:, ::2],
                                 torch.zeros(16, 4).T, torch.zeros(4, 15), torch.zeros(3, 16), torch.zeros(4, 16, dtype=torch.float64)])
def test_outputs_that_are_refused(out):
    """Rows that lie in one another would be written twice, in any order."""
    from tandemllm_b200.kernels import mxfp4, ops
    with pytest.raises(ops.KernelError, match="output"):
        mxfp4._output(out, 4, 16, torch.float32, torch.zeros(4, 8))


@pytest.mark.parametrize("out", [torch.zeros(4, 16), torch.zeros(4, 40)[:, 3:19], torch.zeros(9, 16)[1::2], torch.zeros(4, 2, 16)[:, 0]])
def test_outputs_that_are_taken(out):
    from tandemllm_b200.kernels import mxfp4
    assert mxfp4._output(out, 4, 16, torch.float32, torch.zeros(4, 8)) is out
    row = torch.zeros(1, 16).as_strided((1, 16), (0, 1))
    assert mxfp4._output(row, 1, 16, torch.float32, torch.zeros(1, 8)) is row
