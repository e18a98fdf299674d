"""Rows whose numbers lie far from one another, where the large ones meet weights of nothing."""

import pytest
import torch

from tests import plain_mxfp4 as P
from tests import test_gpu_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m", [9, 12, 16, 17, 40])
def test_products_of_more_than_8_rows_hold_any_row(m):
    """(With up to 8 rows, what is 2^-39 of a row's largest counts as zero; the module says so.)"""
    from tandemllm_b200.kernels import mxfp4, tensorcore
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16)
    tensorcore.enable(rt)
    g = torch.Generator().manual_seed(m)
    x, w = M.rows(g, m, 200), M.weights(g, 48, 200)
    x[:, ::9] *= 2.0 ** 60
    w[:, ::9] = 0
    P.hold(mxfp4.linear(rt, x.to(DEV), mxfp4.quantize(w.to(DEV)), out_dtype=torch.float32), *P.product(x, P.rounded(w)))
