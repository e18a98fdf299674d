"""Blocks of the smallest scale (2^-127) in products of every form: large rows make sums of them that are far from nothing."""

import pytest
import torch

from tests import plain_mxfp4 as P
from tests import test_gpu_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def runtime():
    from tandemllm_b200.kernels import tensorcore
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16)
    tensorcore.enable(rt)
    return rt


def small(g, *shape):
    """Numbers whose blocks' largest is below 2^-124, in some rows below 2^-126."""
    w = torch.rand(*shape, generator=g) * 2.0 ** -124 * torch.where(torch.rand(*shape, generator=g) < 0.5, -1.0, 1.0)
    w[..., 1::3, :] *= 0.2
    return w


@pytest.mark.parametrize("m", [1, 5, 12, 16, 17, 50, 150])
def test_products(runtime, m):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x, w = (M.rows(g, m, 264).float() * 2.0 ** 110).to(torch.bfloat16), small(g, 2, 48, 264)
    v = P.rounded(w)
    assert (v != 0).any(-1).all() and float(v.abs().max()) <= 2.0 ** -124
    want, off = P.product(x, v[0])
    assert float(want.abs().max()) > 2.0 ** -16
    P.hold(mxfp4.linear(runtime, x.to(DEV), mxfp4.quantize(w[0].to(DEV)), out_dtype=torch.float32), want, off)
    P.hold(mxfp4.gated(runtime, x.to(DEV), mxfp4.quantize(w.to(DEV)), "identity"), *P.gated(x, v[0], v[1], "identity"))


@pytest.mark.parametrize("m", [1, 8, 9, 40])
def test_experts_with_such_blocks_among_others(runtime, m):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x = (M.rows(g, m, 96).float() * 2.0 ** 110).to(torch.bfloat16)
    first, down = small(g, 5, 40, 96) * 0.9, M.weights(g, 5, 96, 40)
    ids, wts = M.routed(g, m, 5, 2)
    got = mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV)), "identity",
                        out_dtype=torch.float32)
    want, off = P.experts(x, ids, wts, P.rounded(first).view(5, 1, 40, 96), P.rounded(down), "identity")
    assert float(want.abs().max()) > 2.0 ** -24
    P.hold(got, want, off)


@pytest.mark.parametrize("size,weight", [(-125, 60), (-112, 50), (-111, 0), (-60, -30), (110, -60), (124, -124)])
@pytest.mark.parametrize("m", [1, 8, 9])
def test_rows_of_any_size(runtime, m, size, weight):
    """Token rows from below the smallest normal number to next to the largest one, with weights that bring their products back."""
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x = torch.ldexp(M.rows(g, m, 264).float().clamp(-7, 7), torch.tensor(size)).to(torch.bfloat16)
    x[0, 100:] = 0                              # (a row's largest number may lie anywhere, or there may be none)
    x[m - 1, :] *= 0 if m > 1 else 1
    w = torch.ldexp(M.weights(g, 2, 48, 264).clamp(-0.9, 0.9), torch.tensor(weight))
    v = P.rounded(w)
    want, off = P.product(x, v[0])
    assert float(want.abs().max()) > 2.0 ** (size + weight - 6)
    P.hold(mxfp4.linear(runtime, x.to(DEV), mxfp4.quantize(w[0].to(DEV)), out_dtype=torch.float32), want, off)
    if weight < -90 and m <= mxfp4.EXPERT_ROWS:
        return                                  # (the second half's weights would be beyond 2^95, where sums of up to 8 rows can be infinite)
    down = torch.ldexp(M.weights(g, 2, 264, 48), torch.tensor(-weight))
    ids, wts = M.routed(g, m, 2, 2)
    got = mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), mxfp4.quantize(w.to(DEV)), mxfp4.quantize(down.to(DEV)), "identity",
                        out_dtype=torch.float32)
    P.hold(got, *P.experts(x, ids, wts, v.view(2, 1, 48, 264), P.rounded(down), "identity"))
