"""The sorted experts' tiles of 64 and of 160 rows, on both sides of the border between them and with crowded experts."""

import pytest
import torch

from tests import plain_mxfp4 as P
from tests import test_gpu_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m,e,top", [(20, 4, 4), (21, 4, 4), (32, 8, 5), (33, 8, 5), (100, 16, 2), (161, 16, 2), (700, 3, 1)])
@pytest.mark.parametrize("crowded", [False, True])
def test_tiles(m, e, top, crowded, monkeypatch):
    from tandemllm_b200.kernels import mxfp4, tensorcore
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16)
    tensorcore.enable(rt)
    seen, lib = [], mxfp4.lib()
    plan = lib.tl_mxfp4_plan
    monkeypatch.setattr(lib, "tl_mxfp4_plan", lambda *a: seen.append(a[3]) or plan(*a))
    g = torch.Generator().manual_seed(m + e)
    x = M.rows(g, m, 136)
    ids, wts = M.routed(g, m, e, top)
    if crowded:                                 # most rows have expert 1 (in place of another where they had it already)
        for r in range(0, m, 3):
            ids[r][ids[r] == 1] = ids[r, 0]
            ids[r, 0] = 1
    first, down, v_first, v_down = M.layer(g, e, 2, 72, 136)
    got = mxfp4.experts(rt, x.to(DEV), ids.to(DEV), wts.to(DEV), mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV)), out_dtype=torch.float32)
    P.hold(got, *P.experts(x, ids, wts, v_first, v_down, "silu"))
    assert seen == [64 if m * top <= 20 * e else 160]
