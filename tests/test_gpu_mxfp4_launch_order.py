"""MXFP4 layers behind kernels that are still running when they may begin (programmatic dependent launch switched on)."""

import pytest
import torch

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


@pytest.fixture
def chained():
    from tandemllm_b200.kernels import ops, tensorcore

    def switch(on):
        torch.cuda.synchronize()
        ops.core().tl_set_chained_launches(on)
        tensorcore.lib().tl_tc_set_chained_launches(on)

    yield switch
    switch(0)


@pytest.mark.parametrize("m,e,top,inter,hidden", [(1, 8, 1, 24, 64), (1, 16, 2, 16, 128), (2, 32, 4, 40, 96), (8, 40, 5, 24, 64), (8, 9, 9, 16, 72),
                                                  (20, 16, 2, 40, 64), (90, 8, 3, 72, 136)])
def test_routed_layers_behind_the_router_that_writes_their_ids(runtime, chained, m, e, top, inter, hidden):
    """Small layers, whose first half leaves SMs free for a second half that comes early. The ids' memory holds other experts before."""
    from tandemllm_b200.kernels import mxfp4, ops
    g = torch.Generator().manual_seed(m * e + inter)
    first, down, *_ = M.layer(g, e, 2, inter, hidden)
    q = mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    router, bias = (torch.randn(e, hidden, generator=g) * 0.3).to(DEV), torch.zeros(e, device=DEV)
    xs = [M.rows(g, m, hidden).to(DEV) for _ in range(24)]
    ids, wts = torch.zeros(m, top, dtype=torch.int32, device=DEV), torch.empty(m, top, device=DEV)
    logits = torch.empty(m, e, device=DEV)

    def layers():
        out = []
        for x in xs:
            ops.gemm_simt(x.float(), router, None, logits)
            ops.router_topk(logits, bias, top, True, 0.0, 1.0, ids, wts)
            out.append(mxfp4.experts(runtime, x, ids, wts, *q, out_dtype=torch.float32))
        torch.cuda.synchronize()
        return out

    want = layers()
    chained(1)
    got = layers()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert int(runtime.status.item()) == 0


@pytest.mark.parametrize("name", ["c", "d"])
def test_a_model_with_all_launches_chained(chained, name):
    from tests import test_gpu_mxfp4_models as models
    from tests import test_gpu_puripel as puripel
    from tests import tiny_configs as T
    cfg, spec, W = models.lfm2(name)
    requests = {"a": T.long_tokens(name, 100), "b": T.long_tokens(name, 31, seed=8)}
    schedule = [[("a", 64), ("b", 1)], [("a", 9), ("b", 20)], [("a", 2), ("b", 3)]] + [[("a", 1), ("b", 1)]] * 7 + [[("a", 18)]]
    engine = models.engine_on(spec, W, "bfloat16")
    want = puripel.run_schedule(engine, requests, schedule)
    chained(1)
    for _ in range(3):
        got = puripel.run_schedule(engine, requests, schedule)
        assert all(torch.equal(got[r], want[r]) for r in requests)
