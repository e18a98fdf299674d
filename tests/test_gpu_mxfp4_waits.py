"""The bounded waits of the MXFP4 products. A test hook has a CTA's copies end early, so that a wait runs out without any fault, or has its products
give up: the kernel records status 11, waits for the copies it did ask for, frees its tensor memory and returns by itself; the same call right
after is correct."""

import ctypes

import pytest
import torch

from tests import plain_mxfp4 as P
from tests import test_gpu_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda"
POLLS = 4096


@pytest.fixture(scope="module")
def runtime():
    from tandemllm_b200.kernels import tensorcore
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16)
    tensorcore.enable(rt)
    return rt


@pytest.fixture
def stop(runtime):
    """stop(copies=, products=): from now on the tensor-core products' copies end, or their products give up, at that tile of a CTA's work;
    stop(stage=): the few-row products' copies of that stage of a group's work are left out."""
    from tandemllm_b200.kernels import mxfp4
    lib = mxfp4.lib()._library
    limits = lib.tl_mxfp4_tc_set_wait_limit, lib.tl_mxfp4_few_set_wait_limit
    for f in limits:
        f.argtypes, f.restype = [ctypes.c_uint], ctypes.c_int
    lib.tl_mxfp4_tc_test_stop.argtypes, lib.tl_mxfp4_tc_test_stop.restype = [ctypes.c_int, ctypes.c_int], None
    lib.tl_mxfp4_few_test_skip_stage.argtypes, lib.tl_mxfp4_few_test_skip_stage.restype = [ctypes.c_int], None

    def hook(copies=-1, products=-1, stage=-1, polls=POLLS):
        torch.cuda.synchronize()
        for f in limits:
            assert f(polls) == 0
        lib.tl_mxfp4_tc_test_stop(copies, products)
        lib.tl_mxfp4_few_test_skip_stage(stage)

    def back():
        hook(polls=0)
        runtime.status.zero_()

    hook.back = back
    yield hook
    back()


def gave_up(runtime):
    torch.cuda.synchronize()                     # returns: the kernels ended by their own bound
    return int(runtime.status.item()) == 11


@pytest.mark.parametrize("what", ["copies", "products"])
@pytest.mark.parametrize("tile", [0, 1, 2, 5, 6])
@pytest.mark.parametrize("form", [(16, 1), (64, 1), (128, 1), (32, 2), (128, 2), (64, 0), (160, 0), (256, 0)])
def test_products_of_many_rows(runtime, stop, form, tile, what, monkeypatch):
    from tandemllm_b200.kernels import mxfp4
    if form[1] == 2 and tile > 2:
        tile = 2                                 # (of its share of seven tiles every CTA of a cluster has three)
    monkeypatch.setattr(mxfp4, "shape_of", lambda *a: form)
    g = torch.Generator().manual_seed(tile)
    x, w = M.rows(g, 100, 7 * 128 - 3), M.weights(g, 2, 200, 7 * 128 - 3)
    xd, one, pair, v = x.to(DEV), mxfp4.quantize(w[0].to(DEV)), mxfp4.quantize(w.to(DEV)), P.rounded(w)
    out = torch.full((100, 200), float("nan"), device=DEV)
    for call in (lambda: mxfp4.linear(runtime, xd, one, out=out), lambda: mxfp4.gated(runtime, xd, pair)):
        stop(**{what: tile})
        call()
        assert gave_up(runtime)
        assert out.isnan().all(), "a product that gave up stores nothing"
        stop.back()
        got = call()
        P.hold(got, *(P.product(x, v[0]) if got is out else P.gated(x, v[0], v[1], "silu")))
        assert int(runtime.status.item()) == 0
        out.fill_(float("nan"))


@pytest.mark.parametrize("what", ["copies", "products"])
@pytest.mark.parametrize("tile", [0, 1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("form", [(160, 0), (256, 0)])
def test_a_later_item_of_a_persistent_cta(runtime, stop, form, tile, what, monkeypatch):
    """Of 235 tiles of three times 128 k a CTA has one or two."""
    from tandemllm_b200.kernels import mxfp4
    monkeypatch.setattr(mxfp4, "shape_of", lambda *a: form)
    g = torch.Generator().manual_seed(tile)
    x, w = M.rows(g, 100, 384), M.weights(g, 30000, 384)
    xd, q = x.to(DEV), mxfp4.quantize(w.to(DEV))
    stop(**{what: tile})
    mxfp4.linear(runtime, xd, q)
    assert gave_up(runtime) == (tile < 6)
    stop.back()
    P.hold(mxfp4.linear(runtime, xd, q), *P.product(x, P.rounded(w)))
    assert int(runtime.status.item()) == 0


@pytest.mark.parametrize("what", ["copies", "products"])
@pytest.mark.parametrize("tile", [0, 1, 4, 8, 9, 13])
@pytest.mark.parametrize("m", [30, 300])
def test_experts_of_many_rows(runtime, stop, m, tile, what):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m + tile)
    x = M.rows(g, m, 5 * 128)
    e, inter = (64, 72) if m == 30 else (3, 300)
    ids, wts = M.routed(g, m, e, 2)
    first, down, v_first, v_down = M.layer(g, e, 2, inter, 5 * 128)
    args = x.to(DEV), ids.to(DEV), wts.to(DEV), mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    stop(**{what: tile})
    mxfp4.experts(runtime, *args)
    assert gave_up(runtime) or tile >= 5         # (a CTA may have one item of five tiles, and the second half's three)
    stop.back()
    P.hold(mxfp4.experts(runtime, *args), *P.experts(x, ids, wts, v_first, v_down, "silu"))
    assert int(runtime.status.item()) == 0


@pytest.mark.parametrize("stage", [0, 1, 2])
@pytest.mark.parametrize("m,tiles", [(1, 60), (8, 60), (13, 60), (13, 20)])
def test_products_of_few_rows(runtime, stop, m, tiles, stage):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m + stage)
    k = tiles * 128
    x, w = M.rows(g, m, k), M.weights(g, 2, 72, k)
    xd, one, pair, v = x.to(DEV), mxfp4.quantize(w[0].to(DEV)), mxfp4.quantize(w.to(DEV)), P.rounded(w)
    out = torch.full((m, 72), float("nan"), device=DEV)
    for call in (lambda: mxfp4.linear(runtime, xd, one, out=out), lambda: mxfp4.gated(runtime, xd, pair)):
        stop(stage=stage)
        call()
        # (a group of a team of four has a quarter of a unit's tiles: one stage of 16, or up to four; 13 rows of 60 tiles go to the other kernels)
        assert gave_up(runtime) or stage > 0 or not mxfp4.lib().tl_mxfp4_few_fits(m, 72, k, 0)
        assert int(runtime.status.item()) == 0 or out.isnan().all()
        stop.back()
        got = call()
        P.hold(got, *(P.product(x, v[0]) if got is out else P.gated(x, v[0], v[1], "silu")))
        assert int(runtime.status.item()) == 0
        out.fill_(float("nan"))


@pytest.mark.parametrize("stage", [0, 1])
@pytest.mark.parametrize("m,top", [(1, 1), (3, 4), (8, 6)])
def test_experts_of_few_rows(runtime, stop, m, top, stage):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m + stage)
    x = M.rows(g, m, 640)
    ids, wts = M.routed(g, m, 9, top)
    first, down, v_first, v_down = M.layer(g, 9, 2, 300, 640)
    args = x.to(DEV), ids.to(DEV), wts.to(DEV), mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    stop(stage=stage)
    mxfp4.experts(runtime, *args)
    assert gave_up(runtime) or stage > 0
    stop.back()
    P.hold(mxfp4.experts(runtime, *args), *P.experts(x, ids, wts, v_first, v_down, "silu"))
    assert int(runtime.status.item()) == 0
