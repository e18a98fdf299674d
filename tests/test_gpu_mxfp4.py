"""MXFP4 matrices and the products with them against 64 bits (tests/plain_mxfp4.py has the definition and the bounds)."""

import pytest
import torch

from . import plain_mxfp4 as P

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


@pytest.fixture(scope="module")
def runtime():
    from tandemllm_b200.kernels import tensorcore
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16)
    tensorcore.enable(rt)
    return rt


def weights(g, *shape, scale=0.05):
    return torch.randn(*shape, generator=g) * scale * torch.exp(0.7 * torch.randn(*shape[:-1], 1, generator=g))


def rows(g, m, k):
    return (torch.randn(m, k, generator=g) * torch.exp(0.5 * torch.randn(k, generator=g))).to(torch.bfloat16)


# ---- the quantiser ----

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (8, 32), (9, 33), (7, 128), (16, 130), (130, 264), (3, 5, 7), (2, 16, 256), (4, 9, 1000)])
def test_values_are_the_nearest(dtype, shape):
    from tandemllm_b200.kernels import mxfp4
    w = weights(torch.Generator().manual_seed(sum(shape)), *shape).to(DT[dtype])
    m = mxfp4.quantize(w.to(DEV))
    assert m.shape == shape
    want = P.rounded(w)
    for out in DT.values():
        got = m.values(out)
        assert got.dtype == out and torch.equal(got.cpu().double(), want)


def test_ties_ranges_and_blocks_without_numbers():
    from tandemllm_b200.kernels import mxfp4
    ties = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, -0.0, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -6, -7.9,
                         2 ** -30, .2500001, .7499999, 1.2500001, 4.9999995, 7.9999995])
    blocks = [ties, ties * 2.0 ** 124, ties * 2.0 ** -126, ties * 2.0 ** -100, torch.zeros(32), torch.full((32,), 2.0 ** -149),
              torch.full((32,), 2.0 ** -128), torch.full((32,), 3.3e38), torch.arange(32.0), ties.flip(0) * -8]
    w = torch.stack(blocks)
    got = mxfp4.quantize(w.to(DEV)).values(torch.float32)
    assert torch.equal(got.cpu().double(), P.rounded(w))
    for bad in (float("inf"), float("-inf"), float("nan")):
        w = torch.ones(9, 96)
        w[4, 40] = bad
        got = mxfp4.quantize(w.to(DEV)).values(torch.float32).cpu()
        assert got[4, 32:64].isnan().all() and (got[:4] == 1).all() and (got[5:] == 1).all()
        assert (got[4, :32] == 1).all() and (got[4, 64:] == 1).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment_of_what_is_quantised(dtype):
    from tandemllm_b200.kernels import mxfp4
    w = weights(torch.Generator().manual_seed(5), 2, 40, 264).to(DT[dtype]).to(DEV)
    for view in (w[0, :, :200], w[0, :, 1:], w[1, 3:, 8:136], w[:, ::2], w[0].T, w.transpose(1, 2), w[:, :, ::3], w[:, 5:6, :64],
                 torch.ones(1, device=DEV, dtype=DT[dtype]).expand(7, 65)):
        assert torch.equal(mxfp4.quantize(view).values(torch.float32).cpu().double(), P.rounded(view))


def test_empty_matrices():
    from tandemllm_b200.kernels import mxfp4
    for shape in ((0, 64), (4, 0), (0, 3, 32), (2, 0, 32)):
        assert mxfp4.quantize(torch.empty(*shape, device=DEV)).values().shape == shape


# ---- products ----

SIZES = [(1, 16, 128), (1, 1, 8), (2, 17, 136), (7, 100, 72), (8, 64, 2048), (9, 33, 40), (16, 48, 264), (17, 40, 1000), (32, 130, 512), (33, 64, 256),
         (5, 24, 31), (3, 9, 1), (40, 257, 333), (64, 128, 128), (70, 300, 640), (128, 128, 1024), (129, 144, 200), (257, 130, 384), (300, 520, 136)]


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(runtime, m, n, k, out):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m * n + k)
    x, w, b = rows(g, m, k), weights(g, n, k), torch.randn(n, generator=g)
    q = mxfp4.quantize(w.to(DEV))
    want, off = P.product(x, P.rounded(w))
    P.hold(mxfp4.linear(runtime, x.to(DEV), q, out_dtype=DT[out]), want, off)
    want = want + b.double()
    P.hold(mxfp4.linear(runtime, x.to(DEV), q, b.to(DEV), out_dtype=DT[out]), want, off + 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("act", ["silu", "gelu", "relu2", "identity", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (3, 17, 136), (8, 100, 256), (20, 40, 200), (33, 72, 264), (130, 136, 256), (300, 65, 100)])
def test_gated_product(runtime, m, n, k, act):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m + n + k)
    x, w, b = rows(g, m, k), weights(g, 2, n, k), torch.randn(2 * n, generator=g)
    q, v = mxfp4.quantize(w.to(DEV)), P.rounded(w)
    P.hold(mxfp4.gated(runtime, x.to(DEV), q, act), *P.gated(x, v[0], v[1], act))
    P.hold(mxfp4.gated(runtime, x.to(DEV), q, act, b.to(DEV)), *P.gated(x, v[0], v[1], act, b))


@pytest.mark.parametrize("m", [1, 9, 40, 140])
def test_products_of_far_scales(runtime, m):
    """Blocks of 8 and more (a second factor), of 2^100, and of numbers next to the smallest."""
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x, w = rows(g, m, 288), weights(g, 48, 288)
    w[::3] *= 2.0 ** 9
    w[1::6, 32:64] *= 2.0 ** 100
    w[5::6] *= 2.0 ** -90
    want, off = P.product(x, P.rounded(w))
    P.hold(mxfp4.linear(runtime, x.to(DEV), mxfp4.quantize(w.to(DEV)), out_dtype=torch.float32), want, off)


@pytest.mark.parametrize("m", [1, 12, 50, 150])
def test_a_row_of_a_matrix_that_is_not_a_number(runtime, m):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x, w = rows(g, m, 256), weights(g, 40, 256)
    w[17, 77] = float("nan")
    got = mxfp4.linear(runtime, x.to(DEV), mxfp4.quantize(w.to(DEV))).cpu()
    assert got[:, 17].isnan().all() and got[:, :17].isfinite().all() and got[:, 18:].isfinite().all()


@pytest.mark.parametrize("m", [3, 20, 60, 200])
def test_views_of_rows_and_outputs(runtime, m):
    """Rows and outputs inside larger tensors: what is around them is neither read nor written."""
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    w = weights(g, 72, 200)
    q, v = mxfp4.quantize(w.to(DEV)), P.rounded(w)
    around = torch.full((m + 2, 320), float("nan"), dtype=torch.bfloat16)
    for at in (8, 3, 64):
        whole = around.clone()
        whole[1:m + 1, at:at + 200] = rows(g, m, 200)
        x = whole.to(DEV)[1:m + 1, at:at + 200]
        out = torch.full((m + 2, 100), 7.0, dtype=torch.bfloat16, device=DEV)
        mxfp4.linear(runtime, x, q, out=out[1:m + 1, 5:77])
        P.hold(out[1:m + 1, 5:77], *P.product(whole[1:m + 1, at:at + 200], v))
        out[1:m + 1, 5:77] = 7.0
        assert (out == 7.0).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu2", "identity"])
@pytest.mark.parametrize("m", [1, 9, 40, 70, 300])
def test_an_activation_behind_a_plain_product(runtime, m, act):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x, w, b = rows(g, m, 264), weights(g, 100, 264), torch.randn(100, generator=g)
    want, off = P.product(x, P.rounded(w))
    want = want + b.double()
    want, off = P.activated(want, off + 2.0 ** -24 * want.abs(), act)
    for out in DT.values():
        P.hold(mxfp4.linear(runtime, x.to(DEV), mxfp4.quantize(w.to(DEV)), b.to(DEV), out_dtype=out, act=act), want, off)


@pytest.fixture(scope="module")
def many(runtime):
    """Products with more tiles than SMs, of one to five tiles of k: (rows, matrices, their plain and gated products with bounds)."""
    from tandemllm_b200.kernels import mxfp4
    g, out = torch.Generator().manual_seed(5), []
    for k in (100, 136, 264, 392, 520):
        x, w = rows(g, 700, k), weights(g, 2, 3001, k)
        v = P.rounded(w)
        out.append((x.to(DEV), mxfp4.quantize(w[0].to(DEV)), mxfp4.quantize(w.to(DEV)), P.product(x, v[0]), P.gated(x, v[0], v[1], "silu")))
    return out


@pytest.mark.parametrize("form", [(h, 0) for h in (16, 48, 64, 80, 112, 144, 160, 176, 240, 256)] + [(b, s) for b in (16, 32, 64, 128) for s in (1, 2, 4, 8)])
def test_every_form_of_the_tensor_core_product(runtime, many, form, monkeypatch):
    from tandemllm_b200.kernels import mxfp4
    for x, one, pair, plain, gated in many:
        splits = min(form[1], -(-one.k // 128))
        monkeypatch.setattr(mxfp4, "shape_of", lambda *a: (form[0], splits))
        for out in DT.values():
            P.hold(mxfp4.linear(runtime, x, one, out_dtype=out), *plain)
        P.hold(mxfp4.gated(runtime, x, pair), *gated)


@pytest.mark.parametrize("m", [1, 12, 40, 150])
def test_one_row_seen_as_many(runtime, m):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x, w = rows(g, 1, 136), weights(g, 48, 136)
    P.hold(mxfp4.linear(runtime, x.to(DEV).expand(m, 136), mxfp4.quantize(w.to(DEV))), *P.product(x.expand(m, 136), P.rounded(w)))


# ---- routed experts ----

def routed(g, m, e, top):
    ids = torch.stack([torch.randperm(e, generator=g)[:top] for _ in range(m)]).to(torch.int32)
    return ids, torch.rand(m, top, generator=g) + 0.1


def layer(g, e, gates, inter, hidden):
    first, down = weights(g, gates * e, inter, hidden), weights(g, e, hidden, inter)
    return first, down, P.rounded(first).view(e, gates, inter, hidden), P.rounded(down)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,e,top,inter,hidden,act,gates,weigh", [
    (1, 8, 2, 64, 128, "silu", 2, "output"), (1, 1, 1, 16, 32, "silu", 2, "output"), (3, 6, 3, 40, 72, "gelu", 2, "input"),
    (8, 32, 4, 48, 136, "silu", 2, "output"), (8, 64, 32, 24, 64, "silu", 2, "output"), (5, 40, 8, 37, 131, "relu2", 1, "output"),
    (7, 5, 5, 130, 256, "gelu", 1, "input"), (9, 8, 2, 64, 128, "silu", 2, "output"), (20, 4, 3, 72, 200, "gelu", 2, "output"),
    (33, 16, 4, 61, 77, "silu", 2, "input"), (100, 6, 2, 96, 264, "relu2", 1, "output"), (150, 3, 2, 136, 128, "silu", 2, "output"),
    (300, 2, 1, 40, 64, "silu", 2, "output")])
def test_experts(runtime, m, e, top, inter, hidden, act, gates, weigh, out):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m + e + inter)
    x = rows(g, m, hidden)
    ids, wts = routed(g, m, e, top)
    first, down, v_first, v_down = layer(g, e, gates, inter, hidden)
    got = mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV)), act, weigh,
                        out_dtype=DT[out])
    P.hold(got, *P.experts(x, ids, wts, v_first, v_down, act, weigh))
    assert int(runtime.status.item()) == 0


@pytest.mark.parametrize("m", [1, 4, 8, 11, 90])
def test_all_rows_to_one_expert_and_none_to_others(runtime, m):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x = rows(g, m, 96)
    first, down, v_first, v_down = layer(g, 9, 2, 40, 96)
    q = mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    for ids in (torch.full((m, 1), 8), torch.tensor([[3, 0]]).expand(m, 2), torch.tensor([[7, 1, 4]]).expand(m, 3).flip(0)):
        ids = ids.to(torch.int32).contiguous()
        wts = torch.rand(*ids.shape, generator=g)
        P.hold(mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), *q), *P.experts(x, ids, wts, v_first, v_down, "silu"))


@pytest.mark.parametrize("m", [1, 6, 8, 14, 70])
def test_a_row_that_names_an_expert_twice_and_ids_that_name_none(runtime, m):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(m)
    x = rows(g, m, 64)
    first, down, v_first, v_down = layer(g, 5, 2, 32, 64)
    q = mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    for top in (3, 7):
        ids = torch.randint(0, 5, (m, top), generator=g).to(torch.int32)
        wts = torch.rand(m, top, generator=g)
        P.hold(mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), *q), *P.experts(x, ids, wts, v_first, v_down, "silu"))
    assert int(runtime.status.item()) == 0
    ids[0, 1], ids[m - 1, 2] = 5, -1
    try:
        P.hold(mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), *q), *P.experts(x, ids, wts, v_first, v_down, "silu"))
        assert int(runtime.status.item()) == 6
    finally:
        runtime.status.zero_()


def test_results_repeat_bit_for_bit_and_do_not_depend_on_the_stream(runtime):
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(3)
    first, down, *_ = layer(g, 8, 2, 200, 264)
    q = mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    for m in (2, 8, 30, 200):
        x = rows(g, m, 264).to(DEV)
        ids, wts = (t.to(DEV) for t in routed(g, m, 8, 3))
        once = mxfp4.experts(runtime, x, ids, wts, *q, out_dtype=torch.float32)
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        both = []
        for s in side:
            with torch.cuda.stream(s):
                both.append(mxfp4.experts(runtime, x, ids, wts, *q, out_dtype=torch.float32))
        torch.cuda.synchronize()
        assert all(torch.equal(once, t) for t in both)


@pytest.mark.parametrize("weigh", ["input", "output"])
@pytest.mark.parametrize("m", [3, 8, 9, 60, 500])
def test_rows_that_a_consumer_adds(runtime, m, weigh):
    """With `defer` many rows come as the experts' own; added by the framework's combining kernel they are what the layer gives itself."""
    from tandemllm_b200.kernels import mxfp4, ops
    g = torch.Generator().manual_seed(m)
    first, down, v_first, v_down = layer(g, 6, 2, 72, 136)
    q = mxfp4.quantize(first.to(DEV)), mxfp4.quantize(down.to(DEV))
    x = rows(g, m, 136)
    ids, wts = routed(g, m, 6, 3)
    got = mxfp4.experts(runtime, x.to(DEV), ids.to(DEV), wts.to(DEV), *q, weigh=weigh, out_dtype=torch.float32, defer=True)
    assert isinstance(got, ops.ExpertRows) == (m > mxfp4.EXPERT_ROWS)
    P.hold(ops.materialize(got), *P.experts(x, ids, wts, v_first, v_down, "silu", weigh))


def test_two_captured_graphs_replayed_in_turn(runtime):
    """Products, both forms of the experts and the quantiser captured with inputs of their own: the replays do not disturb one another."""
    from tandemllm_b200.kernels import mxfp4
    g = torch.Generator().manual_seed(9)
    first, down, *_ = layer(g, 8, 2, 200, 264)
    w, w_first, w_down = weights(g, 264, 264).to(DEV), first.to(DEV), down.to(DEV)

    def run(x, ids, wts):
        q = mxfp4.quantize(w), mxfp4.quantize(w_first), mxfp4.quantize(w_down)
        h = mxfp4.linear(runtime, x, q[0])
        return mxfp4.experts(runtime, h, ids, wts, *q[1:], out_dtype=torch.float32)

    inputs = [(rows(g, m, 264).to(DEV), *(t.to(DEV) for t in routed(g, m, 8, 3))) for m in (4, 70, 8)]
    want = [run(*i) for i in inputs]
    graphs, outs = [], []
    for i in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*i))
        graphs.append(graph)
    for order in ((0, 1, 2), (2, 1, 0, 0, 2, 1)):
        for i in order:
            outs[i].zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- refusals ----

def test_refusals(runtime):
    from tandemllm_b200.kernels import mxfp4
    from tandemllm_b200.kernels.ops import KernelError
    from tandemllm_b200.parts.base import Runtime
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    m, pair = mxfp4.quantize(torch.ones(16, 64, device=DEV)), mxfp4.quantize(torch.ones(2, 16, 64, device=DEV))
    up, down = mxfp4.quantize(torch.ones(1, 16, 64, device=DEV)), mxfp4.quantize(torch.ones(1, 64, 16, device=DEV))
    ids, wts = torch.zeros(4, 1, dtype=torch.int32, device=DEV), torch.ones(4, 1, device=DEV)
    for bad in (lambda: mxfp4.quantize(torch.ones(64, device=DEV)), lambda: mxfp4.quantize(torch.ones(2, 2, 2, 2, device=DEV)),
                lambda: mxfp4.quantize(torch.ones(4, 64, dtype=torch.float16, device=DEV)), lambda: mxfp4.quantize(torch.ones(4, 64)),
                lambda: m.values(torch.float16),
                lambda: mxfp4.linear(runtime, x.float(), m), lambda: mxfp4.linear(runtime, x[:, :32], m), lambda: mxfp4.linear(runtime, x[0], m),
                lambda: mxfp4.linear(runtime, x.cpu(), m), lambda: mxfp4.linear(runtime, x.repeat(1, 2)[:, ::2], m), lambda: mxfp4.linear(runtime, x, pair),
                lambda: mxfp4.linear(runtime, x, m, torch.zeros(16, dtype=torch.bfloat16, device=DEV)),
                lambda: mxfp4.linear(runtime, x, m, torch.zeros(15, device=DEV)), lambda: mxfp4.linear(runtime, x, m, out=x),
                lambda: mxfp4.gated(runtime, x, m), lambda: mxfp4.gated(runtime, x, pair, "tanh"), lambda: mxfp4.gated(runtime, x, pair, "swish"),
                lambda: mxfp4.experts(runtime, x, ids.long(), wts, pair, down), lambda: mxfp4.experts(runtime, x, ids[:3], wts[:3], pair, down),
                lambda: mxfp4.experts(runtime, x, ids, wts[:, :0], pair, down), lambda: mxfp4.experts(runtime, x, ids, wts, down, pair),
                lambda: mxfp4.experts(runtime, x, ids, wts, pair, down, "xielu"), lambda: mxfp4.experts(runtime, x, ids, wts, pair, down, weigh="both"),
                lambda: mxfp4.linear(Runtime(torch.device("cpu"), torch.bfloat16), x, m), lambda: mxfp4.linear(runtime, x, m, act="gelu_tanh"),
                lambda: mxfp4.linear(runtime, x, m, act=0), lambda: mxfp4.experts(runtime, x, ids, wts, up, down, "clamped_swish"),
                lambda: mxfp4.experts(runtime, x, ids.expand(4, 40).contiguous(), wts.expand(4, 40).contiguous(), pair, down)):
        with pytest.raises(KernelError):
            bad()


def test_no_rows(runtime):
    from tandemllm_b200.kernels import mxfp4
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV)
    pair, down = mxfp4.quantize(torch.ones(2, 16, 64, device=DEV)), mxfp4.quantize(torch.ones(1, 64, 16, device=DEV))
    assert mxfp4.linear(runtime, x, mxfp4.quantize(torch.ones(16, 64, device=DEV))).shape == (0, 16)
    assert mxfp4.gated(runtime, x, pair).shape == (0, 16)
    none = torch.zeros(0, 2, device=DEV)
    assert mxfp4.experts(runtime, x, none.int(), none, pair, down).shape == (0, 64)
