"""Products with copies of a matrix whose original's bytes are gone."""

import copy
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "torch.save"])
@pytest.mark.parametrize("m", [3, 40])
def test_a_copy_outlives_its_original(m, how):
    from tandemllm_b200.kernels import mxfp4, tensorcore
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16)
    tensorcore.enable(rt)
    g = torch.Generator().manual_seed(m)
    w, x = torch.randn(40, 264, generator=g).to(DEV), torch.randn(m, 264, generator=g).to(DEV, torch.bfloat16)
    q = mxfp4.quantize(w)
    want, values = mxfp4.linear(rt, x, q), q.values()

    def saved(m):
        f = io.BytesIO()
        torch.save(m, f)
        f.seek(0)
        return torch.load(f, weights_only=False)

    c = {"deepcopy": copy.deepcopy, "pickle": lambda m: pickle.loads(pickle.dumps(m)), "torch.save": saved}[how](q)
    q.data.fill_(255)
    del q
    assert torch.equal(mxfp4.linear(rt, x, c), want) and torch.equal(c.values(), values)
