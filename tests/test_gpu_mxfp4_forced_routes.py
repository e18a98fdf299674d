"""Whole bfloat16 models with rounded feed-forwards, row by row against the plain implementation alone, which is given the experts that the engine
chose: what a near tie between two experts does is then in neither's way."""

import numpy as np
import pytest
import torch

from tests import test_gpu_mxfp4_models as models
from tests import test_gpu_puripel as puripel

pytestmark = pytest.mark.gpu
TOL = 3e-2          # of a row's largest logit: nine rows in ten; every row four times that (as the models without the rounding are held)


class Forced:
    """numpy, but for a choice of the largest scores: the next of `rows` comes first (a plain model sorts nothing else)."""

    def __init__(self, rows):
        self.rows, self.used = rows, 0

    def __getattr__(self, name):
        return getattr(np, name)

    def argsort(self, a, axis=-1, kind=None):
        out = []
        for _ in range(1 if a.ndim == 1 else len(a)):
            first = self.rows[self.used].tolist()
            self.used += 1
            out.append(first + [e for e in range(a.shape[-1]) if e not in first])
        return np.array(out[0] if a.ndim == 1 else out)


@pytest.mark.parametrize("family,name", [("dipivik", "d2"), ("dipivik", "d4"), ("gifopel", "f2"), ("gifopel", "f4"), ("niralix", "n2"),
                                         ("puripel", "p1"), ("puripel", "p2"), ("sebilorn", "b2"), ("sebilorn", "b4")])
def test_rows_of_a_bfloat16_model(family, name, monkeypatch):
    import tandemllm_b200.config as config
    module, kind = models.FAMILIES[family]
    cfg, W = module.C.CONFIGS[name], module.C.weights(name, bf16_exact=True)
    spec = getattr(config, kind).from_dict(cfg).to_spec()
    rounded = models.rounded_weights(spec, W)
    engine = models.engine_on(spec, W, "bfloat16")
    toks = module.C.tokens(name, 90, seed=3)
    for requests, schedule in (({"a": toks[:40]}, [[("a", 33)], [("a", 2)]] + [[("a", 1)]] * 5),
                               ({"a": toks, "b": toks[5:40]}, [[("a", 64), ("b", 17)], [("a", 21), ("b", 3)], [("a", 2), ("b", 15)], [("a", 3)]])):
        routes, rows = {}, []
        got = puripel.run_schedule(engine, requests, schedule, routes)
        for r, mine in requests.items():
            if family == "puripel":
                want = module.P.forward(cfg, rounded, mine, routes=routes[r])
            else:
                forced = Forced([row for site in routes.get(r, []) for row in site])
                monkeypatch.setattr(module.P, "np", forced, raising=False)
                want = torch.as_tensor(module.P.forward(cfg, rounded, mine))
                monkeypatch.undo()
                assert forced.used == len(forced.rows)
            rows.append(puripel.rel_rows(got[r], want))
        rows = torch.cat(rows)
        print(family, name, float(rows.quantile(0.5)), float(rows.quantile(0.9)), float(rows.max()))
        assert float(rows.quantile(0.9)) < TOL and float(rows.max()) < 4 * TOL, (float(rows.quantile(0.9)), float(rows.max()))
