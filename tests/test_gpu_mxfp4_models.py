"""Whole models whose feed-forwards' matrices are rounded to 4-bit blocks when they are loaded, against the plain implementations run on
weights rounded by the format's definition (tests/plain_mxfp4.py), with the tolerances that the models have without the rounding: the
rounded weights are exact in both compute dtypes, so the products have no further error."""

import json
import os
import subprocess
import sys

import pytest
import torch

from tests import plain_lfm2, plain_mxfp4, plain_sifupel
from tests import test_gpu_dipivik as dipivik
from tests import test_gpu_gifopel as gifopel
from tests import test_gpu_niralix as niralix
from tests import test_gpu_puripel as puripel
from tests import test_gpu_sebilorn as sebilorn
from tests import tiny_configs as T
from tests.helpers import random_model_weights, write_folder

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOL = {"float32": 1e-4, "bfloat16": 3e-2}


def matrices(part):
    """The names of a feed-forward's matrices that are rounded: all but a router's and a shared part's gate."""
    if hasattr(part, "shared"):
        return matrices(part.routed) + matrices(part.shared)
    router = part.prefix + part.n["router"] + part.suffix if hasattr(part, "top_k") else None
    return [s.name for s in part.weight_specs(None) if s.role == "matrix" and s.name != router]


def rounded_weights(spec, W):
    from tandemllm_b200.parts.model import DecoderModel
    names = [n for layer in DecoderModel(spec).layers for n in matrices(layer.feed_forward)]
    assert names
    return {**W, **{n: plain_mxfp4.rounded(W[n]).float() for n in names}}


def engine_on(spec, W, dtype, weights="mxfp4", **kw):
    from tandemllm_b200.engine import Engine, EngineArgs
    from tandemllm_b200.weights.loader import DictWeights
    args = dict(max_len=4096, parallel=4, block_size=16, kv_blocks=64, graph=False)
    return Engine._build(None, spec, DictWeights({k: v.clone() for k, v in W.items()}),
                         EngineArgs(dtype=dtype, feed_forward_weights=weights, **{**args, **kw}))


FAMILIES = {"dipivik": (dipivik, "DipivikConfig"), "gifopel": (gifopel, "GifopelConfig"), "niralix": (niralix, "NiralixConfig"),
            "puripel": (puripel, "PuripelConfig"), "sebilorn": (sebilorn, "SebilornConfig")}


# gates silu, gelu_tanh with biases, clamped; ungated relu2; experts beside a shared part, weighed in front, without gates; odd widths
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("family,name", [("dipivik", "d2"), ("dipivik", "d4"), ("gifopel", "f2"), ("gifopel", "f4"), ("niralix", "n2"),
                                         ("puripel", "p1"), ("puripel", "p2"), ("sebilorn", "b2"), ("sebilorn", "b4")])
def test_models_agree_with_the_plain_model_on_rounded_weights(family, name, dtype):
    import tandemllm_b200.config as config
    module, kind = FAMILIES[family]
    cfg, W = module.C.CONFIGS[name], module.C.weights(name, bf16_exact=True)
    spec = getattr(config, kind).from_dict(cfg).to_spec()
    rounded = rounded_weights(spec, W)
    engine = engine_on(spec, W, dtype)
    toks = module.C.tokens(name, 90, seed=3)
    for requests, schedule in (({"a": toks[:40]}, [[("a", 33)], [("a", 2)]] + [[("a", 1)]] * 5),
                               ({"a": toks, "b": toks[5:40]}, [[("a", 64), ("b", 17)], [("a", 21), ("b", 3)], [("a", 2), ("b", 15)], [("a", 3)]])):
        if dtype == "float32":
            module.held_to_the_plain_model(engine, cfg, rounded, requests, schedule, dtype, "rounded")
            continue
        # In bfloat16 a routed layer whose two scores lie within rounding may take the other expert, and a recurrent state carries that into
        # every later row (gifopel f2: one choice at a margin of 0.011 in a logit of size one moves its row by half of its largest number and
        # the rows behind it by a tenth, the same to three digits where the rounded weights are plain bfloat16 matrices). So a row is held to
        # the plain model or to the bfloat16 engine on the rounded weights, whichever it is nearer to; nine in ten to the tolerance and all to
        # four times that, as the models without the rounding are.
        got = module.run_schedule(engine, requests, schedule)
        stored = module.run_schedule(engine_on(spec, rounded, dtype, weights="stored"), requests, schedule)
        rows = []
        for r, toks_r in requests.items():
            want = torch.as_tensor(module.P.forward(cfg, rounded, toks_r))
            rows.append(torch.minimum(puripel.rel_rows(got[r], want), puripel.rel_rows(got[r], stored[r])))
        rows = torch.cat(rows)
        assert float(rows.quantile(0.9)) < TOL[dtype] and float(rows.max()) < 4 * TOL[dtype], (float(rows.quantile(0.9)), float(rows.max()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_an_ungated_feed_forward_whose_activation_has_tensors(dtype):
    from tandemllm_b200.config import SifupelConfig
    from tests import sifupel_configs as S
    from tests import test_gpu_sifupel as sifupel
    cfg, W = S.CONFIGS["s2"], S.weights("s2", bf16_exact=True)
    spec = SifupelConfig.from_dict(cfg).to_spec()
    toks = S.tokens("s2", 60, seed=3)
    want = plain_sifupel.forward(cfg, rounded_weights(spec, W), list(toks))
    engine = engine_on(spec, W, dtype)
    for schedule in ([[("a", 60)]], [[("a", 40)]] + [[("a", 1)]] * 20):
        assert sifupel.rel(sifupel.run_schedule(engine, {"a": toks}, schedule)["a"], want) < TOL[dtype]


def lfm2(name):
    from tandemllm_b200.config import Lfm2MoeConfig
    cfg = T.CONFIGS[name]
    return cfg, Lfm2MoeConfig.from_dict(cfg).to_spec(), random_model_weights(cfg, T.SEEDS[name], T.STD[name], bf16_exact=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["b", "c", "d", "e"])
def test_gated_and_routed_layers_follow_the_plain_model_with_the_chosen_experts(name, dtype):
    cfg, spec, W = lfm2(name)
    rounded = rounded_weights(spec, W)
    engine = engine_on(spec, W, dtype)
    requests = {"a": T.long_tokens(name, 100), "b": T.long_tokens(name, 31, seed=8)}
    routes = {}
    got = puripel.run_schedule(engine, requests, [[("a", 64), ("b", 1)], [("a", 9), ("b", 20)], [("a", 2), ("b", 3)]] + [[("a", 1), ("b", 1)]] * 7
                               + [[("a", 18)]], routes)
    routed = [i for i in range(cfg["num_hidden_layers"]) if i >= cfg["num_dense_layers"]]
    for r, toks in requests.items():
        want = plain_lfm2.forward(cfg, rounded, toks, dtype=torch.float64, forced_routes=dict(zip(routed, routes[r])))
        rows = puripel.rel_rows(got[r], want)
        assert float(rows.max()) < TOL[dtype], (r, float(rows.max()))


def test_32_bit_models_run_the_rounded_values_as_plain_matrices():
    cfg, spec, W = lfm2("c")
    toks = {"a": T.long_tokens("c", 50)}
    schedule = [[("a", 30)]] + [[("a", 1)]] * 20
    a = puripel.run_schedule(engine_on(spec, W, "float32"), toks, schedule)["a"]
    b = puripel.run_schedule(engine_on(spec, rounded_weights(spec, W), "float32", weights="stored"), toks, schedule)["a"]
    c = puripel.run_schedule(engine_on(spec, W, "float32", weights="stored"), toks, schedule)["a"]
    assert torch.equal(a, b) and puripel.rel(a, c) > 1e-3


def test_bfloat16_without_the_tensor_core_kernels_runs_the_rounded_values_as_plain_matrices():
    cfg, spec, W = lfm2("c")
    toks = {"a": T.long_tokens("c", 50)}
    schedule = [[("a", 30)]] + [[("a", 1)]] * 20
    a, b = (puripel.run_schedule(engine_on(spec, w, "bfloat16", weights=k, tensorcore=False), toks, schedule)["a"]
            for w, k in ((W, "mxfp4"), (rounded_weights(spec, W), "stored")))
    assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["c", "d"])
def test_generation_from_graphs_is_generation_without_and_counts_its_routing(name):
    from tandemllm_b200.sampling import SamplingParams
    cfg, spec, W = lfm2(name)
    prompts = [T.long_tokens(name, n, seed=n) for n in (40, 3, 21, 1, 70)]
    params = SamplingParams(temperature=0.0, max_tokens=24, ignore_eos=True)
    outs = []
    for graph in (False, True, True):
        engine = engine_on(spec, W, "bfloat16", graph=graph, chunk_size=32, max_batched_tokens=64, record_routing=True)
        first, again = engine.generate(prompts, params), engine.generate(prompts, params)
        assert first == again                   # the second time every decode step is a replay
        records = list(engine.records)
        assert any(r["from_graph"] for r in records) == graph
        layers = cfg["num_hidden_layers"] - cfg["num_dense_layers"]
        assert all(r["pairs_routed"] == r["rows"] * cfg["num_experts_per_tok"] * layers for r in records)
        outs.append(first)
    assert outs[0] == outs[1] == outs[2]


def test_two_engines_side_by_side_do_not_share_a_workspace():
    from tandemllm_b200.engine import StepEntry
    cfg, spec, W = lfm2("c")
    toks = T.long_tokens("c", 60)
    engines = [engine_on(spec, W, "bfloat16", graph=True) for _ in range(2)]
    alone = puripel.run_schedule(engine_on(spec, W, "bfloat16"), {"a": toks}, [[("a", 30)]] + [[("a", 1)]] * 30)["a"][30:]
    for e in engines:
        e.admit("a")
        e.step([StepEntry("a", toks[:30], [29])])
    for i in range(30, 60):
        both = [e.step([StepEntry("a", toks[i:i + 1], [0])]).float().cpu() for e in engines]
        assert torch.equal(both[0], both[1]) and torch.equal(both[0][0], alone[i - 30])
    assert all(e.step_function.graph_replays > 20 for e in engines)


def test_the_byte_accounts_of_rounded_weights():
    cfg, spec, W = lfm2("c")
    stored, small = (engine_on(spec, W, "bfloat16", weights=k).model for k in ("stored", "mxfp4"))
    names = [n for layer in small.layers for n in matrices(layer.feed_forward)]
    numbers = sum(W[n].numel() for n in names)          # (widths of 128 and multiples of 8: no padding)
    padded = sum(-(-W[n].shape[-1] // 128) * 128 * W[n].numel() // W[n].shape[-1] for n in names)
    assert stored.weight_bytes() - small.weight_bytes() == 2 * numbers - padded * 17 // 32
    from tandemllm_b200.kernels.mxfp4 import Mxfp4Matrix
    for a, b in zip(stored.layers, small.layers):
        assert isinstance(b.feed_forward.w_down, Mxfp4Matrix) and isinstance(a.feed_forward.w_down, torch.Tensor)
        n = sum(W[m].numel() for m in matrices(a.feed_forward))
        kw = dict(experts_read=cfg["num_experts"]) if hasattr(a.feed_forward, "top_k") else {}
        assert abs(a.feed_forward.step_bytes(2, **kw) - b.feed_forward.step_bytes(2, **kw) - n * (2 - 17 / 32)) < 2


def test_the_command_line_generates_with_rounded_weights(tmp_path):
    from tandemllm_b200.engine import Engine, EngineArgs
    from tandemllm_b200.sampling import SamplingParams
    cfg, spec, W = lfm2("c")
    folder = write_folder(str(tmp_path / "m"), cfg, W, torch.bfloat16)
    prompt, out = T.long_tokens("c", 20), tmp_path / "out.json"
    r = subprocess.run([sys.executable, "-m", "tandemllm_b200", "generate", "--model", folder, "--feed-forward-weights", "mxfp4", "--prompt-ids",
                        ",".join(map(str, prompt)), "--tokens", "8", "--json", str(out)], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    engine = Engine.from_folder(folder, EngineArgs(dtype="bfloat16", feed_forward_weights="mxfp4"))
    assert json.loads(out.read_text())["outputs"][0] == engine.generate([prompt], SamplingParams(temperature=0.0, max_tokens=8))[0]
