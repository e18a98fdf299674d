"""The benchmark's options that say which weights it runs: taken where they are offered, refused elsewhere, and shown in its lines."""

import ctypes
import os
import subprocess
import sys
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("option", [["--impl", "reference"]] + [["--design", d] for d in ("sifupel", "puripel", "sebilorn", "niralix", "gifopel", "dipivik")])
def test_runs_of_stored_weights_refuse_rounded_ones(option):
    r = subprocess.run([sys.executable, "bench.py", *option, "--feed-forward-weights", "mxfp4"], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "--feed-forward-weights" in r.stderr and not r.stdout


@pytest.mark.parametrize("weights", ["stored", "mxfp4"])
def test_the_mixed_scenario_takes_the_option(weights, monkeypatch):
    import bench
    from tandemllm_b200.engine import Engine

    class Seen(Exception):
        pass

    def from_config(cfg, seed, args):
        raise Seen(args.feed_forward_weights)

    monkeypatch.setattr(Engine, "from_config", from_config)
    a = types.SimpleNamespace(requests=2, longest=256, new_tokens=2, budget_tokens=4096, dtype="bfloat16", graph="on", log=None,
                              feed_forward_weights=weights)
    with pytest.raises(Seen, match=weights):
        bench.mixed_serving(None, "m", a)
    assert bench.dtype_label(a) == ("bf16" if weights == "stored" else "bf16, feed-forward weights mxfp4")


def test_the_profile_table_knows_the_4_bit_launchers():
    import bench
    from tandemllm_b200.kernels import mxfp4
    for name, argtypes in mxfp4._SIGNATURES.items():
        if argtypes[-1] is not ctypes.c_void_p:
            continue
        for tile_group, act in ((None, 0), (None, 1), (5, 0), (5, 1)):
            args = [0] * len(argtypes)
            if name == "tl_mxfp4_tc":
                args[17], args[11] = tile_group, act
            family = bench.LaunchTimer.family(name, tuple(args))
            assert family != name
            if name == "tl_mxfp4_tc":
                assert family.startswith("experts" if tile_group else "dense") and ("gate/up" in family) == (bool(tile_group) and act == 1)
            if name in ("tl_mxfp4_few", "tl_mxfp4_experts_first", "tl_mxfp4_experts_second"):
                assert family.startswith("dense" if name == "tl_mxfp4_few" else "experts")


def test_the_profile_table_times_the_4_bit_library_where_it_is_loaded(monkeypatch):
    import bench
    from tandemllm_b200.kernels import mxfp4, ops, tensorcore
    fake = {m: types.SimpleNamespace() for m in ("core", "tc", "mx")}
    monkeypatch.setattr(ops, "core", lambda: fake["core"])
    monkeypatch.setattr(tensorcore, "lib", lambda: fake["tc"])
    monkeypatch.setattr(mxfp4, "_lib", None)
    assert bench.LaunchTimer().libs == [fake["core"], fake["tc"]]
    monkeypatch.setattr(mxfp4, "_lib", fake["mx"])
    assert bench.LaunchTimer().libs == [fake["core"], fake["tc"], fake["mx"]]
