"""What a routed layer's matrices are rounded from: the stored numbers, whatever types the experts' tensors are stored in."""

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


def bound(types, gated, weights, dtype=BF16):
    """The tensors that an experts part hands to the rounding, and the stored ones. `types`: (expert, which) -> dtype, else bfloat16."""
    from tandemllm_b200.config.spec import PartSpec
    from tandemllm_b200.parts.base import Runtime, make_part
    E, H, I = 3, 64, 40
    spec = PartSpec("sigmoid_topk_experts", {"num_experts": E, "top_k": 2, "intermediate_size": I, "gated": gated, "activation": "silu",
                                             "names": {"router": "r", "bias": "b", "experts": "x", "gate": "g", "up": "u", "down": "d"}})
    part = make_part("feed_forward", spec, prefix="", hidden_size=H)
    runtime = Runtime(torch.device("cpu"), dtype, feed_forward_weights=weights)
    g, stored = torch.Generator().manual_seed(1), {}
    for s in part.weight_specs(None):
        t = torch.randn(*s.shape, generator=g)
        at = next(((e, w) for e in range(E) for w in ("gate", "up", "down") if s.name == part._expert(e, w)) if "x" in s.name else iter(()), None)
        stored[s.name] = t.to(types.get(at, BF16)) if at else t
    seen = []
    runtime.feed_forward_matrix = lambda t, matrices=None: seen.append(t) or t
    part.bind(lambda name: stored[name], runtime)
    want_down = [stored[part._expert(e, "down")] for e in range(E)]
    want_up = [torch.cat([stored[part._expert(e, w)].float() for w in (("gate", "up") if gated else ("up",))]) for e in range(E)]
    return seen, want_up, want_down


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("types", [{}, {(0, "down"): F32}, {(2, "down"): F32}, {(1, "up"): F32}, {(0, "up"): F32}, {(e, "down"): F32 for e in range(3)},
                                   {(2, "gate"): F32, (0, "down"): F32}, {(e, w): F32 for e in range(3) for w in ("gate", "up", "down")},
                                   {(1, "down"): torch.float16}])
def test_the_stored_numbers_reach_the_rounding(types, gated):
    (up, down), want_up, want_down = bound(types, gated, "mxfp4")
    for e in range(3):
        assert torch.equal(up[e].float(), want_up[e]) and torch.equal(down[e].float(), want_down[e].float())
    assert (down.dtype is BF16) == all(w != "down" for _, w in types)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_stored_weights_are_staged_in_the_compute_dtype(dtype):
    (up, down), want_up, want_down = bound({(1, "down"): F32}, True, "stored", dtype)
    assert up.dtype is dtype and down.dtype is dtype
    for e in range(3):
        assert torch.equal(up[e], want_up[e].to(dtype)) and torch.equal(down[e], want_down[e].to(dtype))
