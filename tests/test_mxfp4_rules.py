"""The 4-bit matrices' choices and refusals that need no GPU."""

import subprocess
import sys

import pytest
import torch

from tests import plain_mxfp4


def test_the_definition_rounds_to_the_format_s_values():
    w = torch.tensor([[6.0, 5.0, 2.5, -0.25, 0.3, 7.9, 1.75, -3.5] + [0.0] * 24, [2.0 ** -130] + [0.0] * 31])
    assert plain_mxfp4.rounded(w)[0, :8].tolist() == [6.0, 4.0, 2.0, 0.0, 0.5, 6.0, 2.0, -4.0] and plain_mxfp4.rounded(w)[1, 0] == 0.0


def test_feed_forward_weights_are_named_ones():
    from tandemllm_b200.parts.base import Runtime
    with pytest.raises(ValueError, match="stored, mxfp4"):
        Runtime(torch.device("cpu"), torch.float32, feed_forward_weights="int4")
    assert Runtime(torch.device("cpu"), torch.float32).feed_forward_weights == "stored"
    r = subprocess.run([sys.executable, "-m", "tandemllm_b200", "generate", "--feed-forward-weights", "int4"], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 2 and "mxfp4" in r.stderr


def test_stored_weights_are_what_they_were():
    from tandemllm_b200.parts.base import Runtime
    rt = Runtime(torch.device("cpu"), torch.bfloat16)
    w = torch.randn(4, 6)
    assert torch.equal(rt.feed_forward_matrix(rt.feed_forward_source(w), 2), rt.matrix(w))
    rounding = Runtime(torch.device("cpu"), torch.bfloat16, feed_forward_weights="mxfp4")
    for dtype, kept in ((torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)):
        assert rounding.feed_forward_source(w.to(dtype)).dtype is kept


def test_a_matrix_off_the_gpu_is_refused():
    from tandemllm_b200.kernels import mxfp4, ops
    with pytest.raises(ops.KernelError, match="CUDA tensors only"):
        mxfp4.quantize(torch.zeros(4, 64))
    with pytest.raises(ops.KernelError, match=r"\[n, k\]"):
        mxfp4.quantize(torch.zeros(64))


@pytest.mark.parametrize("gated", [False, True])
def test_the_form_of_a_product_is_one_that_the_kernels_have(gated):
    from tandemllm_b200.kernels.mxfp4 import shape_of
    for rows in [*range(1, 300, 7), 512, 1000, 4097, 100000]:
        for tiles in (1, 2, 16, 57, 112, 300, 5000):
            for k in (1, 31, 128, 129, 600, 2048, 7168, 50000):
                h, splits = shape_of(rows, tiles, k, 148, gated)
                if splits == 0:
                    assert 64 <= h <= 256 and h % 16 == 0
                else:
                    assert h in (16, 32, 64, 128) and splits in (1, 2, 4, 8) and splits <= -(-k // 128)
                    assert splits == 1 or tiles * -(-rows // h) * splits <= 7 * 148 // 4
                    assert -(-rows // h) <= 65535
                assert h == 64 or h < 2 * max(rows, 16)


def test_the_form_of_a_product_follows_its_size():
    from tandemllm_b200.kernels.mxfp4 import shape_of
    assert shape_of(2048, 112, 2048, 148, True)[1] == 0                 # many tiles: persistent
    assert shape_of(256, 16, 7168, 148, False) == (128, 8)              # few tiles of a long k: shared
    assert shape_of(700, 16, 7168, 148, False)[1] in (0, 1)             # no second round of shared ones
