"""What the 4-bit products' launchers refuse before anything is launched."""

import pytest

BAD = 100001


def tc(**kw):
    """The result of the tensor-core product's launcher, given one thing that it has to refuse (so nothing is launched)."""
    from tandemllm_b200.kernels import mxfp4
    a = dict(x=16, ldx=128, x_rows=40, codes=16, scales=16, bias=None, out=16, ldc=256, M=40, N=256, K=128, act=0, a0=0.0, a1=0.0, out_dtype=1, bn=64,
             splits=1, tile_group=None, tile_row0=None, tile_rows=None, n_tiles=None, max_tiles=0, row_weight=None, weight_index=None, status=16,
             stream=None)
    assert set(kw) <= set(a)
    code = mxfp4.lib().tl_mxfp4_tc(*{**a, **kw}.values())
    return code, mxfp4.lib().tl_mx_last_error().decode()


PLAN = dict(tile_group=16, tile_row0=16, tile_rows=16, n_tiles=16, max_tiles=3)


@pytest.mark.parametrize("bad,why", [
    (dict(splits=1, **PLAN), "persistent form"), (dict(splits=2, K=512, ldx=512, **PLAN), "persistent form"), (dict(row_weight=16), "persistent form"),
    (dict(row_weight=16, splits=0), "persistent form"), (dict(splits=0, **{**PLAN, "tile_rows": None}), "incomplete plan"), (dict(bn=48), "48 rows"),
    (dict(bn=0), "0 rows"), (dict(bn=257, splits=0), "257 rows"), (dict(splits=9, K=4096, ldx=4096), "9 runs"), (dict(splits=2), "2 runs"),
    (dict(ldx=129), "row stride"), (dict(x=8), "row stride"), (dict(act=1, out_dtype=0), "type 0"), (dict(act=-5), "activation -5"),
    (dict(act=7), "activation 7")])
def test_the_tensor_core_product_refuses(bad, why):
    code, text = tc(**bad)
    assert code == BAD and why in text
