"""What an `Mxfp4Matrix` is made of, and its copies: they own the bytes that the kernels are pointed at."""

import copy
import pickle

import pytest
import torch


def a_matrix(shape=(3, 9, 130)):
    from tandemllm_b200.kernels import mxfp4
    tiles = shape[0] * -(-shape[1] // 8) * -(-shape[2] // 128)
    return mxfp4.Mxfp4Matrix(torch.arange(tiles * 544).to(torch.uint8), shape)


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "copy"])
def test_a_copy_points_into_its_own_bytes(how):
    from tandemllm_b200.kernels import mxfp4
    m = a_matrix()
    c = {"deepcopy": copy.deepcopy, "pickle": lambda m: pickle.loads(pickle.dumps(m)), "copy": copy.copy}[how](m)
    assert type(c) is mxfp4.Mxfp4Matrix and torch.equal(c.data, m.data)
    assert c.codes == c.data.data_ptr() and c.scales == c.codes + m.scales - m.codes and c.scales - c.codes == 3 * 2 * 2 * 512
    assert (c.data.data_ptr() == m.data.data_ptr()) == (how == "copy")
    assert (c.shape, c.groups, c.n, c.k, c.device, c.index, c.nbytes, c.numel()) == (m.shape, 3, 9, 130, m.device, m.index, m.nbytes, 3 * 9 * 130)


def test_a_part_s_copy_points_into_its_own_bytes():
    class Part:
        pass
    p = Part()
    p.w_down = a_matrix((16, 128, 128))
    q = copy.deepcopy(p)
    assert q.w_down.codes == q.w_down.data.data_ptr() != p.w_down.codes


@pytest.mark.parametrize("data,shape", [
    (torch.zeros(544 * 4, dtype=torch.uint8), (9, 256, 1, 1)), (torch.zeros(544 * 4, dtype=torch.uint8), (256,)), (torch.zeros(543, dtype=torch.uint8), (8, 128)),
    (torch.zeros(544 * 2, dtype=torch.uint8), (8, 128)), (torch.zeros(544), (8, 128)), (torch.zeros(544, dtype=torch.int8), (8, 128)),
    (torch.zeros(544 * 2, dtype=torch.uint8)[::2], (8, 128)), (torch.zeros(561, dtype=torch.uint8)[1:545], (8, 128)),
    (torch.zeros(544, dtype=torch.uint8), (-8, -128))])
def test_bytes_that_are_not_the_matrix_s_are_refused(data, shape):
    from tandemllm_b200.kernels import mxfp4, ops
    with pytest.raises(ops.KernelError, match="mxfp4"):
        mxfp4.Mxfp4Matrix(data, shape)


def test_matrices_without_numbers_are_made():
    from tandemllm_b200.kernels import mxfp4
    for shape in ((0, 64), (4, 0), (0, 3, 32), (2, 0, 32)):
        assert mxfp4.Mxfp4Matrix(torch.zeros(0, dtype=torch.uint8), shape).shape == shape
