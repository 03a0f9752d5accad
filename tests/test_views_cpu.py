"""Views of torch tensors as the operators for training pass them: kept by layout, correct for whichever tensor asks."""
import ctypes as C

import pytest
import torch

from tracea_amd import capi, ops


def fields(t):
    v = ops._plain_view(t)
    n = t.dim()
    return v.ptr, [v.shape[i] for i in range(n)], [v.stride[i] for i in range(n)], v.rank, v.dtype, v.device_id


@pytest.mark.parametrize("make", [
    lambda: torch.zeros(3, 5, 8), lambda: torch.zeros(3, 5, 16)[:, :, :8], lambda: torch.zeros(5, 3, 8).transpose(0, 1),
    lambda: torch.zeros(1, 5, 8).expand(3, 5, 8), lambda: torch.zeros(3, 5, 8, dtype=torch.bfloat16), lambda: torch.zeros(7),
    lambda: torch.zeros(3, 5, 8, dtype=torch.int32)])
def test_a_view_says_what_the_tensor_is(make):
    t = make()
    for x in (t, make(), t):
        ptr, shape, stride, rank, dtype, device = fields(x)
        assert (ptr, shape, stride, rank) == (x.data_ptr(), list(x.shape), list(x.stride()), x.dim())
        assert dtype == ops._DTYPES[x.dtype] and device == x.get_device()


def test_one_layout_for_contiguous_tensors_whatever_stands_for_extents_of_one():
    odd = torch.zeros(1000).as_strided((2, 1, 8), (8, 5, 1))
    plain = torch.zeros(2, 1, 8)
    assert odd.is_contiguous() and odd.stride() != plain.stride()
    assert fields(odd)[2] == fields(plain)[2] == [8, 8, 1]


def test_extents_of_zero_leave_strides_that_share_no_address():
    assert fields(torch.zeros(2, 0, 64))[1:3] == ([2, 0, 64], [64, 64, 1])


def test_a_view_outlives_the_kept_layouts():
    t = torch.zeros(3, 11, 8)
    v = ops._plain_view(t)
    row = torch.zeros(2100)
    for n in range(1, 2100):  # (more layouts than are kept)
        ops._plain_view(row[:n])
    assert [v.shape[i] for i in range(3)] == [3, 11, 8] and [v.stride[i] for i in range(3)] == [88, 8, 1]


def test_types_that_no_operator_has_are_refused():
    with pytest.raises(TypeError):
        ops._plain_view(torch.zeros(3, dtype=torch.complex64))


def test_parameter_blocks_have_the_size_of_the_headers():
    assert C.sizeof(capi.NormParams) == 16
    assert C.sizeof(capi.RotaryParams) == 32  # 4 + 4 * 4, two bytes, padding to 24, a pointer
    assert (capi.RotaryParams.adjacent.offset, capi.RotaryParams.inverse.offset, capi.RotaryParams.stream.offset) == (20, 21, 24)
