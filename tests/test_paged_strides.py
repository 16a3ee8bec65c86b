"""Strides that the paged attentions hand to the C entry points."""

import torch

from iron_b200.common.paged import stride_array


def test_dimensions_of_one_element_have_no_stride():
    shape = (1, 3, 1, 64)
    odd = torch.empty_strided(shape, (5, 64, 7, 1))
    plain = torch.empty(shape)
    assert list(stride_array(odd, shape)) == [0, 64, 0]
    assert stride_array(odd, shape) is stride_array(plain, shape)  # as k_new and v_new must have
    flat = torch.empty(3 * 64 + 10)  # a larger contiguous buffer
    assert stride_array(flat, shape) is stride_array(plain, shape)


def test_other_strides_stay_as_they_are():
    x = torch.empty(2, 5, 6, 64)
    assert list(stride_array(x[:, :, 1:3], (2, 5, 2, 64))) == [1920, 384, 64]
    assert list(stride_array(x[:, :, 1:3].transpose(0, 1), (5, 2, 2, 64))) == [384, 1920, 64]
    assert list(stride_array(x[:1].expand(4, 5, 6, 64), (4, 5, 6, 64))) == [0, 384, 64]
