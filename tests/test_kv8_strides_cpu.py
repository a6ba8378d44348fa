"""Rows as views: a stride that moves nothing, that of an axis of extent 1, is no reason to refuse a call."""
import pytest
import torch

from qcom_htp_b200 import kv8

BF = torch.bfloat16
META = torch.device("meta")


def fields(shape, strides, ragged=False):
    t = torch.empty_strided(shape, strides, dtype=BF, device="meta")
    return kv8._rows_fields("q", t, shape[-2], shape[-1], BF, META, ragged)


@pytest.mark.parametrize("shape,strides,ragged,want", [
    ((1, 1, 4, 64), (999, 256, 64, 1), False, (0, 256, 64)),     # the only sequence
    ((1, 1, 4, 64), (999, 333, 64, 1), False, (0, 0, 64)),
    ((2, 1, 4, 64), (4096, 333, 64, 1), False, (4096, 0, 64)),   # single tokens
    ((2, 3, 1, 64), (4096, 512, 77, 1), False, (4096, 512, 0)),  # a single head
    ((1, 4, 64), (4100, 64, 1), True, (0, 0, 64)),               # the only packed row
    ((0, 3, 4, 64), (770, 256, 64, 1), False, (0, 256, 64)),
])
def test_strides_of_axes_of_extent_one_do_not_matter(shape, strides, ragged, want):
    got = fields(shape, strides, ragged)[1:]
    extent = (1, *shape) if ragged else shape
    for n, g, w in zip(extent, got, want):
        assert g == w or n <= 1
        assert g * 2 % 16 == 0


@pytest.mark.parametrize("shape,strides,ragged", [((2, 1, 4, 64), (999, 256, 64, 1), False), ((1, 2, 4, 64), (999, 257, 64, 1), False),
                                                  ((1, 1, 2, 64), (128, 128, 65, 1), False), ((2, 4, 64), (257, 64, 1), True),
                                                  ((1, 1, 4, 64), (512, 512, 128, 2), False)])
def test_strides_that_matter_are_refused(shape, strides, ragged):
    with pytest.raises(ValueError):
        fields(shape, strides, ragged)
