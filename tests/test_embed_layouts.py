"""How the embedding operators read tensors' layouts, on CPU tensors (no GPU)."""

import pytest
import torch

from browservec_amd import _lib as L
from browservec_amd import embed


@pytest.mark.parametrize("out", [torch.empty(1, 8).expand(5, 8), torch.empty(40).as_strided((5, 8), (4, 1)),
                                 torch.empty(1, 1).expand(5, 1), torch.empty(1, 1, 8).expand(2, 3, 8).view(6, 8)])
def test_an_output_whose_rows_overlap_is_refused(out):
    with pytest.raises(L.BVError) as e:
        embed._out_stride(out, "linear")
    assert e.value.code == L.BV_E_INVALID


@pytest.mark.parametrize("out", [torch.empty(1, 2, 8).expand(5, 2, 8), torch.empty(5, 1, 8).expand(5, 2, 8),
                                 torch.empty(1, 1, 8).expand(1, 2, 8), torch.empty(1, 1, 1).expand(4, 3, 1)])
def test_an_output_whose_heads_overlap_is_refused(out):
    with pytest.raises(L.BVError) as e:
        embed._out_heads(out, "attention")
    assert e.value.code == L.BV_E_INVALID


def test_outputs_that_do_not_overlap_pass():
    assert embed._out_stride(torch.empty(5, 12)[:, 2:10], "linear") == 12
    assert embed._out_stride(torch.empty(5, 8), "linear") == 0
    assert embed._out_stride(torch.empty(1, 8).expand(1, 8), "linear") == 0
    for out in (torch.empty(5, 2, 8), torch.empty(2, 5, 8).transpose(0, 1), torch.empty(5, 40)[:, 3:19].unflatten(1, (2, 8)),
                torch.empty(1, 1, 8).expand(1, 1, 8)):
        embed._out_heads(out, "attention")


def test_an_output_that_is_no_rows_at_one_stride_is_refused():
    for out in (torch.empty(2, 5, 8).transpose(0, 1), torch.empty(4, 5, 8)[:, :3]):
        with pytest.raises(L.BVError) as e:
            embed._flat(out, "linear")
        assert e.value.code == L.BV_E_INVALID
    out = torch.empty(4, 5, 12)[:, :, 2:10]
    rows = embed._flat(out, "linear")
    assert rows.shape == (20, 8) and rows.data_ptr() == out.data_ptr() and embed._out_stride(rows, "linear") == 12


@pytest.mark.parametrize("shape,rows", [((2, 3, 0), 6), ((0,), 1), ((2, 0, 3), 0), ((4, 5, 8), 20), ((8,), 1)])
def test_rows_of_no_elements(shape, rows):
    assert embed._rows(torch.empty(shape))[0].shape == (rows, shape[-1])
    assert embed._flat(torch.empty(shape), "linear").shape == (rows, shape[-1])
