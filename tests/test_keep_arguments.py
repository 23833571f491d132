"""flash_keep_paged's lengths go to memory of their own: other work-groups still read the index tensors when the first one writes.  No GPU needed: every call
here ends before anything is launched."""
import ctypes as C

import pytest
import torch

from test_paged_arguments import E_INVAL, E_NODEVICE
from test_scored_arguments import keep_params, paged  # noqa: F401

# of keep_params: tables 0x300000 (2 rows of 50, 50 apart), path 0x600000 (2 rows of 7, 7 apart); seqlens_out: two words
INSIDE = [{"seqlens_out": 0x600000}, {"seqlens_out": 0x600000 + 4 * 13}, {"seqlens_out": 0x600000 - 4}, {"seqlens_out": 0x600000 + 4 * 26, "path_stride": 20},
          {"seqlens_out": 0x600000 + 4 * 19, "path_stride": 20}, {"max_path": 1, "path_stride": 1, "seqlens_out": 0x600000}, {"seqlens_out": 0x600000 + 4 * 6, "path_stride": 0},
          {"seqlens_out": 0x300000}, {"seqlens_out": 0x300000 + 4 * 99}, {"seqlens_out": 0x300000 - 4}, {"seqlens_out": 0x300000 + 4 * 149, "block_table_stride": 100}, {"seqlens_out": 0x600000 + 4 * 6, "path_stride": 2 ** 62}]
OUTSIDE = [{}, {"seqlens_out": 0x600000 + 4 * 14}, {"seqlens_out": 0x600000 - 8}, {"seqlens_out": 0x600000 + 4 * 27, "path_stride": 20}, {"seqlens_out": 0x600000 + 4 * 7, "path_stride": 0},
           {"seqlens_out": 0x600000 + 4 * 12, "path_stride": 20}, {"seqlens_out": 0x600000 + 4 * 18, "path_stride": 20}, {"seqlens_out": 0x600000 + 4 * 7, "path_stride": 2 ** 62},
           {"seqlens_out": 0x300000 + 4 * 100}, {"seqlens_out": 0x300000 - 8}, {"max_path": 0, "seqlens_out": 0x600000}, {"max_pages": 0, "seqlens_out": 0x300000},
           {"B": 1, "path_stride": 2 ** 62, "block_table_stride": 2 ** 62}]


@pytest.mark.parametrize("kw", INSIDE)
def test_lengths_in_an_index_tensor(paged, kw):  # noqa: F811
    assert paged._lib().flash_keep_paged(C.byref(keep_params(paged, **kw)), None) == E_INVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch with these pointers")
@pytest.mark.parametrize("kw", OUTSIDE)
def test_lengths_beside_them(paged, kw):  # noqa: F811
    assert paged._lib().flash_keep_paged(C.byref(keep_params(paged, **kw)), None) == E_NODEVICE


@pytest.mark.gpu
def test_python_refuses(fa):
    """A path of one column, or a column of the table, is no place for the lengths, either way in."""
    caches = [torch.zeros((4, 2, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
    path, table = (torch.zeros((3, 1), dtype=torch.int32, device="cuda") for _ in range(2))
    lens, cu, accepted = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for out in (path.view(3), table.view(3), lens, accepted):
        for how in ({}, {"stream": torch.cuda.current_stream()}):
            with pytest.raises(fa.FlashError):
                fa.flash_keep_paged(*caches, table, lens, cu, path, accepted, out=out, **how)
