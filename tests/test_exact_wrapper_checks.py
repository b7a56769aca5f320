"""What the exact-attention wrappers make of shapes and strides, on the CPU: device -1 is where a CPU tensor is."""

from __future__ import annotations

import pytest
import torch

from sva_b200 import kernels


def test_rows_of_one_row_pages_have_their_own_size():
    """A dimension of one row may have any stride: what is moved is the row, not the stride."""
    base = torch.zeros(1, 1, 640, 32, dtype=torch.bfloat16)
    for t in (base[:, :, ::64][:, :, :1], base[:, :, 5::64][:, :, :1], base.as_strided((1, 1, 1, 32), (7, 9, 11, 1))):
        assert t.is_contiguous() and t.stride(2) != 32
        at, end, _, _, row, within = kernels._rows_span(-1, t, "rows")
        assert (at, end - at, row, within) == (t.data_ptr(), 64, 64, 64)
    two = torch.zeros(3, 2, 64, 4, 2, dtype=torch.bfloat16)
    at, end, page, head, row, within = kernels._rows_span(-1, two, "rows")
    assert (end - at, page, head, row, within) == (two.numel() * 2, 2048, 1024, 16, 2048)


def test_page_tables_without_columns_are_refused():
    """Their data pointer is null, which the C ABI reads as no table at all."""
    for cols in (0, 1):
        table = torch.zeros(2, cols, dtype=torch.int32)
        if cols:
            assert kernels._page_table(-1, table, 2)[2] == 1
        else:
            with pytest.raises(ValueError, match="page_table"):
                kernels._page_table(-1, table, 2)
    assert kernels._page_table(-1, None, 2) == (0, 0, 0)


def test_tensors_to_write_to_must_not_overlap_themselves():
    base = torch.zeros(4, 6, 8, 16)
    for fine in (base, base[:, ::2], base.transpose(0, 2), base[1:3, :, 3:, :5], base[:1].expand(1, 6, 8, 16), base[..., :1].expand(4, 6, 8, 1),
                 base.view(-1).as_strided((2, 2, 100), (100, 200, 1)), base[:0].expand(0, 6, 8, 16)):
        kernels._unfolded(fine, "out")
    for bad in (base[:1].expand(4, 6, 8, 16), base[:, :1].expand(4, 6, 8, 16), base.view(-1).as_strided((2, 2, 100), (150, 50, 1)),
                base.view(-1).as_strided((4, 64), (63, 1))):
        with pytest.raises(ValueError, match="overlap"):
            kernels._unfolded(bad, "out")
