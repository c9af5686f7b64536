"""int8 rows of fp32 at addresses and strides that are multiples of 16 bytes and not of 32."""

from __future__ import annotations

import pytest
import torch

from test_gpu_int8 import DEV, _check_rows

pytestmark = pytest.mark.gpu


# a wave a row, four waves a row in one to eight pieces, and rows that are read twice
@pytest.mark.parametrize("rows,k", [(2050, 64), (2051, 1040), (2048, 2048), (3, 64), (5, 4112), (9, 16384), (3, 16400)])
def test_rows_at_sixteen_bytes(rows, k):
    print(f"int8 fp32 rows {rows} x {k} at 16 bytes", flush=True)
    stride = k + 12 if k % 8 == 0 else k + 4
    g = torch.Generator(device=DEV).manual_seed(rows + k)
    x = torch.randn(rows * stride + 4, generator=g, device=DEV)[4:].as_strided((rows, k), (stride, 1))
    assert x.data_ptr() % 32 == 16 and stride % 8 == 4
    _check_rows(x)
