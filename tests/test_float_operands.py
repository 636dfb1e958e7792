"""Float experts on CPU: the form of new operand rows, and what the module needs of torch when it is imported."""

import pytest
import torch

from distributedmoellm_b200 import device as D


@pytest.mark.parametrize("dtype", D.OPERAND_TYPES, ids=str)
@pytest.mark.parametrize("n", [0, 1, 3])
@pytest.mark.parametrize("d", [1, 8, 15, 16, 100, 1000, 2048])
def test_new_operand_rows_are_what_the_products_take(dtype, n, d):
    q = D._new_operand(torch.zeros(2, 2), n, d, dtype)
    assert q.shape == (n, d) and q.dtype == dtype and q.stride(1) == 1
    assert q.stride(0) * dtype.itemsize % 16 == 0 and q.data_ptr() % 16 == 0
    assert q.is_contiguous() or d * dtype.itemsize % 16
