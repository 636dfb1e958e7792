"""Float experts on CPU: the form of new operand rows, and what the module needs of torch when it is imported."""

import subprocess
import sys

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


WITHOUT_CUDA = """
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from distributedmoellm_b200 import device, ep, layer, store
ex = store.FloatExperts(2, 24, 16, torch.bfloat16, "cpu")
assert layer.kernel_plan(ex, 4, 12) == [("float", 0)]
try:
    device.operand_rows(torch.zeros(2, 8), torch.bfloat16)
except RuntimeError as e:
    assert "CUDA" in str(e)
else:
    raise AssertionError
print("fine")
"""


def test_package_imports_with_a_torch_that_has_no_cuda():
    """A CPU build of torch has none of its CUDA bindings: import, host-side code and the refusal of CPU tensors work."""
    r = subprocess.run([sys.executable, "-c", WITHOUT_CUDA], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-2000:]
