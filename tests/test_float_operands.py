"""Float experts on CPU: the form of new operand rows, and what the module needs of torch when it is imported."""

import ctypes
import subprocess
import sys
import types

import pytest
import torch

from distributedmoellm_b200 import _build, _lib
from distributedmoellm_b200 import device as D
from distributedmoellm_b200.store import FloatExperts


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


# ---- slices of the experts (expert parallelism) ------------------------------------------------------

def test_a_slice_is_planned_for_its_own_picks(monkeypatch):
    """run_experts passes the picks that these experts get on to every operator, and the range of rows to make."""
    from distributedmoellm_b200 import layer as Lyr
    ex = FloatExperts(4, 200, 136, torch.bfloat16, "cpu")
    calls = []
    for name in ("operand_rows", "grouped_swiglu_t", "grouped_matmul_t"):
        monkeypatch.setattr(D, name, lambda *a, _n=name, **k: calls.append((_n, k)))
    off = torch.zeros(5, dtype=torch.int32)
    r = types.SimpleNamespace(P=64, sorted_rows=torch.zeros(64, dtype=torch.int32), offsets=off)

    def run(picks):
        calls.clear()
        Lyr.run_experts(ex, torch.zeros(8, 200), None, r, torch.zeros(64, 200), lambda n, b: torch.zeros(b, dtype=torch.uint8),
                        None, 12, picks=picks)
        return [k.get("picks") for _, k in calls], calls[0][1].get("offsets")
    assert run(8) == ([None, 8, 8], off)
    assert run(None) == ([None] * 3, None) and run(64) == ([None] * 3, None)


def test_slice_arguments_are_checked():
    bf = torch.bfloat16
    off = torch.zeros(4, dtype=torch.int32)
    x, w = torch.zeros(5, 64, dtype=bf), torch.zeros(3, 32, 64, dtype=bf)
    for bad in (off.long(), off[::2], off[:0], off[None]):
        with pytest.raises(ValueError, match="offsets must"):
            D.operand_rows(torch.zeros(5, 64), bf, offsets=bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.operand_rows(torch.zeros(5, 64), bf, offsets=off)
    for call in (D.grouped_matmul_t, D.grouped_swiglu_t):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(x, w, off, picks=3)
    assert D._picks(0, 5) == 0 and D._picks(5, 5) == 5
    for bad in (-1, 6):
        with pytest.raises(ValueError, match="picks of 5 rows"):
            D._picks(bad, 5)


def test_c_slice_entries_reject_bad_arguments():
    _build.build()
    L = _lib.lib()
    buf = ctypes.create_string_buffer(4096 + 16)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) & ~15)

    def rows(n=8, first=p, last=p):
        return L.mb_operand_rows_slice(p, 0, 64, 4, p, n, 64, 3, p, 64, p, 1, 1, first, last, p, None)
    assert rows(first=None) == 1 and rows(last=None) == 1 and rows(n=-1) == 1 and rows(n=0) == 0

    def mm(P=4, picks=4):
        return L.mb_grouped_matmul_t_slice(p, 3, 64, p, 1, 1, P, p, 4096, 64, p, 2, 64, 64, p, p, 0, 64, picks, None, None)

    def sw(P=4, picks=4):
        return L.mb_grouped_swiglu_t_slice(p, 3, 64, p, 1, 1, P, p, 8192, 64, p, 2, 64, 64, p, p, 64, p, 1, 1, picks, None,
                                           None)
    for f in (mm, sw):
        assert f(picks=5) == 1 and f(picks=-1) == 1 and "picks of 4 rows" in _lib.last_error()
        assert f(P=0, picks=0) == 0
