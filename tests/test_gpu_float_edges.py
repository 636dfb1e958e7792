"""Edges of the float experts' operators: offsets that overlap, groups of NaN,
gates far below zero, quotients of very small scales, f32 accuracy over long K,
rows taken from one operator by the next.  Tolerances as in test_gpu_float.py,
whose helpers these tests use; each is derived beside its test where it differs."""

import pytest
import torch

from test_gpu_float import (BF16, E4M3, F16, F32, G, ceil, check_grouped, close, gen, offsets_of, plain_e4m3, rand_rows,
                            rand_weights, round_tol, same_bits, sum_tol, want_grouped, want_swiglu)
from test_gpu_float import D  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


# ---- offsets ----------------------------------------------------------------------------

def ranges_that_count(offs, P):
    """As the header has it: within 0 .. P, not decreasing, not before the end of an earlier range that counts."""
    end, out = 0, []
    for lo, hi in zip(offs, offs[1:]):
        ok = 0 <= lo <= hi <= P and (lo >= end or lo == hi)
        out.append((lo, hi) if ok else (0, 0))
        if hi > lo and ok:
            end = hi
    return out


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("offs", [[0, 10, 0, 10], [0, 5, 3, 10], [2, 8, 1, 9, 8, 10], [0, 10, 0, 10, 0, 10, 0, 10],
                                  [4, 2, 6, 10], [9, 9, 3, 5, 10], [0, 11, 3, 7, 7, 10], [0, 300, 0, 300, 150, 300]], ids=str)
def test_overlapping_offsets_leave_later_ranges_out(D, dtype, offs):
    """A range that is in order by itself, but overlaps an earlier one: its rows stay the earlier expert's, and the bit
    is set; ranges that overlap nothing are computed."""
    g = gen(len(offs))
    P, K, O, E = max(10, max(offs) // 10 * 10), 256, 136, len(offs) - 1
    x, xs, xw = rand_rows((P, K), dtype, g)
    w, ws, ww = rand_weights((E, O, K), dtype, g)
    want, S = torch.full((P, O), 7.0, dtype=torch.float64, device="cuda"), torch.zeros((P, O), dtype=torch.float64,
                                                                                       device="cuda")
    for e, (lo, hi) in enumerate(ranges_that_count(offs, P)):
        want[lo:hi], S[lo:hi] = xw[lo:hi] @ ww[e].t(), xw[lo:hi].abs() @ ww[e].abs().t()
    off = torch.tensor(offs, dtype=torch.int32, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = torch.full((P, O), 7.0, device="cuda")
    D.grouped_matmul_t(x, w, off, xs, ws, y=y, status=st)
    assert int(st) == 2
    close(y, want, sum_tol(K, S) + round_tol(want, F32), str(offs))
