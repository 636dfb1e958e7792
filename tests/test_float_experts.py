"""Float experts on CPU: what the entry points refuse before they touch a
device, and how FloatExperts holds its matrices."""

import ctypes

import numpy as np
import pytest
import torch

from distributedmoellm_b200 import _build, _lib
from distributedmoellm_b200 import device as D
from distributedmoellm_b200.store import FloatExperts

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def L():
    _build.build()
    return _lib.lib()


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


# ---- the Python entry points ---------------------------------------------------------

def test_operand_rows_refuses():
    with pytest.raises(ValueError, match="rows, columns"):
        D.operand_rows(z(4), E4M3)
    with pytest.raises(ValueError, match="rows, columns"):
        D.operand_rows(z(4, 8, dtype=torch.int8), E4M3)
    with pytest.raises(ValueError, match="operand type"):
        D.operand_rows(z(4, 8), torch.float32)
    with pytest.raises(ValueError, match="int32"):
        D.operand_rows(z(4, 8), E4M3, rows=z(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="int32"):
        D.operand_rows(z(4, 8), E4M3, rows=z(8, dtype=torch.int32)[::2])
    with pytest.raises(ValueError, match="shape"):
        D.operand_rows(z(4, 8), torch.bfloat16, q=z(4, 9, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="no scales"):
        D.operand_rows(z(4, 8), torch.bfloat16, scales=z(4, 1))
    with pytest.raises(ValueError, match="adjacent"):
        D.operand_rows(z(8, 4).t(), E4M3)
    with pytest.raises(ValueError, match="status"):
        D.operand_rows(z(4, 8), E4M3, status=z(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        D.operand_rows(z(4, 8), E4M3)


def test_matmul_t_e4m3_refuses():
    x, w, xs, ws = z(3, 256, dtype=E4M3), z(130, 256, dtype=E4M3), z(3, 2), z(2, 2)
    with pytest.raises(ValueError, match="e4m3"):
        D.matmul_t_e4m3(x.to(torch.bfloat16), xs, w, ws)
    with pytest.raises(ValueError, match="weights of"):
        D.matmul_t_e4m3(x, xs, w.to(torch.bfloat16), ws)
    with pytest.raises(ValueError, match="columns"):
        D.matmul_t_e4m3(x, xs, w[:, :128], ws)
    with pytest.raises(ValueError, match="xs has shape"):
        D.matmul_t_e4m3(x, z(3, 3), w, ws)
    with pytest.raises(ValueError, match="ws has shape"):
        D.matmul_t_e4m3(x, xs, w, z(1, 2))
    with pytest.raises(ValueError, match="xs is missing"):
        D.matmul_t_e4m3(x, None, w, ws)
    with pytest.raises(ValueError, match="contiguous"):
        D.matmul_t_e4m3(x, xs, w, z(2, 2).t())
    with pytest.raises(ValueError, match="result type"):
        D.matmul_t_e4m3(x, xs, w, ws, dtype=E4M3)
    with pytest.raises(ValueError, match="y is"):
        D.matmul_t_e4m3(x, xs, w, ws, y=z(3, 130), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=r"\(O, K\)"):
        D.matmul_t_e4m3(x, xs, w[None], ws)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.matmul_t_e4m3(x, xs, w, ws)


def test_grouped_products_refuse():
    bf = torch.bfloat16
    x, w, off = z(5, 64, dtype=bf), z(3, 32, 64, dtype=bf), z(4, dtype=torch.int32)
    for call in (D.grouped_matmul_t, D.grouped_swiglu_t):
        with pytest.raises(ValueError, match=r"\(E, O, K\)"):
            call(x, w[0], off)
        with pytest.raises(ValueError, match="offsets has shape"):
            call(x, w, off[:3])
        with pytest.raises(ValueError, match="offsets is"):
            call(x, w, off.long())
        with pytest.raises(ValueError, match="offsets must be contiguous"):
            call(x, w, z(8, dtype=torch.int32)[::2])
        with pytest.raises(ValueError, match="no scales"):
            call(x, w, off, xs=z(5, 1))
        with pytest.raises(ValueError, match="weights of"):
            call(x, w.half(), off)
        with pytest.raises(ValueError, match="e4m3, bf16 or f16"):
            call(x.float(), w.float(), off)
        with pytest.raises(ValueError, match="adjacent"):
            call(z(64, 5, dtype=bf).t(), w, off)
        with pytest.raises(RuntimeError, match="CUDA"):
            call(x, w, off)
    with pytest.raises(ValueError, match="even number"):
        D.grouped_swiglu_t(x, z(3, 33, 64, dtype=bf), off)
    with pytest.raises(ValueError, match="q has shape"):
        D.grouped_swiglu_t(x, w, off, q=z(5, 32, dtype=bf))
    xs, ws = z(5, 1), z(3, 2, 1, 1)
    with pytest.raises(ValueError, match="ws has shape"):
        D.grouped_swiglu_t(x.to(E4M3), w.to(E4M3), off, xs, z(3, 1, 1))
    with pytest.raises(ValueError, match="scales has shape"):
        D.grouped_swiglu_t(x.to(E4M3), w.to(E4M3), off, xs, ws, scales=z(5, 2))


# ---- the C ABI: host checks before any device work -----------------------------------------

def _ptr():
    buf = ctypes.create_string_buffer(4096 + 16)
    return buf, ctypes.c_void_p((ctypes.addressof(buf) + 15) & ~15)


def test_c_entries_reject_bad_arguments(L):
    keep, p = _ptr()
    odd = ctypes.c_void_p(p.value + 8)
    F32, BF16, F16, F8 = 0, 1, 2, 3

    def rows(x=p, xt=F32, ldx=64, n_src=4, idx=p, n=8, d=64, t=F8, q=p, ldq=64, s=p, st=p):
        return L.mb_operand_rows(x, xt, ldx, n_src, idx, n, d, t, q, ldq, s, 1, 1, st, None)
    assert rows(xt=F8) == 1 and rows(t=F32) == 1 and rows(d=0) == 1 and rows(n=-1) == 1
    assert rows(idx=None) == 1                              # 8 rows of 4
    assert rows(ldx=63) == 1 and rows(ldq=63) == 1
    assert rows(q=None) == 1 and rows(s=None) == 1 and rows(x=None) == 1
    assert rows(n=0, x=None, q=None) == 0

    def mm(x=p, t=F8, ldx=64, xs=p, P=4, w=p, we=4096, ldw=64, ws=p, E=2, O=64, K=64, off=p, y=p, yt=F32, ldy=64):
        return L.mb_grouped_matmul_t(x, t, ldx, xs, 1, 1, P, w, we, ldw, ws, E, O, K, off, y, yt, ldy, None, None)

    def sw(x=p, t=F8, ldx=64, xs=p, P=4, w=p, we=8192, ldw=64, ws=p, E=2, I=64, K=64, off=p, q=p, ldq=64, qs=p):
        return L.mb_grouped_swiglu_t(x, t, ldx, xs, 1, 1, P, w, we, ldw, ws, E, I, K, off, q, ldq, qs, 1, 1, None, None)
    for f in (mm, sw):
        assert f(t=F32) == 1 and f(E=0) == 1 and f(E=1025) == 1 and f(K=0) == 1 and f(P=1 << 31) == 1 and f(P=-1) == 1
        assert f(ldx=63) == 1 and f(ldx=72) == 1 and f(ldw=72) == 1 and f(we=8200) == 1 and f(we=1024) == 1
        assert "16 bytes" in _lib.last_error() or "overlap" in _lib.last_error()
        assert f(x=odd) == 1 and f(w=odd) == 1
        assert "aligned" in _lib.last_error()
        assert f(x=None) == 1 and f(off=None) == 1 and f(xs=None) == 1 and f(ws=None) == 1
        assert f(P=0, x=None, off=None) == 0                # no rows: nothing to do
    assert mm(yt=F8) == 1 and mm(y=None) == 1 and mm(ldy=63) == 1 and mm(O=0) == 1
    assert sw(q=None) == 1 and sw(qs=None) == 1 and sw(ldq=63) == 1 and sw(I=0) == 1
    assert L.mb_matmul_t_e4m3(p, 64, p, 1, 1, 4, p, 72, p, 64, 64, p, F32, 64, None, None) == 1
    assert L.mb_matmul_t_e4m3(p, 64, None, 1, 1, 4, p, 64, p, 64, 64, p, F32, 64, None, None) == 1
    assert L.mb_matmul_t_e4m3(None, 64, None, 1, 1, 0, None, 64, None, 64, 64, None, F32, 64, None, None) == 0


# ---- FloatExperts ------------------------------------------------------------------------

def test_float_experts_hold_what_was_put():
    ex = FloatExperts(3, 200, 136, E4M3, "cpu")
    assert ex.gu.shape == (3, 272, 200) and ex.gu.stride() == (272 * 208, 208, 1)      # rows a multiple of 16 bytes
    assert ex.down.shape == (3, 200, 136) and ex.down.stride(1) == 144
    assert ex.gu_s.shape == (3, 2, 2, 2) and ex.dn_s.shape == (3, 2, 2)
    g = torch.Generator().manual_seed(0)
    gu, dn = torch.randn((272, 200), generator=g).to(E4M3), torch.randn((200, 136), generator=g).to(E4M3)
    gs, ds = torch.rand((2, 2, 2), generator=g), torch.rand((2, 2), generator=g)
    ex.put(1, gu.view(torch.uint8).numpy(), dn, gs.numpy(), ds)
    assert torch.equal(ex.gu[1].view(torch.uint8), gu.view(torch.uint8)) and torch.equal(ex.dn_s[1], ds)
    assert torch.equal(ex.gu_s[1], gs) and ex.present == {1}
    b = FloatExperts(2, 24, 16, torch.bfloat16, "cpu")
    bits = torch.randn(32, 24, generator=g).bfloat16()
    b.put(0, bits.view(torch.uint16).numpy(), torch.zeros(24, 16, dtype=torch.bfloat16))
    assert torch.equal(b.gu[0], bits) and b.gu_s is None and b.nbytes == 2 * 2 * (32 * 24 + 24 * 16)


def test_float_experts_refuse():
    with pytest.raises(ValueError, match="float experts"):
        FloatExperts(2, 64, 64, torch.float32, "cpu")
    ex = FloatExperts(2, 64, 64, torch.float16, "cpu")
    gu, dn = torch.zeros(128, 64, dtype=torch.float16), torch.zeros(64, 64, dtype=torch.float16)
    with pytest.raises(KeyError):
        ex.put(2, gu, dn)
    with pytest.raises(ValueError, match="no scales"):
        ex.put(0, gu, dn, torch.ones(2, 1, 1), torch.ones(1, 1))
    with pytest.raises(ValueError, match="experts of"):
        ex.put(0, gu.bfloat16(), dn)
    with pytest.raises(ValueError, match="does not match"):
        ex.put(0, gu[:64], dn)
    assert not ex.present
    with pytest.raises(ValueError, match="need block scales"):
        FloatExperts(2, 64, 64, E4M3, "cpu").put(0, gu, dn)


def test_layer_runs_float_experts_through_the_grouped_products(monkeypatch):
    """run_experts over FloatExperts, at every size: rows, gate|up with the activation, down, on one workspace whose
    parts do not overlap; the packed experts' kernels are not called."""
    from distributedmoellm_b200 import layer as Lyr
    ex = FloatExperts(4, 200, 136, E4M3, "cpu")
    assert Lyr.kernel_plan(ex, 1, 12) == Lyr.kernel_plan(ex, 100000, 12) == [("float", 0)]
    calls = []
    monkeypatch.setattr(D, "operand_rows", lambda x, dt, rows, q, s, st: calls.append(("rows", q, s)))
    monkeypatch.setattr(D, "grouped_swiglu_t", lambda x, w, o, xs, ws, q, s, st: calls.append(("gu", x, xs, q, s)))
    monkeypatch.setattr(D, "grouped_matmul_t", lambda x, w, o, xs, ws, y, status: calls.append(("down", x, xs, y)))
    P = 7
    import types
    r = types.SimpleNamespace(P=P, sorted_rows=torch.zeros(P, dtype=torch.int32), offsets=None)
    bufs = {}

    def workspace(name, n):
        return bufs.setdefault(name, torch.zeros(n, dtype=torch.uint8))
    y = torch.zeros(P, 200)
    Lyr.run_experts(ex, torch.zeros(3, 200), None, r, y, workspace, None, 12)
    assert [c[0] for c in calls] == ["rows", "gu", "down"] and list(bufs) == ["float"]
    (_, q, s), (_, q2, s2, a, as_), (_, a2, as2, y2) = calls
    assert q is q2 and s is s2 and a is a2 and as_ is as2 and y2.shape == (P, 200)
    assert q.shape == (P, 200) and s.shape == (P, 2) and a.shape == (P, 136) and as_.shape == (P, 2)
    spans = sorted((t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))
                    * t.element_size()) for t in (q, s, a, as_))
    assert all(b <= c for (_, b), (c, _) in zip(spans, spans[1:]))
    assert spans[-1][1] <= bufs["float"].data_ptr() + bufs["float"].numel()
    assert all((t.data_ptr() - bufs["float"].data_ptr()) % 16 == 0 and t.stride(0) % 16 == 0 for t in (q, a))
    assert np.prod(r.sorted_rows.shape) == P
    r.P = 0
    Lyr.run_experts(ex, torch.zeros(0, 200), None, r, y, workspace, None, 12)
    assert len(calls) == 3


def test_peer_layer_refuses_float_experts(monkeypatch):
    from distributedmoellm_b200 import ep
    monkeypatch.setattr(ep.dist, "get_world_size", lambda g=None: 1)
    monkeypatch.setattr(ep.dist, "get_rank", lambda g=None: 0)
    with pytest.raises(ValueError, match="EPGatherLayer"):
        ep.EPPeerLayer(torch.zeros(2, 64), FloatExperts(2, 64, 64, torch.bfloat16, "cpu"), 2, 1)
