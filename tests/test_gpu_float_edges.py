"""Edges of the float experts' operators: offsets that overlap, groups of NaN,
gates far below zero, quotients of very small scales, f32 accuracy over long K,
rows taken from one operator by the next.  Tolerances as in test_gpu_float.py,
whose helpers these tests use; each is derived beside its test where it differs."""

import pytest
import torch

import test_gpu_float as base
from test_gpu_float import (BF16, E4M3, F16, F32, G, ceil, close, float_layer, gen, layer_reference, offsets_of,
                            plain_e4m3, rand_rows, rand_weights, round_tol, same_bits, sum_tol, want_grouped, want_swiglu)
from test_gpu_float import D  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def padded_ones(n, d, dtype):
    return torch.ones((n, d), device="cuda").to(dtype)


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


# ---- quotients of very small scales ------------------------------------------------------

# (largest value of a group, a value of it): next to a border of e4m3 with scales of 2^-97 and below, where the remainder
# of an f32 division has bits below the smallest f32
NEXT_TO_BORDERS = [("0x1.c0000ap-89", "0x1.800008p-106"), ("0x1.c00010p-90", "0x1.80000ep-107"),
                   ("0x1.bfffd8p-90", "0x1.ffffd4p-109"), ("0x1.bfffeap-90", "0x1.ffffe8p-109"),
                   ("0x1.500004p-89", "0x1.b00006p-105"), ("0x1.500002p-90", "0x1.e00004p-107"),
                   ("0x1.500002p-89", "0x1.e00004p-106")]


def test_operand_rows_quotients_of_small_scales_bit_exact(D):
    x = torch.zeros((len(NEXT_TO_BORDERS), 256), dtype=torch.float64)
    for i, (m, v) in enumerate(NEXT_TO_BORDERS):
        x[i, 0], x[i, 1:128] = float.fromhex(m), float.fromhex(v)
        x[i, 128], x[i, 129:] = -float.fromhex(m), -float.fromhex(v)
    x = x.float().cuda()
    q, s = D.operand_rows(x, E4M3)
    wq, ws = plain_e4m3(x)
    assert torch.equal(s, ws) and same_bits(q, wq)


@pytest.mark.parametrize("low,high", [(-126, -76), (-80, -70), (-10, 10), (90, 110)])
def test_operand_rows_next_to_every_border_bit_exact(D, low, high):
    """Values whose quotients lie half an f32 step from a border between two e4m3 values, for scales of every size."""
    g = gen(low + 1000)
    n = 20000
    m = torch.rand(n, generator=g, device="cuda") + 1
    m = m * torch.exp2(torch.randint(low + 9, high + 9, (n,), generator=g, device="cuda").float())
    s = (m / torch.full_like(m, 448.0)).double()
    k = torch.arange(128, device="cuda")
    borders = torch.where(k < 16, (k // 2 + 0.5) * 2.0 ** -9, (8 + (k // 2) % 8 + 0.5) / 8 * 2.0 ** (-6 + (k - 16) // 16))
    step = torch.nextafter(borders.float(), torch.full_like(k, 1000.0, dtype=F32)).double() - borders.double()
    mid = borders.double() + (k % 2 - 0.5) * step
    x = (s[:, None] * mid).float()
    x[:, 0] = m
    q, sc = D.operand_rows(x, E4M3)
    wq, ws = plain_e4m3(x)
    assert torch.equal(sc, ws) and same_bits(q, wq)


# ---- groups of NaN ------------------------------------------------------------------------

@pytest.mark.parametrize("T,k", [(6, 0), (0, 4)], ids=["each pick", "made once"])
@pytest.mark.parametrize("d", [256, 200, 513])
def test_operand_rows_groups_of_nothing_but_nan_have_scale_one(D, T, k, d):
    """Whole groups of NaN (the last, shorter one too), groups with one value among NaN, and rows beside them; k: so many
    rows and picks that each row is made once."""
    if k:
        T = 16 * torch.cuda.get_device_properties(0).multi_processor_count
        d = 512 + ceil(d, 16) * 16
    g = gen(d)
    x = torch.randn((T, d), generator=g, device="cuda")
    x[0] = float("nan")
    x[2, :128] = float("nan")
    x[3, 128:] = float("nan")
    x[4, 1:] = float("nan")
    x[4, 0] = -3.0
    rows = torch.arange(T, device="cuda", dtype=torch.int32).repeat(max(k, 1))
    q, s = D.operand_rows(x, E4M3, rows=rows)
    wq, ws = plain_e4m3(x[rows.long()])
    assert (ws[0] == 1).all() and ws[2, 0] == 1 and (ws[3, 1:] == 1).all()
    assert torch.equal(s, ws) and same_bits(q, wq)


def test_swiglu_nan_groups_have_the_same_scale_as_operand_rows(D):
    """The activation of a NaN row, put into operand form, is what operand_rows makes of a row of NaN."""
    g = gen(5)
    x, xs, _ = rand_rows((20, 128), E4M3, g)
    x[5] = float("nan")
    w, ws, _ = rand_weights((1, 2, 200, 128), E4M3, g)
    q, s = D.grouped_swiglu_t(x, w.reshape(1, 400, 128), offsets_of([20]), xs, ws)
    q2, s2 = D.operand_rows(torch.full((1, 200), float("nan"), device="cuda"), E4M3)
    assert same_bits(q[5:6], q2) and torch.equal(s[5:6], s2)


# ---- gates far below zero -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("rows", [3, 40])
def test_swiglu_gates_far_below_zero(D, dtype, rows):
    """Gates of -112 .. 112 with ups of 2^60 and 2^-60: below -87.3 the activation is tiny, but no zero once the up is
    large.  Tolerance: as want_swiglu's, and exp(g) off by a step of the smallest f32 (2^-149), times |g u|; one product per
    sum, which is exact."""
    v = torch.arange(-448, 449, 1, device="cuda").float().to(E4M3).float().unique() / 4          # exact in both types
    v = torch.cat([v, torch.linspace(-112, -80, 65, device="cuda")]) if dtype == BF16 else v
    v = v.to(BF16).float()
    I = v.numel()
    x = padded_ones(rows, 128, dtype)
    for up in (60, -60):
        w = torch.zeros((1, 2, I, 128), device="cuda")
        w[0, 0, :, 0] = v * (4 if dtype == E4M3 else 1)
        w[0, 1, :, 0] = 1.0 if dtype == E4M3 else 2.0 ** up
        xs = ws = None
        if dtype == E4M3:
            xs = torch.ones((rows, 1), device="cuda")
            ws = torch.full((1, 2, ceil(I, G), 1), 0.25, device="cuda")
            ws[0, 1] = 2.0 ** up
        q, s = D.grouped_swiglu_t(x, w.to(dtype).view(1, 2 * I, 128), offsets_of([rows]), xs, ws)
        g64, u = v.double(), 2.0 ** up
        a = g64 / (1 + torch.exp(-g64)) * u
        tol = (g64.abs() + 8) * 2.0 ** -22 * a.abs() + g64.abs() * u * 2.0 ** -149 + 2.0 ** -149
        a, tol = a.expand(rows, I), tol.expand(rows, I)
        if dtype != E4M3:
            close(q, a, tol + round_tol(a, dtype), f"up 2^{up}")
            continue
        sw = s.double().repeat_interleave(G, 1)[:, :I]
        close(q.double() * sw, a, tol * 17 / 16 + 2.0 ** -4 * a.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * sw, f"up 2^{up}")


@pytest.mark.parametrize("rows", [3, 40])
def test_swiglu_groups_of_tiny_activations(D, rows):
    """A whole group of gates near -88 with ups of 1: its scale follows the activations, which are normal numbers."""
    gate = torch.tensor([-87.0, -87.5, -88.0, -88.5], device="cuda").repeat(32)
    x = padded_ones(rows, 128, E4M3)
    w = torch.zeros((1, 2, 128, 128), device="cuda")
    w[0, 0, :, 0], w[0, 0, :, 1], w[0, 1, :, 0] = -352.0, (gate * 4 + 352.0), 1.0     # -352 + (4, 2, 0, -2)
    ws = torch.ones((1, 2, 1, 1), device="cuda")
    ws[0, 0] = 0.25
    q, s = D.grouped_swiglu_t(x, w.to(E4M3).view(1, 256, 128), offsets_of([rows]), torch.ones((rows, 1), device="cuda"), ws)
    g64 = gate.double()
    a = (g64 / (1 + torch.exp(-g64))).expand(rows, 128)
    tol = (g64.abs() + 8) * 2.0 ** -22 * a.abs() + g64.abs() * 2.0 ** -149
    m = a.abs().amax(1, keepdim=True) / 448
    close(s, m, tol.amax(1, keepdim=True) / 448 + 2.0 ** -23 * m + 2.0 ** -149, "scales")
    close(q.double() * s.double(), a, tol * 17 / 16 + 2.0 ** -4 * a.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * s.double()
          + 448 * 2.0 ** -149, "values")


# ---- rows taken from one operator by the next ---------------------------------------------------

@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("H,I", [(1000, 715), (24, 1), (129, 4), (272, 208)])
def test_operators_take_each_others_rows_at_any_width(D, dtype, H, I):
    """Operand rows, gate|up and down with the results that the operators make themselves, widths that are no multiple of
    16 bytes among them."""
    g = gen(H + I)
    off = offsets_of([3, 0, 40])
    x = torch.randn((43, H), generator=g, device="cuda")
    q, s = D.operand_rows(x, dtype)
    w, ws, ww = rand_weights((3, 2, I, H), dtype, g, scale=2.0 / H ** 0.5)
    wv = torch.as_strided(w, (3, 2 * I, H), (2 * I * w.stride(2), w.stride(2), 1), w.storage_offset())
    a, as_ = D.grouped_swiglu_t(q, wv, off, s, ws)
    d, ds, dw = rand_weights((3, H, I), dtype, g)
    y = D.grouped_matmul_t(a, d, off, as_, ds)

    def wide(v, sc):
        return v.double() if sc is None else v.double() * sc.double().repeat_interleave(G, 1)[:, :v.shape[1]]
    want, S, _ = want_grouped(wide(a, as_), dw, off)
    close(y, want, sum_tol(I, S) + round_tol(want, F32))
    act, tol, _ = want_swiglu(wide(q, s), ww.reshape(3, 2 * I, H), off, I, H)
    if dtype != E4M3:
        close(a, act, tol + round_tol(act, dtype))
    else:
        sw = as_.double().repeat_interleave(G, 1)[:, :I]
        close(a.double() * sw, act, tol * 17 / 16 + 2.0 ** -4 * act.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * sw)
        m, ms, mw = rand_weights((I, H), E4M3, g)
        want, S = wide(q, s) @ mw.t(), wide(q, s).abs() @ mw.abs().t()
        close(D.matmul_t_e4m3(q, s, m, ms), want, sum_tol(H, S) + round_tol(want, F32))


# ---- slices of the experts (expert parallelism) ------------------------------------------------------

@pytest.mark.parametrize("picks", [0, 1, 40, 300, 700])
@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_products_are_right_whatever_picks_says(D, dtype, picks):
    """A slice's offsets within many rows: passes and splits follow `picks`, results do not depend on it beyond the order of
    sums; rows outside stay."""
    g = gen(picks)
    P, K, O, E = 700, 272, 256, 4
    off = offsets_of([33, 0, 150, 5], 100)
    x, xs, xw = rand_rows((P, K), dtype, g)
    w, ws, ww = rand_weights((E, O, K), dtype, g)
    y = torch.full((P, O), 7.0, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    D.grouped_matmul_t(x, w, off, xs, ws, y=y, status=st, picks=picks)
    want, S, real = want_grouped(xw, ww, off)
    close(y[real], want[real], (sum_tol(K, S) + round_tol(want, F32))[real])
    assert (y[~real] == 7.0).all() and int(st) == 0
    g2, gs2, gw2 = rand_weights((E, 2, 128, K), dtype, g, scale=3.0 / K ** 0.5)
    q = torch.full((P, 128), 7.0, device="cuda").to(dtype)
    s = torch.full((P, 1), 7.0, device="cuda") if dtype == E4M3 else None
    D.grouped_swiglu_t(x, g2.reshape(E, 256, K), off, xs, gs2, q=q, scales=s, status=st, picks=picks)
    a, tol, _ = want_swiglu(xw, gw2.reshape(E, 256, K), off, 128, K)
    assert (q[~real].float() == 7.0).all() and int(st) == 0
    if dtype != E4M3:
        close(q[real], a[real], (tol + round_tol(a, dtype))[real])
        return
    assert (s[~real] == 7.0).all()
    sw = s.double().expand(P, 128)
    close(q[real].double() * sw[real], a[real],
          (tol * 17 / 16 + 2.0 ** -4 * a.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * sw)[real])


@pytest.mark.parametrize("dst", [E4M3, BF16])
@pytest.mark.parametrize("blocks,k", [(0, 8), (1, 8)], ids=["few rows", "many rows"])
@pytest.mark.parametrize("first,last", [(0, -1), (100, 3000), (3, 4), (700, 700), (2047, 10 ** 9), (-5, 60), (900, 20)])
def test_operand_rows_of_a_slice_only(D, dst, blocks, k, first, last):
    """Only the rows within the offsets are made (and only their indices looked at); the others keep what they held."""
    T = 16 * torch.cuda.get_device_properties(0).multi_processor_count if blocks else 500
    d = 1024
    g = gen(T + first)
    x = torch.randn((T, d), generator=g, device="cuda")
    n = T * k
    rows = torch.randint(0, T, (n,), generator=g, device="cuda", dtype=torch.int32)
    last = n if last == -1 else last
    lo, hi = max(first, 0), max(min(last, n), max(first, 0))
    rows[:lo], rows[hi:] = 2 ** 31 - 1, -7                       # nothing looks at these
    q = torch.full((n, d), 3.0, device="cuda").to(dst)
    s = torch.full((n, d // G), 3.0, device="cuda") if dst == E4M3 else None
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    off = torch.tensor([first, lo, last], dtype=torch.int32, device="cuda")
    D.operand_rows(x, dst, rows=rows, q=q, scales=s, status=st, offsets=off)
    assert int(st) == 0
    assert (q[:lo].float() == 3).all() and (q[hi:].float() == 3).all()
    assert s is None or ((s[:lo] == 3).all() and (s[hi:] == 3).all())
    if hi > lo:
        want = x[rows[lo:hi].long()]
        wq, ws = plain_e4m3(want) if dst == E4M3 else (want.to(dst), None)
        assert same_bits(q[lo:hi], wq) and (s is None or torch.equal(s[lo:hi], ws))


class OneProcess:
    """torch.distributed for the ranks of a group that run one after the other in this process: a first pass of every rank
    records what it gathers, a second one hands all ranks' parts out."""

    def __init__(self, world):
        self.world, self.rank, self.sent, self.play, self.at = world, 0, {}, False, 0

    def start(self, rank, play):
        self.rank, self.play, self.at = rank, play, 0

    def get_world_size(self, group=None):
        return self.world

    def get_rank(self, group=None):
        return self.rank

    def _coalescing_manager(self, group=None, device=None):
        import contextlib
        return contextlib.nullcontext()

    def all_gather_into_tensor(self, out, inp, group=None):
        if not self.play:
            self.sent[self.rank, self.at] = inp.clone()
        parts = [self.sent[r, self.at] if self.play else inp for r in range(self.world)]
        out.copy_(torch.cat([p.reshape(inp.shape) for p in parts]).view(out.shape))
        self.at += 1

    def all_to_all_single(self, out, inp, out_rows, in_rows, group=None):
        assert self.world == 1
        out.copy_(inp)

    def reduce_scatter_tensor(self, out, inp, group=None):
        T = out.shape[0]
        out.copy_(inp[self.rank * T:(self.rank + 1) * T])


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("world", [1, 2, 4])
def test_gather_layer_of_float_experts(D, monkeypatch, dtype, T, world):
    """EPGatherLayer with a slice of the float experts on each of `world` ranks, run one after the other: the ranks' partial
    sums add up to the layer (tolerance as in test_layer_of_float_experts, and an addition for each rank)."""
    from distributedmoellm_b200 import ep
    from distributedmoellm_b200.store import FloatExperts
    E, H, I, k = 8, 272, 208, 3
    layer, wide = float_layer(dtype, E, H, I, k, 97)
    x = torch.randn((world * T, H), generator=gen(T), device="cuda")
    layer(x)
    want, mag = layer_reference(D, layer, wide, x, dtype, layer.buffers(world * T))
    fake = OneProcess(world)
    monkeypatch.setattr(ep, "dist", fake)
    ranks = []
    El = E // world
    for r in range(world):
        fake.start(r, False)
        ex = FloatExperts(El, H, I, dtype, "cuda")
        for j in range(El):
            e = r * El + j
            ex.put(j, layer.experts.gu[e], layer.experts.down[e], None if dtype != E4M3 else layer.experts.gu_s[e],
                   None if dtype != E4M3 else layer.experts.dn_s[e])
        ranks.append(ep.EPGatherLayer(layer.router, ex, E, k))
    for play in (False, True):
        for r, l in enumerate(ranks):
            fake.start(r, play)
            if l._bufs:                     # whatever earlier calls left in workspaces and results is not seen
                b = l.buffers(T)
                b.y.fill_(float("nan"))
                for w in b.ws.values():
                    w.fill_(0x7F)
            l(x[r * T:(r + 1) * T])
            assert l.status(T) == 0
    got = sum(l.buffers(T).partial.double() for l in ranks)
    half = {E4M3: 2.0 ** -4, BF16: 2.0 ** -8}[dtype]
    close(got, want, half * mag * 1.01 + 1e-4 * mag.amax(1, keepdim=True), f"{world} ranks")


@pytest.mark.parametrize("dtype", [E4M3, F16])
@pytest.mark.parametrize("T", [1, 50])
def test_exchange_layer_of_float_experts(D, monkeypatch, dtype, T):
    """EPLayer (rows exchanged and regrouped by local expert) over float experts, as a single rank: the layer's results."""
    from distributedmoellm_b200 import ep
    E, H, I, k = 8, 272, 208, 3
    layer, wide = float_layer(dtype, E, H, I, k, 98)
    x = torch.randn((T, H), generator=gen(T), device="cuda")
    whole = layer(x).clone()
    monkeypatch.setattr(ep, "dist", OneProcess(1))
    ops = ep.DeviceOps(layer.router, layer.experts, E, k)
    got = ep.EPLayer(ops, E, k, H)(x)
    assert torch.equal(got, whole) and int(ops._ws["status"]) == 0


# ---- accuracy of f32 results -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("K", [2048, 7168])
@pytest.mark.parametrize("counts", [[3], [40], [300, 0, 130], [5] * 40], ids=["3", "40", "300+130", "40x5"])
def test_f32_results_over_long_columns(D, dtype, K, counts):
    """Few rows (split over K), ordinary ones and many, against 64 bits, relative in norm.

    The tensor cores cut an f32 sum at each step of 32 bytes of columns: by 0.36 of 2^-23 of the sum so far on average, and
    over n steps of random products the sums so far add up to 2 n / 3 of the last.  16-bit types: n = 16 steps between two
    f32 additions (256 columns): 4.6e-7; the additions behind them, rounded, come to 2.5e-8 sqrt(K / 512) <= 1e-7, added as
    squares: below 5e-7.  (Sums over all of K, n = 128 from 2048 columns, would be at 3.7e-6.)  e4m3: n = 4 steps a group:
    1.15e-7, the scaled additions 2.5e-8 sqrt(K / 256) <= 1.35e-7 and the scales' products 3e-8: 1.8e-7, and a bound of 3e-7
    for what chance adds."""
    g = gen(K + len(counts))
    off = offsets_of(counts)
    x, xs, xw = rand_rows((int(off[-1]), K), dtype, g)
    w, ws, ww = rand_weights((len(counts), 384, K), dtype, g)
    y = D.grouped_matmul_t(x, w, off, xs, ws)
    want, _, _ = want_grouped(xw, ww, off)
    error = float((y.double() - want).norm() / want.norm())
    assert error < (3e-7 if dtype == E4M3 else 5e-7), error


# ---- rows made once and copied, wherever that way begins ---------------------------------------------

def rows_for_every_sm():
    return 16 * torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("more", [-1, 0, 3, 100])
@pytest.mark.parametrize("src,dst,k,d", [(F32, E4M3, 8, 1024), (F32, E4M3, 5, 656), (BF16, E4M3, 4, 2048), (F16, E4M3, 6, 784),
                                         (F32, BF16, 6, 768), (F16, F16, 4, 1032)])
def test_operand_rows_of_many_picks_around_the_rule(D, src, dst, k, d, more):
    """From sixteen rows of x for every SM on, each e4m3 row of enough columns is made once; one row fewer, for every pick."""
    base.test_operand_rows_of_many_picks(D, src, dst, rows_for_every_sm() + more, k, d)


@pytest.mark.parametrize("d", [5440, 5456, 5472, 5488])
def test_operand_rows_made_once_at_the_shared_memory_limit(D, d):
    """Rows of up to 5456 columns fit sixteen at a time (d bytes and a scale per 128 columns each, 88 KB in all); wider ones
    are made for every pick."""
    T = rows_for_every_sm()
    x = torch.randn((T, d), generator=gen(d), device="cuda")
    rows = torch.arange(T, device="cuda", dtype=torch.int32).repeat(4)
    q, s = D.operand_rows(x, E4M3, rows=rows)
    wq, ws = plain_e4m3(x)
    assert same_bits(q, wq[rows.long()]) and torch.equal(s, ws[rows.long()])


def test_operand_rows_made_once_with_the_most_rows_a_column(D):
    """Four rows of x a column, and one more, which is made for every pick."""
    for T in (4096, 4097):
        x = torch.randn((T, 1024), generator=gen(T), device="cuda")
        rows = torch.randint(0, T, (4 * T,), generator=gen(1), device="cuda", dtype=torch.int32)
        q, s = D.operand_rows(x, E4M3, rows=rows)
        wq, ws = plain_e4m3(x)
        assert same_bits(q, wq[rows.long()]) and torch.equal(s, ws[rows.long()])


@pytest.mark.parametrize("dtype", [E4M3, F16])
def test_captured_slice_follows_its_offsets(D, dtype):
    """run_experts over a slice, captured: replays on new picks, whose range begins and ends elsewhere, equal eager calls,
    and rows outside the range stay."""
    from distributedmoellm_b200 import layer as Lyr
    from distributedmoellm_b200.store import FloatExperts
    E, H, I, k, T, e0, El = 8, 272, 144, 2, 60, 2, 3
    layer, _ = float_layer(dtype, E, H, I, k, 99)
    ex = FloatExperts(El, H, I, dtype, "cuda")
    for j in range(El):
        e = e0 + j
        ex.put(j, layer.experts.gu[e], layer.experts.down[e], None if dtype != E4M3 else layer.experts.gu_s[e],
               None if dtype != E4M3 else layer.experts.dn_s[e])
    P = T * k
    x = torch.randn((T, H), generator=gen(1), device="cuda")
    idx = torch.zeros((T, k), dtype=torch.int32, device="cuda")
    w = torch.ones((T, k), device="cuda")
    r = D.Routing(T, k, E, "cuda")
    local = D.Routing.from_plan(r.counts[e0:e0 + El], r.offsets[e0:e0 + El + 1], r.sorted_rows[:P])
    bufs, st = {}, torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(y):
        D.permute(idx, w, E, r)
        Lyr.run_experts(ex, x, None, local, y, lambda n, b: bufs.setdefault(n, torch.empty(b, dtype=torch.uint8, device="cuda")),
                        st, 12, picks=P // 2)

    def route(seed):
        idx.copy_(torch.rand((T, E), generator=gen(seed), device="cuda").topk(k, dim=1).indices)
    route(1)
    got, want = torch.empty((P, H), device="cuda"), torch.empty((P, H), device="cuda")
    step(got)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(got)
    for seed in (2, 3):
        route(seed)
        got.fill_(5.0)
        want.fill_(5.0)
        g.replay()
        step(want)
        assert torch.equal(got, want) and int(st) == 0
        lo, hi = int(local.offsets[0]), int(local.offsets[-1])
        assert 0 < lo < hi < P and (got[:lo] == 5).all() and (got[hi:] == 5).all() and (got[lo:hi] != 5).any()
