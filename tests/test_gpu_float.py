"""GPU parity of the float experts' operators against plain 64-bit arithmetic.

Tolerances, per element, for f32 sums of exactly represented products (e4m3 x
e4m3 has 8 significant bits, bf16 x bf16 16, f16 x f16 22: all exact in f32):
each of at most K additions (and, for e4m3, the K / 128 scalings and their
sums) is off by at most 2^-24 of the sum of magnitudes S = sum |x w| (scaled),
twice that where the adder truncates, so |y - exact| <= 2 (K + 8) 2^-24 S.  A
result rounded to a shorter type adds eps / 2 of its value (and half the
smallest subnormal).

SiLU(g) u: with errors dg, du of g and u as above, |silu'| <= 1.1 and |silu(g)|
<= |g|: 1.1 |u| dg + |g| du (+ 1.1 dg du); exp(-g) is taken with a relative
error of at most (|g| + 8) 2^-22, and the few operations behind it stay below
that too: + (|g| + 8) 2^-22 |a|.  An e4m3 value of the result is off by half a
step more: 2^-4 of the value, at least 2^-10 (half the smallest subnormal) of the
scale; the scale by the largest error of its group / 448 and two roundings.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3, BF16, F16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32
G = 128


@pytest.fixture(scope="module")
def D():
    from distributedmoellm_b200 import _build
    _build.build()
    from distributedmoellm_b200 import device
    device.require_device()
    return device


def ceil(a, b):
    return -(-a // b)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- inputs: rows with a distance of 16 bytes' multiple, as the products need them --------------

def padded(shape, dtype):
    """Zeros (..., rows, columns) whose rows lie a multiple of 16 bytes apart, with 0x7f bytes (NaN in e4m3 and bf16) in
    the padding."""
    step = 16 // dtype.itemsize
    t = torch.zeros((*shape[:-1], ceil(shape[-1], step) * step), dtype=dtype, device="cuda")
    t.view(torch.uint8).fill_(0x7F)
    return t[..., :shape[-1]]


def rand_rows(shape, dtype, g, scale=1.0):
    """(rows, scales or None, both in f64 as the rows they stand for)."""
    t = padded(shape, dtype)
    t.copy_(torch.randn(shape, generator=g, device="cuda") * (scale if dtype != E4M3 else 60.0))
    if dtype != E4M3:
        return t, None, t.double()
    s = (torch.rand((*shape[:-1], ceil(shape[-1], G)), generator=g, device="cuda") + 0.5) * scale / 60.0
    return t, s, t.double() * s.double().repeat_interleave(G, -1)[..., :shape[-1]]


def rand_weights(shape, dtype, g, scale=0.05):
    w = padded(shape, dtype)
    w.copy_(torch.randn(shape, generator=g, device="cuda") * (scale if dtype != E4M3 else 60.0))
    if dtype != E4M3:
        return w, None, w.double()
    *lead, O, K = shape
    s = (torch.rand((*lead, ceil(O, G), ceil(K, G)), generator=g, device="cuda") + 0.5) * scale / 60.0
    wide = s.double().repeat_interleave(G, -2)[..., :O, :].repeat_interleave(G, -1)[..., :K]
    return w, s, w.double() * wide


def offsets_of(counts, first=0):
    off = [first]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


def sum_tol(K, S):
    return 2 * (K + 8) * 2.0 ** -24 * S


def round_tol(want, dtype):
    if dtype == F32:
        return 2.0 ** -24 * want.abs() + 2.0 ** -150
    tiny = {BF16: 2.0 ** -134, F16: 2.0 ** -25}[dtype]
    return torch.finfo(dtype).eps / 2 * want.abs() + tiny


def close(got, want, tol, what=""):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {d.numel()} off, worst {float((d / tol.clamp(min=1e-300)).max())}"


# ---- operand rows ------------------------------------------------------------------------

def plain_e4m3(x):
    """The definition in f32 (IEEE divisions, one rounding): bit-exact."""
    n, d = x.shape
    p = torch.zeros((n, ceil(d, G) * G), device=x.device)
    p[:, :d] = x.float()
    p = p.view(n, -1, G)
    m = p.abs().nan_to_num(nan=0.0, posinf=float("inf")).amax(2)
    s = m / torch.full_like(m, 448.0)                     # a tensor: torch divides by a number through its reciprocal
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (p / s[:, :, None]).clamp(-448, 448).view(n, -1)[:, :d].to(E4M3)
    return q, s


def same_bits(a, b):
    """Equal bytes, any NaN equal to any other."""
    a, b = a.contiguous(), b.contiguous()
    n = torch.isnan(a.float()) & torch.isnan(b.float())
    return bool((n | (a.view(torch.uint8) == b.view(torch.uint8))).all()) if a.dtype == E4M3 else \
        torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


@pytest.mark.parametrize("src", [F32, BF16, F16])
@pytest.mark.parametrize("dst", [E4M3, BF16, F16])
@pytest.mark.parametrize("T,d", [(1, 1), (3, 31), (5, 128), (2, 129), (7, 200), (33, 2048), (300, 768), (2, 4100)])
def test_operand_rows(D, src, dst, T, d):
    g = gen(T * 7 + d)
    x = (torch.randn((T, d), generator=g, device="cuda") * 3).to(src)
    rows = torch.randint(0, T, (2 * T + 1,), generator=g, device="cuda", dtype=torch.int32)
    for r in (None, rows):
        q, s = D.operand_rows(x, dst, rows=r)
        want = x if r is None else x[r.long()]
        if dst == E4M3:
            wq, ws = plain_e4m3(want)
            assert torch.equal(s, ws) and same_bits(q, wq)
        else:
            assert s is None and torch.equal(q, want.float().to(dst))


def test_operand_rows_strides_and_neighbours(D):
    """Rows and scales with other strides, unaligned starts; nothing outside the result is written."""
    g = gen(3)
    x = torch.randn((40, 301), generator=g, device="cuda")[::2, 1:260]          # odd start, odd distance
    rows = torch.tensor([19, 0, 0, 7], dtype=torch.int32, device="cuda")
    buf = torch.full((4, 300), 99, dtype=torch.uint8, device="cuda")
    q = buf.view(E4M3)[:, 3:262]
    sbuf = torch.full((9, 8), 5.0, device="cuda")
    s = sbuf[1:9:2, 1:7:2]
    D.operand_rows(x, E4M3, rows=rows, q=q, scales=s)
    wq, ws = plain_e4m3(x[rows.long()])
    assert torch.equal(s, ws) and same_bits(q, wq)
    assert (buf[:, :3] == 99).all() and (buf[:, 262:] == 99).all()
    s.fill_(5.0)
    assert (sbuf == 5.0).all()
    xb = torch.randn((9, 77), generator=g, device="cuda").to(BF16)[:, 1:]
    qb = torch.full((9, 99), 1.0, dtype=F16, device="cuda")
    D.operand_rows(xb, F16, q=qb[:, 7:83])
    assert torch.equal(qb[:, 7:83], xb.float().to(F16)) and (qb[:, :7] == 1).all() and (qb[:, 83:] == 1).all()


def test_operand_rows_edge_values(D):
    """Zero groups (scale 1), signed zeros, values next to the rounding borders, tiny and huge groups, NaN and infinity."""
    x = torch.zeros((12, 256), device="cuda")
    x[1, 5] = -0.0
    g = gen(9)
    x[2, :128] = torch.arange(128, device="cuda") * 0.5 + 448 - 64                # scale 1-ish: halves of steps
    x[2, 0] = 448.0
    x[3] = torch.randn(256, generator=g, device="cuda") * 1e-38
    x[4] = torch.randn(256, generator=g, device="cuda") * 1e-41                   # subnormal values and scales
    x[5, :3] = torch.tensor([1e-45, -1e-45, 2e-45])                               # scale underflows to 0: 1
    x[6] = torch.randn(256, generator=g, device="cuda") * 1e38
    x[6, 0] = 3.4e38
    x[7, 3] = float("nan")
    x[7, 4] = 2.0
    x[8, 200] = float("inf")
    x[8, 201] = -1.0
    x[9, :128] = 2.0 ** -6 / 448 * torch.arange(128, device="cuda")
    x[9, 127] = 1.0
    k = torch.arange(256, device="cuda")
    x[10] = (448.0 - k) * (1 + 2.0 ** -23 * (k % 3))
    x[11] = torch.randn(256, generator=g, device="cuda").exp()
    q, s = D.operand_rows(x, E4M3)
    wq, ws = plain_e4m3(x)
    wq[7, 3] = float("nan")
    assert torch.equal(s, ws) and same_bits(q, wq)
    assert s[0, 0] == 1 and torch.isinf(s[8, 1]) and torch.isnan(q[8, 72 + 128].float()) and s[5, 0] == 1
    y, _ = D.operand_rows(x, F16)
    assert same_bits(y, x.to(F16))


def test_operand_rows_random_exponents_bit_exact(D):
    """Groups of every magnitude: the quotient rounds as an IEEE division does."""
    g = gen(10)
    e = torch.randint(-126, 118, (2000, 1), generator=g, device="cuda").float()
    x = torch.randn((2000, 256), generator=g, device="cuda") * torch.exp2(e)
    x = x * torch.exp2(torch.randint(-12, 1, x.shape, generator=g, device="cuda").float())
    q, s = D.operand_rows(x, E4M3)
    wq, ws = plain_e4m3(x)
    assert torch.equal(s, ws) and same_bits(q, wq)


def test_operand_rows_bad_index_sets_status(D):
    x = torch.ones((4, 160), device="cuda")
    rows = torch.tensor([0, 4, -1, 3], dtype=torch.int32, device="cuda")
    for dst in (E4M3, BF16):
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        q, s = D.operand_rows(x, dst, rows=rows, status=st)
        assert int(st) == 2
        assert (q[1:3].float() == 0).all() and (q[0].float() != 0).all() and (q[3].float() != 0).all()
        if s is not None:
            assert (s[1:3] == 1).all()
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    D.operand_rows(x, E4M3, rows=rows[:1], status=st)
    assert int(st) == 0
    q, s = D.operand_rows(x, E4M3, rows=rows[:0])
    assert q.shape == (0, 160) and s.shape == (0, 2)
    q, s = D.operand_rows(x[:0], BF16)
    assert q.shape == (0, 160)


# ---- one matrix -----------------------------------------------------------------------------

@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("n,O,K", [(1, 1, 1), (1, 128, 128), (2, 100, 16), (17, 129, 144), (5, 8, 1000), (129, 300, 272),
                                   (16, 1000, 2048), (300, 257, 1424), (1, 2048, 4096), (257, 128, 640), (0, 64, 64)])
def test_matmul_t_e4m3(D, out, n, O, K):
    g = gen(n + 3 * O + 7 * K)
    x, xs, xw = rand_rows((n, K), E4M3, g)
    w, ws, ww = rand_weights((O, K), E4M3, g)
    y = D.matmul_t_e4m3(x, xs, w, ws, dtype=out)
    want, S = xw @ ww.t(), xw.abs() @ ww.abs().t()
    assert y.shape == (n, O) and y.dtype == out
    if n:
        close(y, want, sum_tol(K, S) + round_tol(want, out), f"{n} x {O} x {K}")


def test_matmul_t_e4m3_result_strides(D):
    g = gen(5)
    x, xs, xw = rand_rows((37, 320), E4M3, g)
    w, ws, ww = rand_weights((70, 320), E4M3, g)
    want, S = xw @ ww.t(), xw.abs() @ ww.abs().t()
    for out in (F32, BF16):
        buf = torch.full((80, 91), 3.0, dtype=out, device="cuda")
        y = buf[1:75:2, 5:75]                      # odd start, odd distance
        assert D.matmul_t_e4m3(x, xs.t().contiguous().t(), w, ws, y=y) is y
        close(y, want, sum_tol(320, S) + round_tol(want, out))
        y.fill_(3.0)
        assert (buf == 3.0).all()


# ---- grouped products -----------------------------------------------------------------------

def want_grouped(xw, ww, off):
    off = off.tolist()
    want = torch.zeros((xw.shape[0], ww.shape[1]), dtype=torch.float64, device="cuda")
    S = torch.zeros_like(want)
    real = torch.zeros(xw.shape[0], dtype=torch.bool, device="cuda")
    for e in range(len(off) - 1):
        r = slice(off[e], off[e + 1])
        want[r], S[r] = xw[r] @ ww[e].t(), xw[r].abs() @ ww[e].abs().t()
        real[r] = True
    return want, S, real


def check_grouped(D, counts, O, K, dtype, out, seed, first=0, tail=0):
    g = gen(seed)
    off = offsets_of(counts, first)
    P = int(off[-1]) + tail
    x, xs, xw = rand_rows((P, K), dtype, g)
    w, ws, ww = rand_weights((len(counts), O, K), dtype, g)
    y = torch.full((P, O), 7.0, dtype=out, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    D.grouped_matmul_t(x, w, off, xs, ws, y=y, status=st)
    want, S, real = want_grouped(xw, ww, off)
    assert int(st) == 0
    close(y[real], want[real], (sum_tol(K, S) + round_tol(want, out))[real], f"{counts} {O} {K}")
    assert (y[~real] == 7.0).all(), "rows outside every group were written"


RAGGED = [[3], [0, 0, 5, 0], [1, 1, 1, 1, 1, 1, 1, 1], [130, 0, 17, 1, 64, 33, 128, 255], [0, 700, 2], [256, 257, 258],
          [16, 15, 31, 32, 48, 47]]


@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("counts", RAGGED, ids=str)
def test_grouped_ragged(D, dtype, counts):
    check_grouped(D, counts, 200, 272, dtype, F32, 11)
    check_grouped(D, counts, 128, 128, dtype, BF16, 12, first=3, tail=9)


@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("O,K", [(1, 1), (7, 8), (64, 64), (127, 100), (129, 136), (768, 520), (100, 2056), (512, 1664),
                                 (2048, 768)])
def test_grouped_shapes(D, dtype, O, K):
    for out in (F32, BF16, F16):
        check_grouped(D, [5, 0, 40, 1], O, K, dtype, out, O + K)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_grouped_many_experts(D, dtype):
    """1024 experts, most of them empty, one with most rows."""
    counts = [0] * 1024
    counts[0], counts[511], counts[700], counts[1023] = 3, 1, 300, 2
    check_grouped(D, counts, 48, 80, dtype, F32, 21, tail=1)
    check_grouped(D, [1] * 1024, 48, 80, dtype, F32, 22)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_grouped_no_rows_at_all(D, dtype):
    check_grouped(D, [0, 0, 0], 64, 64, dtype, F32, 1, tail=33)
    check_grouped(D, [0, 0, 0], 64, 64, dtype, F32, 1)


@pytest.mark.parametrize("dtype", [E4M3, F16])
def test_grouped_strided_operands(D, dtype):
    """Rows of x and of w and the experts' matrices further apart than they need be, experts taken every second."""
    g = gen(31)
    step = 16 // dtype.itemsize
    xb, xs, xw = rand_rows((60, 256 + 2 * step), dtype, g)
    wb, ws, ww = rand_weights((6, 70, 256 + 2 * step), dtype, g)
    off = offsets_of([7, 20, 33])
    if dtype == E4M3:                          # whole groups of columns
        x, w, k0 = xb[:, :256], wb[::2, :64, :256], 0
        xs, ws = xs[:, :2], ws[::2, :1, :2].contiguous()
    else:
        x, w, k0 = xb[:, step:step + 256], wb[::2, :64, step:step + 256], step
    y = D.grouped_matmul_t(x, w, off, xs, ws)
    want, S, _ = want_grouped(xw[:, k0:k0 + 256], ww[::2, :64, k0:k0 + 256], off)
    close(y, want, sum_tol(256, S) + round_tol(want, F32))


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_grouped_non_finite_rows_stay_alone(D, dtype):
    """A NaN or infinity in one row reaches that row's results only, whatever else shares its tile; rows behind the last
    group may hold anything."""
    g = gen(41)
    off = offsets_of([40, 3, 90], 2)
    x, xs, xw = rand_rows((140, 200), dtype, g)
    w, ws, ww = rand_weights((3, 150, 200), dtype, g)
    want, S, real = want_grouped(xw, ww, off)
    bad = [0, 1, 5, 41, 44, 100, 135, 139]
    x[bad] = float("nan")
    if dtype == BF16:
        x[100] = float("inf")
    y = D.grouped_matmul_t(x, w, off, xs, ws)
    fine = real.clone()
    fine[bad] = False
    close(y[fine], want[fine], (sum_tol(200, S) + round_tol(want, F32))[fine])
    assert not torch.isfinite(y[[5, 41, 44, 100]]).any()


@pytest.mark.parametrize("offs", [[0, 5, 3, 10], [0, 5, 11, 11], [-1, 2, 4, 10], [0, 4, 4, 2000000000]])
def test_grouped_bad_offsets_set_status(D, offs):
    """Ranges that decrease, start before 0 or pass the rows are reported and left out; nothing is read or written outside."""
    g = gen(51)
    x, xs, xw = rand_rows((10, 128), E4M3, g)
    w, ws, ww = rand_weights((3, 64, 128), E4M3, g)
    off = torch.tensor(offs, dtype=torch.int32, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    buf = torch.full((30, 64), 7.0, device="cuda")
    D.grouped_matmul_t(x, w, off, xs, ws, y=buf[10:20], status=st)
    assert int(st) == 2
    st.zero_()
    w2, ws2, _ = rand_weights((3, 2, 32, 128), E4M3, g)
    D.grouped_swiglu_t(x, w2.reshape(3, 64, 128), off, xs, ws2.view(3, 2, 1, 1), status=st)
    assert int(st) == 2
    assert (buf[:10] == 7).all() and (buf[20:] == 7).all()
    for e in range(3):
        if 0 <= offs[e] <= offs[e + 1] <= 10:
            r = slice(offs[e], offs[e + 1])
            want, S = xw[r] @ ww[e].t(), xw[r].abs() @ ww[e].abs().t()
            # a later, overlapping range may write the same rows: only ranges that nothing else covers are compared
            if not any(i != e and 0 <= offs[i] <= offs[i + 1] <= 10 and offs[i] < offs[e + 1] and offs[e] < offs[i + 1]
                       for i in range(3)):
                close(buf[10:20][r], want, sum_tol(128, S) + round_tol(want, F32))


# ---- gate|up with the activation ----------------------------------------------------------------

def want_swiglu(xw, ww, off, I, K):
    h, S, real = want_grouped(xw, ww, off)
    g, u = h[:, :I], h[:, I:]
    dg, du = sum_tol(K, S[:, :I]), sum_tol(K, S[:, I:])
    a = g / (1 + torch.exp(-g)) * u
    tol = 1.1 * u.abs() * dg + g.abs() * du + 1.1 * dg * du + (g.abs() + 8) * 2.0 ** -22 * a.abs() + 2.0 ** -140
    return a, tol, real


def check_swiglu(D, counts, I, K, dtype, seed, first=0, tail=0):
    g = gen(seed)
    off = offsets_of(counts, first)
    P, E = int(off[-1]) + tail, len(counts)
    x, xs, xw = rand_rows((P, K), dtype, g)
    w, ws, ww = rand_weights((E, 2, I, K), dtype, g, scale=3.0 / K ** 0.5)
    wv = torch.as_strided(w, (E, 2 * I, K), (2 * I * w.stride(2), w.stride(2), 1), w.storage_offset())
    q = torch.full((P, I), 7.0, device="cuda").to(dtype)
    s = torch.full((P, ceil(I, G)), 7.0, device="cuda") if dtype == E4M3 else None
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    D.grouped_swiglu_t(x, wv, off, xs, ws, q=q, scales=s, status=st)
    assert int(st) == 0
    a, tol, real = want_swiglu(xw, ww.reshape(E, 2 * I, K), off, I, K)
    assert (q[~real].float() == 7.0).all()
    if dtype != E4M3:
        close(q[real], a[real], (tol + round_tol(a, dtype))[real], f"{counts} {I} {K}")
        return
    assert (s[~real] == 7.0).all()
    pad = ceil(I, G) * G - I
    m = torch.nn.functional.pad(a, (0, pad)).view(P, -1, G).abs().amax(2) / 448
    mt = torch.nn.functional.pad(tol, (0, pad)).view(P, -1, G).amax(2) / 448
    close(s[real], m[real], (mt + 2.0 ** -23 * m)[real], "scales")
    sw = s.double().repeat_interleave(G, 1)[:, :I]
    close(q[real].double() * sw[real], a[real],
          (tol * 17 / 16 + 2.0 ** -4 * a.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * sw)[real], "values")


@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("counts", RAGGED, ids=str)
def test_swiglu_ragged(D, dtype, counts):
    check_swiglu(D, counts, 200, 272, dtype, 61)
    check_swiglu(D, counts, 128, 128, dtype, 62, first=2, tail=5)


@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("I,K", [(1, 1), (8, 16), (64, 64), (127, 100), (129, 136), (384, 520), (768, 2048), (712, 1000),
                                 (130, 1664)])
def test_swiglu_shapes(D, dtype, I, K):
    check_swiglu(D, [5, 0, 40, 1], I, K, dtype, I + K)


def test_swiglu_large_values(D):
    """Gates far from zero on both sides: exp(-g) overflows to infinity (the activation is -0) or vanishes."""
    x = torch.ones((4, 16), dtype=BF16, device="cuda")
    w = torch.zeros((1, 4, 16), dtype=BF16, device="cuda")
    w[0, 0] = -20.0          # gate -320
    w[0, 1] = 20.0           # gate 320
    w[0, 2:] = 1.0           # up 16
    q, _ = D.grouped_swiglu_t(x, w, offsets_of([4]))
    assert (q[:, 0] == 0).all() and (q[:, 1] == 5120).all()


def test_swiglu_zero_rows_have_scale_one(D):
    g = gen(71)
    x, xs, _ = rand_rows((9, 128), E4M3, g)
    x[3] = 0.0
    w, ws, _ = rand_weights((1, 2, 130, 128), E4M3, g)
    q, s = D.grouped_swiglu_t(x, w.reshape(1, 260, 128), offsets_of([9]), xs, ws)
    assert (q[3].float() == 0).all() and (s[3] == 1).all() and (s[4] != 1).any()


def test_swiglu_nan_rows_stay_alone(D):
    g = gen(72)
    for dtype in (E4M3, F16):
        x, xs, _ = rand_rows((20, 128), dtype, g)
        w, ws, _ = rand_weights((2, 2, 100, 128), dtype, g)
        off = offsets_of([7, 13])
        q, s = D.grouped_swiglu_t(x, w.reshape(2, 200, 128), off, xs, ws)
        x[5] = float("nan")
        q2, s2 = D.grouped_swiglu_t(x, w.reshape(2, 200, 128), off, xs, ws)
        keep = [i for i in range(20) if i != 5]
        assert same_bits(q2[keep], q[keep]) and torch.isnan(q2[5].float()).all()
        assert s is None or torch.equal(s[keep], s2[keep])


# ---- the same results again, other streams, graphs -------------------------------------------------

def _product_inputs(dtype, seed=81, counts=(9, 0, 140, 33), O=256, K=640):
    g = gen(seed)
    off = offsets_of(counts)
    x, xs, _ = rand_rows((int(off[-1]), K), dtype, g)
    w, ws, _ = rand_weights((len(counts), O, K), dtype, g)
    return x, w, off, xs, ws


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_repeats_and_streams_are_bit_identical(D, dtype):
    a = _product_inputs(dtype)
    b = _product_inputs(dtype, seed=82, counts=(1, 1, 2, 0), O=2048, K=4096)     # few rows: split over K
    first = [D.grouped_matmul_t(*i) for i in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    out = []
    for s in streams:                       # both products on three streams at the same time
        with torch.cuda.stream(s):
            out += [(i, D.grouped_matmul_t(*inp)) for _ in range(5) for i, inp in enumerate((a, b))]
    torch.cuda.synchronize()
    assert all(torch.equal(y, first[i]) for i, y in out)


def test_captured_products_follow_their_inputs(D):
    """Two captured graphs of the same shapes, replayed in turn and at the same time, with new rows and new offsets."""
    x, w, off, xs, ws = _product_inputs(E4M3)
    wg, wgs, _ = rand_weights((4, 2, 320, 640), E4M3, gen(83))
    wg = wg.reshape(4, 640, 640)

    def step(out):
        out[0] = D.grouped_matmul_t(x, w, off, xs, ws)
        out[1], out[2] = D.grouped_swiglu_t(x, wg, off, xs, wgs)
    warm = {}
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(warm)
    torch.cuda.synchronize()
    outs, graphs = [{}, {}], []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(o)
        graphs.append(g)
    for counts in ((9, 0, 140, 33), (0, 100, 1, 81), (182, 0, 0, 0)):
        off.copy_(offsets_of(counts))
        x.view(torch.uint8).copy_(x.view(torch.uint8).flip(0).clone())
        want = {}
        step(want)
        torch.cuda.synchronize()
        for k, g in enumerate(graphs):
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and same_bits(o[1], want[1]) and torch.equal(o[2], want[2])


# ---- a layer of float experts --------------------------------------------------------------------

def float_layer(dtype, E, H, I, k, seed):
    from distributedmoellm_b200.layer import MoELayer
    from distributedmoellm_b200.store import FloatExperts
    g = gen(seed)
    ex = FloatExperts(E, H, I, dtype, "cuda")
    wide = []
    for e in range(E):
        gu, gus, guw = rand_weights((2, I, H), dtype, g, scale=2 / H ** 0.5)
        dn, dns, dnw = rand_weights((H, I), dtype, g, scale=1 / I ** 0.5)
        ex.put(e, gu.reshape(2 * I, H), dn, gus, dns)
        wide.append((guw.reshape(2 * I, H), dnw))
    router = torch.randn((E, H), generator=g, device="cuda") * 0.05
    return MoELayer(router, ex, k, True), wide


def layer_reference(D, layer, wide, x, dtype, b):
    """The layer in 64 bits on the kernels' own operand rows: (out, error bound without the activation's rounding)."""
    q, s = D.operand_rows(x, dtype)
    xw = q.double() if s is None else q.double() * s.double().repeat_interleave(G, 1)[:, :x.shape[1]]
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    I = layer.I
    for t in range(x.shape[0]):
        for e, wt in zip(b.idx[t].tolist(), b.w[t].tolist()):
            guw, dnw = wide[e]
            h = guw @ xw[t]
            a = h[:I] / (1 + torch.exp(-h[:I])) * h[I:]
            out[t] += wt * (dnw @ a)
            mag[t] += wt * (dnw.abs() @ a.abs())
    return out, mag


@pytest.mark.parametrize("dtype", [E4M3, BF16, F16])
@pytest.mark.parametrize("T", [1, 7, 150])
def test_layer_of_float_experts(D, dtype, T):
    """Router, permute, operand rows, gate|up, down and combine together.  Against 64 bits on the same operand rows the
    activation's rounding dominates: half a step of its type on every product (2^-4, 2^-8 or 2^-11 of sum |a w|, and for
    e4m3 half the smallest subnormal, 2^-10 of scale = 2^-10 / 448 of the group's largest, on top)."""
    E, H, I, k = 8, 272, 208, 3
    layer, wide = float_layer(dtype, E, H, I, k, 91)
    assert layer.kernel_plan(T) == [("float", 0)]
    x = torch.randn((T, H), generator=gen(T), device="cuda")
    out = layer(x)
    b = layer.buffers(T)
    want, mag = layer_reference(D, layer, wide, x, dtype, b)
    half = {E4M3: 2.0 ** -4, BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
    tol = half * mag * 1.01 + 1e-4 * mag.amax(1, keepdim=True)
    close(out, want, tol, str(dtype))
    assert layer.status(T) == 0


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_captured_layer_of_float_experts(D, dtype):
    layer, _ = float_layer(dtype, 8, 256, 128, 2, 92)
    x = torch.randn((9, 256), generator=gen(1), device="cuda")
    g = layer.capture(x)
    for seed in (2, 3):
        x.copy_(torch.randn((9, 256), generator=gen(seed), device="cuda"))
        g.replay()
        got = layer.buffers(9).out.clone()
        fresh = layer(x).clone()
        assert torch.equal(got, fresh)


def test_layer_equals_packed_experts_of_the_same_weights(D):
    """Int8 experts whose group scales are powers of two are f16 numbers: the same layer as FloatExperts(f16) agrees with
    the packed experts' decode kernels up to the f16 rounding of the rows and activations (2^-11 each on every product,
    and the router's picks are the same)."""
    import numpy as np
    from distributedmoellm_b200 import layout as L
    from distributedmoellm_b200.layer import MoELayer
    from distributedmoellm_b200.store import FloatExperts, LayerExperts
    rng = np.random.default_rng(4)
    E, H, I, k, gs, T = 8, 256, 128, 2, 32, 20
    packed = LayerExperts(E, H, I, gs, L.FMT_Q8_F32, L.FMT_Q8_F32, "cuda")
    flt = FloatExperts(E, H, I, F16, "cuda")
    for e in range(E):
        def mat(o, i):
            q = rng.integers(-127, 128, (o, i), dtype=np.int8)
            s = np.exp2(rng.integers(-13, -9, (o, i // gs))).astype(np.float32)
            return q, s, (q.astype(np.float32) * np.repeat(s, gs, 1)).astype(np.float16)
        gq, gsc, gw = mat(2 * I, H)
        dq, ds, dw = mat(H, I)
        packed.put_int8(e, gq, gsc, dq, ds)
        flt.put(e, gw, dw)
    packed.publish()
    router = torch.from_numpy((rng.standard_normal((E, H)) * 0.1).astype(np.float32)).cuda()
    x = torch.randn((T, H), generator=gen(4), device="cuda")
    a = MoELayer(router, packed, k, True, gemm_min_rows=0)
    b = MoELayer(router, flt, k, True)
    ya, yb = a(x).double(), b(x).double()
    assert torch.equal(a.buffers(T).idx, b.buffers(T).idx)
    # rows off by 2^-11 move gate and up by 2^-11 sum |x w|; bounded here through the largest output of the row
    assert float(((ya - yb).abs().amax(1) / ya.abs().amax(1)).max()) < 1e-2


# ---- operand rows of many picks (each row of x made once, then copied to its picks) ------------------

@pytest.mark.parametrize("src,dst,T,k,d", [(F32, E4M3, 1200, 8, 512), (F32, E4M3, 1187, 5, 400), (BF16, E4M3, 1300, 4, 2048),
                                           (F32, BF16, 1200, 6, 768), (F16, F16, 1250, 4, 1032)])
def test_operand_rows_of_many_picks(D, src, dst, T, k, d):
    """Every token k times in random order, one token another 5000 times, and some indices outside x."""
    g = gen(T + k + d)
    x = (torch.randn((T, d), generator=g, device="cuda") * 3).to(src)
    rows = torch.arange(T, device="cuda", dtype=torch.int32).repeat(k)
    rows = torch.cat([rows, torch.full((5000,), 7, dtype=torch.int32, device="cuda")])
    rows = rows[torch.randperm(rows.numel(), generator=g, device="cuda")].contiguous()
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, s = D.operand_rows(x, dst, rows=rows, status=st)
    assert int(st) == 0

    def want(r):
        return plain_e4m3(x[r.long()]) if dst == E4M3 else (x[r.long()].float().to(dst), None)
    wq, ws = want(rows)
    assert same_bits(q, wq) and (s is None or torch.equal(s, ws))
    bad = torch.tensor([0, 4100, rows.numel() - 1], device="cuda")
    rows[bad] = torch.tensor([-1, T, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    q, s = D.operand_rows(x, dst, rows=rows, status=st)
    assert int(st) == 2
    rows[bad] = 0
    wq, ws = want(rows)
    wq[bad] = torch.zeros((3, d), device="cuda").to(dst)
    assert same_bits(q, wq)
    if s is not None:
        ws[bad] = 1.0
        assert torch.equal(s, ws)


# ---- results whose rows no vector fits, and splits of every size ---------------------------------------

@pytest.mark.parametrize("dtype", [E4M3, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_grouped_unaligned_rows_of_results(D, dtype, out):
    """Odd O: rows of y start anywhere; large passes and small ones, full quarters and rests of them."""
    check_grouped(D, [160, 35, 8, 1, 77], 1001, 272, dtype, out, 101, first=1, tail=3)
    check_grouped(D, [3, 0, 17], 333, 144, dtype, out, 102, tail=2)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 32])
def test_few_rows_long_columns_are_split(D, dtype, n):
    """One expert's few rows over long columns: the K split, for passes of 16 and of 32 rows, and gate|up."""
    check_grouped(D, [n], 130, 7168, dtype, F32, 110 + n)
    check_grouped(D, [0, n, 0], 600, 2064, dtype, BF16, 111 + n)
    check_swiglu(D, [n], 200, 4112, dtype, 112 + n)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("n", [33, 64, 65, 100, 128, 200])
def test_ordinary_rows_long_columns_are_split(D, dtype, n):
    """Large passes on few items: clusters of two over K, every lane quarter full, ragged or empty."""
    check_grouped(D, [n], 300, 4096, dtype, F32, 130 + n, tail=1)
    check_grouped(D, [0, n, 3], 260, 2064, dtype, BF16, 131 + n, first=2)


# ---- slices of a layer, captured splits, other streams ---------------------------------------------------

@pytest.mark.parametrize("dtype", [E4M3, F16])
def test_slices_of_experts_add_up_to_the_layer(D, dtype):
    """run_experts over a slice of the experts and the matching slice of the routing (expert parallelism): the slices write
    their own picks' rows only, and together every row as the whole layer has it."""
    from distributedmoellm_b200 import layer as Lyr
    from distributedmoellm_b200.store import FloatExperts
    E, H, I, k, T = 8, 272, 144, 3, 40
    layer, _ = float_layer(dtype, E, H, I, k, 93)
    x = torch.randn((T, H), generator=gen(7), device="cuda")
    layer(x)
    b = layer.buffers(T)
    P = T * k
    whole = b.y[:P].clone()
    off = b.routing.offsets.tolist()
    y = torch.full((P, H), 5.0, device="cuda")
    bufs = {}
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    for e0, e1 in ((0, 3), (3, 8)):
        ex = FloatExperts(e1 - e0, H, I, dtype, "cuda")
        ex.gu, ex.down = layer.experts.gu[e0:e1], layer.experts.down[e0:e1]
        if dtype == E4M3:
            ex.gu_s, ex.dn_s = layer.experts.gu_s[e0:e1], layer.experts.dn_s[e0:e1]
        r = D.Routing.from_plan(b.routing.counts[e0:e1], b.routing.offsets[e0:e1 + 1], b.routing.sorted_rows[:P])
        Lyr.run_experts(ex, x, b.row_exp, r, y,
                        lambda name, n: bufs.setdefault((name, n), torch.empty(n, dtype=torch.uint8, device="cuda")),
                        st, 12)
        assert torch.equal(y[off[e0]:off[e1]], whole[off[e0]:off[e1]])
        if e1 < E:
            assert (y[off[e1]:] == 5.0).all()
    assert torch.equal(y, whole) and int(st) == 0


def test_captured_split_replays_on_several_streams(D):
    """A call split over K (clusters), captured without a call before it at this size, replayed on two streams at once."""
    x, w, off, xs, ws = _product_inputs(E4M3, seed=95, counts=(3, 0, 2), O=392, K=5008)
    y = [torch.zeros((5, 392), device="cuda") for _ in range(2)]
    graphs = []
    for o in y:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            D.grouped_matmul_t(x, w, off, xs, ws, y=o)
        graphs.append(g)
    want = D.grouped_matmul_t(x, w, off, xs, ws)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y[0], want) and torch.equal(y[1], want)


def test_one_row_may_be_asked_for_twice_and_rows_shared(D):
    """The same pick several times, and x's rows taken from an expanded row: every copy is the same."""
    x = torch.randn((1, 256), generator=gen(96), device="cuda").expand(6, 256)
    q, s = D.operand_rows(x.contiguous(), E4M3, rows=torch.tensor([5, 5, 0, 5], dtype=torch.int32, device="cuda"))
    assert all(same_bits(q[i], q[0]) and torch.equal(s[i], s[0]) for i in range(4))
    with pytest.raises(RuntimeError, match="closer"):
        D.operand_rows(x, E4M3)                    # a row distance of 0 is refused
    w = torch.zeros((1, 64, 256), dtype=BF16, device="cuda").expand(3, 64, 256)
    with pytest.raises(RuntimeError, match="overlap"):
        D.grouped_matmul_t(x.to(BF16).contiguous(), w, offsets_of([2, 2, 2]))
    with pytest.raises(RuntimeError, match="16 bytes"):
        D.grouped_matmul_t(torch.zeros((6, 100), dtype=BF16, device="cuda"), torch.zeros((3, 64, 100), dtype=BF16,
                                                                                      device="cuda"), offsets_of([2, 2, 2]))


def test_1024_experts_with_long_columns(D):
    """Large tables beside the stages and a split's partial sums."""
    counts = [0] * 1024
    counts[3], counts[1023] = 2, 20
    for dtype in (E4M3, BF16):
        check_grouped(D, counts, 40, 2064, dtype, F32, 141)
        check_swiglu(D, counts, 40, 1040, dtype, 142)
        counts[5] = 300
        check_swiglu(D, counts, 40, 528, dtype, 143)


@pytest.mark.parametrize("d", [2480, 2496, 2504, 2520, 2536])
def test_operand_rows_of_many_picks_at_the_shared_memory_limit(D, d):
    x = torch.randn((1200, d), generator=gen(d), device="cuda")
    rows = torch.arange(1200, device="cuda", dtype=torch.int32).repeat(4)
    q, _ = D.operand_rows(x, BF16, rows=rows)
    assert torch.equal(q, x[rows.long()].to(BF16))


@pytest.mark.parametrize("src,dst,T,k,d", [(F32, E4M3, 2368, 8, 512), (F32, E4M3, 2367, 8, 512), (F32, E4M3, 2371, 5, 400),
                                           (BF16, E4M3, 2500, 4, 2048), (F32, BF16, 2400, 6, 768), (F16, F16, 2433, 4, 1032)])
def test_operand_rows_of_many_picks_of_many_rows(D, src, dst, T, k, d):
    """Rows for every SM's blocks of sixteen, the last block ragged, and one row fewer than that."""
    test_operand_rows_of_many_picks(D, src, dst, T, k, d)


@pytest.mark.parametrize("d", [2752, 2760, 2768, 2776, 2784])
def test_operand_rows_of_many_rows_at_the_shared_memory_limit(D, d):
    x = torch.randn((2400, d), generator=gen(d), device="cuda")
    rows = torch.arange(2400, device="cuda", dtype=torch.int32).repeat(4)
    q, _ = D.operand_rows(x, BF16, rows=rows)
    assert torch.equal(q, x[rows.long()].to(BF16))


# ---- results of more than 2^31 values -----------------------------------------------------------------

ENDS = (slice(0, 130), slice(-130, None))


@pytest.mark.parametrize("T,P", [(100, 1_060_000), (2400, 1_060_000)])
def test_operand_rows_past_32_bits(D, T, P):
    """Made for each pick, and made once and copied."""
    x = torch.randn((T, 2048), generator=gen(T), device="cuda")
    rows = torch.randint(0, T, (P,), generator=gen(P), device="cuda", dtype=torch.int32)
    q, s = D.operand_rows(x, E4M3, rows=rows)
    assert q.numel() > 2 ** 31
    for r in ENDS:
        wq, ws = plain_e4m3(x[rows[r].long()])
        assert same_bits(q[r], wq) and torch.equal(s[r], ws)


@pytest.mark.parametrize("dtype,O", [(E4M3, 14336), (E4M3, 14337), (F16, 14336)])
def test_grouped_past_32_bits(D, dtype, O):
    """Results by TMA, one at a time, and by vectors."""
    g = gen(O)
    P, K, E = 151_000, 64, 2
    x, xs, xw = rand_rows((P, K), dtype, g)
    w, ws, ww = rand_weights((E, O, K), dtype, g)
    off = offsets_of([70_001, P - 70_001])
    y = D.grouped_matmul_t(x, w, off, xs, ws, dtype=BF16)
    assert y.numel() > 2 ** 31
    for e, r in enumerate(ENDS):
        want, S = xw[r] @ ww[e].t(), xw[r].abs() @ ww[e].abs().t()
        close(y[r], want, sum_tol(K, S) + round_tol(want, BF16), str(r))


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_swiglu_past_32_bits(D, dtype):
    g = gen(81)
    P, K, I = 151_000, 64, 14336
    x, xs, xw = rand_rows((P, K), dtype, g)
    w, ws, ww = rand_weights((1, 2, I, K), dtype, g, scale=3.0 / K ** 0.5)
    q, s = D.grouped_swiglu_t(x, w.view(1, 2 * I, K), offsets_of([P]), xs, ws)
    assert q.numel() > 2 ** 31
    for r in ENDS:
        a, tol, _ = want_swiglu(xw[r], ww.view(1, 2 * I, K), offsets_of([130]), I, K)
        if dtype != E4M3:
            close(q[r], a, tol + round_tol(a, dtype), str(r))
            continue
        sw = s[r].double().repeat_interleave(G, 1)
        close(q[r].double() * sw, a, tol * 17 / 16 + 2.0 ** -4 * a.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * sw, str(r))


FIRST_CALL = """
import torch
from distributedmoellm_b200 import device as D
torch.manual_seed(0)
x = torch.randn(40, 2048, device="cuda")
w = torch.randn(4, 1536, 2048, device="cuda").to(torch.float8_e4m3fn)
ws = torch.rand(4, 2, 6, 16, device="cuda")
wd = torch.randn(4, 2048, 768, device="cuda").to(torch.float8_e4m3fn)
wds = torch.rand(4, 16, 6, device="cuda")
off = torch.tensor([0, 1, 9, 9, 40], dtype=torch.int32, device="cuda")
one = torch.randn(1, 2048, device="cuda")
torch.cuda.synchronize()

def run():
    q, s = D.operand_rows(x, torch.float8_e4m3fn)
    a, t = D.grouped_swiglu_t(q, w, off, s, ws)
    y = D.grouped_matmul_t(a, wd, off, t, wds)
    q1, s1 = D.operand_rows(one, torch.float8_e4m3fn)
    return y, D.matmul_t_e4m3(q1, s1, w[0], ws[0].reshape(12, 16))

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    captured = run()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, run()))

# several threads, each on a stream of its own
import threading
want, bad = run(), []
def work():
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(50):
            got = run()
        torch.cuda.current_stream().synchronize()
        if not all(torch.equal(a, b) for a, b in zip(got, want)):
            bad.append(1)
torch.cuda.synchronize()
ts = [threading.Thread(target=work) for _ in range(4)]
[t.start() for t in ts]; [t.join() for t in ts]
assert not bad
print("fine")
"""


def test_first_calls_of_a_process_captured_and_from_threads(D):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stderr[-2000:]
