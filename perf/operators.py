"""What is measured of the float-expert operators: their cases, the inputs,
their plain form in elementary torch operations, and their definition in 64
bits.

* operand_rows: rows of x picked by index and put into the form the products
  take (e4m3 with one f32 scale per 128 columns, or bf16 / f16);
* matmul_t_e4m3: x @ W.T with e4m3 rows (a scale per 128 columns) and e4m3
  weights (a scale per 128 x 128 block);
* grouped_matmul_t: rows grouped by expert times each expert's matrix, e4m3
  with scales or bf16 / f16;
* grouped_swiglu_t: the same for gate|up matrices, with SiLU(gate) * up put
  into operand form.
"""

import math

import torch

own = False

G = 128                                  # columns (and weight rows) per scale
E4M3 = torch.float8_e4m3fn
TYPES = {"e4m3": E4M3, "bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"e4m3": 1, "bf16": 2, "f16": 2, "f32": 4}


def ceil(a, b):
    return -(-a // b)


def _over_448(m):
    """m / 448 (e4m3's largest value), one rounding: torch divides by a plain number through its reciprocal."""
    return m / torch.full_like(m, 448.0)


# ---- the cases -------------------------------------------------------------------------

def listed():
    return [
        # a decode step's 64 tokens, each to 8 experts of the 128-expert layer, on the way into gate|up
        dict(name="rows_e4m3_T64", op="rows", T=64, k=8, d=2048, src="f32", dst="e4m3", skew=0.5),
        # the same for a long prompt of 4096 tokens
        dict(name="rows_e4m3_T4096", op="rows", T=4096, k=8, d=2048, src="f32", dst="e4m3", skew=0.5),
        # one token through one wide matrix (the 14336 x 4096 gate of an 8-expert layer)
        dict(name="mm_e4m3_n1", op="mm", n=1, O=14336, K=4096, out="f32"),
        # odd sizes: 333 rows, row and column counts that end inside a block
        dict(name="mm_e4m3_odd", op="mm", n=333, O=1000, K=1424, out="bf16"),
        # a long prompt through the wide matrix
        dict(name="mm_e4m3_n4096", op="mm", n=4096, O=14336, K=4096, out="bf16"),
        # down products of a decode step: 64 tokens, 8 of 128 experts each, about 4 rows an expert
        dict(name="grouped_e4m3_T64", op="grouped", T=64, k=8, E=128, O=2048, K=768, type="e4m3", out="f32", skew=0.5,
             tail=0),
        # down products of a 2048-token prompt
        dict(name="grouped_e4m3_T2048", op="grouped", T=2048, k=8, E=128, O=2048, K=768, type="e4m3", out="f32",
             skew=0.5, tail=0),
        # 16-bit experts, one token: eight matrices of 1536 x 2048
        dict(name="grouped_bf16_T1", op="grouped", T=1, k=8, E=128, O=1536, K=2048, type="bf16", out="f32", skew=0.5,
             tail=0),
        # 16-bit experts, a 2048-token prompt, loads that differ much between experts and unused rows at the end
        dict(name="grouped_f16_T2048", op="grouped", T=2048, k=8, E=128, O=1536, K=2048, type="f16", out="f16",
             skew=1.0, tail=77),
        # gate|up with the activation, a decode step of 8 tokens
        dict(name="swiglu_e4m3_T8", op="swiglu", T=8, k=8, E=128, I=768, K=2048, type="e4m3", skew=0.5, tail=0),
        # gate|up with the activation, a 4096-token prompt
        dict(name="swiglu_e4m3_T4096", op="swiglu", T=4096, k=8, E=128, I=768, K=2048, type="e4m3", skew=0.5, tail=0),
        # gate|up of 16-bit experts at an odd token count, an intermediate size that ends inside a block
        dict(name="swiglu_bf16_odd", op="swiglu", T=555, k=4, E=24, I=712, K=1000, type="bf16", skew=1.0, tail=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: rows 1 .. 4096, experts 1 .. 128, 1 .. 8 picks a token, any odd sizes (columns
    of an operand row whose byte length is a multiple of 16)."""
    op = rng.choice(["rows", "mm", "grouped", "grouped", "swiglu"])
    T = _log(rng, 1, 4096)
    if op == "rows":
        return dict(op=op, T=T, k=rng.randint(1, 8), d=_log(rng, 32, 4096), src=rng.choice(["f32", "bf16", "f16"]),
                    dst=rng.choice(["e4m3", "e4m3", "bf16", "f16"]), skew=rng.choice([0.0, 0.5, 1.0]))
    if op == "mm":
        return dict(op=op, n=T, O=_log(rng, 64, 14336), K=16 * _log(rng, 4, 256), out=rng.choice(["f32", "bf16", "f16"]))
    E = _log(rng, 2, 128)
    k = rng.randint(1, min(E, 8))
    ty = rng.choice(["e4m3", "e4m3", "bf16", "f16"])
    K = 16 * _log(rng, 4, 128) if ty == "e4m3" else 8 * _log(rng, 8, 256)
    common = dict(T=T, k=k, E=E, K=K, type=ty, skew=rng.choice([0.0, 0.5, 1.0]), tail=rng.choice([0, 0, 1, 77]))
    if op == "grouped":
        return dict(op=op, O=_log(rng, 64, 2048), out=rng.choice(["f32", "bf16", "f16"]), **common)
    return dict(op=op, I=_log(rng, 64, 768), **common)


# ---- inputs ----------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weights(shape, type_, g):
    """Weights ~N(0, 0.02) (moelan's tiny checkpoints), as a checkpoint of that type holds them: 16-bit values, or e4m3
    with the scale max / 448 of each 128 x 128 block.  Returns (w, block scales or None)."""
    w = torch.randn(shape, generator=g, device="cuda") * 0.02
    if type_ != "e4m3":
        return w.to(TYPES[type_]), None
    *lead, O, K = shape
    Ob, Kb = ceil(O, G), ceil(K, G)
    p = torch.zeros((*lead, Ob * G, Kb * G), device="cuda")
    p[..., :O, :K] = w
    p = p.view(*lead, Ob, G, Kb, G)
    s = _over_448(p.abs().amax(dim=(-3, -1)))
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (p / s[..., :, None, :, None]).clamp(-448, 448).view(*lead, Ob * G, Kb * G)[..., :O, :K].to(E4M3)
    return q.contiguous(), s


def _picks(T, k, E, skew, g):
    """Top-k of random router logits (an offset per expert makes loads differ), sorted by expert as mb_permute does."""
    logits = torch.randn((T, E), generator=g, device="cuda") + skew * torch.randn((E,), generator=g, device="cuda")
    idx = logits.topk(k, dim=1).indices.reshape(-1)
    order = torch.sort(idx, stable=True).indices
    counts = torch.bincount(idx, minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return (order // k).to(torch.int32), offsets, int(counts.max())


def _operand(x, type_):
    if type_ != "e4m3":
        return x.to(TYPES[type_]), None
    return _encode(x)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "rows":
        E = max(8, case["k"])
        rows, _, _ = _picks(case["T"], case["k"], E, case["skew"], g)
        x = torch.randn((case["T"], case["d"]), generator=g, device="cuda").to(TYPES[case["src"]])
        return dict(op=op, x=x, rows=rows, dst=TYPES[case["dst"]])
    if op == "mm":
        x, xs = _operand(torch.randn((case["n"], case["K"]), generator=g, device="cuda"), "e4m3")
        w, ws = _weights((case["O"], case["K"]), "e4m3", g)
        return dict(op=op, x=x, xs=xs, w=w, ws=ws, out=TYPES[case["out"]])
    T, k, E, K, ty, tail = (case[n] for n in ("T", "k", "E", "K", "type", "tail"))
    _, offsets, most = _picks(T, k, E, case["skew"], g)
    P = T * k + tail                         # rows behind the last expert's are not touched
    x, xs = _operand(torch.randn((P, K), generator=g, device="cuda"), ty)
    if op == "grouped":
        w, ws = _weights((E, case["O"], K), ty, g)
        y = torch.full((P, case["O"]), 7.0, device="cuda").to(TYPES[case["out"]])
        return dict(op=op, x=x, xs=xs, w=w, ws=ws, offsets=offsets, most=most, y=y)
    I = case["I"]
    w, ws = _weights((E, 2, I, K), ty, g)    # gate rows, then up rows, each with its own grid of blocks
    w = w.view(E, 2 * I, K)
    q = torch.full((P, I), 7.0, device="cuda").to(TYPES[ty])
    s = torch.full((ceil(I, G), P), 7.0, device="cuda").t() if ty == "e4m3" else None
    return dict(op=op, x=x, xs=xs, w=w, ws=ws, offsets=offsets, most=most, q=q, s=s)


# ---- plain forms -----------------------------------------------------------------------

def _encode(x):
    """(q, s): s = max|group| / 448 (1 for a group of zeros), q = e4m3(x / s); s is (n, groups), stored group by group."""
    n, d = x.shape
    Kb = ceil(d, G)
    p = torch.zeros((n, Kb * G), device=x.device)
    p[:, :d] = x.float()
    p = p.view(n, Kb, G)
    s = _over_448(p.abs().amax(dim=2))
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (p / s[:, :, None]).clamp(-448, 448).view(n, Kb * G)[:, :d].to(E4M3)
    return q.contiguous(), s.t().contiguous().t()


def _wide(x, xs):
    """Operand rows in f32: values times their group's scale."""
    x = x.float()
    return x if xs is None else x * xs.repeat_interleave(G, dim=1)[:, :x.shape[1]]


def _wide_w(w, ws, rows):
    """Weights (..., rows, K) in f32: values times their block's scale."""
    w = w.float()
    if ws is None:
        return w
    return w * ws.repeat_interleave(G, dim=-2)[..., :rows, :].repeat_interleave(G, dim=-1)[..., :w.shape[-1]]


def _padded(s):
    """Each expert's rows of x, padded to the largest load: (rows (E, most, K), their index, which of them exist)."""
    off = s["offsets"].long()
    at = off[:-1, None] + torch.arange(s["most"], device=off.device)[None, :]
    real = at < off[1:, None]
    x = _wide(s["x"], s["xs"])
    return x[torch.where(real, at, torch.zeros_like(at))], at, real


def _plain_grouped(s):
    x, at, real = _padded(s)
    y = x @ _wide_w(s["w"], s["ws"], s["w"].shape[1]).transpose(1, 2)
    s["y"][at[real]] = y[real].to(s["y"].dtype)
    return s["y"]


def _plain_swiglu(s):
    x, at, real = _padded(s)
    E, I2, K = s["w"].shape
    w = _wide_w(s["w"].view(E, 2, I2 // 2, K), s["ws"], I2 // 2).view(E, I2, K)
    h = (x @ w.transpose(1, 2))[real]
    g, u = h[:, :I2 // 2], h[:, I2 // 2:]
    a = g / (1 + torch.exp(-g)) * u
    if s["s"] is None:
        s["q"][at[real]] = a.to(s["q"].dtype)
        return s["q"]
    q, sc = _encode(a)
    s["q"].view(torch.uint8)[at[real]] = q.view(torch.uint8)
    s["s"][at[real]] = sc
    return s["q"], s["s"]


def _plain(s):
    if s["op"] == "rows":
        x = s["x"][s["rows"].long()]
        return _encode(x) if s["dst"] == E4M3 else x.float().to(s["dst"])
    if s["op"] == "mm":
        return (_wide(s["x"], s["xs"]) @ _wide_w(s["w"], s["ws"], s["w"].shape[0]).t()).to(s["out"])
    return _plain_grouped(s) if s["op"] == "grouped" else _plain_swiglu(s)


def _own(s):
    from distributedmoellm_b200 import device as D
    if s["op"] == "rows":
        q, sc = D.operand_rows(s["x"], s["dst"], rows=s["rows"])
        return q if sc is None else (q, sc)
    if s["op"] == "mm":
        return D.matmul_t_e4m3(s["x"], s["xs"], s["w"], s["ws"], dtype=s["out"])
    if s["op"] == "grouped":
        return D.grouped_matmul_t(s["x"], s["w"], s["offsets"], xs=s["xs"], ws=s["ws"], y=s["y"])
    q, sc = D.grouped_swiglu_t(s["x"], s["w"], s["offsets"], xs=s["xs"], ws=s["ws"], q=s["q"], scales=s["s"])
    return q if sc is None else (q, sc)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "rows":
        T, P, d = case["T"], case["T"] * case["k"], case["d"]
        b = T * d * SIZE[case["src"]] + P * 4 + P * d * SIZE[case["dst"]]
        return {"bytes": b + (P * ceil(d, G) * 4 if case["dst"] == "e4m3" else 0), "flops": 0}
    K = case["K"]
    if op == "mm":
        n, O = case["n"], case["O"]
        b = O * K + n * K + (n + ceil(O, G)) * ceil(K, G) * 4 + n * O * SIZE[case["out"]]
        return {"bytes": b, "flops": 2 * n * O * K}
    ty = case["type"]
    P, E = case["T"] * case["k"], case["E"]
    O = case["O"] if op == "grouped" else 2 * case["I"]
    # experts that at least one of the picks meets, if every expert were as likely as another
    act = E * (1 - (1 - case["k"] / E) ** case["T"])
    b = act * O * K * SIZE[ty] + P * K * SIZE[ty] + (E + 1) * 4
    if ty == "e4m3":
        b += (P + act * ceil(O, G)) * ceil(K, G) * 4
    if op == "grouped":
        b += P * O * SIZE[case["out"]]
    else:
        b += P * case["I"] * SIZE[ty] + (P * ceil(case["I"], G) * 4 if ty == "e4m3" else 0)
    return {"bytes": int(b), "flops": 2 * P * O * K}


# ---- the definition in 64 bits -----------------------------------------------------------

def _exact_rows(a, typed):
    """Rows in operand form before the last rounding: values divided by their group's scale, and the scales; or the rows
    themselves for a 16-bit type."""
    if typed != E4M3:
        return a
    n, d = a.shape
    q, s = torch.empty_like(a), torch.empty((n, ceil(d, G)), dtype=torch.float64, device=a.device)
    for g in range(ceil(d, G)):
        cols = slice(g * G, min(d, (g + 1) * G))
        m = a[:, cols].abs().max(dim=1).values / 448
        s[:, g] = torch.where(m > 0, m, 1.0)
        q[:, cols] = a[:, cols] / s[:, g, None]
    return q, s


def _exact_product(x, xs, w, ws):
    """x (n, K) @ w (O, K).T in float64, block by block of 128 columns where there are scales."""
    x, w = x.double(), w.double()
    if xs is None:
        return x @ w.t()
    y = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device=x.device)
    row_block = torch.arange(w.shape[0], device=x.device) // G
    for g in range(xs.shape[1]):
        cols = slice(g * G, min(x.shape[1], (g + 1) * G))
        y += (x[:, cols] @ w[:, cols].t()) * xs[:, g, None].double() * ws[row_block, g][None, :].double()
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rows":
        return _exact_rows(s["x"][s["rows"].long()].double(), s["dst"])
    if op == "mm":
        return _exact_product(s["x"], s["xs"], s["w"], s["ws"])
    off = s["offsets"].tolist()
    if op == "grouped":
        y = s["y"].double()
        for e in range(case["E"]):
            r = slice(off[e], off[e + 1])
            if off[e + 1] > off[e]:
                y[r] = _exact_product(s["x"][r], None if s["xs"] is None else s["xs"][r], s["w"][e],
                                      None if s["ws"] is None else s["ws"][e])
        return y
    I = case["I"]
    q = s["q"].double()
    sc = None if s["s"] is None else s["s"].double()
    for e in range(case["E"]):
        r = slice(off[e], off[e + 1])
        if off[e + 1] == off[e]:
            continue
        xs = None if s["xs"] is None else s["xs"][r]
        h = [_exact_product(s["x"][r], xs, s["w"][e, i * I:(i + 1) * I], None if s["ws"] is None else s["ws"][e, i])
             for i in (0, 1)]
        a = h[0] / (1 + torch.exp(-h[0])) * h[1]
        if sc is None:
            q[r] = a
        else:
            q[r], sc[r] = _exact_rows(a, E4M3)
    return q if sc is None else (q, sc)
