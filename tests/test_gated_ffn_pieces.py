"""gated_ffn where every piece of an operand counts: calls of every tile of the large products, with real values in every bit.

The operands are such that a sum has few terms: a row of X and of dY has one entry, a column of Wd has one, Wg and Wu are full.  G, U, Y
and dA are then single products and dX sums of two, so that a bound by the number of terms n is a few roundings, where
one by the length of the sum would hide a lost piece.  E = 2^-24, B = 2^-8 (half a step of fp32 / bf16):

* fp32.  An operand is three bf16 pieces, the second at most 2^-9, the third at most 2^-18 of it; six products of pieces are added (the
  three left out are below 2^-26).  The first term's roundings are of its small pieces but for the last one; a further term adds six
  to a sum of full size: (6 n - 4) E of the sum of the terms' absolute values.  A piece product that is missing is off by up to
  2^-18 = 64 E (m m') or more.
* bf16 calls with more than 16384 elements of A: A, dG and dU are rounded (B each), P = U act'(G) and Q = act(G) keep 24 bits (2^-16).

relu throughout: its activation is exact, its slope is 0 or 1 but where the error of G reaches its sign (the whole term, then)."""
import re

import pytest
import torch

E, B8 = 2.0 ** -24, 2.0 ** -8
f32, bf16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def amd():
    import agcn_amd
    if agcn_amd._build.is_stale():
        agcn_amd._build.build()
    return agcn_amd


def case(seed, M, F, H, O, dtype, device="cuda"):
    g = torch.Generator().manual_seed(seed)

    def one(rows, cols):
        t = torch.zeros(rows, cols)
        t[torch.arange(rows), torch.randint(0, cols, (rows,), generator=g)] = 1 + torch.rand(rows, generator=g)
        return t
    full = lambda r, c: torch.randn(r, c, generator=g)  # noqa: E731
    X, Wg, Wu, Wd, dY = one(M, F), full(F, H), full(F, H), one(O, H).t().contiguous(), one(M, O)
    return [t.to(dtype).to(device) for t in (X, Wg, Wu, Wd, dY)]


def reference(X, Wg, Wu, Wd, dY, dtype):
    """float64 results and their bounds"""
    b, pq = (B8, 2.0 ** -16) if dtype == bf16 else (0.0, 0.0)
    X, Wg, Wu, Wd, dY = (t.double() for t in (X, Wg, Wu, Wd, dY))

    def product(x, w, ex=None, ew=None, nx=None, nw=None):
        """x w, |its errors|: those of the operands, and its own roundings by the number of terms that are not zero"""
        n = (x != 0 if nx is None else nx).double() @ (w != 0 if nw is None else nw).double()
        e = (6 * n - 4).clamp(min=0) * E * (x.abs() @ w.abs())
        if ex is not None:
            e = e + ex @ w.abs()
        if ew is not None:
            e = e + x.abs() @ ew
        return x @ w, e
    G, eG = product(X, Wg)
    U, eU = product(X, Wu)
    on = G > -eG                                             # where relu may let something through
    a, P = G.clamp(min=0), U * (G > 0)
    A = a * U
    eA = U.abs() * eG * on + a * eU + (b + E) * A.abs()
    eP = U.abs() * (G.abs() <= eG) * (eG > 0) + eU * on + (pq + E) * P.abs()
    eQ = eG * on + pq * a
    dA, eDA = product(dY, Wd.t())
    dG, dU = dA * P, dA * a
    eDG = dA.abs() * eP + P.abs() * eDA + (b + E) * dG.abs()
    eDU = dA.abs() * eQ + a * eDA + (b + E) * dU.abs()
    nd, na = (dA != 0) & on, (U != 0) & on
    res = {"Y": product(A, Wd, ex=eA, nx=na),
           "dX": product(torch.cat((dG, dU), 1), torch.cat((Wg, Wu), 1).t(), ex=torch.cat((eDG, eDU), 1), nx=torch.cat((nd, nd), 1)),
           "dWg": product(X.t(), dG, ew=eDG, nw=nd), "dWu": product(X.t(), dU, ew=eDU, nw=nd),
           "dWd": product(A.t(), dY, ex=eA.t(), nx=na.t())}
    s = B8 if dtype == bf16 else E
    return {k: v for k, (v, _) in res.items()}, {k: 1.01 * e + s * v.abs() + 1e-37 for k, (v, e) in res.items()}


def worst(got, want, bound):
    return {k: float(((got[k].double() - want[k]).abs() / bound[k]).max()) for k in want}


# ---- the bounds notice what they are for (CPU; the mistakes are in this emulation) --------------------------------------
def pieces(x):
    h = x.to(bf16).float()
    m = (x - h).to(bf16).float()
    return h, m, (x - h - m).to(bf16).float()


PAIRS = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]


def emulate(X, Wg, Wu, Wd, dY, dtype, drop=None, low=True):
    """The passes as the kernels make them.  drop: (product, pair of pieces that it leaves out); low=False: P and Q without their
    lower eight bits."""
    def mm(name, x, w):
        if dtype == bf16:
            return (x.double() @ w.double()).float()
        xs, ws = pieces(x), pieces(w)
        s = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
        for p in PAIRS:
            if drop != (name, p):
                s += xs[p[0]].double() @ ws[p[1]].double()
        return s.float()

    def kept(x):
        if dtype == f32:
            return x
        bits = x.view(torch.int32) + 0x80
        return (bits & (-256 if low else -65536)).view(f32)
    stored = lambda t: t.to(dtype).float()  # noqa: E731
    X, Wg, Wu, Wd, dY = (t.float() for t in (X, Wg, Wu, Wd, dY))
    G, U = mm("GU", X, Wg), mm("GU", X, Wu)
    a, da = G.clamp(min=0), (G > 0).float()
    A, P, Q = stored(a * U), kept(da * U), kept(a)
    dA = mm("DH", dY, Wd.t())
    dG, dU = stored(dA * P), stored(dA * Q)
    out = {"Y": mm("Y", A, Wd), "dX": mm("DX", torch.cat((dG, dU), 1), torch.cat((Wg, Wu), 1).t()),
           "dWg": mm("DW", X.t(), dG), "dWu": mm("DW", X.t(), dU), "dWd": mm("DWD", A.t(), dY)}
    return {k: stored(v) for k, v in out.items()}


def test_bounds_hold_for_all_pieces_and_break_without_any_one():
    args = case(1, 400, 30, 120, 50, f32, "cpu")
    want, bound = reference(*args, f32)
    assert max(worst(emulate(*args, f32), want, bound).values()) <= 1.0
    for name in ("GU", "Y", "DH", "DX", "DW", "DWD"):
        for pair in PAIRS:
            w = worst(emulate(*args, f32, drop=(name, pair)), want, bound)
            assert max(w.values()) > 1.2, (name, pair, w)


def test_bounds_hold_for_24_bits_and_break_for_16():
    args = case(2, 400, 30, 120, 50, bf16, "cpu")
    want, bound = reference(*args, bf16)
    assert max(worst(emulate(*args, bf16), want, bound).values()) <= 1.0
    w = worst(emulate(*args, bf16, low=False), want, bound)
    assert min(w["dX"], w["dWg"], w["dWu"]) > 1.2, w


# ---- the kernels ---------------------------------------------------------------------------------------------------------
# rows, features, hidden, outputs: together every product of a training pass on its large, middle and small tile, whole and cut along k
PLANES = [(2052, 22, 347, 927), (229, 2117, 1092, 1368), (1652, 840, 623, 1704), (851, 95, 2864, 834), (22678, 70, 129, 254), (843, 2338, 614, 104),
          (17150, 1425, 33, 260), (810, 1358, 2542, 2512), (1171, 460, 2099, 1102), (2300, 200, 3000, 160), (2304, 200, 3000, 160)]
BF16 = [(43, 18, 431, 21), (1986, 1210, 22, 1934), (6389, 82, 1293, 19), (22965, 137, 145, 452), (41, 1134, 2000, 1765), (16550, 2075, 16, 2449),
        (4625, 37, 2126, 213), (33, 60, 3295, 2515), (33, 2344, 2011, 54), (8491, 472, 2392, 22), (4782, 27, 3288, 1214), (2300, 200, 3000, 160)]


# operands split in registers (whole chunks of 16 bytes and not), both products in one kernel, few rows
SMALLER = [(100, 300, 200, 152), (101, 301, 203, 151), (33, 1027, 90, 1033), (5000, 60, 300, 64), (20000, 100, 200, 120), (3, 300, 2000, 70), (1, 2051, 700, 300)]


def run(amd, X, Wg, Wu, Wd, dY):
    ts = [t.detach().requires_grad_(True) for t in (X, Wg, Wu, Wd)]
    Y = amd.gated_ffn(*ts, activation="relu")
    return dict(zip(("Y", "dX", "dWg", "dWu", "dWd"), (Y.detach(),) + torch.autograd.grad(Y, ts, dY)))


@pytest.mark.gpu
@pytest.mark.parametrize("size,dtype", [(s, f32) for s in PLANES + SMALLER] + [(s, bf16) for s in BF16 + SMALLER])
def test_every_piece_counts(amd, size, dtype):
    args = case(sum(size), *size, dtype)
    want, bound = reference(*args, dtype)
    w = worst(run(amd, *args), want, bound)
    assert max(w.values()) <= 1.0, w
    Y = amd.gated_ffn(*args[:4], activation="relu")          # the form that keeps nothing
    assert worst({"Y": Y}, {"Y": want["Y"]}, bound)["Y"] <= 1.0


# a product by its template arguments: transposed A, transposed B, matrices of B, epilogue
PRODUCTS = {("false", "true", "2", "0"): "GU", ("false", "true", "1", "1"): "Y", ("false", "false", "1", "2"): "DH",
            ("false", "false", "1", "1"): "DX", ("true", "true", "2", "1"): "DW", ("true", "true", "1", "1"): "DWD"}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sizes,form", [(f32, PLANES, "3"), (bf16, BF16, "1")])
def test_sizes_reach_every_tile(amd, dtype, sizes, form):
    """The sizes above are no good if the choice of tiles moves away from them: what they launch, by the kernels' names."""
    from torch.profiler import ProfilerActivity, profile
    seen = set()
    for size in sizes:
        args = case(0, *size, dtype)
        run(amd, *args)
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            run(amd, *args)
            torch.cuda.synchronize()
        names = [e.name for e in p.events()]
        if not any("ffn_" in n for n in names):
            pytest.skip("no kernel names from the profiler here")
        found = [m for m in (re.search(r"ffn_gemm_kernel<(\d), (\d+), \d+, \d, \d, (\w+), (\w+), (\d), (\d), \d>", n) for n in names) if m]
        assert len(found) == 6 and {m.group(1) for m in found} == {form}, (size, names)
        seen |= {(PRODUCTS[m.groups()[2:]], m.group(2)) for m in found}
        if any("ffn_reduce_kernel<2" in n for n in names):
            seen.add(("two sums", "reduce"))
    assert seen >= {(name, rows) for name in PRODUCTS.values() for rows in ("256", "128", "64")}, sorted(seen)
    assert ("two sums", "reduce") in seen
