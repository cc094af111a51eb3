"""gated_ffn (csrc/gated_ffn.hip): Y = (act(X Wg) * (X Wu)) Wd and its gradients against float64.

Two kinds of checks.  (1) Exact: with small integers and relu every inner value is an integer that bf16 holds and every sum one
that fp32 holds, so results must EQUAL the float64 ones (rounded once where they are stored in bf16): a term that is
missing, doubled or misplaced shows at any size.  (2) Bounds, E = 2^-24, B = 2^-8 (half a step of fp32 / bf16): a sum of K terms
is within (K + 8) E of the sum of their absolute values (the six piece products of an fp32 product are within 4 E of it), the
activations within 16 E of themselves, an error e of G moves act by at most 1.2 e and act' by at most 0.8 e (sup |act'|,
sup |act''| over silu, gelu, sigmoid; relu: the whole term where e reaches |G|); bf16 calls store G, U, A, dG, dU with an error
of B each.  The bounds are carried through the formulas with absolute values; 5 per cent for products of errors."""
import ctypes as C
import math

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


def act64(name, g):
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    s = torch.sigmoid(g)
    if name == "sigmoid":
        return s, s * torch.sigmoid(-g)
    if name == "silu":
        return g * s, s * (1 + g * torch.sigmoid(-g))
    c = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def reference(X, Wg, Wu, Wd, dY, act, dtype, b=None, act_err=16 * E):
    X, Wg, Wu, Wd, dY = (t.double() for t in (X, Wg, Wu, Wd, dY))
    if b is None:
        b = B8 if dtype == bf16 else 0.0
    M, F = X.shape
    H, O = Wd.shape
    G, U = X @ Wg, X @ Wu
    a, da = act64(act, G)
    A = a * U
    aX, aWg, aWu, aWd = X.abs(), Wg.abs(), Wu.abs(), Wd.abs()
    eG, eU = (F + 8) * E * (aX @ aWg), (F + 8) * E * (aX @ aWu)
    ea = 1.2 * eG + act_err * a.abs()
    eA = U.abs() * ea + a.abs() * eU + (b + 2 * E) * A.abs()
    out, err = {"Y": A @ Wd}, {"Y": eA @ aWd + (H + 8) * E * (A.abs() @ aWd)}
    dA = dY @ Wd.t()
    eDA = (O + 8) * E * (dY.abs() @ aWd.t())
    eGs, eUs = eG + b * G.abs(), eU + b * U.abs()
    eda = ((G.abs() <= eGs).double() if act == "relu" else 0.8 * eGs) + act_err * da.abs()
    dG, dU = dA * U * da, dA * a
    eDG = (dA * U).abs() * eda + (dA * da).abs() * eUs + (U * da).abs() * eDA + (b + 4 * E) * dG.abs()
    eDU = dA.abs() * (1.2 * eGs + act_err * a.abs()) + a.abs() * eDA + (b + 2 * E) * dU.abs()
    out["dX"] = dG @ Wg.t() + dU @ Wu.t()
    err["dX"] = eDG @ aWg.t() + eDU @ aWu.t() + (2 * H + 8) * E * (dG.abs() @ aWg.t() + dU.abs() @ aWu.t())
    out["dWg"], out["dWu"], out["dWd"] = X.t() @ dG, X.t() @ dU, A.t() @ dY
    err["dWg"] = aX.t() @ eDG + (M + 8) * E * (aX.t() @ dG.abs())
    err["dWu"] = aX.t() @ eDU + (M + 8) * E * (aX.t() @ dU.abs())
    err["dWd"] = eA.t() @ dY.abs() + (M + 8) * E * (A.abs().t() @ dY.abs())
    inner = max(float(t.abs().max()) if t.numel() else 0.0 for t in (G, U, A, dG, dU))
    return out, err, inner


def run(amd, X, Wg, Wu, Wd, dY, act):
    ts = [t.detach().clone().requires_grad_(True) for t in (X, Wg, Wu, Wd)]
    Y = amd.gated_ffn(*ts, activation=act)
    g = torch.autograd.grad(Y, ts, dY)
    with torch.no_grad():
        serving = amd.gated_ffn(X, Wg, Wu, Wd, activation=act)                   # the form that keeps nothing
    return dict(zip(("Y", "dX", "dWg", "dWu", "dWd", "serving"), (Y.detach(),) + g + (serving,)))


def check(got, out, err, dtype):
    out, err = dict(out, serving=out["Y"]), dict(err, serving=err["Y"])
    b = B8 if dtype == bf16 else E
    for k in out:
        assert got[k].shape == out[k].shape and got[k].dtype == dtype
        bound = 1.05 * err[k] + b * out[k].abs() + 1e-37
        worst = float(((got[k].double() - out[k]).abs() / bound).max()) if out[k].numel() else 0.0
        assert worst <= 1.0 and bool(torch.isfinite(got[k]).all()), "%s: %.3f of its bound" % (k, worst)


def real(seed, M, F, H, O, dtype):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [t.to(dtype).cuda() for t in (rn(M, F), rn(F, H) / math.sqrt(F), rn(F, H) / math.sqrt(F), rn(H, O) / math.sqrt(H), rn(M, O))]


def integers(seed, M, F, H, O, dtype):
    """Each row of X has up to five entries in {-2 .. 2}, dY up to three of +-1, the weights are +-1 and zeros: |G|, |U| <= 10,
    |dA| <= 3, so that A <= 100 and dG <= 30."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def sparse(rows, cols, per, hi):
        t = torch.zeros(rows, cols, device="cuda")
        if rows:
            at = torch.randint(0, cols, (rows, per), generator=g, device="cuda")
            t.scatter_(1, at, torch.randint(-hi, hi + 1, (rows, per), generator=g, device="cuda").float())
        return t
    w = lambda r, c: torch.randint(-1, 2, (r, c), generator=g, device="cuda").float()  # noqa: E731
    return [t.to(dtype) for t in (sparse(M, F, 5, 2), w(F, H), w(F, H), w(H, O), sparse(M, O, 3, 1))]


def check_exact(amd, args, dtype):
    got = run(amd, *args, "relu")
    out, _, inner = reference(*args, "relu", dtype)
    assert inner <= 256
    out["serving"] = out["Y"]
    for k in out:
        assert float(out[k].abs().max()) < 2 ** 24
        assert torch.equal(got[k], out[k].to(dtype)), k


# rows, F, H, F_out: one of everything, odd sizes, sizes around the tiles' edges, and (last) each of the kernel's tile shapes
SMALL = [(1, 1, 1, 1), (1, 64, 128, 64), (7, 75, 33, 12), (18, 64, 256, 64), (63, 65, 66, 67), (65, 8, 7, 9), (130, 200, 129, 257), (300, 128, 512, 128), (100, 36, 44, 28)]
LARGE = [(4608, 64, 256, 64), (4100, 257, 1000, 250), (8200, 1500, 4200, 1500), (5003, 1001, 2731, 1001), (1, 2048, 8192, 2048), (40000, 30, 50, 20), (128, 516, 2052, 260), (129, 1024, 2052, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", SMALL + LARGE)
def test_integers_come_out_exactly(amd, size, dtype):
    check_exact(amd, integers(sum(size), *size, dtype), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("size", SMALL + [(1030, 257, 300, 130)])
def test_matches_float64(amd, size, act, dtype):
    args = real(sum(size) + len(act), *size, dtype)
    out, err, _ = reference(*args, act, dtype)
    check(run(amd, *args, act), out, err, dtype)


@pytest.mark.gpu
def test_the_same_bits_again(amd):
    for dtype in (f32, bf16):
        args = real(3, 4608, 64, 256, 64, dtype)
        a, b = run(amd, *args, "gelu"), run(amd, *args, "gelu")
        for k in a:
            assert torch.equal(a[k], b[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_far_gates(amd, act):
    """Gates of 0 and of +-1, 90, 1e4, 1e30 and the smallest numbers: activations and slopes stay finite (bf16 and fp32).
    (Not dWu = sum x act(x): its true value, 1e60, is beyond fp32.)"""
    v = torch.tensor([0.0, 1.0, -1.0, 90.0, -90.0, 1e4, -1e4, 1e30, -1e30, 1e-40, -1e-40])
    for dtype in (f32, bf16):
        X = v.to(dtype).cuda()[:, None]
        one = torch.ones(1, 1, dtype=dtype, device="cuda")
        Wu = torch.zeros(1, 1, dtype=dtype, device="cuda")
        got = run(amd, X, one, Wu, one, torch.ones(11, 1, dtype=dtype, device="cuda"), act)
        for k in ("Y", "dX", "dWg", "dWd"):
            assert bool(torch.isfinite(got[k]).all()), k


@pytest.mark.gpu
def test_a_row_that_is_not_finite_stays_alone(amd):
    for dtype in (f32, bf16):
        X, Wg, Wu, Wd, _ = real(5, 200, 96, 64, 40, dtype)
        want = amd.gated_ffn(X, Wg, Wu, Wd)
        for bad in (float("nan"), float("inf")):
            Z = X.clone()
            Z[77, 5] = bad
            got = amd.gated_ffn(Z, Wg, Wu, Wd)
            keep = torch.arange(200, device="cuda") != 77
            assert torch.equal(got[keep], want[keep]) and not bool(torch.isfinite(got[77]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(70, 64, 96, 72), (70, 68, 100, 76), (1500, 68, 1100, 76)])
def test_strides_alignment_and_what_lies_around(amd, dtype, size):
    M, F, H, O = size
    X, Wg, Wu, Wd, dY = integers(11, M, F, H, O, dtype)
    out, _, _ = reference(X, Wg, Wu, Wd, dY, "relu", dtype)
    wide = torch.full((M, F + 9), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:1 + F] = X                                       # rows start at odd addresses, NaN between them
    buf = torch.full((F * H + 1,), float("nan"), dtype=dtype, device="cuda")
    wg = buf[1:].view(F, H)
    wg.copy_(Wg)                                               # an aligned partner (Wu) and a misaligned one
    ts = [wide[:, 1:1 + F].detach().requires_grad_(True), wg.detach().requires_grad_(True), Wu.t().contiguous().t().requires_grad_(True),
          Wd.clone().requires_grad_(True)]
    Y = amd.gated_ffn(*ts, activation="relu")
    grads = torch.autograd.grad(Y, ts, dY.t().contiguous().t())
    for g, k in zip((Y,) + grads, ("Y", "dX", "dWg", "dWu", "dWd")):
        assert torch.equal(g, out[k].to(dtype)), k
    ones = torch.autograd.grad(amd.gated_ffn(*ts, activation="relu").sum(), ts)          # an expanded gradient
    ref, _, _ = reference(X, Wg, Wu, Wd, torch.ones_like(dY), "relu", dtype)
    if dtype == f32:
        for g, k in zip(ones, ("dX", "dWg", "dWu", "dWd")):
            assert torch.equal(g, ref[k].to(dtype)), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_rows_of_zeros_and_no_rows(amd, dtype):
    X, Wg, Wu, Wd, dY = real(2, 40, 75, 60, 31, dtype)
    X[10:20] = 0
    Y = amd.gated_ffn(X, Wg, Wu, Wd, activation="sigmoid")
    assert torch.equal(Y[10:20], torch.zeros_like(Y[10:20]))
    got = run(amd, X[:0], Wg, Wu, Wd, dY[:0], "silu")
    assert got["Y"].shape == (0, 31) and got["dX"].shape == (0, 75)
    for k in ("dWg", "dWu", "dWd"):
        assert torch.equal(got[k], torch.zeros_like(got[k]))


@pytest.mark.gpu
def test_only_some_gradients(amd):
    X, Wg, Wu, Wd, dY = integers(9, 90, 40, 50, 30, f32)
    out, _, _ = reference(X, Wg, Wu, Wd, dY, "relu", f32)
    names = ("dX", "dWg", "dWu", "dWd")
    for pick in ((0,), (1,), (2,), (3,), (0, 3), (1, 2)):
        ts = [t.clone().requires_grad_(i in pick) for i, t in enumerate((X, Wg, Wu, Wd))]
        amd.gated_ffn(*ts, activation="relu").backward(dY)
        for i, t in enumerate(ts):
            assert (t.grad is None) if i not in pick else torch.equal(t.grad, out[names[i]].float())


@pytest.mark.gpu
def test_gradient_against_differences(amd):
    """Along a random direction of all inputs, central difference with t = 2^-6 in fp32.  Rounding: 320 outputs within 2e-6 of
    numbers of order 1, weighted by order 1, over 2 t: 36 * 2e-6 / 2^-5 = 2e-3; truncation: t^2 / 6 of a third derivative of
    order 100: 4e-3.  Bound 0.02 against a derivative of order 10."""
    X, Wg, Wu, Wd, dY = real(21, 20, 24, 40, 16, f32)
    got = run(amd, X, Wg, Wu, Wd, dY, "gelu")
    g = torch.Generator().manual_seed(4)
    v = [0.3 * torch.randn(t.shape, generator=g).cuda() for t in (X, Wg, Wu, Wd)]
    v[1:] = [x * 0.3 for x in v[1:]]
    want = sum(float((got[k].double() * d.double()).sum()) for k, d in zip(("dX", "dWg", "dWu", "dWd"), v))

    def loss(t):
        return float((amd.gated_ffn(*[a + t * d for a, d in zip((X, Wg, Wu, Wd), v)], activation="gelu").double() * dY.double()).sum())
    t = 2.0 ** -6
    assert abs((loss(t) - loss(-t)) / (2 * t) - want) <= 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_other_stream_and_replayed_graph(amd, dtype):
    size = (333, 75, 100, 64)
    args = integers(1, *size, dtype)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(amd, *args, "relu")
    torch.cuda.current_stream().wait_stream(s)
    out, _, _ = reference(*args, "relu", dtype)
    for k in out:
        assert torch.equal(got[k], out[k].to(dtype)), k
    del got
    ts = [t.clone().requires_grad_(True) for t in args[:4]]
    dY = args[4].clone()

    def step():
        Y = amd.gated_ffn(*ts, activation="relu")
        return (Y,) + torch.autograd.grad(Y, ts, dY)
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in range(3):
        fresh = integers(70 + seed, *size, dtype)
        with torch.no_grad():
            for t, v in zip(ts + [dY], fresh):
                t.copy_(v)
        graph.replay()
        out, _, _ = reference(*fresh, "relu", dtype)
        torch.cuda.synchronize()
        for r, k in zip(res, ("Y", "dX", "dWg", "dWu", "dWd")):
            assert torch.equal(r, out[k].to(dtype)), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(1, 600, 2100, 80), (3, 40, 64, 24), (500, 64, 1000, 60), (17000, 96, 160, 100), (90, 300, 200, 150)])
def test_replayed_serving_calls(amd, size, dtype):
    """Two calls in one graph, so that the second's scratch may lie where the first's was; replayed between eager calls."""
    a, b = integers(80, *size, dtype)[:4], integers(81, *size, dtype)[:4]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        amd.gated_ffn(*a, activation="relu")
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ya = amd.gated_ffn(*a, activation="relu")
        yb = amd.gated_ffn(*b, activation="relu")
    for seed in range(3):
        for args, off in ((a, 0), (b, 50)):
            for t, v in zip(args, integers(90 + seed + off, *size, dtype)):
                t.copy_(v)
        graph.replay()
        eager = amd.gated_ffn(*a, activation="relu")
        torch.cuda.synchronize()
        for args, y in ((a, ya), (b, yb), (a, eager)):
            X, Wg, Wu, Wd = (t.double() for t in args)
            assert torch.equal(y, (((X @ Wg).clamp(min=0) * (X @ Wu)) @ Wd).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(2300, 32, 40, 16), (2300, 200, 40, 16), (2300, 200, 3000, 160)])
def test_offsets_beyond_32_bits(amd, size, dtype):
    """rows 2^20 elements apart: the last ones lie more than 2^31 elements behind the first"""
    X, Wg, Wu, Wd, dY = real(9, *size, dtype)
    far = torch.empty((size[0], 1 << 20), dtype=dtype, device="cuda")[:, :size[1]]
    far.copy_(X)
    assert torch.equal(amd.gated_ffn(far, Wg, Wu, Wd), amd.gated_ffn(X, Wg, Wu, Wd))
    both = []
    for x in (far, X):
        ts = [t.detach().requires_grad_(True) for t in (x, Wg, Wu, Wd)]
        Y = amd.gated_ffn(*ts)
        both.append((Y,) + torch.autograd.grad(Y, ts, dY))
    for a, b in zip(*both):
        assert torch.equal(a, b)


# few rows have kernels of their own; the sizes cut k in parts in neither, one or both of their products, strips end inside a chunk
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(9, 5, 3), (64, 40, 24), (520, 4104, 1000), (1030, 2057, 90), (1100, 1500, 70)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5])
def test_few_rows(amd, rows, size, dtype):
    check_exact(amd, integers(rows + sum(size), rows, *size, dtype), dtype)
    args = real(rows * sum(size), rows, *size, dtype)
    out, err, _ = reference(*args, "silu", dtype)
    check(run(amd, *args, "silu"), out, err, dtype)


# features of at most 128 have a forward of their own that keeps nothing: both widths of it, rows and chunks of H that end inside a tile, H
# in one part and in several, odd numbers of chunks
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(5, 64, 32, 64), (70, 33, 97, 17), (1500, 64, 1000, 50), (20000, 16, 40, 64), (33, 8, 1, 1), (4200, 100, 520, 128), (17000, 65, 130, 9), (33000, 128, 70, 128), (2100, 7, 1100, 127)])
def test_narrow_features(amd, size, dtype):
    check_exact(amd, integers(sum(size), *size, dtype), dtype)
    args = real(sum(size) + 1, *size, dtype)
    for act in ("gelu", "sigmoid"):
        out, err, _ = reference(*args, act, dtype)
        check(run(amd, *args, act), out, err, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(700, 50, 330, 30), (17000, 90, 130, 70)])
def test_narrow_features_at_any_address(amd, size, dtype):
    rows, F, H, O = size
    X, Wg, Wu, Wd, _ = real(7, *size, dtype)
    want = amd.gated_ffn(X, Wg, Wu, Wd)
    wide = torch.full((rows + 1, F + 9), float("nan"), dtype=dtype, device="cuda")
    wide[:rows, 3:3 + F] = X
    moved = []
    for w in (Wg, Wu, Wd):
        flat = torch.full((w.numel() + 12,), float("nan"), dtype=dtype, device="cuda")
        flat[1:1 + w.numel()] = w.reshape(-1)
        moved.append(flat[1:1 + w.numel()].view(w.shape))
    assert torch.equal(amd.gated_ffn(wide[:rows, 3:3 + F], *moved), want)
    X[rows // 2] = float("nan")                               # a row is a row of its own
    got = amd.gated_ffn(X, Wg, Wu, Wd)
    keep = torch.arange(rows, device="cuda") != rows // 2
    assert torch.equal(got[keep], want[keep]) and bool(got[rows // 2].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("rows", [1, 3])
def test_few_rows_at_any_address(amd, rows, dtype):
    F, H, O = 75, 1101, 130
    X, Wg, Wu, Wd, dY = real(5, rows, F, H, O, dtype)
    want = amd.gated_ffn(X, Wg, Wu, Wd)
    wide = torch.full((rows, F + 9), float("nan"), dtype=dtype, device="cuda")          # what is around the operands is not read as one
    wide[:, 3:3 + F] = X
    moved = []
    for w in (Wg, Wu, Wd):
        flat = torch.full((w.numel() + 12,), float("nan"), dtype=dtype, device="cuda")
        flat[1:1 + w.numel()] = w.reshape(-1)
        moved.append(flat[1:1 + w.numel()].view(w.shape))
    assert torch.equal(amd.gated_ffn(wide[:, 3:3 + F], *moved), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_few_rows_do_not_touch_each_other(amd, dtype):
    X, Wg, Wu, Wd, _ = real(6, 3, 70, 2600, 90, dtype)
    want = amd.gated_ffn(X, Wg, Wu, Wd)
    X[1] = float("nan")
    got = amd.gated_ffn(X, Wg, Wu, Wd)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and bool(got[1].isnan().all())


# bf16 calls of up to 16384 elements of A keep it, dG and dU in two pieces (2^-16), P and Q in 24 bits (2^-16): b = 2^-15.  Their
# activations: the fit of the normal distribution is within 3e-5 < 2^-15 of its tail, exp2 within (1 + |g|) 2^-23: 2^-14.
@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("size", [(2, 40, 72, 24), (6, 40, 72, 24), (9, 33, 130, 50), (60, 100, 272, 64), (300, 20, 50, 30)])
def test_small_bf16_calls_round_their_results_alone(amd, size, act):
    args = real(sum(size), *size, bf16)
    out, err, _ = reference(*args, act, bf16, b=2.0 ** -15, act_err=2.0 ** -14)
    check(run(amd, *args, act), out, err, bf16)


@pytest.mark.gpu
def test_a_value_beyond_bf16_stays_infinite(amd):
    X = torch.full((6, 8), 2.0 ** 60, device="cuda", dtype=bf16)
    W = torch.full((8, 16), 2.0 ** 4, device="cuda", dtype=bf16)
    Y = amd.gated_ffn(X, W, W, torch.ones(16, 4, device="cuda", dtype=bf16), activation="relu")      # A = (2^67)^2 > 2^128
    assert bool((Y == float("inf")).all())


@pytest.mark.gpu
def test_a_second_derivative_is_refused(amd):
    ts = [t.requires_grad_(True) for t in real(1, 6, 8, 16, 8, f32)[:4]]
    (g,) = torch.autograd.grad(amd.gated_ffn(*ts).sum(), ts[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|twice|differentiat"):
        g.sum().backward()
    loss = amd.gated_ffn(*ts).sum()                           # ... nor dropped next to a loss that has a derivative
    (g,) = torch.autograd.grad(loss, ts[:1], create_graph=True)
    with pytest.raises(amd.AgcnError, match="differentiated again"):
        (loss + (g * g).sum()).backward()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 700])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_two_backward_passes_of_one_forward(amd, rows, dtype):
    X, Wg, Wu, Wd, dY = real(2, rows, 40, 72, 24, dtype)
    ts = [t.requires_grad_(True) for t in (X, Wg, Wu, Wd)]
    Y = amd.gated_ffn(*ts)
    first = torch.autograd.grad(Y, ts, dY, retain_graph=True)
    other = torch.autograd.grad(Y, ts, -2 * dY, retain_graph=True)
    again = torch.autograd.grad(Y, ts, dY)
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, c)
    fresh = torch.autograd.grad(amd.gated_ffn(*ts), ts, -2 * dY)
    for b, f in zip(other, fresh):                            # (not -2 x the first: the matrix instruction's sums need not be
        assert torch.equal(b, f)                              # rounded the same way for both signs)


def test_refusals(amd):
    lib = amd._ffi.lib()
    z = torch.zeros
    with pytest.raises(amd.AgcnError, match="GPU"):
        amd.gated_ffn(z(3, 4), z(4, 5), z(4, 5), z(5, 4))
    with pytest.raises(ValueError, match="activation"):
        amd.gated_ffn(z(3, 4), z(4, 5), z(4, 5), z(5, 4), activation="tanh")
    D = amd._ffi.FfnDesc
    ok = dict(rows=4, Fin=8, H=16, Fout=8, activation=4, dtype=0, ldx=8, training=1, reserved=0)
    mk = lambda **k: D(*[{**ok, **k}[f[0]] for f in D._fields_])  # noqa: E731
    for bad, text in ((mk(rows=-1), b"rows"), (mk(rows=1 << 31), b"rows"), (mk(Fin=0), b"1..65536"), (mk(H=65537), b"1..65536"), (mk(Fout=0), b"1..65536"),
                      (mk(dtype=2), b"f32 or bf16"), (mk(activation=0), b"activation"), (mk(activation=2), b"activation"), (mk(ldx=7), b"ldx")):
        assert lib.agcn_gated_ffn_reserve_bytes(C.byref(bad)) == 0 and text in lib.agcn_last_error()
        assert lib.agcn_gated_ffn_forward_workspace_bytes(C.byref(bad)) == 0 and lib.agcn_gated_ffn_backward_workspace_bytes(C.byref(bad)) == 0
    for rows in (0, 1):                                  # size queries answer for no rows as well
        e = mk(rows=rows)
        assert lib.agcn_gated_ffn_reserve_bytes(C.byref(e)) >= 256 and lib.agcn_gated_ffn_forward_workspace_bytes(C.byref(e)) >= 256
        assert lib.agcn_gated_ffn_backward_workspace_bytes(C.byref(e)) >= 256
    d, p, n = mk(), 4096, 1 << 30
    assert lib.agcn_gated_ffn_forward(C.byref(d), p, None, p, p, p, p, n, p, n, None) == -1
    assert lib.agcn_gated_ffn_forward(C.byref(d), p, p, p, p, p, p, 64, p, n, None) == -2 and b"reserve" in lib.agcn_last_error()
    assert lib.agcn_gated_ffn_forward(C.byref(d), p, p, p, p, p, p + 8, n, p, n, None) == -2
    assert lib.agcn_gated_ffn_backward(C.byref(d), p, p, p, p, p, p, p, p, p, p, n, p, 64, None) == -2 and b"workspace" in lib.agcn_last_error()
    assert lib.agcn_gated_ffn_backward(C.byref(mk(training=0)), p, p, p, p, p, p, p, p, p, p, n, p, n, None) == -1
    assert lib.agcn_gated_ffn_backward(C.byref(d), p, p, p, p, p, p, p, None, p, p, n, p, n, None) == -1 and b"together" in lib.agcn_last_error()


@pytest.mark.gpu
def test_refusals_of_tensors(amd):
    X, Wg, Wu, Wd, _ = real(1, 6, 8, 16, 8, f32)
    for bad, args in ((TypeError, (X.half(), Wg, Wu, Wd)), (TypeError, (X, Wg.bfloat16(), Wu, Wd)), (ValueError, (X[0], Wg, Wu, Wd)),
                      (ValueError, (X, Wg[:7], Wu, Wd)), (ValueError, (X, Wg, Wu[:, :9], Wd)), (ValueError, (X, Wg, Wu, Wd[:9])),
                      (amd.AgcnError, (X, Wg.cpu(), Wu, Wd))):
        with pytest.raises(bad):
            amd.gated_ffn(*args)


def _gate_values(act, g):
    """act(g), act'(g) and the terms that they are made of, float64"""
    if act == "sigmoid":
        s, ns = torch.sigmoid(g), torch.sigmoid(-g)
        return s, s * ns, s, s * ns
    if act == "silu":
        s, ns = torch.sigmoid(g), torch.sigmoid(-g)
        return g * s, s * (1 + g * ns), (g * s).abs(), s * (1 + g.abs() * ns)
    c = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    phi = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g * c, c + g * phi, (g * c).abs(), c + g.abs() * phi


# The gate alone: X = (v, 1), Wg picks v, Wu the one, so that G = v and U = 1 exactly, Y = act(v), dX = (act'(v), act(v)).
# fp32: 16 E of the terms; gelu's functions of g^2 / 2 and g / sqrt 2 move by g^2 times the roundings of their arguments (3 in all).
# bf16: e^-|g| from one rounded exponent, 2 |g| E; the fit of the normal distribution 2^-14 of its tail; the results 2^-8; with more
# than 16384 elements of A it, dG and dU are rounded too (2^-8).  Below 2^-126 numbers, or pieces of them (2^-9 and 2^-18 of the whole),
# may be flushed to zero: 2^-107 where the matrix pipe reads them.
@pytest.mark.gpu
@pytest.mark.parametrize("H,dtype", [(1, f32), (1, bf16), (64, f32), (64, bf16)])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_gates_by_value(amd, act, H, dtype):
    v = torch.cat((torch.linspace(-100, 100, 401), torch.linspace(-6, 6, 173), torch.tensor([0.0, -0.0, 1e-3, -1e-3, 1e-30, -1e-30]))).to(dtype)
    X = torch.stack((v, torch.ones_like(v)), 1).cuda()
    Wg, Wu, Wd = torch.zeros(2, H), torch.zeros(2, H), torch.zeros(H, 1)
    Wg[0], Wu[1], Wd[0] = 1, 1, 1
    Wg, Wu, Wd = (t.to(dtype).cuda() for t in (Wg, Wu, Wd))
    g = v.double()
    a, da, ta, tda = _gate_values(act, g)
    rel = 16 * E + (3 * g * g * E if act == "gelu" else 0)
    if dtype == bf16:
        rel = rel + 2 * g.abs() * E + 2.0 ** -14 + (2 if H > 1 else 1) * B8 * 1.01
    for rows in (len(v), 3):
        for at in range(0, len(v), rows):
            cut = slice(at, at + rows)
            x, dY = X[cut], torch.ones(len(X[cut]), 1, dtype=dtype, device="cuda")
            got = run(amd, x, Wg, Wu, Wd, dY, act)
            for o, want, terms in ((got["Y"][:, 0], a, ta), (got["serving"][:, 0], a, ta), (got["dX"][:, 0], da, tda), (got["dX"][:, 1], a, ta)):
                err = (o.double().cpu() - want[cut]).abs()
                bound = (rel[cut] if torch.is_tensor(rel) else rel) * terms[cut] + 2.0 ** -107
                assert bool((err <= bound).all()), (at, float((err / bound).max()))
            if rows == 3 and at > 60:
                break                                        # (the far ones; 20 calls)


def test_more_rows_than_a_launch_holds(amd):
    """2^32 threads and more: refused before anything is launched (both products in one kernel; as two; the backward)."""
    lib = amd._ffi.lib()
    p, n = 4096, (1 << 63) - 1
    for rows, F, H, O, dtype, training in ((1 << 30, 8, 8, 8, 1, 0), (1 << 30, 64, 32, 8, 0, 0), (1 << 30, 8, 8, 8, 1, 1),
                                           ((1 << 31) - 257, 1, 1, 1, 1, 1)):
        d = amd._ffi.FfnDesc(rows, F, H, O, 4, dtype, F, training, 0)
        assert lib.agcn_gated_ffn_forward(C.byref(d), p, p, p, p, p, p, n, p, n, None) == -1
        assert b"more than one launch holds" in lib.agcn_last_error()
        if training:
            assert lib.agcn_gated_ffn_backward(C.byref(d), p, p, p, p, p, p, p, p, p, p, n, p, n, None) == -1
            assert b"more than one launch holds" in lib.agcn_last_error()
