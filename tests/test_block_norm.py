"""norm_gate_residual (csrc/block_norm.hip): y = x + s a(g) N(z), h = N'(y) and every gradient against the definition in
float64.

Bounds.  E = 2^-24 (half a step of fp32), B = 2^-8 (of bf16).  A row's statistics are sums of F terms added in at most 16 + 14
fp32 steps, the square root and the products add a handful of roundings: every fp32 chain below is within 64 E of the sum of
the absolute values of its terms.  A result stored in bf16 adds B of itself; nothing else is rounded to bf16 (the backward forms y again).  A column sum over n rows adds at most n E."""
import ctypes as C

import numpy as np
import pytest
import torch

E, B8 = 2.0 ** -24, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def amd():
    import agcn_amd
    if agcn_amd._build.is_stale():
        agcn_amd._build.build()
    return agcn_amd


def _norm64(v, w, b, kind, eps):
    if w is None:
        return v, v, torch.ones_like(v[:, :1])
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    o = c * r * w
    return (o if b is None else o + b), c * r, r


def _act64(name, g):
    if name == "tanh":
        return torch.tanh(g), 1 - torch.tanh(g) ** 2
    if name == "sigmoid":
        return torch.sigmoid(g), torch.sigmoid(g) * (1 - torch.sigmoid(g))
    return g, torch.ones_like(g)


def make(seed, rows, F, xt="f32", zt="f32", kind="rms", gate="none", ns=None, z=True, post=True, pre=True, scale=True, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = {"x": (rn(rows, F) * (1 + 10 * (torch.rand(F, generator=g) < 0.05).float())).to(DT[xt]), "dh": rn(rows, F).to(DT[zt])}
    if z:
        d["z"] = (0.7 * rn(rows, F) + 0.1).to(DT[zt])
        d["dy"] = rn(rows, F).to(DT[xt])
        if scale:
            d["scale"] = 0.5 + 0.2 * rn(F)
        if post:
            d["post_weight"] = 1 + 0.2 * rn(F)
            if kind == "layer":
                d["post_bias"] = 0.2 * rn(F)
        if gate == "row":
            d["gate"] = rn(rows, F).to(DT[zt])
        elif gate == "graph":
            d["gate"] = rn(len(ns), F).to(DT[zt])
    if pre:
        d["pre_weight"] = 1 + 0.2 * rn(F)
        if kind == "layer":
            d["pre_bias"] = 0.2 * rn(F)
    else:
        d.pop("dh")
    return {k: v.to(dev) for k, v in d.items()}


LEAVES = ("z", "x", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


def reference(d, kind, eps, act, graph_of_row=None):
    """Outputs, gradients and, for each, the sum of the absolute values of its terms (what its bound scales with): float64, CPU."""
    v = {k: t.double().cpu() for k, t in d.items()}
    z, x = v.get("z"), v["x"]
    out, mag = {}, {}
    F = x.shape[1]
    gor = None if graph_of_row is None else torch.as_tensor(graph_of_row)
    one = torch.ones(F, dtype=torch.float64)
    if z is not None:
        s = v.get("scale", one)
        w, b = v.get("post_weight"), v.get("post_bias")
        u, zh, rz = _norm64(z, w, b, kind, eps)
        w_, b_ = (one if w is None else w), (0 * one if b is None else b)
        if "gate" in v:
            a, da = _act64(act, v["gate"])
            if gor is not None:
                a, da = a[gor], da[gor]
        else:
            a, da = torch.ones_like(z), None
        y = x + s * a * u
        # |v - mean|'s terms: |v| + mean |v|
        zabs = z.abs() + (z.abs().mean(1, keepdim=True) if kind == "layer" and w is not None else 0)
        out["y"], mag["y"] = y, x.abs() + (s * a).abs() * (zabs * rz * w_.abs() + b_.abs())
    else:
        y = x
        mag["y"] = x.abs()
    if "pre_weight" in v:
        w2, b2 = v["pre_weight"], v.get("pre_bias")
        h, yh, ry = _norm64(y, w2, b2, kind, eps)
        # h moves with every y of its row: through its own element, and through the row's statistics
        spread = (mag["y"] * yh.abs()).mean(1, keepdim=True) * ry * yh.abs()
        spread = spread + (mag["y"].mean(1, keepdim=True) * ry if kind == "layer" else 0)
        out["h"], mag["h"] = h, ((mag["y"] * ry + spread) * w2.abs() + (0 if b2 is None else b2.abs()))
    # gradients
    D, Da = v.get("dy", torch.zeros_like(y)), v.get("dy", torch.zeros_like(y)).abs()
    if "dh" in v:
        e = v["dh"] * w2
        t = e - yh * (e * yh).mean(1, keepdim=True)
        ta = e.abs() + yh.abs() * (e * yh).abs().mean(1, keepdim=True) + (e.abs() * yh.abs()).mean(1, keepdim=True) * yh.abs()
        if kind == "layer":
            t = t - e.mean(1, keepdim=True)
            ta = ta + e.abs().mean(1, keepdim=True)
        # (yh itself is y's error magnified by r: |y|'s terms over |y|)
        ya = (mag["y"] * ry).clamp(min=1e-30)
        ta = ta + ya * (e * yh).mean(1, keepdim=True).abs() + yh.abs() * (e.abs() * ya).mean(1, keepdim=True)
        D, Da = D + t * ry, Da + ta * ry
        out["dpre_weight"], mag["dpre_weight"] = (v["dh"] * yh).sum(0), (v["dh"].abs() * (yh.abs() + ya)).sum(0)
        if b2 is not None:
            out["dpre_bias"], mag["dpre_bias"] = v["dh"].sum(0), v["dh"].abs().sum(0)
    out["dx"], mag["dx"] = D, Da
    if z is not None:
        za = zabs * rz
        ua = za * w_.abs() + b_.abs()
        if da is not None:
            dg, dga = D * s * u * da, Da * (s * da).abs() * ua
            if gor is not None:
                zero = torch.zeros_like(v["gate"])
                dg, dga = zero.clone().index_add_(0, gor, dg), zero.index_add_(0, gor, dga)
            out["dgate"], mag["dgate"] = dg, dga
        if "scale" in v:
            out["dscale"], mag["dscale"] = (D * a * u).sum(0), (Da * a.abs() * ua).sum(0)
        f, fa = D * s * a, Da * (s * a).abs()
        if w is not None:
            out["dpost_weight"], mag["dpost_weight"] = (f * zh).sum(0), (fa * za).sum(0)
            if b is not None:
                out["dpost_bias"], mag["dpost_bias"] = f.sum(0), fa.sum(0)
            f, fa = f * w, fa * w.abs()
            t = f - zh * (f * zh).mean(1, keepdim=True)
            ta = fa + za * (fa * za).mean(1, keepdim=True)
            if kind == "layer":
                t, ta = t - f.mean(1, keepdim=True), ta + fa.mean(1, keepdim=True)
            f, fa = t * rz, ta * rz
        out["dz"], mag["dz"] = f, fa
    return out, mag


def check(got, ref, mag, xt, zt, rows):
    for k, r in ref.items():
        g = got[k].detach().double().cpu()
        assert tuple(g.shape) == tuple(r.shape), k
        tol = 64 * E
        if k not in ("y", "h"):
            tol += 64 * E
        if k in ("dscale", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias") or (k == "dgate" and r.shape[0] != rows):
            tol += rows * E
        stored = {"y": xt, "dx": xt}.get(k, zt if k in ("h", "dz", "dgate") else "f32")
        bound = tol * mag[k] + (B8 if stored == "bf16" else E) * r.abs() + 1e-30
        worst = float(((g - r).abs() / bound).max()) if g.numel() else 0.0
        assert torch.isfinite(g).all() and worst <= 1.0, "%s: %.3f of its bound" % (k, worst)


def run(amd, d, kind, act, plan=None, eps=1e-6, use=("y", "h")):
    t = {k: (v.clone().requires_grad_(True) if k in LEAVES else v) for k, v in d.items()}
    y, h = amd.norm_gate_residual(t.get("z"), t["x"], post_weight=t.get("post_weight"), post_bias=t.get("post_bias"), gate=t.get("gate"),
                                  scale=t.get("scale"), pre_weight=t.get("pre_weight"), pre_bias=t.get("pre_bias"), norm=kind, eps=eps,
                                  gate_activation=act, plan=plan)
    outs, ups = [], []
    if y is not None and "y" in use:
        outs.append(y), ups.append(t["dy"])
    if h is not None and "h" in use:
        outs.append(h), ups.append(t["dh"])
    names = [k for k in LEAVES if k in t]
    grads = torch.autograd.grad(outs, [t[k] for k in names], ups, allow_unused=True)
    got = {"d" + k: g for k, g in zip(names, grads)}
    if y is not None:
        got["y"] = y
    if h is not None:
        got["h"] = h
    return got


SHAPES = [(1, 1), (3, 7), (18, 64), (5, 65), (33, 200), (17, 513), (70, 1001), (9, 1024), (4, 2050), (3, 4096), (5, 5001), (2, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,F", SHAPES)
@pytest.mark.parametrize("xt,zt", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("kind,gate,act", [("rms", "none", "linear"), ("layer", "row", "sigmoid")])
def test_norm_gate_residual_matches_float64(amd, rows, F, xt, zt, kind, gate, act):
    d = make(rows * 31 + F, rows, F, xt, zt, kind, gate)
    ref, mag = reference(d, kind, 1e-6, act)
    check(run(amd, d, kind, act), ref, mag, xt, zt, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["linear", "tanh", "sigmoid"])
@pytest.mark.parametrize("ns", [[1], [18, 5, 48, 1], [130, 7, 64, 65, 200], [3] * 300])
@pytest.mark.parametrize("kind,F", [("rms", 96), ("layer", 300), ("rms", 2049)])
def test_gate_per_graph(amd, act, ns, kind, F):
    plan = amd.Plan(ns, device="cuda")
    gor = np.repeat(np.arange(len(ns)), ns)
    d = make(len(ns) + F, sum(ns), F, "f32", "f32", kind, "graph", ns)
    ref, mag = reference(d, kind, 1e-6, act, gor)
    got = run(amd, d, kind, act, plan)
    check(got, ref, mag, "f32", "f32", sum(ns))
    again = run(amd, d, kind, act, plan)
    for k in got:                                   # fixed-order sums: the same bits
        assert torch.equal(got[k], again[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("opts", [dict(post=False), dict(scale=False), dict(post=False, scale=False), dict(pre=False), dict(z=False),
                                  dict(pre=False, scale=False)])
@pytest.mark.parametrize("kind,zt", [("rms", "f32"), ("layer", "bf16")])
def test_parts_left_out(amd, opts, kind, zt):
    d = make(5, 37, 129, zt, zt, kind, "none", **opts)
    ref, mag = reference(d, kind, 1e-6, "linear")
    check(run(amd, d, kind, "linear"), ref, mag, zt, zt, 37)


@pytest.mark.gpu
@pytest.mark.parametrize("use", [("y",), ("h",)])
def test_an_output_nobody_uses(amd, use):
    d = make(6, 21, 257, "f32", "f32", "layer", "row")
    got = run(amd, d, "layer", "tanh", use=use)
    d2 = dict(d)
    d2["dy" if use == ("h",) else "dh"] = torch.zeros_like(d["dy" if use == ("h",) else "dh"])
    ref, mag = reference(d2, "layer", 1e-6, "tanh")
    check(got, ref, mag, "f32", "f32", 21)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "row", "graph"])
def test_pad_rows_give_zeros_and_take_part_in_nothing(amd, gate):
    ns, stride, F = [4, 9, 1, 17, 20], 20, 70
    plan = amd.Plan(ns, stride, device="cuda")
    real = np.concatenate([np.arange(n) + b * stride for b, n in enumerate(ns)])
    rows = plan.rows
    d = make(9, rows, F, "f32", "f32", "layer", gate, ns)
    pad = np.setdiff1d(np.arange(rows), real)
    for k in ("x", "z", "dy", "dh") + (("gate",) if gate == "row" else ()):
        d[k][pad] = float("nan")
    got = run(amd, d, "layer", "sigmoid", plan)
    gor = np.repeat(np.arange(len(ns)), ns) if gate == "graph" else None
    dr = {k: (v[real] if k in ("x", "z", "dy", "dh") or (k == "gate" and gate == "row") else v) for k, v in d.items()}
    ref, mag = reference(dr, "layer", 1e-6, "sigmoid", gor)
    for k in ("y", "h", "dx", "dz") + (("dgate",) if gate == "row" else ()):
        assert torch.equal(got[k][pad], torch.zeros_like(got[k][pad])), k
        got[k] = got[k][real]
    check(got, ref, mag, "f32", "f32", len(real))


@pytest.mark.gpu
def test_strided_rows_and_odd_alignment(amd):
    rows, F = 41, 75
    for zt in ("f32", "bf16"):
        d = make(3, rows, F, zt, zt, "rms", "row")
        wide = {k: torch.full((rows, F + 6), 7.0, dtype=d[k].dtype, device="cuda") for k in ("x", "z", "gate")}
        for k in wide:
            wide[k][:, 3:3 + F] = d[k]
        ref, mag = reference(d, "rms", 1e-6, "tanh")
        view = {k: w[:, 3:3 + F] for k, w in wide.items()}
        t = {k: view.get(k, v).detach() for k, v in d.items()}
        y, h = amd.norm_gate_residual(t["z"], t["x"], post_weight=t["post_weight"], gate=t["gate"], scale=t["scale"],
                                      pre_weight=t["pre_weight"], gate_activation="tanh")
        check({"y": y, "h": h}, {k: ref[k] for k in ("y", "h")}, mag, zt, zt, rows)
        lv = {k: view[k].requires_grad_(True) for k in view}
        y, h = amd.norm_gate_residual(lv["z"], lv["x"], post_weight=t["post_weight"], gate=lv["gate"], scale=t["scale"],
                                      pre_weight=t["pre_weight"], gate_activation="tanh")
        g = torch.autograd.grad((y, h), [lv["z"], lv["x"], lv["gate"]], (d["dy"], d["dh"]))
        check(dict(zip(("dz", "dx", "dgate"), g)), {k: ref[k] for k in ("dz", "dx", "dgate")}, mag, zt, zt, rows)


@pytest.mark.gpu
def test_no_rows(amd):
    d = make(1, 0, 33, "f32", "bf16", "layer", "row")
    got = run(amd, d, "layer", "linear")
    assert got["y"].shape == (0, 33) and got["h"].dtype == torch.bfloat16
    for k in ("dscale", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias"):
        assert torch.equal(got[k], torch.zeros(33, device="cuda")), k


@pytest.mark.gpu
def test_zero_and_extreme_rows(amd):
    """A row of zeros has deviation sqrt(eps): finite everywhere.  A NaN stays in its row (and in the column sums)."""
    d = make(4, 6, 100, "f32", "f32", "layer", "none")
    d["x"][2] = 0
    d["z"][2] = 0
    d["z"][3] = 5.0                                     # no variance
    ref, mag = reference(d, "layer", 1e-6, "linear")
    got = run(amd, d, "layer", "linear")
    for k in ("y", "h", "dx", "dz"):
        assert torch.isfinite(got[k]).all()
    check({k: got[k][:3] if got[k].dim() == 2 else got[k] for k in ("y", "h")}, {k: ref[k][:3] for k in ("y", "h")},
          {k: mag[k][:3] for k in ("y", "h")}, "f32", "f32", 6)
    d["z"][4, 7] = float("nan")
    got2 = run(amd, d, "layer", "linear")
    keep = [0, 1, 2, 3, 5]
    for k in ("y", "h", "dx", "dz"):
        assert torch.equal(got2[k][keep], got[k][keep]) and torch.isnan(got2[k][4]).any()


@pytest.mark.gpu
def test_gradient_against_differences(amd):
    """d/dt of sum(y dy) + sum(h dh) along a random direction, by a central difference with t = 2^-7.  Its rounding: 1280 outputs,
    each within 64 E of terms that add up to about 5, weighted by numbers of order 1: 36 * 64 E * 5 = 7e-4 in each sum, 0.05
    after the division by 2 t.  Its truncation: t^2 / 6 of a third derivative of order 100: 1e-3.  Bound: 0.06 (the derivative
    itself is of order 30)."""
    d = make(8, 10, 64, "f32", "f32", "layer", "row")
    got = run(amd, d, "layer", "tanh")
    g = torch.Generator().manual_seed(1)
    names = [k for k in LEAVES if k in d]
    v = {k: torch.randn(d[k].shape, generator=g).cuda() * 0.3 for k in names}
    want = sum(float((got["d" + k].double() * v[k].double()).sum()) for k in names)

    def loss(t):
        e = {k: (x + t * v[k] if k in v else x) for k, x in d.items()}
        y, h = amd.norm_gate_residual(e["z"], e["x"], post_weight=e["post_weight"], post_bias=e["post_bias"], gate=e["gate"],
                                      scale=e["scale"], pre_weight=e["pre_weight"], pre_bias=e["pre_bias"], norm="layer", gate_activation="tanh")
        return float((y.double() * d["dy"].double()).sum() + (h.double() * d["dh"].double()).sum())
    t = 2.0 ** -7
    num = (loss(t) - loss(-t)) / (2 * t)
    assert abs(num - want) <= 0.06, (num, want)


@pytest.mark.gpu
def test_other_stream_and_replayed_graph(amd):
    d = make(12, 100, 192, "f32", "f32", "rms", "none")
    want = run(amd, d, "rms", "linear")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(amd, d, "rms", "linear")
    torch.cuda.current_stream().wait_stream(s)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    del got, want
    leaves = {k: (v.clone().requires_grad_(True) if k in LEAVES else v) for k, v in d.items()}
    names = [k for k in LEAVES if k in d]

    def step():
        y, h = amd.norm_gate_residual(leaves["z"], leaves["x"], post_weight=leaves["post_weight"], scale=leaves["scale"],
                                      pre_weight=leaves["pre_weight"])
        return (y, h) + torch.autograd.grad((y, h), [leaves[k] for k in names], (leaves["dy"], leaves["dh"]))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        fresh = make(50 + seed, 100, 192, "f32", "f32", "rms", "none")
        with torch.no_grad():
            for k in fresh:
                leaves[k].copy_(fresh[k])
        graph.replay()
        eager = run(amd, fresh, "rms", "linear")
        torch.cuda.synchronize()
        for o, k in zip(out, ["y", "h"] + ["d" + n for n in names]):
            assert torch.equal(o, eager[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("kind,gate", [("rms", "none"), ("layer", "row")])
def test_offsets_beyond_32_bits(amd, kind, gate):
    """more than 2^31 elements: the last rows' results are those of a call on the last rows alone"""
    rows, F, last = 132000, 16384, 7
    g = torch.Generator(device="cuda").manual_seed(1)
    t = {k: torch.randn(rows, F, generator=g, device="cuda", dtype=torch.bfloat16) for k in ("z", "x") + (("gate",) if gate == "row" else ())}
    v = {k: 1 + 0.1 * torch.randn(F, generator=g, device="cuda") for k in ("scale", "post_weight", "pre_weight")}
    if kind == "layer":
        v.update({k: 0.1 * torch.randn(F, generator=g, device="cuda") for k in ("post_bias", "pre_bias")})
    dy, dh = t["x"].flip(1), t["z"].flip(1)

    def call(cut):
        ts = {k: a[cut].detach().requires_grad_(True) for k, a in t.items()}
        out = amd.norm_gate_residual(**ts, **v, norm=kind, gate_activation="tanh" if gate == "row" else "linear")
        return out + torch.autograd.grad(out, list(ts.values()), (dy[cut], dh[cut]))
    for a, b in zip(call(slice(None)), call(slice(rows - last, rows))):
        assert torch.equal(a[rows - last:], b)


@pytest.mark.gpu
def test_a_second_derivative_is_refused(amd):
    d = make(30, 6, 32)
    x = d["x"].requires_grad_(True)
    y, h = amd.norm_gate_residual(d["z"], x, post_weight=d["post_weight"], pre_weight=d["pre_weight"])
    loss = y.sum() + h.sum()
    (g,) = torch.autograd.grad(loss, [x], create_graph=True)
    with pytest.raises(amd.AgcnError, match="differentiated again"):
        (loss + (g * g).sum()).backward()


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "row", "graph"])
def test_two_backward_passes_of_one_forward(amd, gate):
    ns = [18, 5, 48, 1]
    plan = amd.Plan(ns, device="cuda") if gate == "graph" else None
    d = make(31, sum(ns), 96, gate=gate, ns=ns)
    names = [k for k in ("z", "x", "gate", "scale", "post_weight", "pre_weight") if k in d]
    ts = [d[k].requires_grad_(True) for k in names]
    out = amd.norm_gate_residual(**{k: d[k] for k in names}, gate_activation="tanh", plan=plan)
    first = torch.autograd.grad(out, ts, (d["dy"], d["dh"]), retain_graph=True)
    other = torch.autograd.grad(out, ts, (-2 * d["dy"], -2 * d["dh"]), retain_graph=True)
    again = torch.autograd.grad(out, ts, (d["dy"], d["dh"]))
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, c)
        assert torch.equal(-2 * a, b)


def test_refusals(amd):
    """Before any launch: shapes, types, combinations (CPU; the C entries see addresses only)."""
    lib = amd._ffi.lib()
    with pytest.raises(amd.AgcnError, match="GPU"):
        amd.norm_gate_residual(None, torch.zeros(3, 4), pre_weight=torch.ones(4))
    with pytest.raises(ValueError, match="norm"):
        amd.norm_gate_residual(None, torch.zeros(3, 4), norm="batch")
    with pytest.raises(ValueError, match="gate_activation"):
        amd.norm_gate_residual(None, torch.zeros(3, 4), gate_activation="relu")
    p = 4096                                             # any address: no call below gets as far as a launch

    def fwd(desc, inputs, y=p, h=p, plan=None):
        return lib.agcn_norm_gate_residual_forward(C.byref(desc), plan, plan, C.byref(inputs), y, h, None, None)
    N, I = amd._ffi.NormDesc, amd._ffi.NormInputs
    good = I(p, p, None, None, p, None, p, None)
    ok = dict(rows=4, F=8, norm=0, gate=0, gate_activation=0, x_dtype=0, z_dtype=0, ldx=8, ldz=8, ldg=8, eps=1e-6)
    mk = lambda **k: N(*[{**ok, **k}[f[0]] for f in N._fields_])  # noqa: E731
    for bad, inputs, text in ((mk(F=0), good, b"F in 1"), (mk(F=16385), good, b"F in 1"), (mk(rows=-1), good, b"rows"),
                              (mk(norm=2), good, b"unknown norm"), (mk(eps=0.0), good, b"eps"), (mk(eps=float("nan")), good, b"eps"),
                              (mk(gate=3), good, b"unknown gate"), (mk(gate_activation=1), good, b"activation"),
                              (mk(x_dtype=1, z_dtype=0), good, b"types"), (mk(x_dtype=2), good, b"types"),
                              (mk(gate=2), I(p, p, p, None, p, None, p, None), b"needs a plan"),
                              (mk(gate=1), good, b"do not agree"), (mk(ldx=7), good, b"leading dimension"),
                              (mk(ldz=3), good, b"leading dimension"), (mk(), I(p, None, None, None, p, None, p, None), b"null"),
                              (mk(), I(p, p, None, None, p, p, p, None), b"no bias"),
                              (mk(norm=1), I(p, p, None, None, None, p, p, None), b"bias without"),
                              (mk(), I(None, p, None, p, None, None, p, None), b"need a block output"),
                              (mk(), I(None, p, None, None, None, None, None, None), b"nothing to compute")):
        assert fwd(bad, inputs) == -1 and text in lib.agcn_last_error(), (text, lib.agcn_last_error())
    assert fwd(mk(), good, y=None) == -1 and fwd(mk(), good, h=None) == -1
    plan = amd.Plan([3, 2])
    assert fwd(mk(), good, plan=plan.host_ptr) == -1 and b"the plan has 5" in lib.agcn_last_error()
    G = amd._ffi.NormGrads

    def bwd(desc, inputs, grads, ws=p, n=1 << 20, dy=p, dh=p):
        return lib.agcn_norm_gate_residual_backward(C.byref(desc), None, None, C.byref(inputs), p, dy, dh, C.byref(grads), ws, n, None)
    full = G(p, p, None, None, p, None, p, None)
    assert lib.agcn_norm_gate_residual_backward_workspace_bytes(C.byref(mk()), None) >= 4 * 4 * 8
    assert bwd(mk(), good, full, n=16) == -2 and b"workspace" in lib.agcn_last_error()
    assert bwd(mk(), good, G(None, p, None, None, p, None, p, None)) == -1
    assert bwd(mk(), good, G(p, p, p, None, p, None, p, None)) == -1 and b"do not agree" in lib.agcn_last_error()
    assert bwd(mk(), good, G(p, p, None, p, p, None, p, None)) == -1


@pytest.mark.gpu
def test_refusals_of_tensors(amd):
    x, z = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad, kw in ((TypeError, dict(z=z.half())), (TypeError, dict(x=x.bfloat16())), (ValueError, dict(z=z[:3])),
                    (ValueError, dict(z=z[:, :7])), (ValueError, dict(pre_weight=w[:7])), (TypeError, dict(pre_weight=w.bfloat16())),
                    (ValueError, dict(gate=z[:2])), (TypeError, dict(gate=z.bfloat16())), (ValueError, dict(z=None, gate=z)),
                    (ValueError, dict(plan=amd.Plan([3], device="cuda"))), (ValueError, dict(plan=amd.Plan([4]))),
                    (amd.AgcnError, dict(z=z.cpu())), (amd.AgcnError, dict(post_bias=w)), (amd.AgcnError, dict(z=None, pre_weight=None))):
        kw = {**dict(z=z, x=x, pre_weight=w), **kw}
        with pytest.raises((bad, ValueError) if bad is amd.AgcnError else bad):
            amd.norm_gate_residual(kw.pop("z"), kw.pop("x"), **kw)


def _skewed(big, small=20, count=4095):
    """one large graph among thousands of small ones"""
    return [small] * (count // 2) + [big] + [small] * (count - count // 2)


def test_workspace_grows_with_the_rows_and_the_graphs_not_with_their_product(amd):
    """A graph leaves one set of four sums per strip of its own rows (strips of eight rows or more at 256 features): at most
    rows / 8 + B of them."""
    lib = amd._ffi.lib()
    F = 256
    for ns in ([18] * 4096, _skewed(1024), _skewed(1600), [1600] * 3 + [1] * 30000, [1], [1600]):
        plan = amd.Plan(ns)
        d = amd._ffi.NormDesc(plan.rows, F, 0, 2, 2, 0, 0, F, F, F, 1e-6)
        got = lib.agcn_norm_gate_residual_backward_workspace_bytes(C.byref(d), plan.host_ptr)
        assert 0 < got <= (plan.rows // 8 + len(ns)) * 4 * F * 4 + 256, (len(ns), got)
    many = amd.Plan(np.ones(4300000, dtype=np.int32))        # 1024 threads each: more than the 2^32 threads of a launch
    d = amd._ffi.NormDesc(many.rows, 16384, 0, 2, 2, 0, 0, 16384, 16384, 16384, 1e-6)
    assert lib.agcn_norm_gate_residual_backward_workspace_bytes(C.byref(d), many.host_ptr) == 0
    assert b"graphs are more than one launch holds" in lib.agcn_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("F,kind,zt", [(64, "layer", "f32"), (300, "rms", "bf16"), (2050, "rms", "f32")])
@pytest.mark.parametrize("ns", [_skewed(1600, 3, 900), [1] * 5000 + [700], [700] + [1] * 70, [2, 1, 1] * 700 + [33, 64, 65] * 40])
def test_gate_per_graph_of_graphs_of_very_different_sizes(amd, ns, F, kind, zt):
    plan = amd.Plan(ns, device="cuda")
    gor = np.repeat(np.arange(len(ns)), ns)
    d = make(len(ns) + F, sum(ns), F, "f32", zt, kind, "graph", ns)
    ref, mag = reference(d, kind, 1e-6, "sigmoid", gor)
    check(run(amd, d, kind, "sigmoid", plan), ref, mag, "f32", zt, sum(ns))


@pytest.mark.gpu
@pytest.mark.parametrize("per_graph", [False, True])
@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
def test_gates_by_value(amd, act, per_graph):
    """The gate alone: x = 0, z = 1, no norms: y = a(g), dgate = a'(g) where the rows are alone in their graphs.  16 E of the value,
    far gates and small ones included.  An e^-2|g| (e^-|g|) below 2^-126 may be flushed, and tanh's slope is 4 e / (1 + e)^2: 2^-124."""
    g = torch.cat((torch.linspace(-100, 100, 401), torch.linspace(-6, 6, 173), torch.linspace(-0.3, 0.3, 121),
                   torch.tensor([0.0, 1e-3, -1e-3, 1e-20, -1e-20, 1e4, -1e4, 1e30, -1e30])))
    F = 8
    rows = -(-len(g) // F)
    gate = torch.cat((g, torch.zeros(rows * F - len(g)))).view(rows, F).cuda().requires_grad_(True)
    plan = amd.Plan([1] * rows, device="cuda") if per_graph else None
    x, z = torch.zeros(rows, F, device="cuda"), torch.ones(rows, F, device="cuda")
    y, _ = amd.norm_gate_residual(z, x, gate=gate, gate_activation=act, plan=plan)
    (dg,) = torch.autograd.grad(y, [gate], torch.ones_like(y))
    v = gate.detach().double().cpu()
    a = torch.tanh(v) if act == "tanh" else torch.sigmoid(v)
    s, ns = torch.sigmoid(2 * v if act == "tanh" else v), torch.sigmoid(-2 * v if act == "tanh" else -v)
    da = (4 if act == "tanh" else 1) * s * ns
    for got, want in ((y.detach(), a), (dg, da)):
        assert bool(((got.double().cpu() - want).abs() <= 16 * E * want.abs() + 2.0 ** -124).all())


@pytest.mark.gpu
@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("kind,F", [("rms", 96), ("layer", 300), ("rms", 2049)])
def test_gate_per_graph_in_bf16(amd, kind, F, xt):
    ns = [18, 5, 48, 1, 70]
    plan = amd.Plan(ns, device="cuda")
    d = make(F, sum(ns), F, xt, "bf16", kind, "graph", ns)
    ref, mag = reference(d, kind, 1e-6, "tanh", np.repeat(np.arange(len(ns)), ns))
    check(run(amd, d, kind, "tanh", plan), ref, mag, xt, "bf16", sum(ns))
