"""What is measured of the row operators around the graph-convolution layers: the gated feed-forward block, the norms with
gate and residual scale around a block, and the clipping of a network's gradients by their global norm.

`run` makes ONE pass: in plain torch operations in 32 bits where `own` is false, through this package's entry points where
it is true.  `exact` states the same from the definitions in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one node (or token) through a wide block while serving: the weights have to stream in once, nothing else counts
        {"name": "ffn_single_row", "op": "ffn", "train": False, "rows": 1, "F": 2048, "H": 8192, "t": "bf16", "act": "silu"},
        # the benchmark's batch of 256 molecules (about 18 atoms each) behind a 64-filter layer: launch latency counts
        {"name": "ffn_molecules_train", "op": "ffn", "train": True, "rows": 4608, "F": 64, "H": 256, "t": "f32", "act": "gelu"},
        # 32 point clouds of 1024 points behind a 128-filter layer, prediction
        {"name": "ffn_clouds", "op": "ffn", "train": False, "rows": 32768, "F": 128, "H": 512, "t": "f32", "act": "silu"},
        # sizes that nothing divides: every row starts at another alignment
        {"name": "ffn_ragged_train", "op": "ffn", "train": True, "rows": 5003, "F": 1001, "H": 2731, "t": "bf16", "act": "gelu"},
        # a training step of a wide block: the matrix pipe
        {"name": "ffn_wide_train", "op": "ffn", "train": True, "rows": 8192, "F": 2048, "H": 8192, "t": "bf16", "act": "silu"},
        # the frame of a block for one molecule while serving: latency
        {"name": "norm_molecule", "op": "norm", "train": False, "graphs": 1, "nodes": 18, "F": 64, "x": "f32", "z": "f32",
         "kind": "rms", "gate": "none", "gate_act": "linear"},
        # 256 molecules, each with a gate vector of its own (a condition of the graph), training
        {"name": "norm_molecules_train", "op": "norm", "train": True, "graphs": 256, "nodes": 18, "F": 256, "x": "f32",
         "z": "f32", "kind": "layer", "gate": "graph", "gate_act": "tanh"},
        # fp32 residual rows around bf16 blocks, a gate for every element, odd width
        {"name": "norm_ragged_train", "op": "norm", "train": True, "graphs": 53, "nodes": 377, "F": 1001, "x": "f32",
         "z": "bf16", "kind": "rms", "gate": "row", "gate_act": "sigmoid"},
        # a training step's rows of a wide network: memory bandwidth
        {"name": "norm_wide_train", "op": "norm", "train": True, "graphs": 32, "nodes": 1024, "F": 4096, "x": "bf16",
         "z": "bf16", "kind": "rms", "gate": "none", "gate_act": "linear"},
        # the gradients of the reference's four-layer molecule network with its dense layer and 12 heads: latency
        {"name": "clip_network", "op": "clip", "tensors": 31, "scale": 4542, "types": "f32", "clip": 0.5},
        # many tensors of odd sizes and both types, below the limit (nothing to clip)
        {"name": "clip_ragged", "op": "clip", "tensors": 331, "scale": 50021, "types": "mixed", "clip": 1e6},
        # the gradients of a wide network in bf16: memory bandwidth
        {"name": "clip_wide", "op": "clip", "tensors": 96, "scale": 6000000, "types": "bf16", "clip": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "norm", "clip"])
    if op == "ffn":
        while True:
            c = {"op": op, "train": rng.random() < 0.5, "rows": _log(rng, 1, 32768), "F": _log(rng, 16, 2048),
                 "H": _log(rng, 32, 8192), "act": rng.choice(["silu", "gelu", "sigmoid"])}
            c["t"] = rng.choice(["f32", "bf16"])
            if rng.random() < 0.5:                       # widths of half of the cases are multiples of 8
                c["F"], c["H"] = max(8, c["F"] // 8 * 8), max(8, c["H"] // 8 * 8)
            # products in fp32 cost several times what they cost in bf16
            if work(c)["flops"] * (6 if c["t"] == "f32" else 1) <= work(listed()[4])["flops"]:
                return c
    if op == "norm":
        while True:
            c = {"op": op, "train": rng.random() < 0.7, "graphs": _log(rng, 1, 400), "nodes": _log(rng, 1, 1024),
                 "F": _log(rng, 8, 4096), "kind": rng.choice(["rms", "layer"]), "gate": rng.choice(["none", "row", "graph"])}
            c["x"], c["z"] = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
            c["gate_act"] = rng.choice(["linear", "tanh", "sigmoid"]) if c["gate"] != "none" else "linear"
            if work(c)["bytes"] <= work(listed()[8])["bytes"]:
                return c
    while True:
        c = {"op": op, "tensors": _log(rng, 1, 400), "scale": _log(rng, 100, 1000000),
             "types": rng.choice(["f32", "bf16", "mixed"]), "clip": rng.choice([0.01, 1.0, 1e6])}
        if work(c)["bytes"] <= work(listed()[11])["bytes"]:
            return c


def _nodes(case):
    """Node counts of the graphs: `nodes` on the average, between half and one and a half of it."""
    g, n = case["graphs"], case["nodes"]
    return [max(1, n // 2 + (i * 7919 + 13 * i * i) % (n + 1)) if g > 1 else n for i in range(g)]


def _sizes(case):
    """Element counts of the gradient tensors: matrices and small vectors in turn, around `scale` on the average."""
    out = []
    for i in range(case["tensors"]):
        out.append(max(1, case["scale"] * (1 + (i * 37) % 11) // 4) if i % 3 != 2 else 1 + (i * 61) % 257)
    return out


def _types(case):
    n = case["tensors"]
    if case["types"] == "mixed":
        return ["f32" if i % 2 else "bf16" for i in range(n)]
    return [case["types"]] * n


def work(case):
    if case["op"] == "ffn":
        M, F, H = case["rows"], case["F"], case["H"]
        size = 4 if case["t"] == "f32" else 2
        if case["train"]:
            return {"bytes": (4 * M * F + 6 * F * H) * size, "flops": 18 * M * F * H}
        return {"bytes": (2 * M * F + 3 * F * H) * size, "flops": 6 * M * F * H}
    if case["op"] == "norm":
        n = _nodes(case)
        M, F = sum(n), case["F"]
        xs, zs = (4 if case["x"] == "f32" else 2), (4 if case["z"] == "f32" else 2)
        gate = {"none": 0, "row": M * F * zs, "graph": len(n) * F * zs}[case["gate"]]
        one = M * F * (2 * xs + 2 * zs) + gate          # z, x, gate in; y, h out
        if case["train"]:                               # ... dy, dh in; dx, dz, dgate out
            return {"bytes": 2 * one, "flops": 40 * M * F}
        return {"bytes": one, "flops": 12 * M * F}
    b = sum(s * (4 if t == "f32" else 2) for s, t in zip(_sizes(case), _types(case)))
    return {"bytes": 2 * b, "flops": 3 * sum(_sizes(case))}


# ---------------------------------------------------------------- inputs

def _inputs(case, seed):
    """The inputs from the seed alone, on the GPU."""
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * (seed + 1) + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    def uniform(r, *shape):
        return (torch.rand(*shape, generator=g, device=DEV, dtype=torch.float32) * 2 - 1) * r

    if case["op"] == "ffn":
        M, F, H = case["rows"], case["F"], case["H"]
        t = DT[case["t"]]
        r = math.sqrt(6.0 / (F + H))                    # glorot, as the package's layers draw their weights
        s = {"X": normal(M, F).to(t), "Wg": uniform(r, F, H).to(t), "Wu": uniform(r, F, H).to(t), "Wd": uniform(r, H, F).to(t)}
        if case["train"]:
            s["dY"] = normal(M, F).to(t)
        return s
    if case["op"] == "norm":
        n = _nodes(case)
        M, F = sum(n), case["F"]
        xt, zt = DT[case["x"]], DT[case["z"]]
        # residual rows carry a few channels that are far larger than the rest
        loud = 1.0 + 20.0 * (torch.rand(F, generator=g, device=DEV) < 0.02).float()
        s = {"x": (normal(M, F) * loud).to(xt), "z": (0.5 * normal(M, F)).to(zt),
             "w_post": 1.0 + 0.2 * normal(F), "w_pre": 1.0 + 0.2 * normal(F), "scale": 0.3 + 0.1 * normal(F)}
        if case["kind"] == "layer":
            s["b_post"], s["b_pre"] = 0.1 * normal(F), 0.1 * normal(F)
        if case["gate"] == "row":
            s["gate"] = normal(M, F).to(zt)
        elif case["gate"] == "graph":
            s["gate"] = normal(len(n), F).to(zt)
        if case["train"]:
            s["dy"], s["dh"] = normal(M, F).to(xt), normal(M, F).to(zt)
        return s
    ts = []
    for i, (size, t) in enumerate(zip(_sizes(case), _types(case))):
        mag = 10.0 ** (-4 + (i * 5) % 4)                # gradients of different layers differ by orders of magnitude
        ts.append((normal(size) * mag).to(DT[t]))
    return {"grads": ts}


def _flat(case, tensors):
    """One buffer for each type, the tensors of that type one after the other (what a bucket of gradients is)."""
    groups = {k: [t.reshape(-1) for t, k2 in zip(tensors, _types(case)) if k2 == k] for k in DT}
    return {k: torch.cat(g) for k, g in groups.items() if g}


_LEAVES = {"ffn": ("X", "Wg", "Wu", "Wd"), "norm": ("z", "x", "w_post", "b_post", "gate", "scale", "w_pre", "b_pre")}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "norm":
        n = _nodes(case)
        s["graph_of_row"] = torch.repeat_interleave(torch.arange(len(n), device=DEV), torch.tensor(n, device=DEV))
        if own:                                         # the batch's plan, which a program keeps beside the batch
            import agcn_amd
            s["plan"] = agcn_amd.Plan(n, device=DEV)
    if case["op"] == "clip":                            # the clipped gradients' buffers are the program's own
        s["flat"] = _flat(case, [torch.zeros_like(t) for t in s["grads"]])
        at, s["out"] = {k: 0 for k in DT}, []
        for t, k in zip(s["grads"], _types(case)):
            s["out"].append(s["flat"][k][at[k]:at[k] + t.numel()])
            at[k] += t.numel()
    if case.get("train"):
        for k in _LEAVES[case["op"]]:
            if k in s:
                s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if own:
        return {"ffn": _own_ffn, "norm": _own_norm, "clip": _own_clip}[case["op"]](state, case)
    with torch.no_grad():
        return {"ffn": _plain_ffn, "norm": _plain_norm, "clip": _plain_clip}[case["op"]](state, case)


def _own_ffn(s, case):
    import agcn_amd
    if not case["train"]:
        return {"Y": agcn_amd.gated_ffn(s["X"], s["Wg"], s["Wu"], s["Wd"], activation=case["act"])}
    Y = agcn_amd.gated_ffn(s["X"], s["Wg"], s["Wu"], s["Wd"], activation=case["act"])
    dX, dWg, dWu, dWd = torch.autograd.grad(Y, (s["X"], s["Wg"], s["Wu"], s["Wd"]), s["dY"])
    return {"Y": Y.detach(), "dX": dX, "dWg": dWg, "dWu": dWu, "dWd": dWd}


def _own_norm(s, case):
    import agcn_amd
    y, h = agcn_amd.norm_gate_residual(s["z"], s["x"], post_weight=s["w_post"], post_bias=s.get("b_post"), gate=s.get("gate"),
                                       scale=s["scale"], pre_weight=s["w_pre"], pre_bias=s.get("b_pre"), norm=case["kind"],
                                       eps=1e-6, gate_activation=case["gate_act"], plan=s["plan"])
    if not case["train"]:
        return {"y": y, "h": h}
    names = [k for k in _LEAVES["norm"] if k in s]
    grads = torch.autograd.grad((y, h), [s[k] for k in names], (s["dy"], s["dh"]))
    out = {"y": y.detach(), "h": h.detach()}
    out.update({"d" + k: v for k, v in zip(names, grads)})
    return out


def _own_clip(s, case):
    import agcn_amd
    _, norm = agcn_amd.clip_by_global_norm(s["grads"], case["clip"], out=s["out"])
    return {"norm": norm, **s["flat"]}


def _act(name, g):
    """activation and its derivative"""
    sig = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return sig, sig * (1.0 - sig)
    if name == "silu":
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_ffn(s, case):
    X, Wg, Wu, Wd = s["X"].float(), s["Wg"].float(), s["Wu"].float(), s["Wd"].float()
    G, U = X @ Wg, X @ Wu
    a, da = _act(case["act"], G)
    A = a * U
    t = s["X"].dtype
    out = {"Y": (A @ Wd).to(t)}
    if case["train"]:
        dY = s["dY"].float()
        dA = dY @ Wd.t()
        dG, dU = dA * U * da, dA * a
        out.update({"dX": (dG @ Wg.t() + dU @ Wu.t()).to(t), "dWg": (X.t() @ dG).to(t), "dWu": (X.t() @ dU).to(t),
                    "dWd": (A.t() @ dY).to(t)})
    return out


def _norm_fwd(kind, v, eps):
    """normalised rows and 1 / deviation"""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    return v * r, r


def _norm_bwd(kind, g, hat, r):
    """gradient of the rows from the gradient of the normalised rows"""
    t = g - hat * (g * hat).mean(1, keepdim=True)
    if kind == "layer":
        t = t - g.mean(1, keepdim=True)
    return t * r


def _gate(name, g):
    if name == "tanh":
        t = torch.tanh(g)
        return t, 1.0 - t * t
    if name == "sigmoid":
        t = 1.0 / (1.0 + torch.exp(-g))
        return t, t * (1.0 - t)
    return g, torch.ones_like(g)


def _plain_norm(s, case):
    kind, eps = case["kind"], 1e-6
    z, x = s["z"].float(), s["x"].float()
    zhat, rz = _norm_fwd(kind, z, eps)
    u = zhat * s["w_post"]
    if "b_post" in s:
        u = u + s["b_post"]
    if "gate" in s:
        a, da = _gate(case["gate_act"], s["gate"].float())
        if case["gate"] == "graph":
            a, da = a[s["graph_of_row"]], da[s["graph_of_row"]]
        y = x + s["scale"] * a * u
    else:
        a, da = None, None
        y = x + s["scale"] * u
    yhat, ry = _norm_fwd(kind, y, eps)
    h = yhat * s["w_pre"]
    if "b_pre" in s:
        h = h + s["b_pre"]
    out = {"y": y.to(s["x"].dtype), "h": h.to(s["z"].dtype)}
    if not case["train"]:
        return out
    dh = s["dh"].float()
    D = s["dy"].float() + _norm_bwd(kind, dh * s["w_pre"], yhat, ry)
    Da = D if a is None else D * a
    du = Da * s["scale"]
    out["dz"] = _norm_bwd(kind, du * s["w_post"], zhat, rz).to(s["z"].dtype)
    out["dx"] = D.to(s["x"].dtype)
    out["dw_post"] = (du * zhat).sum(0)
    if "b_post" in s:
        out["db_post"] = du.sum(0)
    if a is not None:
        dg = D * s["scale"] * u * da
        if case["gate"] == "graph":
            dg = torch.zeros(s["gate"].shape, dtype=torch.float32, device=dg.device).index_add_(0, s["graph_of_row"], dg)
        out["dgate"] = dg.to(s["gate"].dtype)
    out["dscale"] = (Da * u).sum(0)
    out["dw_pre"] = (dh * yhat).sum(0)
    if "b_pre" in s:
        out["db_pre"] = dh.sum(0)
    return out


def _plain_clip(s, case):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for t in s["grads"]:
        f = t.float()
        total = total + (f * f).sum().double()
    norm = torch.sqrt(total).float()
    scale = case["clip"] / torch.clamp(norm, min=case["clip"])
    scale = torch.where(torch.isfinite(norm), scale, torch.full_like(scale, float("nan")))
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * scale)
    return {"norm": norm, **s["flat"]}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "clip":
        g = [t.double() for t in s["grads"]]
        n = math.sqrt(math.fsum(float(torch.dot(t, t)) for t in g))
        k = 1.0 if n <= case["clip"] else case["clip"] / n
        return {"norm": torch.tensor(n, dtype=torch.float64, device=DEV), **_flat(case, [t * k for t in g])}
    if case["op"] == "ffn":
        leaves = [s[k].double().requires_grad_(case["train"]) for k in ("X", "Wg", "Wu", "Wd")]
        X, Wg, Wu, Wd = leaves
        g = torch.mm(X, Wg)
        gated = {"silu": lambda t: t * torch.sigmoid(t), "sigmoid": torch.sigmoid,
                 "gelu": lambda t: t * 0.5 * torch.special.erfc(-t / math.sqrt(2.0))}[case["act"]](g)
        Y = torch.mm(gated * torch.mm(X, Wu), Wd)
        out = {"Y": Y.detach()}
        if case["train"]:
            out.update(zip(("dX", "dWg", "dWu", "dWd"), torch.autograd.grad(Y, leaves, s["dY"].double())))
        return out
    names = [k for k in _LEAVES["norm"] if k in s]
    v = {k: s[k].double().requires_grad_(case["train"]) for k in names}

    def norm(t, w, b):
        c = t - t.mean(1, keepdim=True) if case["kind"] == "layer" else t
        o = w * c * torch.rsqrt(c.pow(2).sum(1, keepdim=True) / t.shape[1] + 1e-6)
        return o if b is None else o + b

    u = v["scale"] * norm(v["z"], v["w_post"], v.get("b_post"))
    if "gate" in v:
        a = {"linear": lambda t: t, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[case["gate_act"]](v["gate"])
        if case["gate"] == "graph":
            a = torch.cat([a[i:i + 1].expand(k, -1) for i, k in enumerate(_nodes(case))])
        u = a * u
    y = v["x"] + u
    h = norm(y, v["w_pre"], v.get("b_pre"))
    out = {"y": y.detach(), "h": h.detach()}
    if case["train"]:
        grads = torch.autograd.grad((y, h), [v[k] for k in names], (s["dy"].double(), s["dh"].double()))
        out.update({"d" + k: t for k, t in zip(names, grads)})
    return out
