"""The operators as a network uses them: SGC_LL -> NodeNorm -> [GatedFeedForward -> NormBlockEnd] x 2 -> GraphGatherMol through
ResidualGraphMol, its loss's gradients into one bucket, clipped by their global norm, and a step on them.

Bounds: the float64 composition of the definitions starts from the SGC_LL layer's own fp32 output, so what is compared are five
layers of row operators.  Each is within 1e-6 of its result's scale for these widths (tests/test_gated_ffn.py,
tests/test_block_norm.py bound them term by term: sums of at most 80 terms, 88 E = 5e-6 of the sum of absolute values at the
worst), a norm divides by a deviation of order 1; five layers and the way back: 2e-5 of each tensor's largest element."""
import numpy as np
import pytest
import torch

import agcn_oracle as orc
from helpers import synth_case

DEV = "cuda:0"
F, H = 64, 80


@pytest.fixture(scope="module")
def amd():
    import agcn_amd
    if agcn_amd._build.is_stale():
        agcn_amd._build.build()
    return agcn_amd


def _batch(amd, ns=(9, 17, 5, 24, 12)):
    _, X, _, csr, _, _ = synth_case(71, list(ns), 75, 8, 2, orc.SGC_LL, atoms=True)
    return amd.GraphBatch.from_arrays(np.asarray(ns, np.int32), np.concatenate(X, 0), csr, DEV)


def _model(amd, B, norm="rms", act="silu"):
    g = lambda s: torch.Generator().manual_seed(s)  # noqa: E731
    m = amd.ResidualGraphMol(75, B, 24)
    m.add(amd.SGC_LL(F, 75, B, K=2, activation="relu", laplacian_mode="paper", device=DEV, generator=g(0)))
    m.add(amd.NodeNorm(F, norm=norm, device=DEV))
    for i in (1, 2):
        m.add(amd.GatedFeedForward(H, F, activation=act, device=DEV, generator=g(i)))
        m.add(amd.NormBlockEnd(i, F, norm=norm, gate_activation="sigmoid", scale=0.5, pre_norm=(i == 1), device=DEV))
    m.add(amd.GraphGatherMol(B, activation="tanh"))
    return m


def _norm64(v, w, b, kind):
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    o = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-6) * w
    return o if b is None else o + b


def _tail64(x, layers, gate, plan, kind, act):
    """the network behind its SGC_LL layer, in float64 on the CPU: (output, parameters)"""
    P = [{k: v.detach().double().cpu().requires_grad_(True) for k, v in l.vars.items()} for l in layers]
    gor = torch.as_tensor(np.repeat(np.arange(plan.B), plan.n))
    h = _norm64(x, P[0]["weight"], P[0].get("bias"), kind)
    for i in (1, 3):
        f, e = P[i], P[i + 1]
        gv = h @ f["w_gate"]
        a = gv * torch.sigmoid(gv) if act == "silu" else gv * 0.5 * torch.special.erfc(-gv / 2 ** 0.5)
        z = (a * (h @ f["w_up"])) @ f["w_down"]
        x = x + e["scale"] * (1.0 if gate is None else torch.sigmoid(gate)[gor]) * _norm64(z, e["post_weight"], e.get("post_bias"), kind)
        h = _norm64(x, e["pre_weight"], e.get("pre_bias"), kind) if "pre_weight" in e else x
    out = torch.zeros(plan.B, x.shape[1], dtype=torch.float64).index_add_(0, gor, h)
    return torch.tanh(out), P


def _close(got, want, what):
    scale = float(want.detach().abs().max())
    err = float((got.detach().double().cpu() - want.detach()).abs().max())
    assert err <= 2e-5 * max(scale, 1e-6), (what, err, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("norm,act,gated", [("rms", "silu", False), ("layer", "gelu", True), ("rms", "silu", True)])
def test_network_against_float64(amd, norm, act, gated):
    gb = _batch(amd)
    B = gb.plan.B
    model = _model(amd, B, norm, act)
    gate = torch.randn(B, F, generator=torch.Generator().manual_seed(5)).to(DEV).requires_grad_(True) if gated else None
    feed = gb
    if gated:
        feed = {"graph_batch": gb, "node_features": gb.X, "data_slice": None, "original_laplacian": None, "lap_slice": None, "gate": gate}
    out = model(feed)
    first, _, _ = model.layers[0]({"node_features": gb.X, "graph_batch": gb})
    tail = model.layers[1:-1]
    x64 = first.data.detach().double().cpu().requires_grad_(True)
    g64 = None if gate is None else gate.detach().double().cpu().requires_grad_(True)
    want, P = _tail64(x64, tail, g64, gb.plan, norm, act)
    _close(out, want, "output")
    up = torch.randn(B, F, generator=torch.Generator().manual_seed(6))
    (out * up.to(DEV)).sum().backward()
    (want * up.double()).sum().backward()
    for l, p in zip(tail, P):
        for k in p:
            _close(l.vars[k].grad, p[k].grad, type(l).__name__ + "." + k)
    if gated:
        _close(gate.grad, g64.grad, "gate")


@pytest.mark.gpu
def test_training_steps_with_a_clipped_bucket(amd):
    gb = _batch(amd)
    model = _model(amd, gb.plan.B)
    model(gb)
    params = [p for p in model.parameters() if p.requires_grad]
    bucket = amd.dist.GradBucket(params)
    for _ in range(3):
        bucket.zero()
        (model(gb) ** 2).sum().backward()
        before = bucket.flat.clone()
        norm = bucket.clip(0.25)
        n = float(before.double().norm())
        assert abs(float(norm) - n) <= 1e-6 * n and n > 0.25
        assert abs(float(bucket.flat.double().norm()) - 0.25) <= 1e-6
        assert all(p.grad.data_ptr() == v.data_ptr() for p, v in zip(bucket.params, bucket.views))
        with torch.no_grad():
            for p in params:
                p -= 0.01 * p.grad


@pytest.mark.gpu
def test_step_captures_into_one_graph(amd):
    gb = _batch(amd)
    model = _model(amd, gb.plan.B, "layer", "gelu")
    with torch.no_grad():                               # (builds the parameters; no graph of theirs outlives it)
        model(gb)
    params = [p for p in model.parameters() if p.requires_grad]
    bucket = amd.dist.GradBucket(params)

    def step():
        bucket.zero()
        (model(gb) ** 2).sum().backward()
        return bucket.clip(0.25)
    graphed = amd.GraphedStep(step, DEV)
    for scale in (1.0, 0.5, 2.0):
        with torch.no_grad():
            model.layers[2].vars["w_down"].mul_(scale)
        n = graphed.replay().clone()
        got = bucket.flat.clone()
        eager = step()
        torch.cuda.synchronize()
        assert float((got - bucket.flat).abs().max()) <= 1e-5 * float(bucket.flat.abs().max())
        assert abs(float(n) - float(eager)) <= 1e-5 * float(n)


@pytest.mark.gpu
def test_layers_in_bf16_and_from_the_padded_feed(amd):
    ns, stride = [4, 9, 5, 17], 20
    plan_rows = torch.randn(4, stride, F, generator=torch.Generator().manual_seed(1)).to(DEV)
    for b, n in enumerate(ns):
        plan_rows[b, n:] = 0
    feed = {"node_features": plan_rows, "data_slice": np.array([[n, -1] for n in ns]), "original_laplacian": None}
    lay = amd.GatedFeedForward(H, F, device=DEV, generator=torch.Generator().manual_seed(2))
    norm = amd.NodeNorm(F, device=DEV)
    lap = [torch.eye(stride, device=DEV) for _ in ns]
    feed["original_laplacian"] = lap
    out = lay(feed)
    assert len(out) == 4 and tuple(out[0].shape) == (stride, F)
    ref = amd.gated_ffn(plan_rows.reshape(-1, F), lay.vars["w_gate"], lay.vars["w_up"], lay.vars["w_down"])
    assert torch.equal(torch.stack(list(out)).reshape(-1, F), ref)            # pad rows of zeros give zeros
    h = norm(feed)
    assert all(bool((h[b][n:] == 0).all()) for b, n in enumerate(ns))
    # bf16: fp32 parameters widen the features, bf16 ones keep them
    X = torch.randn(35, F, generator=torch.Generator().manual_seed(3)).to(DEV).bfloat16()
    plan = amd.Plan(ns, device=DEV)
    gb = amd.GraphBatch(plan, X)
    y = lay({"node_features": X, "graph_batch": gb})
    assert y.data.dtype == torch.bfloat16 and torch.equal(y.data, amd.gated_ffn(X.float(), *lay.parameters()).bfloat16())
    low = amd.GatedFeedForward(H, F, dtype="bfloat16", device=DEV, generator=torch.Generator().manual_seed(2))
    y = low({"node_features": X, "graph_batch": gb})
    assert low.vars["w_gate"].dtype == torch.bfloat16 and torch.equal(y.data, amd.gated_ffn(X, *low.parameters()))
    with pytest.raises(TypeError):
        low({"node_features": X.float(), "graph_batch": gb})
    end = amd.NormBlockEnd(1, F, device=DEV)
    res, h = end({"node_features": y, "block_outputs": X.float(), "graph_batch": gb})
    assert res.data.dtype == torch.float32 and h.data.dtype == torch.bfloat16
    res, h = end({"node_features": y.data.float(), "block_outputs": X, "graph_batch": gb})
    assert res.data.dtype == torch.bfloat16 and h.data.dtype == torch.bfloat16


def test_views_of_a_padded_feed_end_with_the_last_graph(amd):
    """Iterating over the per-graph views stops after the last graph, whichever layout they are cut from."""
    class Feed(object):
        pad_stride = 4
    plan = amd.Plan([2, 3])
    views = amd.RowViews(torch.zeros(5, 2), plan, Feed())
    views._padded = torch.zeros(8, 2)
    assert len(list(views)) == 2 and len(list(amd.RowViews(torch.zeros(5, 2), plan))) == 2
    for bad in (2, -3):
        with pytest.raises(IndexError):
            views[bad]


def test_layer_contract(amd):
    with pytest.raises(ValueError):
        amd.GatedFeedForward(8, 4, activation="tanh")
    with pytest.raises(ValueError):
        amd.GatedFeedForward(8, 4, dtype="float16")
    with pytest.raises(ValueError):
        amd.NodeNorm(4, norm="batch")
    with pytest.raises(ValueError):
        amd.NormBlockEnd(1, 4, gate_activation="relu")
    lay = amd.NormBlockEnd(1, 4, norm="layer")
    assert [tuple(p.shape) for p in lay.parameters()] == [(4,)] * 5 and list(lay.vars) == ["scale", "post_weight", "post_bias", "pre_weight", "pre_bias"]
    with pytest.raises(ValueError):
        lay.load_vars({"scale": np.ones(4)})
    f = amd.GatedFeedForward(6, 4, 3)
    f.load_vars({"w_gate": np.zeros((4, 6)), "w_up": np.ones((4, 6)), "w_down": np.ones((6, 3))})
    with pytest.raises(ValueError):
        f.load_vars({"w_gate": np.zeros((4, 5)), "w_up": np.ones((4, 6)), "w_down": np.ones((6, 3))})
    with pytest.raises(amd.AgcnError):
        f({"node_features": torch.zeros(3, 4), "graph_batch": amd.GraphBatch(amd.Plan([3]), torch.zeros(3, 4))})
