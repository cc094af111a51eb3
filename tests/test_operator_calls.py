"""What autograd may do with the calls of norm_gate_residual and gated_ffn between forward and backward: saved tensors that
come back at other addresses and in other layouts.  The CPU tests put a recorder in the library's place: it holds every pointer that a call hands over
against the tensor that lies there."""
import ctypes as C

import pytest
import torch

f32, bf16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def amd():
    import agcn_amd
    if agcn_amd._build.is_stale():
        agcn_amd._build.build()
    return agcn_amd


class Recorder(object):
    """Answers every entry with success and keeps the arguments; size queries ask the library itself (they need no GPU)."""

    def __init__(self, lib):
        self.lib, self.calls = lib, {}

    def __getattr__(self, name):
        if name.endswith("_bytes") or name == "agcn_last_error":
            return getattr(self.lib, name)

        def entry(*args):
            self.calls.setdefault(name, []).append([getattr(a, "_obj", a) for a in args])
            return 0
        return entry


@pytest.fixture
def recorder(amd, monkeypatch):
    rec = Recorder(amd._ffi.lib())
    f = amd.functional
    monkeypatch.setattr(amd._ffi, "lib", lambda: rec)
    monkeypatch.setattr(f, "_require_gpu", lambda t, what: None)
    monkeypatch.setattr(f, "_stream", lambda dev: 0)
    monkeypatch.setattr(f, "_on_device_of", lambda t, fn, *args: fn(*args))
    return rec


class Hook(object):
    """A pack / unpack pair; `back` makes what a saved tensor comes back as, and `seen` keeps it, by address."""

    def __init__(self, back):
        self.back, self.seen = back, {}

    def unpack(self, t):
        t = self.back(t)
        self.seen[t.data_ptr()] = t
        return t

    def __enter__(self):
        self.ctx = torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), self.unpack)
        self.ctx.__enter__()
        return self

    def __exit__(self, *exc):
        self.ctx.__exit__(*exc)


def odd(t):
    """the same values, one element behind an allocation's start"""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return flat[1:].view(t.shape).copy_(t)


def wider(t):
    """the same values with more room between the rows"""
    return t.new_empty(t.shape[0], t.shape[1] + 24)[:, :t.shape[1]].copy_(t) if t.dim() == 2 else t.clone()


def turned(t):
    """the same values, columns first"""
    return t.t().contiguous().t() if t.dim() == 2 else t.clone()


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


BACK = {"dense": dense, "odd": odd, "wider": wider, "turned": turned}


def cut(rows, cols, dtype, seed, device="cpu", at=64):
    """columns of a wider matrix"""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, 2 * at + cols, generator=g).to(device=device, dtype=dtype)[:, at:at + cols]


@pytest.mark.parametrize("back", sorted(BACK))
@pytest.mark.parametrize("xt,zt", [(f32, f32), (f32, bf16), (bf16, bf16)])
def test_norm_backward_reads_saved_tensors_as_they_come_back(amd, recorder, back, xt, zt):
    rows, F = 7, 64
    t = {"z": cut(rows, F, zt, 1), "x": cut(rows, F, xt, 2), "gate": cut(rows, F, zt, 3)}
    v = {k: torch.ones(F) for k in ("scale", "post_weight", "pre_weight")}
    leaves = [a.requires_grad_(True) for a in list(t.values()) + list(v.values())]
    with Hook(BACK[back]) as hook:
        y, h = amd.norm_gate_residual(**t, **v)
        torch.autograd.grad((y, h), leaves, (torch.ones_like(y), torch.ones_like(h)))
    (desc, _, _, inputs, stats, _, _, _, _, _, _), = recorder.calls["agcn_norm_gate_residual_backward"]
    for name, ld, dt in (("x", desc.ldx, xt), ("z", desc.ldz, zt), ("gate", desc.ldg, zt)):
        p = getattr(inputs, name)
        if p in hook.seen:                                   # read as it came back: with ITS leading dimension
            s = hook.seen[p]
            assert s.dtype is dt and s.stride() == (ld, 1), name
        else:                                                # or a copy of it
            assert ld == F, name
    forward = recorder.calls["agcn_norm_gate_residual_forward"][0][0]
    assert (forward.ldx, forward.ldz, forward.ldg) == (F + 128,) * 3


@pytest.mark.gpu
@pytest.mark.parametrize("back", sorted(BACK) + ["save_on_cpu"])
@pytest.mark.parametrize("xt,zt", [(f32, f32), (f32, bf16), (bf16, bf16)])
@pytest.mark.parametrize("gate", ["row", "graph"])
def test_norm_gradients_under_saved_tensor_hooks(amd, gate, back, xt, zt):
    ns, F = [18, 5, 48, 1], 64
    plan = amd.Plan(ns, device="cuda") if gate == "graph" else None
    rows = sum(ns)
    t = {"z": cut(rows, F, zt, 1, "cuda"), "x": cut(rows, F, xt, 2, "cuda"), "gate": cut(len(ns) if plan else rows, F, zt, 3, "cuda")}
    v = {k: 1 + 0.1 * cut(1, F, f32, 4 + i, "cuda")[0] for i, k in enumerate(("scale", "post_weight", "post_bias", "pre_weight", "pre_bias"))}
    leaves = [a.requires_grad_(True) for a in list(t.values()) + list(v.values())]

    def grads():
        y, h = amd.norm_gate_residual(**t, **v, norm="layer", gate_activation="tanh", plan=plan)
        return torch.autograd.grad((y, h), leaves, (cut(rows, F, xt, 8, "cuda"), cut(rows, F, zt, 9, "cuda")))
    want = grads()
    with torch.autograd.graph.save_on_cpu() if back == "save_on_cpu" else Hook(BACK[back]):
        got = grads()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_norm_refuses_a_saved_tensor_that_is_another(amd, recorder):
    for back in (lambda t: t[:1], lambda t: t.double()):
        x = cut(5, 16, f32, 1).requires_grad_(True)
        with Hook(back):
            y, h = amd.norm_gate_residual(cut(5, 16, f32, 2), x, pre_weight=torch.ones(16))
            with pytest.raises((TypeError, ValueError), match="saved"):
                (y.sum() + h.sum()).backward()
    assert "agcn_norm_gate_residual_backward" not in recorder.calls


@pytest.mark.parametrize("back", sorted(BACK))
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_ffn_backward_reads_saved_tensors_as_they_come_back(amd, recorder, back, dtype):
    """Features of whole 16-byte chunks: the forward reads such bf16 matrices in place, so the backward must find them so."""
    rows, F, H, O = 50, 64, 96, 72
    ts = [cut(rows, F, dtype, 1)] + [cut(a, b, dtype, 2 + i, at=0) for i, (a, b) in enumerate(((F, H), (F, H), (H, O)))]
    ts = [t.requires_grad_(True) for t in ts]
    with Hook(BACK[back]) as hook:
        Y = amd.gated_ffn(*ts)
        torch.autograd.grad(Y, ts, torch.ones_like(Y))
    (desc, X, Wg, Wu, Wd, *_), = recorder.calls["agcn_gated_ffn_backward"]
    (forward, *_), = recorder.calls["agcn_gated_ffn_forward"]
    assert forward.ldx == F + 128
    for name, p, cols, ld in (("X", X, F, desc.ldx), ("Wg", Wg, H, H), ("Wu", Wu, H, H), ("Wd", Wd, O, O)):
        if p in hook.seen:
            assert hook.seen[p].stride() == (ld, 1), name
        else:
            assert ld == cols, name
        assert dtype == f32 or (p % 16 == 0 and ld % 8 == 0), name


@pytest.mark.parametrize("back", [lambda t: t[:1], lambda t: t.double()])
def test_ffn_refuses_a_saved_tensor_that_is_another(amd, recorder, back):
    X = cut(5, 16, f32, 1).requires_grad_(True)
    with Hook(back):
        Y = amd.gated_ffn(X, torch.ones(16, 8), torch.ones(16, 8), torch.ones(8, 4))
        with pytest.raises(ValueError, match="saved"):
            Y.sum().backward()
    assert "agcn_gated_ffn_backward" not in recorder.calls


# (rows, H): few rows; A in two pieces; one piece / planes of fp32 pieces.  72: whole chunks of 16 bytes, 75: an image in the forward
@pytest.mark.gpu
@pytest.mark.parametrize("back", sorted(BACK) + ["save_on_cpu"])
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("size", [(3, 72, 96, 40), (50, 72, 96, 40), (50, 75, 96, 41), (700, 200, 3000, 160), (700, 203, 3001, 161)])
def test_ffn_gradients_under_saved_tensor_hooks(amd, size, back, dtype):
    rows, F, H, O = size
    ts = [cut(rows, F, dtype, 1, "cuda")] + [cut(a, b, dtype, 2 + i, "cuda", 0) / a ** 0.5 for i, (a, b) in enumerate(((F, H), (F, H), (H, O)))]
    ts = [t.requires_grad_(True) for t in ts]
    dY = cut(rows, O, dtype, 7, "cuda", 0)
    want = torch.autograd.grad(amd.gated_ffn(*ts), ts, dY)
    with torch.autograd.graph.save_on_cpu() if back == "save_on_cpu" else Hook(BACK[back]):
        got = torch.autograd.grad(amd.gated_ffn(*ts), ts, dY)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_ffn_gradients_when_some_weights_move(amd):
    """Both projections are read in place or neither is: one that comes back at an odd address beside one that stayed, and an odd
    one that comes back aligned."""
    rows, F, H, O = 300, 72, 96, 40
    X, dY = cut(rows, F, bf16, 1, "cuda"), cut(rows, O, bf16, 7, "cuda", 0)
    W = [cut(a, b, bf16, 2 + i, "cuda", 0) / a ** 0.5 for i, (a, b) in enumerate(((F, H), (F, H), (H, O)))]
    for start in (0, 1, 2, 4, 7):
        ts = [X] + [odd(w) if start >> i & 1 else w for i, w in enumerate(W)]
        ts = [t.detach().requires_grad_(True) for t in ts]
        want = torch.autograd.grad(amd.gated_ffn(*ts), ts, dY)
        for moved in range(8):
            turn = iter(range(-1, 8))

            def back(t):
                i = next(turn)                               # saved in the order X, w_gate, w_up, w_down, reserve
                return t if not 0 <= i < 3 or not moved >> i & 1 else (dense(t) if t.data_ptr() & 15 else odd(t))
            with Hook(back):
                got = torch.autograd.grad(amd.gated_ffn(*ts), ts, dY)
            for a, b in zip(want, got):
                assert torch.equal(a, b), (start, moved)


def _operators(amd):
    """name -> (call of a list of tensors, the tensors)"""
    vec = torch.ones(8)
    return {"norm": (lambda ts: amd.norm_gate_residual(ts[0], ts[1], gate=ts[2], post_weight=ts[3], pre_weight=vec),
                     [cut(4, 8, f32, i) for i in range(3)] + [torch.ones(8)]),
            "ffn": (lambda ts: amd.gated_ffn(*ts), [cut(4, 8, f32, 1), torch.ones(8, 6), torch.ones(8, 6), torch.ones(6, 3)])}


@pytest.mark.parametrize("op", ["norm", "ffn"])
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("mode", ["plain", "no_grad", "requires_grad", "jvp"])
def test_forward_mode_is_refused(amd, recorder, op, which, mode):
    """A tangent has no way through the kernels: dropped in silence it would be a derivative of zero."""
    call, ts = _operators(amd)[op]
    with pytest.raises(amd.AgcnError, match="forward-mode"):
        if mode == "jvp":
            torch.func.jvp(lambda t: call(ts[:which] + [t] + ts[which + 1:]), (ts[which],), (torch.ones_like(ts[which]),))
        else:
            with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
                if mode == "requires_grad":
                    ts = [t.requires_grad_(True) for t in ts]
                ts[which] = torch.autograd.forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
                call(ts)
    assert not recorder.calls


@pytest.mark.parametrize("op", ["norm", "ffn"])
def test_calls_without_a_tangent_run_in_a_forward_mode_level(amd, recorder, op):
    call, ts = _operators(amd)[op]
    with torch.autograd.forward_ad.dual_level():
        call(ts)
    assert len(recorder.calls) == 1


@pytest.mark.parametrize("op", ["norm", "ffn"])
@pytest.mark.parametrize("create_graph", [False, True])
def test_a_tangent_of_the_upstream_gradient_is_refused(amd, recorder, op, create_graph):
    call, ts = _operators(amd)[op]
    ts = [t.requires_grad_(True) for t in ts]
    out = call(ts)
    out = out[0] if isinstance(out, tuple) else out
    with torch.autograd.forward_ad.dual_level():
        up = torch.autograd.forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(amd.AgcnError, match="forward-mode"):
            torch.autograd.grad(out, ts, up, create_graph=create_graph)
    assert len(recorder.calls) == 1


# (tensors without memory: the recorder reads nothing)
def far(rows, cols, ld, dtype=f32):
    return torch.empty_strided((rows, cols), (ld, 1), dtype=dtype, device="meta")


@pytest.mark.parametrize("ld", [1 << 20, (1 << 20) + 8, (1 << 31) - 1, 1 << 31, (1 << 32) + 128])
@pytest.mark.parametrize("grad", [False, True])
def test_leading_dimensions_reach_the_library_whole(amd, recorder, ld, grad):
    """The descriptors hold 32 bits, and gated_ffn takes up to 2^20: rows farther apart are copied together first."""
    F = 64
    t = {k: far(3, F, ld).requires_grad_(grad) for k in ("x", "z", "gate")}
    out = amd.norm_gate_residual(**t, pre_weight=torch.ones(F, device="meta"))
    X = far(3, F, ld).requires_grad_(grad)
    W = [torch.ones(s, device="meta") for s in ((F, 32), (F, 32), (32, 8))]
    Y = amd.gated_ffn(X, *W)
    if grad:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
            out = amd.norm_gate_residual(**t, pre_weight=torch.ones(F, device="meta"))
            Y = amd.gated_ffn(X, *W)
        torch.autograd.grad(out, list(t.values()), [torch.ones_like(o) for o in out])
        torch.autograd.grad(Y, X, torch.ones_like(Y))
    for name, calls in recorder.calls.items():
        for desc, *_ in calls:
            if "ffn" in name:
                assert desc.ldx == (ld if ld <= 1 << 20 else F), name
            else:
                assert (desc.ldx, desc.ldz, desc.ldg) == ((ld if ld < 1 << 31 else F),) * 3, name
    assert len(recorder.calls) == (4 if grad else 2)


def test_sizes_beyond_32_bits_are_refused(amd, monkeypatch):
    """... and not taken for what their lower halves say."""
    f = amd.functional
    monkeypatch.setattr(f, "_require_gpu", lambda t, what: None)
    monkeypatch.setattr(f, "_stream", lambda dev: 0)
    monkeypatch.setattr(f, "_on_device_of", lambda t, fn, *args: fn(*args))
    n = (1 << 32) + 64
    x = far(2, n, n)
    with pytest.raises(amd.AgcnError, match="F in 1..16384"):
        amd.norm_gate_residual(None, x, pre_weight=torch.empty(n, device="meta"))
    for F, H, O in ((n, 8, 8), (8, n, 8), (8, 8, n)):
        with pytest.raises(amd.AgcnError, match="1..65536"):
            amd.gated_ffn(far(2, F, F), far(F, H, H), far(F, H, H), far(H, O, O))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_rows_farther_apart_than_the_descriptors_hold(amd, dtype):
    ld, F = (1 << 31) + 64, 40
    buf = torch.empty(2 * ld + F, dtype=dtype, device="cuda")
    x = buf.as_strided((3, F), (ld, 1))
    near = cut(3, F, dtype, 1, "cuda")
    x.copy_(near)
    w = torch.ones(F, device="cuda")
    W = [cut(a, b, dtype, 2 + i, "cuda", 0) for i, (a, b) in enumerate(((F, 32), (F, 32), (32, 8)))]
    for a, b in zip(amd.norm_gate_residual(x, x, gate=x, pre_weight=w), amd.norm_gate_residual(near, near, gate=near, pre_weight=w)):
        assert torch.equal(a, b)
    assert torch.equal(amd.gated_ffn(x, *W), amd.gated_ffn(near, *W))


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_a_block_that_is_computed_again_in_the_backward(amd, dtype, reentrant):
    """Checkpointing: the backward reads what a second forward kept, at other addresses."""
    from torch.utils.checkpoint import checkpoint
    rows, F, H = 90, 72, 96
    X = cut(rows, F, dtype, 1, "cuda").requires_grad_(True)
    W = [(cut(a, b, dtype, 2 + i, "cuda", 0) / a ** 0.5).requires_grad_(True) for i, (a, b) in enumerate(((F, H), (F, H), (H, 3 * F)))]
    v = [(1 + 0.1 * cut(1, F, f32, 6 + i, "cuda")[0]).requires_grad_(True) for i in range(3)]

    def block(x, *p):
        wide = amd.gated_ffn(x, *p[:3])                      # z, gate: columns of one wide product
        return amd.norm_gate_residual(wide[:, :F], x, gate=wide[:, 2 * F:], scale=p[3], post_weight=p[4], pre_weight=p[5], gate_activation="sigmoid")
    ts = [X] + W + v
    up = cut(rows, F, dtype, 9, "cuda"), cut(rows, F, dtype, 10, "cuda")

    def grads(out):
        for t in ts:
            t.grad = None
        torch.autograd.backward(out, up)
        return [t.grad for t in ts]
    want = grads(block(*ts))
    for a, b in zip(want, grads(checkpoint(block, *ts, use_reentrant=reentrant))):
        assert torch.equal(a, b)
