"""global_norm / clip_by_global_norm / GradBucket.clip (csrc/clip.hip) against float64.

Bounds: the squares are exact in 64 bits and added there, so the norm is within one fp32 rounding (and 2^-40 of it for the
64-bit sums); the factor is one fp32 rounding of a 64-bit quotient, the product another, the stored value a last one."""
import ctypes as C

import numpy as np
import pytest
import torch

E, B8 = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def amd():
    import agcn_amd
    if agcn_amd._build.is_stale():
        agcn_amd._build.build()
    return agcn_amd


def tensors(seed, sizes, types, mag=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=g) * mag * 10.0 ** (i % 5 - 2)).to(t).cuda()
            for i, (s, t) in enumerate(zip(sizes, types))]


def norm64(ts):
    return float(np.sqrt(sum(float((t.double().cpu() ** 2).sum()) for t in ts)))


def check(ts, out, norm, clip):
    n = norm64(ts)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - n) <= 2 * E * n
    k = min(1.0, clip / n) if n else 1.0
    for t, o in zip(ts, out):
        want = t.double().cpu() * k
        bound = (2 * E + (B8 if t.dtype == torch.bfloat16 else E)) * want.abs() + 1e-45
        if k == 1.0:
            assert torch.equal(o, t)
        assert o.shape == t.shape and o.dtype == t.dtype and bool(((o.double().cpu() - want).abs() <= bound).all())


f32, bf16 = torch.float32, torch.bfloat16
LISTS = [([1], [f32]), ([1], [bf16]), ([7, (3, 5)], [bf16, f32]), ([0, 5, 0], [f32, bf16, bf16]), ([1023, 1024, 1025, 4096, 4097], [f32] * 5),
         ([2047, 2048, 2049, 8191], [bf16] * 4), ([(64, 75), 64, (75, 75), 1, (128, 256)], [f32] * 5), ([3000001], [bf16]), ([2000003, 17], [f32, bf16]),
         ([3 + (i * 37) % 900 for i in range(300)], [f32 if i % 3 else bf16 for i in range(300)]),
         ([40000 + i for i in range(250)], [bf16 if i % 2 else f32 for i in range(250)])]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(LISTS)))
@pytest.mark.parametrize("clip", [0.37, 1e9, float("inf")])
def test_clip_matches_float64(amd, case, clip):
    ts = tensors(case, *LISTS[case])
    keep = [t.clone() for t in ts]
    out, norm = amd.clip_by_global_norm(ts, clip)
    check(keep, out, norm, clip)
    assert all(torch.equal(a, b) for a, b in zip(ts, keep))              # the inputs stay
    again, norm2 = amd.clip_by_global_norm(ts, clip)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(out, again))
    assert torch.equal(amd.global_norm(ts), norm)
    res, norm3 = amd.clip_by_global_norm(ts, clip, out=ts)               # in place
    assert all(a is b for a, b in zip(res, ts)) and torch.equal(norm3, norm)
    assert all(torch.equal(a, b) for a, b in zip(ts, out))


@pytest.mark.gpu
def test_unaligned_views_and_what_lies_around_them(amd):
    for t in (f32, bf16):
        flat = torch.randn(10000, device="cuda").to(t)
        dst = torch.full((10000,), 3.0, device="cuda", dtype=t)
        spans = [(1, 18), (19, 20), (21, 4121), (4123, 9997)]
        ts, os_ = [flat[a:b] for a, b in spans], [dst[a:b] for a, b in spans]
        out, norm = amd.clip_by_global_norm(ts, 0.5, out=os_)
        check(ts, out, norm, 0.5)
        outside = torch.ones(10000, dtype=torch.bool)
        for a, b in spans:
            outside[a:b] = False
        assert bool((dst.cpu()[outside] == 3.0).all())


@pytest.mark.gpu
def test_sizes_of_values(amd):
    """Squares that leave fp32's range at either end, exact zeros."""
    for mag in (1e30, 1e-30):
        ts = [torch.full((1000,), mag, device="cuda"), torch.full((3,), -mag, device="cuda")]
        out, norm = amd.clip_by_global_norm(ts, 1e-3 * mag)
        check(ts, out, norm, 1e-3 * mag)
    z = [torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda", dtype=bf16)]
    out, norm = amd.clip_by_global_norm(z, 1.0)
    assert float(norm) == 0.0 and all(torch.equal(a, b) for a, b in zip(z, out))
    empty = [torch.empty(0, device="cuda")]
    out, norm = amd.clip_by_global_norm(empty, 1.0)
    assert float(norm) == 0.0 and out[0].numel() == 0 and float(amd.global_norm(empty)) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n", [100, 6000000])
def test_a_norm_that_is_not_finite(amd, bad, n):
    ts = [torch.ones(n, device="cuda"), torch.ones(9, device="cuda", dtype=bf16)]
    ts[0][n // 2] = bad
    out, norm = amd.clip_by_global_norm(ts, 1.0)
    assert not bool(torch.isfinite(norm)) and all(bool(torch.isnan(o).all()) for o in out)


@pytest.mark.gpu
def test_none_entries_strides_and_bucket(amd):
    ts = tensors(1, [(40, 30), 17], [f32, f32])
    out, norm = amd.clip_by_global_norm([None, ts[0], None, ts[1]], 0.1)
    assert out[0] is None and out[2] is None
    check(ts, [out[1], out[3]], norm, 0.1)
    tr = ts[0].t()
    out, norm = amd.clip_by_global_norm([tr], 0.1)
    check([tr], out, norm, 0.1)
    ps = [torch.nn.Parameter(torch.randn(75, 64, device="cuda")), torch.nn.Parameter(torch.randn(64, device="cuda"))]
    bucket = amd.dist.GradBucket(ps)
    ((ps[0] ** 2).sum() + (ps[1] * 3).sum()).backward()
    before = [p.grad.clone() for p in ps]
    norm = bucket.clip(2.0)
    check(before, [p.grad for p in ps], norm, 2.0)


@pytest.mark.gpu
def test_a_tensor_of_more_than_2_to_the_31_elements(amd):
    n = (1 << 31) + 1003
    t = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    t[-5:] = 3.0
    norm64_ = float(np.sqrt((n - 5) + 45.0))
    (out,), norm = amd.clip_by_global_norm([t], norm64_ / 2)
    assert abs(float(norm) - norm64_) <= 2 * E * norm64_
    assert bool((out[:-5] == 0.5).all()) and bool((out[-5:] == 1.5).all())      # (k = 0.5 within 2 E: a bf16 rounds to the same)


@pytest.mark.gpu
def test_clip_in_a_replayed_graph_and_on_another_stream(amd):
    ts = tensors(2, [5000, 3, 70001], [f32, bf16, f32])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out, norm = amd.clip_by_global_norm(ts, 0.3)
    torch.cuda.current_stream().wait_stream(s)
    check(ts, out, norm, 0.3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, norm = amd.clip_by_global_norm(ts, 0.3)
    for i in range(3):
        fresh = tensors(20 + i, [5000, 3, 70001], [f32, bf16, f32], mag=10.0 ** -i)
        for a, b in zip(ts, fresh):
            a.copy_(b)
        graph.replay()
        eager, n2 = amd.clip_by_global_norm(fresh, 0.3)
        torch.cuda.synchronize()
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_an_overwritten_tensor_is_seen_as_such(amd):
    w = torch.ones(5, device="cuda", requires_grad=True)
    v = torch.full((5,), 3.0, device="cuda")
    y = (w * v).sum()
    amd.clip_by_global_norm([v], 1.0, out=[v])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_refusals(amd):
    lib = amd._ffi.lib()
    with pytest.raises(amd.AgcnError, match="GPU"):
        amd.clip_by_global_norm([torch.ones(3)], 1.0)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="positive"):
            amd.clip_by_global_norm([torch.ones(3)], bad)
    for none in ([], [None]):
        with pytest.raises(ValueError, match="no tensors"):
            amd.clip_by_global_norm(none, 1.0)
        with pytest.raises(ValueError, match="no tensors"):
            amd.global_norm(none)

    def call(ins, outs, numel, dtype, clip=1.0, ws=4096, wn=1 << 20, norm=4096):
        n = len(ins)
        P, L, D = (C.c_void_p * n)(*ins), (C.c_int64 * n)(*numel), (C.c_int32 * n)(*dtype)
        O = None if outs is None else (C.c_void_p * n)(*outs)
        return lib.agcn_clip_by_global_norm(n, P, O, L, D, clip, norm, ws, wn, None)
    A, B = 1 << 20, 1 << 21                               # addresses that no call below reaches
    for rc, text, args in ((-1, b"positive", ([A], [B], [4], [0], 0.0)), (-1, b"bad tensor table", ([A], [B], [-1], [0])),
                           (-1, b"bad tensor table", ([A], [B], [4], [2])), (-1, b"is null", ([A], [None], [4], [0])),
                           (-1, b"not aligned", ([A + 2], [B], [4], [0])), (-1, b"not aligned", ([A], [B + 1], [4], [1])),
                           (-1, b"overlap", ([A, A + 64], [B, B + 12], [4, 4], [0, 0])),
                           (-1, b"overlap", ([A, A], [A, A], [4, 4], [0, 0])),
                           (-1, b"overlaps output", ([A], [A + 4], [4], [0])),
                           (-1, b"overlaps output", ([A, A + 4], [A, B], [4, 4], [0, 0])),
                           (-2, b"workspace", ([A], [B], [4], [0], 1.0, 4096, 8)), (-2, b"workspace", ([A], [B], [4], [0], 1.0, None, 4096)),
                           (-1, b"null table", ([A], [B], [4], [0], 1.0, 4096, 4096, None))):
        assert call(*args) == rc and text in lib.agcn_last_error(), (text, lib.agcn_last_error())
    assert lib.agcn_clip_workspace_bytes(0, None, None) == 0


@pytest.mark.gpu
def test_refusals_of_tensors(amd):
    a = torch.ones(4, 4, device="cuda")
    with pytest.raises(TypeError):
        amd.clip_by_global_norm([a.half()], 1.0)
    for out in ([], [a[:2]], [a.bfloat16()], [a.t()], [None], [torch.ones(4, 4)]):
        with pytest.raises(ValueError):
            amd.clip_by_global_norm([a], 1.0, out=out)
    with pytest.raises(amd.AgcnError, match="overlap"):
        amd.clip_by_global_norm([a, a], 1.0, out=[a, a])
    with pytest.raises(ValueError):
        amd.clip_by_global_norm([a, torch.ones(3)], 1.0)


def _calls(amd, ts, out):
    yield lambda: amd.global_norm(ts)
    yield lambda: amd.clip_by_global_norm(ts, 1.0)
    yield lambda: amd.clip_by_global_norm(ts, 1.0, out=ts)
    yield lambda: amd.clip_by_global_norm(ts, 1.0, out=out)


def test_a_derivative_is_refused_not_lost(amd):
    """Gradients that are themselves differentiable (create_graph=True), parameters, tangents: the results would carry no graph."""
    a, b = torch.ones(4, requires_grad=True), torch.ones(4)
    (g,) = torch.autograd.grad((a ** 3).sum(), [a], create_graph=True)
    for first, ts, out in ((0, [b, g], [b, b]), (0, [a], [b]), (0, [None, a], [None, b]), (3, [b], [a])):
        for call in list(_calls(amd, ts, out))[first:]:     # (the last: its input asks for nothing, its output does)
            with pytest.raises(amd.AgcnError, match="no_grad"):
                call()
            with torch.no_grad(), pytest.raises(amd.AgcnError, match="GPU"):
                call()                                      # (as far as the device check)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        d = torch.autograd.forward_ad.make_dual(b, b)
        for call in _calls(amd, [b, d], [b, b]):
            with pytest.raises(amd.AgcnError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_clip_of_differentiable_gradients_without_a_graph(amd):
    p = torch.nn.Parameter(torch.randn(500, device="cuda"))
    (p ** 3).sum().backward(create_graph=True)
    keep = [p.grad.detach().clone()]
    with pytest.raises(amd.AgcnError, match="no_grad"):
        amd.clip_by_global_norm([p.grad], 0.5)
    with torch.no_grad():
        out, norm = amd.clip_by_global_norm([p.grad], 0.5)
    check(keep, out, norm, 0.5)
    assert not out[0].requires_grad and not norm.requires_grad
    p.grad = None                                           # (its graph holds p: a cycle)


@pytest.mark.gpu
@pytest.mark.parametrize("n,t", [(100, f32), (100, bf16), (3000001, f32), (3000001, bf16)])
def test_a_norm_beyond_fp32_is_one_that_is_not_finite(amd, n, t):
    """Finite gradients whose norm no fp32 holds: the norm that is handed back is infinite, and the results agree with it.  Just
    below, both are numbers."""
    big = torch.finfo(t).max
    below = [torch.zeros(n, device="cuda", dtype=t), torch.zeros(4, device="cuda", dtype=t)]
    below[0][n // 2] = big / 2                              # norm = the largest number of the type
    below[1][:3] = big / 2
    out, norm = amd.clip_by_global_norm(below, 1.0)
    check(below, out, norm, 1.0)
    assert bool(torch.isfinite(norm))
    below[1][3] = big
    out, norm = amd.clip_by_global_norm(below, 1.0)         # sqrt 2 of it
    assert float(norm) == float("inf") and all(bool(torch.isnan(o).all()) for o in out)
    assert float(amd.global_norm(below)) == float("inf")
    res, norm = amd.clip_by_global_norm(below, float("inf"), out=below)
    assert float(norm) == float("inf") and all(bool(torch.isnan(o).all()) for o in res)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [50, 3000001])
@pytest.mark.parametrize("clip", [1.0, 2.0 ** -20, 2.0 ** -100])
def test_a_factor_below_the_normal_numbers(amd, n, clip):
    """clip / norm down to 2^-226 is no normal fp32 number, the results are: within the bounds of check() (and half a step of the
    smallest numbers, 2^-150; of bf16, 2^-134)."""
    g = torch.Generator().manual_seed(n)
    ts = [(torch.randn(k, generator=g) * 2.0 ** 110).to(t).cuda() for k, t in ((n, f32), (77, bf16), (3, f32))]
    ts[0][1], ts[0][n // 2], ts[1][5] = 2.0 ** 126, 0.0, 1.0
    for dst in (None, [t.clone() for t in ts]):
        out, norm = amd.clip_by_global_norm(ts, clip, out=dst)
        n64 = norm64(ts)
        assert abs(float(norm) - n64) <= 2 * E * n64
        for t, o in zip(ts, out):
            want = t.double().cpu() * (clip / n64)
            bound = (2 * E + (B8 if t.dtype == bf16 else E)) * want.abs() + 2.0 ** -150 + (2.0 ** -134 if t.dtype == bf16 else 0.0)
            assert bool(((o.double().cpu() - want).abs() <= bound).all())
