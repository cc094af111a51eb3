"""torch.autograd bridge to the C ABI: one forward / one backward call per layer for the
whole batch.  PyTorch is used for device memory, streams and autograd bookkeeping only --
all arithmetic happens in the HIP library (there is no eager fallback)."""
import ctypes as C
import functools
import threading

import torch
from torch.autograd import forward_ad

from . import _ffi


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    # (what torch.cuda.current_stream(device).cuda_stream returns, without the stream object: 0.1 instead of 1.9 us)
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device.index is None else device.index)


def _on_tensor_device(fn):
    """Runs an autograd Function's forward / backward with the device of its first GPU tensor made current: the
    library resolves per-device state (dynamic-LDS caps, the mixed-dispatch side stream) through hipGetDevice(), and
    a launch on a stream of another device than the current one would fail."""
    @functools.wraps(fn)
    def wrapped(ctx, *args):
        dev = next((a.device for a in args if torch.is_tensor(a) and a.is_cuda), None)
        if dev is None or dev.index == torch.cuda.current_device():
            return fn(ctx, *args)
        with torch.cuda.device(dev):
            return fn(ctx, *args)
    return wrapped


def _require_gpu(t, what):
    if not t.is_cuda:
        raise _ffi.AgcnError("%s must live on the GPU: the AGCN layer path has no CPU fallback" % what)


def _f32c(t, what):
    if t.dtype != torch.float32:
        raise TypeError("%s must be float32" % what)
    return t if t.is_contiguous() else t.contiguous()


_DT = {torch.float32: 0, torch.bfloat16: 1}
_TYPES = {i: t for t, i in _DT.items()}


class CastRowsFunction(torch.autograd.Function):
    """Storage-dtype conversion of a feature matrix (bf16 <-> f32) through the C ABI; the gradient is cast back."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, X, dtype):
        _require_gpu(X, "features")
        if X.dtype not in _DT or dtype not in _DT:
            raise TypeError("features must be float32 or bfloat16")
        ctx.src = X.dtype
        if X.dtype == dtype:
            return X
        X = X if X.is_contiguous() else X.contiguous()
        out = torch.empty(X.shape, dtype=dtype, device=X.device)
        cols = X.shape[-1]
        _ffi.check(_ffi.lib().agcn_cast_rows(X.data_ptr(), _DT[X.dtype], out.data_ptr(), _DT[dtype],
                                             X.numel() // cols, cols, cols, cols, _stream(X.device)))
        return out

    @staticmethod
    @_on_tensor_device
    def backward(ctx, g):
        return CastRowsFunction.apply(g, ctx.src), None


class PackRowsFunction(torch.autograd.Function):
    """Reference feed -> packed rows: [B * stride, F] (graph b at rows b*stride .. b*stride + n_b) -> [N1, F].
    `batch.plan` is the PACKED plan.  Backward unpacks the gradient (pad rows get 0)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, Xpad, batch, stride):
        _require_gpu(Xpad, "node features")
        Xpad = _f32c(Xpad, "node features")
        plan, F = batch.plan, Xpad.shape[1]
        if Xpad.shape[0] != plan.B * stride:
            raise ValueError("padded node features must be [B * max_atom, F]")
        out = torch.empty((plan.N1, F), dtype=torch.float32, device=Xpad.device)
        _ffi.check(_ffi.lib().agcn_rows_pack(plan.host_ptr, plan.dev_ptr, Xpad.data_ptr(), int(stride), F, F,
                                             out.data_ptr(), F, _stream(Xpad.device)))
        ctx.batch, ctx.stride = batch, int(stride)
        return out

    @staticmethod
    @_on_tensor_device
    def backward(ctx, g):
        return UnpackRowsFunction.apply(g, ctx.batch, ctx.stride, None), None, None


class UnpackRowsFunction(torch.autograd.Function):
    """Packed rows -> the reference's padded layout [B * stride, F]; pad rows are 0, or `fill` [F] (DenseMol's
    bias lands on pad rows too, dense_layer.py:42-50).  Backward packs the gradient."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, Xp, batch, stride, fill):
        _require_gpu(Xp, "node features")
        Xp = _f32c(Xp, "node features")
        plan, F = batch.plan, Xp.shape[1]
        out = torch.empty((plan.B * int(stride), F), dtype=torch.float32, device=Xp.device)
        if fill is not None:
            fill = _f32c(fill.detach(), "fill")
        _ffi.check(_ffi.lib().agcn_rows_unpack(plan.host_ptr, plan.dev_ptr, Xp.data_ptr(), F, F, out.data_ptr(),
                                               int(stride), F, _ptr(fill), _stream(Xp.device)))
        ctx.batch, ctx.stride = batch, int(stride)
        return out

    @staticmethod
    @_on_tensor_device
    def backward(ctx, g):
        return PackRowsFunction.apply(g, ctx.batch, ctx.stride), None, None, None


class _Cfg(object):
    __slots__ = ("Fin", "Fout", "K", "mode", "variant", "activation", "lsum", "prev_sym", "bf16")

    def __init__(self, Fin, Fout, K, mode, variant, activation, lsum=True, prev_sym=False, bf16=False):
        # bf16: X / Y / dY / dX are bf16 tensors read and written by the kernels themselves (AgcnLayerDesc.feat_dtype)
        self.bf16 = bool(bf16)
        # prev_sym: the caller vouches that L_prev is symmetric (AgcnGraphBatch.L_prev_symmetric)
        self.prev_sym = bool(prev_sym)
        self.Fin, self.Fout, self.K = int(Fin), int(Fout), int(K)
        self.mode, self.variant, self.activation = mode, variant, activation
        # lsum=False: an SGC_LL call whose combined Laplacian nobody reads (the reference's SGC_LL returns three
        # outputs, graphconv.py:252) -- the L_sum tile is then neither allocated nor written
        self.lsum = bool(lsum) or variant == "SGC_LL_Reslap"


# Per-call dispatch flags (include/agcn.h: AgcnLayerDesc.flags): which of the equivalent kernel paths serves the calls THIS
# thread issues inside a `with dispatch(...)` block.  Nothing process-wide is touched; other threads keep their own flags.
_tls = threading.local()


def current_flags():
    return getattr(_tls, "flags", 0)


class dispatch(object):
    """`with agcn_amd.dispatch(spec_mode=3):` -- the layer calls issued by this thread inside the block carry these per-call
    dispatch overrides (names and values as the agcn_set_* functions of include/agcn.h: spec_mode, fused_mode, pg_onepass,
    spec_small, rows_split, slab_mode, fused_gb, spec_tail, coop_members).  The backward of an autograd call uses the flags
    its forward ran with, whichever thread runs it.  Step objects (SgcLLStep, ...) take the flags current at construction."""

    def __init__(self, **knobs):
        self.knobs = knobs

    def __enter__(self):
        self.prev = current_flags()
        _tls.flags = _ffi.dispatch_flags(self.prev, **self.knobs)
        return self

    def __exit__(self, *exc):
        _tls.flags = self.prev
        return False


def no_member_flags(base=None):
    """`base` (default: this thread's current flags) with everything switched off in which one workgroup WAITS for another
    inside a launch: the member workgroups that share a large graph (every graph then runs in one workgroup, or on the slab
    kernels) and the tagged hand-off of the parameter-gradient kernel (the arrival-counter kernel instead: its last arriver
    adds the partials, nobody polls) -- the dispatch a call is re-issued on when a bounded wait ran out."""
    base = current_flags() if base is None else int(base)
    sm = (base & 15) - 1 if (base & 15) else _ffi.lib().agcn_get_spec_mode()
    pg = ((base >> 7) & 3) - 1 if ((base >> 7) & 3) else _ffi.lib().agcn_get_param_grad_onepass()
    return _ffi.dispatch_flags(base, spec_mode=sm & 3, pg_onepass=min(pg, 1))


# Parameter gradients beside the backward chain (include/agcn.h: agcn_sgc_ll_backward_forked).  In a multi-layer step the
# parameter-gradient kernel of layer l depends on that layer's per-graph backward kernel only; nothing downstream of it is needed by
# the backward of layer l - 1.  Inside `with param_grad_fork(device):` every SGC layer's backward enqueues its parameter gradients
# on ONE side stream (an event edge per layer), the main stream goes straight on to the previous layer, and the two streams are
# joined once when the block ends.  Process-wide per device (autograd runs backward() on its own thread), so one training step at
# a time per device.  Parameters' .grad must be None (or untouched) until the block ends: the gradient tensors are filled on the
# side stream -- autograd only STORES them (no kernel) when .grad is None.
_forks = {}


class param_grad_fork(object):
    def __init__(self, device):
        dev = torch.device(device)
        self.idx = dev.index if dev.index is not None else torch.cuda.current_device()
        st = _forks.get(self.idx)
        if st is None:
            st = _forks[self.idx] = {"stream": torch.cuda.Stream(torch.device("cuda", self.idx)), "keep": [], "active": False}
        self.st = st

    def __enter__(self):
        self.st["active"] = True
        self.st["used"] = False
        return self

    def __exit__(self, *exc):
        st = self.st
        st["active"] = False
        if st["used"]:
            torch.cuda.current_stream(torch.device("cuda", self.idx)).wait_stream(st["stream"])      # the ONE join of the step
        if torch.cuda.is_current_stream_capturing():
            # a captured graph replays on these buffers: they belong to the capturing object (engine.GraphedStep's capture_scope)
            # for as long as its graph lives, like the pooled reserves a capture pins
            (_capture_scopes[-1].held if _capture_scopes else _unscoped_captures).extend((None, k) for k in st["keep"])
        del st["keep"][:]
        return False


def _active_fork(dev):
    st = _forks.get(dev.index if dev.index is not None else torch.cuda.current_device())
    return st if (st is not None and st["active"]) else None


# how many calls were re-issued on the non-member dispatch after a cooperative wait ran out (engine.*.check(recover=True),
# functional.run_checked)
recovered_calls = [0]


def _desc(cfg, ldx, ldy, flags=None):
    return _ffi.LayerDesc(cfg.Fin, cfg.Fout, cfg.K, _ffi.MODE[cfg.mode], _ffi.VARIANT[cfg.variant],
                          _ffi.ACT[cfg.activation], int(ldx), int(ldy), 1 if getattr(cfg, "bf16", False) else 0,
                          current_flags() if flags is None else int(flags))


def _gbatch(batch, X, L_prev, prev_symmetric=False):
    p = batch.plan
    return _ffi.GraphBatch(p.host_ptr, p.dev_ptr, X.data_ptr(), _ptr(batch.l0_dense), batch.l0_ld,
                           1 if batch.l0_symmetric else 0,
                           _ptr(batch.l0_rowptr), _ptr(batch.l0_col), _ptr(batch.l0_val), _ptr(L_prev),
                           1 if (prev_symmetric and L_prev is not None) else 0, 0)


def _sizes(plan, cfg, ldx, ldy, flags=None):
    """(desc, reserve bytes, forward workspace bytes, backward workspace bytes) of a layer on a plan: three host-side
    FFI calls, cached on the plan (a plan is immutable)."""
    lib = _ffi.lib()
    flags = current_flags() if flags is None else int(flags)
    # the per-call flags and, where they leave a field alone, the process defaults change which kernels (and so which
    # workspaces) a call takes
    knobs = (flags, lib.agcn_get_lds_limit(), lib.agcn_get_fused_mode(), lib.agcn_get_slab_mode(),
             lib.agcn_get_fused_global_b(), lib.agcn_get_param_grad_onepass(), lib.agcn_get_spec_mode(),
             lib.agcn_get_spec_small(), lib.agcn_get_spec_tail(), lib.agcn_get_rows_split(), lib.agcn_get_coop_members())
    key = (cfg.Fin, cfg.Fout, cfg.K, cfg.mode, cfg.variant, cfg.activation, int(ldx), int(ldy), bool(cfg.bf16)) + knobs
    cache = plan.__dict__.setdefault("_size_cache", {})
    hit = cache.get(key)
    if hit is None:
        lib = _ffi.lib()
        desc = _desc(cfg, ldx, ldy, flags)
        hit = (desc, lib.agcn_sgc_ll_reserve_bytes(C.byref(desc), plan.host_ptr),
               lib.agcn_sgc_ll_forward_workspace_bytes(C.byref(desc), plan.host_ptr),
               lib.agcn_sgc_ll_backward_workspace_bytes(C.byref(desc), plan.host_ptr))
        cache[key] = hit
    return hit


# One persistent status word per device, registered with the library (include/agcn.h: agcn_set_device_status_word): a wait
# between the workgroups that share a large graph that runs out counts itself there.  The reserves of the autograd path die
# with their autograd graph -- right after backward() --, so the count has to live somewhere that outlives them (the weak
# references this module kept until round 3 were all dead by the time a training loop looked at them).
_status_words = {}


def _status_word(device):
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _status_words.get(idx)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _ffi.check(_ffi.lib().agcn_set_device_status_word(idx, w.data_ptr()))
        _status_words[idx] = w
    return w


def device_timeouts(clear=True):
    """Synchronises the devices that ran SGC_LL autograd calls; returns how many cooperative waits ran out since the words
    were last cleared (0: every result is good) and, by default, clears them."""
    total = 0
    for idx, w in list(_status_words.items()):
        with torch.cuda.device(idx):
            t = C.c_int32(0)
            _ffi.lib().agcn_device_status(idx, torch.cuda.current_stream(idx).cuda_stream, C.byref(t))
            if t.value and clear:
                w.zero_()
            total += int(t.value)
    return total


def run_checked(fn):
    """A step that cannot be lost: runs `fn()` (the calls of one training / evaluation step on this thread: forward, loss,
    backward -- it must be re-runnable: same inputs, gradients zeroed or overwritten inside), synchronises, and if a wait between
    the workgroups that share a large graph ran out anywhere in it -- results NaN, include/agcn.h: agcn_device_status --
    RE-ISSUES the same calls on the non-member dispatch (fresh launches, per-call flags: no workgroup of those kernels waits
    for another) and returns that run's result.  `recovered_calls[0]` counts such re-runs."""
    device_timeouts()           # (whatever an earlier, unchecked step left behind is not this step's)
    out = fn()
    if device_timeouts() == 0:
        return out
    nm = no_member_flags()
    with dispatch(spec_mode=(nm & 15) - 1, pg_onepass=((nm >> 7) & 3) - 1):
        out = fn()
    recovered_calls[0] += 1
    if device_timeouts() != 0:
        raise _ffi.AgcnError("a cooperative wait ran out on the non-member dispatch (which has none): device fault")
    return out


def check_device_status():
    """Synchronises the devices that ran SGC_LL autograd calls and raises AgcnError if a wait between the workgroups that share
    a large graph ran out in any call since the last check -- forward OR backward: the count is kept in a persistent word per
    device, not in the reserves (which autograd frees once backward has run).  The gradients of such a step are NaN.  Call it
    where the training loop synchronises anyway (reading the loss).  Returns the number of devices checked; the word is
    cleared when an error is raised, so that one bad step is reported once."""
    n = 0
    for idx, w in list(_status_words.items()):
        with torch.cuda.device(idx):
            t = C.c_int32(0)
            rc = _ffi.lib().agcn_device_status(idx, torch.cuda.current_stream(idx).cuda_stream, C.byref(t))
            if rc != 0:
                msg = _ffi.lib().agcn_last_error().decode()
                w.zero_()
                raise _ffi.AgcnError("agcn error %d: %s" % (rc, msg))
        n += 1
    return n


# Reserve buffers of the autograd path are LEASED from a pool per (device, stream, size class) instead of allocated -- and their
# 64 KB exchange header zero-filled, one fill kernel per layer call: 3.7 us, 5 % of a molecule network's step -- on every forward.
# A reserve may serve any batch after any other (the header is self-maintaining: include/agcn.h), so a buffer that comes back
# from the pool needs nothing.  A lease goes back when the autograd node that holds it dies (after backward(), or when the outputs
# of a forward-only call are dropped).  Under stream capture: a pooled buffer (allocated eagerly, e.g. by the warm-up steps
# GraphedStep runs on its capture stream) is used at its fixed address by every replay, so it belongs to the CAPTURING OBJECT for
# as long as its graph lives (capture_scope(): engine.GraphedStep owns the list and frees the buffers when it is
# reset or deleted; a capture outside any scope pins its buffers in _unscoped_captures until release_reserve_pool(force=True));
# a buffer allocated INSIDE a capture belongs to the graph's own memory pool and never enters this one.
_reserve_pool = {}
_reserve_pool_bytes = [0]
_RESERVE_POOL_CAP = 2 << 30
_unscoped_captures = []
_capture_scopes = []


def _size_class(rbytes):
    """256 KB classes below 64 MB, 1/8-octave classes (at most +12.5 %) above: a point-cloud reserve of ~256 MB that grows by a
    few KB with the batch finds the buffer of the previous batch instead of pinning a new one."""
    if rbytes < (64 << 20):
        return (rbytes + 262143) // 262144 * 262144
    step = 1 << (int(rbytes - 1).bit_length() - 4)
    return (rbytes + step - 1) // step * step


def _pool_put(key, tensor):
    if _reserve_pool_bytes[0] + tensor.numel() <= _RESERVE_POOL_CAP:
        _reserve_pool.setdefault(key, []).append(tensor)
        _reserve_pool_bytes[0] += tensor.numel()


class capture_scope(object):
    """Owner of the pooled reserves a stream capture pins.  `with capture_scope() as scope:` around the capture; the buffers
    stay out of the pool until `scope.release()` (call it once the captured graph is gone)."""

    def __init__(self):
        self.held = []

    def __enter__(self):
        _capture_scopes.append(self)
        return self

    def __exit__(self, *exc):
        _capture_scopes.remove(self)
        return False

    def release(self):
        # (back to the torch caching allocator, not to the lease pool: the pool is keyed by stream, and the side stream of a
        # GraphedStep that is gone may never ask again)
        self.held = []

    @property
    def nbytes(self):
        return sum(t.numel() for _, t in self.held if torch.is_tensor(t))


def reserve_pool_bytes():
    """(bytes idle in the pool, bytes pinned by captures outside any capture_scope)."""
    return _reserve_pool_bytes[0], sum(t.numel() for _, t in _unscoped_captures if torch.is_tensor(t))


def release_reserve_pool(force=False):
    """Drops every idle reserve buffer of the pool (the torch caching allocator gets them back; torch.cuda.empty_cache() then
    returns them to the device).  `force=True` also drops the buffers pinned by captures that ran outside a capture_scope --
    only once those graphs are gone.  Returns the number of bytes dropped."""
    n = _reserve_pool_bytes[0]
    _reserve_pool.clear()
    _reserve_pool_bytes[0] = 0
    if force:
        n += sum(t.numel() for _, t in _unscoped_captures if torch.is_tensor(t))
        del _unscoped_captures[:]
    return n


class _ReserveLease(object):
    __slots__ = ("tensor", "key", "pooled")

    def __del__(self):
        try:
            if self.pooled:
                _pool_put(self.key, self.tensor)
        except Exception:          # (interpreter shutdown)
            pass


def _lease_reserve(dev, rbytes):
    size = _size_class(rbytes)
    capturing = torch.cuda.is_current_stream_capturing()
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    key = (idx, torch.cuda.current_stream(dev).cuda_stream, size)
    lease = _ReserveLease()
    lease.key = key
    lst = _reserve_pool.get(key)
    if lst:
        lease.tensor = lst.pop()
        _reserve_pool_bytes[0] -= lease.tensor.numel()
        lease.pooled = not capturing
        if capturing:
            (_capture_scopes[-1].held if _capture_scopes else _unscoped_captures).append((key, lease.tensor))
    else:
        lease.tensor = torch.empty(size, dtype=torch.uint8, device=dev)
        lease.tensor[:min(size, _ffi.RESERVE_HEADER_BYTES)].zero_()      # (must be zero when a reserve is first used)
        lease.pooled = not capturing
    return lease


class SgcLLFunction(torch.autograd.Function):
    """(Y, res_L, res_W, L_sum) = SGC_LL[_Reslap](X; weight, bias, M_L, alpha, beta, L_prev)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, X, weight, bias, M_L, alpha, beta, L_prev, batch, cfg):
        lib = _ffi.lib()
        _require_gpu(X, "node features")
        fdt = torch.bfloat16 if cfg.bf16 else torch.float32
        if cfg.bf16:
            if X.dtype != torch.bfloat16:
                raise TypeError("a bf16 layer call needs bf16 node features")
            X = X if X.is_contiguous() else X.contiguous()
        else:
            X = _f32c(X, "node features")
        weight, bias, M_L, alpha = (_f32c(weight, "weight"), _f32c(bias, "bias"), _f32c(M_L, "M_L"),
                                    _f32c(alpha, "alpha"))
        plan = batch.plan
        if X.dim() != 2 or X.shape[0] != plan.rows or X.shape[1] < cfg.Fin:
            raise ValueError("node features must be [rows=%d, >=%d], got %s" % (plan.rows, cfg.Fin, tuple(X.shape)))
        if tuple(weight.shape) != (cfg.Fin * cfg.K, cfg.Fout) or tuple(M_L.shape) != (cfg.Fin, cfg.Fin):
            raise ValueError("parameter shapes do not match the layer")
        reslap = cfg.variant == "SGC_LL_Reslap"
        if L_prev is not None:
            L_prev = _f32c(L_prev, "L_prev")
            if L_prev.numel() != plan.tile_elems:
                raise ValueError("L_prev must be a packed tile tensor of %d floats" % plan.tile_elems)
            if beta is None:
                raise ValueError("L_prev given without beta")
            beta = _f32c(beta, "beta")
        dev = X.device
        _status_word(dev)
        ldx, ldy = X.shape[1], cfg.Fout
        Y = torch.empty((plan.rows, ldy), dtype=fdt, device=dev)
        res_L = torch.empty(plan.tile_elems, dtype=torch.float32, device=dev)
        res_W = torch.empty(plan.tile_elems, dtype=torch.float32, device=dev)
        L_sum = torch.empty(plan.tile_elems if cfg.lsum else 0, dtype=torch.float32, device=dev)
        flags = current_flags()
        desc, rbytes, wbytes, _ = _sizes(plan, cfg, ldx, ldy, flags)
        # (the reserve starts with the exchange header of the cooperative kernels, which must be zero when a reserve is FIRST
        # used -- include/agcn.h: AGCN_RESERVE_HEADER_BYTES; only that: at point-cloud sizes the reserve holds n x n tiles, and
        # zero-filling all of it was 75 us per layer call -- and only then: see _lease_reserve)
        lease = _lease_reserve(dev, rbytes)
        reserve = lease.tensor
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        gb = _gbatch(batch, X, L_prev if reslap else None, cfg.prev_sym)
        pr = _ffi.Params(weight.data_ptr(), bias.data_ptr(), M_L.data_ptr(), alpha.data_ptr(), _ptr(beta))
        out = _ffi.Outputs(Y.data_ptr(), res_L.data_ptr(), res_W.data_ptr(), L_sum.data_ptr() if cfg.lsum else None)
        _ffi.check(lib.agcn_sgc_ll_forward(C.byref(desc), C.byref(gb), C.byref(pr), C.byref(out),
                                           reserve.data_ptr(), reserve.numel(), ws.data_ptr(), wbytes, _stream(dev)))
        ctx.batch, ctx.cfg, ctx.has_prev, ctx.has_beta = batch, cfg, (reslap and L_prev is not None), beta is not None
        ctx.reserve_lease, ctx.flags = lease, flags
        ctx.save_for_backward(X, weight, bias, M_L, alpha, beta, L_prev if reslap else None,
                              Y, res_L, res_W, L_sum)
        ctx.mark_non_differentiable(res_L, res_W)
        ctx.set_materialize_grads(False)      # an unused L_sum must reach the library as "no upstream gradient"
        return Y, res_L, res_W, L_sum

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dY, _dres_L, _dres_W, dL_sum):
        lib = _ffi.lib()
        X, weight, bias, M_L, alpha, beta, L_prev, Y, res_L, res_W, L_sum = ctx.saved_tensors
        reserve = ctx.reserve_lease.tensor
        batch, cfg, plan = ctx.batch, ctx.cfg, ctx.batch.plan
        dev = X.device
        paper = cfg.mode == "paper"
        if dY is None:
            dY = torch.zeros_like(Y)
        if cfg.bf16:
            dY = dY.to(torch.bfloat16)
            dY = dY if dY.is_contiguous() else dY.contiguous()
        else:
            dY = _f32c(dY, "dY")
        if dL_sum is not None:
            dL_sum = _f32c(dL_sum, "dL_sum")
        ldx, ldy = X.shape[1], cfg.Fout
        desc, _, _, wbytes = _sizes(plan, cfg, ldx, ldy, ctx.flags)     # (the forward's flags: autograd runs this on its own thread)
        dX = torch.empty_like(X)
        if ldx > cfg.Fin:
            dX.zero_()
        dweight = torch.empty_like(weight)
        dbias = torch.empty_like(bias)
        dM = torch.empty_like(M_L) if paper else None
        dalpha = torch.empty_like(alpha)
        dbeta = torch.empty_like(beta) if ctx.has_prev else None
        dLp = torch.empty_like(L_prev) if ctx.has_prev else None
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        gb = _gbatch(batch, X, L_prev, ctx.cfg.prev_sym)
        pr = _ffi.Params(weight.data_ptr(), bias.data_ptr(), M_L.data_ptr(), alpha.data_ptr(), _ptr(beta))
        fw = _ffi.Outputs(Y.data_ptr(), res_L.data_ptr(), res_W.data_ptr(), L_sum.data_ptr() if cfg.lsum else None)
        gr = _ffi.Grads(dX.data_ptr(), dweight.data_ptr(), dbias.data_ptr(), _ptr(dM), dalpha.data_ptr(),
                        _ptr(dbeta), _ptr(dLp))
        fk = _active_fork(dev)
        if fk is not None:
            main = torch.cuda.current_stream(dev)
            ev = torch.cuda.Event()
            ev.record(main)                                   # (creates the handle; the library records it again where it forks)
            _ffi.check(lib.agcn_sgc_ll_backward_forked(C.byref(desc), C.byref(gb), C.byref(pr), C.byref(fw),
                                                       dY.data_ptr(), _ptr(dL_sum), C.byref(gr), reserve.data_ptr(),
                                                       reserve.numel(), ws.data_ptr(), wbytes, main.cuda_stream,
                                                       fk["stream"].cuda_stream, int(ev.cuda_event)))
            # what the side stream still reads when this function returns: alive until the join (NOT the gradient tensors: a
            # second reference would make autograd copy them -- on the main stream, before they are written)
            fk["keep"].append((ws, ev, ctx.reserve_lease, X, Y, dY))
            fk["used"] = True
        else:
            _ffi.check(lib.agcn_sgc_ll_backward(C.byref(desc), C.byref(gb), C.byref(pr), C.byref(fw),
                                                dY.data_ptr(), _ptr(dL_sum), C.byref(gr), reserve.data_ptr(),
                                                reserve.numel(), ws.data_ptr(), wbytes, _stream(dev)))
        if ctx.has_beta and dbeta is None:
            dbeta = None   # beta unused (no L_prev): TF reports no gradient either
        return dX, dweight, dbias, dM, dalpha, dbeta, dLp, None, None


class GraphGatherFunction(torch.autograd.Function):
    """out[b] = act(sum of graph b's real rows)   (graphgather.py:40-77)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, X, batch, activation):
        lib = _ffi.lib()
        _require_gpu(X, "node features")
        X = _f32c(X, "node features")
        plan = batch.plan
        if X.dim() != 2 or X.shape[0] != plan.rows:
            raise ValueError("node features must be [rows=%d, F]" % plan.rows)
        F = X.shape[1]
        out = torch.empty((plan.B, F), dtype=torch.float32, device=X.device)
        _ffi.check(lib.agcn_graph_gather_forward(plan.host_ptr, plan.dev_ptr, X.data_ptr(), F, F,
                                                 _ffi.ACT[activation], out.data_ptr(), _stream(X.device)))
        ctx.batch, ctx.activation, ctx.F = batch, activation, F
        ctx.save_for_backward(out)
        return out

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dOut):
        lib = _ffi.lib()
        (out,) = ctx.saved_tensors
        plan = ctx.batch.plan
        dOut = _f32c(dOut, "dOut")
        dX = torch.empty((plan.rows, ctx.F), dtype=torch.float32, device=out.device)
        _ffi.check(lib.agcn_graph_gather_backward(plan.host_ptr, plan.dev_ptr, out.data_ptr(), dOut.data_ptr(),
                                                  ctx.F, ctx.F, _ffi.ACT[ctx.activation], dX.data_ptr(),
                                                  _stream(out.device)))
        return dX, None, None


class RowsDenseFunction(torch.autograd.Function):
    """Y = act([scale *] A . W [+ bias] [+ Add]) over the row space: DenseMol (dense_layer.py:33-50),
    BlockEnd (blockend.py:67-86) and, with the device scalar `scale`, one term of DenseBlockEnd
    (densenet_block.py:113-123)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, A, W, bias, Add, batch, activation, keep_pad_rows, scale=None):
        lib = _ffi.lib()
        _require_gpu(A, "node features")
        A, W = _f32c(A, "node features"), _f32c(W, "weight")
        plan = batch.plan
        Fin, Fout = W.shape
        if A.dim() != 2 or A.shape[0] != plan.rows or A.shape[1] < Fin:
            raise ValueError("node features must be [rows=%d, >=%d]" % (plan.rows, Fin))
        if bias is not None:
            bias = _f32c(bias, "bias")
        if Add is not None:
            Add = _f32c(Add, "Add")
            if tuple(Add.shape) != (plan.rows, Fout):
                raise ValueError("Add must be [rows, Fout]")
        if scale is not None:
            scale = _f32c(scale, "scale")
            if scale.numel() != 1:
                raise ValueError("scale must hold one element")
        Y = torch.empty((plan.rows, Fout), dtype=torch.float32, device=A.device)
        desc = _ffi.DenseDesc(Fin, Fout, _ffi.ACT[activation], 1 if keep_pad_rows else 0, A.shape[1], Fout, Fout, current_flags())
        # (point-cloud row counts: the product runs on the split-bf16 row kernels, which build a parameter image per call)
        wbytes = lib.agcn_rows_dense_forward_workspace_bytes(C.byref(desc), plan.host_ptr)
        ws = torch.empty(wbytes, dtype=torch.uint8, device=A.device) if wbytes else None
        _ffi.check(lib.agcn_rows_dense_scaled_forward_ws(C.byref(desc), plan.host_ptr, plan.dev_ptr, A.data_ptr(),
                                                         W.data_ptr(), _ptr(scale), _ptr(bias), _ptr(Add), Y.data_ptr(),
                                                         _ptr(ws), wbytes, _stream(A.device)))
        ctx.batch, ctx.desc, ctx.has_bias, ctx.has_add = batch, desc, bias is not None, Add is not None
        ctx.has_scale = scale is not None
        if scale is not None:
            ctx.save_for_backward(A, W, Y, scale)
        else:
            ctx.save_for_backward(A, W, Y)
        return Y

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dY):
        lib = _ffi.lib()
        saved = ctx.saved_tensors
        A, W, Y = saved[:3]
        scale = saved[3] if ctx.has_scale else None
        plan, desc = ctx.batch.plan, ctx.desc
        dY = _f32c(dY, "dY")
        dA = torch.empty_like(A)
        if A.shape[1] > desc.Fin:
            dA.zero_()
        dW = torch.empty_like(W)
        db = torch.empty(desc.Fout, dtype=torch.float32, device=A.device) if ctx.has_bias else None
        dAdd = torch.empty((plan.rows, desc.Fout), dtype=torch.float32, device=A.device) if ctx.has_add else None
        ds = torch.empty_like(scale) if scale is not None else None
        wbytes = lib.agcn_rows_dense_backward_workspace_bytes(C.byref(desc), plan.host_ptr)
        ws = torch.empty(wbytes, dtype=torch.uint8, device=A.device)
        _ffi.check(lib.agcn_rows_dense_scaled_backward(
            C.byref(desc), plan.host_ptr, plan.dev_ptr, A.data_ptr(), W.data_ptr(), _ptr(scale), Y.data_ptr(),
            dY.data_ptr(), dA.data_ptr(), _ptr(dAdd), dW.data_ptr(), _ptr(db), _ptr(ds), ws.data_ptr(), wbytes,
            _stream(A.device)))
        return dA, dW, db, dAdd, None, None, None, ds


class MultitaskCEFunction(torch.autograd.Function):
    """T two-class heads + the weighted sigmoid cross-entropy training loss
    (model_operatos.py:710-759,792-864; multitask_classifier.py:41-44,187-209).
    Returns (loss [1], logits [T, B, 2]); the gradient flows through the loss only."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, feat, W, bias, labels, weights, batch_size):
        lib = _ffi.lib()
        _require_gpu(feat, "graph features")
        feat, W, bias = _f32c(feat, "graph features"), _f32c(W, "head weights"), _f32c(bias, "head biases")
        labels, weights = _f32c(labels, "labels"), _f32c(weights, "weights")
        T, F = W.shape[0], W.shape[1]
        B = feat.shape[0]
        if feat.dim() != 2 or feat.shape[1] < F or tuple(W.shape) != (T, F, 2) or tuple(bias.shape) != (T, 2):
            raise ValueError("feat [B, >=F], W [T, F, 2], bias [T, 2] expected")
        if tuple(labels.shape) != (B, T) or tuple(weights.shape) != (B, T):
            raise ValueError("labels and weights must be [B, T]")
        dev = feat.device
        logits = torch.empty((T, B, 2), dtype=torch.float32, device=dev)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        wbytes = lib.agcn_multitask_ce_workspace_bytes(B, F, T)
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        inv = 1.0 / float(batch_size)
        _ffi.check(lib.agcn_multitask_ce_forward(B, F, T, feat.data_ptr(), feat.shape[1], W.data_ptr(), bias.data_ptr(),
                                                 labels.data_ptr(), weights.data_ptr(), inv, logits.data_ptr(),
                                                 loss.data_ptr(), ws.data_ptr(), wbytes, _stream(dev)))
        ctx.dims, ctx.inv = (B, F, T), inv
        ctx.save_for_backward(feat, W, logits, labels, weights)
        ctx.mark_non_differentiable(logits)
        return loss, logits

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dloss, _dlogits):
        lib = _ffi.lib()
        feat, W, logits, labels, weights = ctx.saved_tensors
        B, F, T = ctx.dims
        dev = feat.device
        dloss = _f32c(dloss.reshape(1), "dloss")
        dfeat = torch.empty_like(feat)
        if feat.shape[1] > F:
            dfeat.zero_()
        dW = torch.empty_like(W)
        db = torch.empty((T, 2), dtype=torch.float32, device=dev)
        wbytes = lib.agcn_multitask_ce_workspace_bytes(B, F, T)
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        _ffi.check(lib.agcn_multitask_ce_backward(B, F, T, feat.data_ptr(), feat.shape[1], W.data_ptr(),
                                                  logits.data_ptr(), labels.data_ptr(), weights.data_ptr(), ctx.inv,
                                                  dloss.data_ptr(), dfeat.data_ptr(), dW.data_ptr(), db.data_ptr(),
                                                  ws.data_ptr(), wbytes, _stream(dev)))
        return dfeat, dW, db, None, None, None


class GraphPoolFunction(torch.autograd.Function):
    """GraphPoolMol (graphpool.py:55-110).  grad='reference': no gradient, like the reference's py_func;
    grad='argmax': route the gradient to the arg-max rows (extension)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, X, batch, grad):
        lib = _ffi.lib()
        _require_gpu(X, "node features")
        X = _f32c(X, "node features")
        plan = batch.plan
        if X.dim() != 2 or X.shape[0] != plan.rows:
            raise ValueError("node features must be [rows=%d, F]" % plan.rows)
        F = X.shape[1]
        out = torch.empty((plan.rows, F), dtype=torch.float32, device=X.device)
        argmax = torch.empty((plan.rows, F), dtype=torch.int32, device=X.device) if grad == "argmax" else None
        gb = _gbatch(batch, X, None)
        _ffi.check(lib.agcn_graph_pool_forward(plan.host_ptr, plan.dev_ptr, C.byref(gb), X.data_ptr(), F, F,
                                               out.data_ptr(), _ptr(argmax), _stream(X.device)))
        ctx.batch, ctx.grad, ctx.F = batch, grad, F
        if argmax is not None:
            ctx.save_for_backward(argmax)
        else:
            ctx.mark_non_differentiable(out)     # like tf.py_func: no gradient
        return out

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dOut):
        if ctx.grad != "argmax":
            return None, None, None
        lib = _ffi.lib()
        (argmax,) = ctx.saved_tensors
        plan = ctx.batch.plan
        dOut = _f32c(dOut, "dOut")
        dX = torch.empty((plan.rows, ctx.F), dtype=torch.float32, device=dOut.device)
        gb = _gbatch(ctx.batch, dOut, None)
        _ffi.check(lib.agcn_graph_pool_backward(plan.host_ptr, plan.dev_ptr, C.byref(gb), argmax.data_ptr(),
                                                dOut.data_ptr(), ctx.F, ctx.F, dX.data_ptr(), _stream(dOut.device)))
        return dX, None, None


def _rows_ptr(t):
    """Data pointer of a row matrix; torch gives an EMPTY tensor the null pointer, which the library reads as "no such tensor"
    (the kernels touch no row of it)."""
    return None if t is None else (t.data_ptr() or 256)


_I32 = 0x7fffffff               # descriptors hold 32 bits: a size beyond goes in as this, which every entry refuses
_FFN_LD = 1 << 20               # agcn_gated_ffn_*: ldx


def _row_matrix(t, what, F=None, most=_I32):
    """`t` as a [rows, F] matrix of f32 or bf16 whose rows are contiguous, with a leading dimension of at most `most`."""
    _require_gpu(t, what)
    if t.dtype not in _DT:
        raise TypeError("%s must be float32 or bfloat16" % what)
    if t.dim() != 2 or t.shape[1] < 1 or (F is not None and t.shape[1] != F):
        raise ValueError("%s must be [rows, %s], got %s" % (what, "F" if F is None else F, tuple(t.shape)))
    if t.stride(1) != 1 or not t.shape[1] <= t.stride(0) <= most:
        return t.contiguous()
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _vector(t, what, F, like):
    """`t` as a contiguous float32 vector of F elements on the device of `like`."""
    if t is None:
        return None
    if t.dtype is torch.float32 and t.shape == (F,) and t.get_device() == like.get_device() and t.is_contiguous():
        return t
    _require_gpu(t, what)
    t = _f32c(t, what)
    if t.shape != (F,):
        raise ValueError("%s must be [%d], got %s" % (what, F, tuple(t.shape)))
    if t.device != like.device:
        raise ValueError("%s is on %s, the rows are on %s" % (what, t.device, like.device))
    return t


def _no_tangents(tensors):
    """Refuses tensors that carry a forward-mode tangent: the kernels would drop it, which reads as a derivative of zero."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _ffi.AgcnError("this operator has no forward-mode derivative")


def _wants_grad(tensors):
    _no_tangents(tensors)
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _on_device_of(t, fn, *args):
    """fn(*args) with the device of `t` made current (see _on_tensor_device)."""
    i = t.get_device()
    if i < 0 or i == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(i):
        return fn(*args)


def _saved(t, what, shape, dtype, index, most=_I32):
    """A saved tensor for a backward on GPU `index`.  Saved-tensor hooks (save_on_cpu, a pack hook that clones) give back the
    values, not the layout: sizes, type and device are held against the forward's, and leading dimensions are taken from the
    tensor that is returned here."""
    if t.dtype is dtype and t.get_device() == index and t.shape == shape:
        if t.is_contiguous() or (len(shape) == 2 and t.stride(1) == 1 and shape[1] <= t.stride(0) <= most):
            return t
        return t.contiguous()
    raise ValueError("%s: saved as %s %s on GPU %d, but came back as %s %s on %s" %
                     (what, tuple(shape), dtype, index, tuple(t.shape), t.dtype, t.device))


def _norm_forward(z, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias, plan, norm, eps, gate_activation, keep):
    """-> (y, h, what a backward needs: the tensors as the kernel read them, its row statistics, the descriptor)"""
    x = _row_matrix(x, "residual rows")
    rows, F = x.shape
    dev = x.device
    if plan is not None:
        if plan.dev is None or plan.dev.get_device() != x.get_device():
            raise ValueError("the plan is not on the rows' device")
        if plan.rows != rows:
            raise ValueError("the rows are %d, the plan has %d" % (rows, plan.rows))
    kind = 0
    if z is not None:
        z = _row_matrix(z, "block output", F)
        if z.get_device() != x.get_device():
            raise ValueError("block output is on %s, the rows are on %s" % (z.device, dev))
        if z.shape[0] != rows:
            raise ValueError("block output and residual rows differ in length (%d, %d)" % (z.shape[0], rows))
        if x.dtype is torch.bfloat16 and z.dtype is not torch.bfloat16:
            raise TypeError("bfloat16 residual rows need a bfloat16 block output")
    if gate is not None:
        if z is None:
            raise ValueError("a gate needs a block output")
        if gate.dtype is not z.dtype:
            raise TypeError("gate and block output must have one type")
        gate = _row_matrix(gate, "gate", F)
        if gate.get_device() != x.get_device():
            raise ValueError("gate is on %s, the rows are on %s" % (gate.device, dev))
        if plan is not None and gate.shape[0] == plan.B:
            kind = 2
        elif gate.shape[0] == rows:
            kind = 1
        else:
            raise ValueError("gate must have one row per row (%d)%s, got %d" %
                             (rows, "" if plan is None else " or one per graph (%d)" % plan.B, gate.shape[0]))
    scale = _vector(scale, "scale", F, x)
    post_weight, post_bias = _vector(post_weight, "post_weight", F, x), _vector(post_bias, "post_bias", F, x)
    pre_weight, pre_bias = _vector(pre_weight, "pre_weight", F, x), _vector(pre_bias, "pre_bias", F, x)
    zt = x.dtype if z is None else z.dtype
    if F > _I32:
        raise _ffi.AgcnError("F in 1..16384 (%d)" % F)
    desc = _ffi.NormDesc(rows, F, _ffi.NORM[norm], kind, _ffi.GATE_ACT[gate_activation], _DT[x.dtype], _DT[zt], _ld(x),
                         0 if z is None else _ld(z), 0 if gate is None else _ld(gate), eps)
    inputs = _ffi.NormInputs(_rows_ptr(z), _rows_ptr(x), _rows_ptr(gate), _ptr(scale), _ptr(post_weight), _ptr(post_bias),
                             _ptr(pre_weight), _ptr(pre_bias))
    y = torch.empty((rows, F), dtype=x.dtype, device=dev) if z is not None else None
    h = torch.empty((rows, F), dtype=zt, device=dev) if pre_weight is not None else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=dev) if keep else None
    host, devp = (None, None) if plan is None else (plan.host_ptr, plan.dev_ptr)
    _ffi.check(_ffi.lib().agcn_norm_gate_residual_forward(C.byref(desc), host, devp, C.byref(inputs), _rows_ptr(y), _rows_ptr(h),
                                                          _ptr(stats), _stream(dev)))
    return y, h, (z, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias, stats), desc


class _NoSecondDerivative(torch.autograd.Function):
    """A gradient that may be used, but not differentiated: without it, a penalty on a gradient would silently lose the terms
    that a kernel's backward does not carry on."""

    @staticmethod
    def forward(ctx, grad, mark):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad):
        raise _ffi.AgcnError("this operator's gradient cannot be differentiated again")


def _first_order(backward):
    @functools.wraps(backward)
    def run(ctx, *grads):
        _no_tangents(grads)
        if not torch.is_grad_enabled():                       # the usual case: no graph of the backward pass is wanted
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
            mark = torch.empty(0, requires_grad=True)
        return tuple(None if g is None else _NoSecondDerivative.apply(g, mark) for g in out)
    return run


class NormGateResidualFunction(torch.autograd.Function):
    """(y, h) = (x + scale * a(gate) * N(z), N'(y)); see norm_gate_residual."""

    @staticmethod
    def forward(ctx, z, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias, plan, norm, eps, gate_activation):
        y, h, saved, desc = _on_device_of(x, _norm_forward, z, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias, plan,
                                          norm, eps, gate_activation, True)
        ctx.desc, ctx.plan = desc, plan
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @_first_order
    def backward(ctx, dy, dh):
        if dy is None and dh is None:
            return (None,) * 12
        saved = ctx.saved_tensors
        return _on_device_of(dh if dy is None else dy, NormGateResidualFunction._backward, ctx.desc, ctx.plan, saved, dy, dh) + (None,) * 4

    @staticmethod
    def _backward(desc, plan, saved, dy, dh):
        lib = _ffi.lib()
        z, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias, stats = saved
        rows, F = desc.rows, desc.F
        dev = (dh if dy is None else dy).device
        at, xt, zt, shape = (dh if dy is None else dy).get_device(), _TYPES[desc.x_dtype], _TYPES[desc.z_dtype], (rows, F)
        x = _saved(x, "residual rows", shape, xt, at)
        ldx, ldz, ldg = _ld(x), 0, 0
        if z is not None:
            z = _saved(z, "block output", shape, zt, at)
            ldz = _ld(z)
        if gate is not None:
            gate = _saved(gate, "gate", shape if desc.gate == 1 else (plan.B, F), zt, at)
            ldg = _ld(gate)
        f32, where = torch.float32, []
        stats = _saved(stats, "row statistics", (rows, 4), f32, at).contiguous()
        vectors = [scale, post_weight, post_bias, pre_weight, pre_bias]
        for i, p in enumerate(vectors):
            if p is not None and not (p.dtype is f32 and p.is_contiguous() and p.numel() == F and p.get_device() == at):
                p = vectors[i] = _saved(p, "a vector", (F,), f32, at)
            where.append(0 if p is None else p.data_ptr())
        if (ldx, ldz, ldg) != (desc.ldx, desc.ldz, desc.ldg):
            desc = _ffi.NormDesc(rows, F, desc.norm, desc.gate, desc.gate_activation, desc.x_dtype, desc.z_dtype, ldx, ldz, ldg, desc.eps)
        dy = None if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        dx = torch.empty((rows, F), dtype=x.dtype, device=dev)
        dz = None if z is None else torch.empty((rows, F), dtype=z.dtype, device=dev)
        dgate = None if gate is None else torch.empty(gate.shape, dtype=gate.dtype, device=dev)
        # (the vectors' gradients: rows of one small matrix)
        given = [i for i, p in enumerate(vectors) if p is not None]
        params = [None] * 5
        for i, g in zip(given, torch.empty((len(given), F), dtype=torch.float32, device=dev).unbind(0)):
            params[i] = g
        inputs = _ffi.NormInputs(_rows_ptr(z), _rows_ptr(x), _rows_ptr(gate), *where)
        grads = _ffi.NormGrads(_rows_ptr(dz), _rows_ptr(dx), _rows_ptr(dgate), *[0 if p is None else p.data_ptr() for p in params])
        host, devp = (None, None) if plan is None else (plan.host_ptr, plan.dev_ptr)
        wbytes = lib.agcn_norm_gate_residual_backward_workspace_bytes(C.byref(desc), host)
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        _ffi.check(lib.agcn_norm_gate_residual_backward(
            C.byref(desc), host, devp, C.byref(inputs), _rows_ptr(stats), _rows_ptr(dy), _rows_ptr(dh), C.byref(grads),
            ws.data_ptr(), wbytes, _stream(dev)))
        return (dz, dx, dgate) + tuple(params)


def norm_gate_residual(z, x, post_weight=None, post_bias=None, gate=None, scale=None, pre_weight=None, pre_bias=None, norm="rms",
                       eps=1e-6, gate_activation="linear", plan=None):
    """The frame of a residual block in one pass over the node rows:

        u = N(z; post_weight, post_bias)            z [rows, F]: the block's output (no post_weight: u = z)
        y = x + scale * a(gate) * u                 x [rows, F]: the residual rows
        h = N(y; pre_weight, pre_bias)              what the next block reads (no pre_weight: h is None)

    norm: 'rms' (no biases) or 'layer'.  gate: [rows, F], or [B, F] with `plan` (a Plan or GraphBatch): one vector per graph;
    gate_activation: 'linear', 'tanh' or 'sigmoid'.  Rows are float32, bfloat16, or float32 x with bfloat16 z (h and gate have
    z's type); the vectors are float32.  z=None: h = N(x) alone.  With `plan`, pad rows come out zero.  Returns (y, h)."""
    if norm not in _ffi.NORM:
        raise ValueError("norm must be 'rms' or 'layer'")
    if gate_activation not in _ffi.GATE_ACT:
        raise ValueError("gate_activation must be 'linear', 'tanh' or 'sigmoid'")
    if x is None or not torch.is_tensor(x):
        raise TypeError("residual rows must be a tensor")
    plan = getattr(plan, "plan", plan)
    args = (z, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    if _wants_grad(args):
        return NormGateResidualFunction.apply(*args, plan, norm, float(eps), gate_activation)
    return _on_device_of(x, _norm_forward, *args, plan, norm, float(eps), gate_activation, False)[:2]


def _ffn_forward(X, Wg, Wu, Wd, activation, keep):
    """-> (Y, what a backward needs: the tensors as the kernels read them and the reserve, the descriptor)"""
    lib = _ffi.lib()
    X = _row_matrix(X, "node features", most=_FFN_LD)
    rows, Fin = X.shape
    dev = X.device
    Ws = []
    for W, what in ((Wg, "w_gate"), (Wu, "w_up"), (Wd, "w_down")):
        if W.dtype is not X.dtype:
            raise TypeError("%s is %s, the node features are %s" % (what, W.dtype, X.dtype))
        _require_gpu(W, what)
        if W.dim() != 2 or W.get_device() != X.get_device():
            raise ValueError("%s must be a matrix on %s" % (what, dev))
        Ws.append(W if W.is_contiguous() else W.contiguous())
    Wg, Wu, Wd = Ws
    H, Fout = Wg.shape[1], Wd.shape[1]
    if Wg.shape[0] != Fin or Wu.shape != Wg.shape or Wd.shape[0] != H:
        raise ValueError("w_gate and w_up must be [%d, H] and w_down [H, F_out], got %s, %s, %s" %
                         (Fin, tuple(Wg.shape), tuple(Wu.shape), tuple(Wd.shape)))
    desc = _ffi.FfnDesc(rows, min(Fin, _I32), min(H, _I32), min(Fout, _I32), _ffi.FFN_ACT[activation], _DT[X.dtype], min(_ld(X), _I32),
                        1 if keep else 0, 0)
    rbytes, wbytes = lib.agcn_gated_ffn_reserve_bytes(C.byref(desc)), lib.agcn_gated_ffn_forward_workspace_bytes(C.byref(desc))
    if not rbytes:
        _ffi.check(-1)
    reserve = torch.empty(rbytes, dtype=torch.uint8, device=dev)
    ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
    Y = torch.empty((rows, Fout), dtype=X.dtype, device=dev)
    _ffi.check(lib.agcn_gated_ffn_forward(C.byref(desc), X.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), Wd.data_ptr(), Y.data_ptr(),
                                          reserve.data_ptr(), rbytes, ws.data_ptr(), wbytes, _stream(dev)))
    return Y, (X, Wg, Wu, Wd, reserve), desc


class GatedFfnFunction(torch.autograd.Function):
    """Y = (act(X Wg) * (X Wu)) Wd; see gated_ffn."""

    @staticmethod
    def forward(ctx, X, Wg, Wu, Wd, activation):
        Y, saved, ctx.desc = _on_device_of(X, _ffn_forward, X, Wg, Wu, Wd, activation, True)
        ctx.save_for_backward(*saved)
        ctx.read_at = [t.data_ptr() for t in saved[:4]] if Y.dtype is torch.bfloat16 else None
        return Y

    @staticmethod
    @_first_order
    def backward(ctx, dY):
        return _on_device_of(dY, GatedFfnFunction._backward, ctx.desc, ctx.saved_tensors, ctx.read_at, dY, ctx.needs_input_grad)

    @staticmethod
    def _backward(desc, saved, read_at, dY, need):
        lib = _ffi.lib()
        X, Wg, Wu, Wd, reserve = saved
        dev, dtype, rows, Fin, H, Fout = dY.device, dY.dtype, desc.rows, desc.Fin, desc.H, desc.Fout
        at = dY.get_device()
        X = _saved(X, "node features", (rows, Fin), dtype, at, _FFN_LD)
        Wg, Wu = _saved(Wg, "w_gate", (Fin, H), dtype, at).contiguous(), _saved(Wu, "w_up", (Fin, H), dtype, at).contiguous()
        Wd = _saved(Wd, "w_down", (H, Fout), dtype, at).contiguous()
        ldx = _ld(X)
        if read_at is not None:
            # Where the forward could read a bf16 matrix in place it left no aligned copy of it.  One that has moved since and
            # whose rows do not start at 16 bytes is copied to where they do.
            now = [(X.data_ptr() | 2 * ldx) & 15, Wg.data_ptr() & 15, Wu.data_ptr() & 15, Wd.data_ptr() & 15]
            if any(now):
                X, Wg, Wu, Wd = [t.clone(memory_format=torch.contiguous_format) if odd and (t.data_ptr() != was or t is X and ldx != desc.ldx) else t
                                 for t, odd, was in zip((X, Wg, Wu, Wd), now, read_at)]
                ldx = _ld(X)
        if reserve.get_device() != at:
            raise ValueError("what the forward kept came back on %s" % reserve.device)
        if reserve.data_ptr() & 255 or not reserve.is_contiguous():
            reserve = reserve.clone(memory_format=torch.contiguous_format)
        if ldx != desc.ldx:
            desc = _ffi.FfnDesc(rows, Fin, H, Fout, desc.activation, desc.dtype, ldx, desc.training, 0)
        dY = dY.contiguous()
        dX = torch.empty((desc.rows, desc.Fin), dtype=X.dtype, device=dev) if need[0] else None
        dWg, dWu = (torch.empty_like(Wg), torch.empty_like(Wu)) if need[1] or need[2] else (None, None)
        dWd = torch.empty_like(Wd) if need[3] else None
        wbytes = lib.agcn_gated_ffn_backward_workspace_bytes(C.byref(desc))
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        _ffi.check(lib.agcn_gated_ffn_backward(C.byref(desc), X.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), Wd.data_ptr(), dY.data_ptr(),
                                               _ptr(dX), _ptr(dWg), _ptr(dWu), _ptr(dWd), reserve.data_ptr(), reserve.numel(),
                                               ws.data_ptr(), wbytes, _stream(dev)))
        return dX, dWg if need[1] else None, dWu if need[2] else None, dWd, None


def gated_ffn(X, w_gate, w_up, w_down, activation="silu"):
    """Gated feed-forward block over node rows: (act(X w_gate) * (X w_up)) w_down.  X [rows, F], w_gate and w_up [F, H], w_down
    [H, F_out], all float32 or all bfloat16; activation: 'silu', 'gelu' (the erf form), 'relu' or 'sigmoid'.  Every row is a
    row of its own: pad rows that are zero come out zero.  The kernels are chosen by the sizes and by whether a gradient is wanted: a
    row's last bits may differ between batch sizes, and between serving and training."""
    if activation not in _ffi.FFN_ACT:
        raise ValueError("activation must be one of %s" % ", ".join(sorted(_ffi.FFN_ACT)))
    if _wants_grad((X, w_gate, w_up, w_down)):
        return GatedFfnFunction.apply(X, w_gate, w_up, w_down, activation)
    return _on_device_of(X, _ffn_forward, X, w_gate, w_up, w_down, activation, False)[0]
