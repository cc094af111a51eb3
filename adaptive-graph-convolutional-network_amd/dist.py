"""Data parallelism over the GPUs of one node: graphs are independent units, only the
parameter gradients couple them.  Each rank packs its own shard; the single exchange step is
one RCCL all-reduce (SUM) over the flat gradient bucket.  The reference has no multi-GPU code;
SUM (not mean) is right because its loss divides by the GLOBAL batch size
(models/tf_modules/multitask_classifier.py:207-208).

Consequence for callers: anything that divides by the batch size -- `MultitaskHead(..., batch_size=...)`, a hand-written
loss scale -- must be given the GLOBAL batch size (per-rank graphs x world size) on every rank; the SGC layers
themselves are built with the LOCAL graph count (it is the length of their output lists).  `global_batch_size()`
returns the number to use."""
from array import array

import numpy as np
import torch
import torch.distributed as dist

from . import _ffi
from .functional import _no_tangents


def graph_cost(n, Fin, Fout, K):
    """Work model of one graph: n^2 Fin (pairwise distances, L X) + n K Fin Fout (filter GEMM)."""
    n = np.asarray(n, dtype=np.int64)
    return n * n * int(Fin) + n * int(K) * int(Fin) * int(Fout)


def shard_graphs(costs, world_size):
    """Greedy longest-processing-time binning with EQUAL graph counts per rank (weak scaling
    keeps the per-GPU batch fixed).  Deterministic; returns a list of index arrays whose
    concatenation is a permutation of range(len(costs))."""
    costs = np.asarray(costs, dtype=np.int64)
    B = costs.shape[0]
    cap = -(-B // world_size)
    order = np.argsort(-costs, kind="stable")
    load = np.zeros(world_size, dtype=np.int64)
    count = np.zeros(world_size, dtype=np.int64)
    bins = [[] for _ in range(world_size)]
    for g in order:
        open_ranks = np.nonzero(count < cap)[0]
        r = open_ranks[np.argmin(load[open_ranks])]
        bins[r].append(int(g))
        load[r] += costs[g]
        count[r] += 1
    return [np.sort(np.asarray(b, dtype=np.int64)) for b in bins]


def init_from_env(backend=None):
    """torchrun-style rendezvous (RANK / LOCAL_RANK / WORLD_SIZE / MASTER_*).  backend 'nccl'
    is RCCL on ROCm; CPU tests use 'gloo'."""
    import os
    rank = int(os.environ.get("RANK", "0"))
    world = int(os.environ.get("WORLD_SIZE", "1"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    if world > 1 and not dist.is_initialized():
        if backend is None:
            backend = "nccl" if torch.cuda.is_available() else "gloo"
        if backend == "nccl":
            torch.cuda.set_device(local)
            dist.init_process_group(backend, rank=rank, world_size=world,
                                    device_id=torch.device("cuda", local))
        else:
            dist.init_process_group(backend, rank=rank, world_size=world)
    return rank, local, world


def global_batch_size(local_batch_size, group=None):
    """Batch size the loss must divide by under data parallelism (SUM all-reduce): local x world size."""
    if dist.is_available() and dist.is_initialized():
        return int(local_batch_size) * dist.get_world_size(group)
    return int(local_batch_size)


def allreduce_bucket(bucket, group=None):
    """One collective per step over the flat fp32 gradient bucket (61 KB for a 75->64 layer:
    latency-bound on xGMI, so never split it)."""
    if dist.is_available() and dist.is_initialized() and dist.get_world_size(group) > 1:
        dist.all_reduce(bucket, op=dist.ReduceOp.SUM, group=group)
    return bucket


def flatten_grads(tensors):
    """Pack a list of gradient tensors into one flat buffer and return (flat, views)."""
    flat = torch.cat([t.reshape(-1) for t in tensors])
    views, o = [], 0
    for t in tensors:
        views.append(flat[o:o + t.numel()].view_as(t))
        o += t.numel()
    return flat, views


_CLIP_DT = {torch.float32: 0, torch.bfloat16: 1}
_T = torch.Tensor


def _each(method, ts):
    return list(map(method, ts))


def _no_graph(ts):
    """Clipping has no derivative: a loss built on its results would lose these tensors' part in silence."""
    if torch.is_grad_enabled() and True in map(_T.requires_grad.__get__, ts):
        raise _ffi.AgcnError("the results of clipping carry no graph, but a tensor requires grad: call it under torch.no_grad()")
    _no_tangents(ts)


def _looked_over(ts):
    """devices, types, element counts (lists of a hundred tensors and more: each is one pass over the list, made once)"""
    return _each(_T.get_device, ts), [t.dtype for t in ts], _each(_T.numel, ts)


def _clip(ts, clip_norm, out, looked_over):
    lib = _ffi.lib()
    where, types, sizes = looked_over
    if where.count(where[0]) != len(where):
        raise ValueError("all gradients must be on one device")
    if where[0] < 0:
        raise _ffi.AgcnError("gradients must live on the GPU: the clipping kernels have no CPU fallback")
    n = len(ts)
    try:
        dtype = array("i", [_CLIP_DT[t] for t in types])
    except KeyError:
        raise TypeError("gradients must be float32 or bfloat16")
    numel = array("q", sizes)
    ins = array("Q", map(_T.data_ptr, ts))
    outs = None
    if out is not None:
        outs = ins if out is ts else array("Q", map(_T.data_ptr, out))
    dev = ts[0].device
    with torch.cuda.device(dev):
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ln, ld = numel.buffer_info()[0], dtype.buffer_info()[0]
        wbytes = lib.agcn_clip_workspace_bytes(n, ln, ld)
        ws = torch.empty(wbytes, dtype=torch.uint8, device=dev)
        _ffi.check(lib.agcn_clip_by_global_norm(n, ins.buffer_info()[0], None if outs is None else outs.buffer_info()[0], ln, ld,
                                                clip_norm, norm.data_ptr(), ws.data_ptr(), wbytes,
                                                torch._C._cuda_getCurrentRawStream(where[0])))
    return norm


def global_norm(tensors):
    """sqrt of the sum of squares over every element of every tensor (float32 or bfloat16, one device; None entries are
    skipped): a 0-dim device tensor, no synchronisation.  It has no derivative: tensors that require grad are refused outside
    torch.no_grad()."""
    ts = [t.contiguous() for t in tensors if t is not None]
    if not ts:
        raise ValueError("no tensors")
    _no_graph(ts)
    return _clip(ts, 1.0, None, _looked_over(ts))


def clip_by_global_norm(tensors, clip_norm, out=None):
    """Scales a list of gradient tensors (float32 or bfloat16, one device) so that their global norm is at most `clip_norm`:
    out_t = t * clip_norm / max(norm, clip_norm).  Returns (list of clipped tensors, norm before clipping as a 0-dim device tensor);
    nothing synchronises.  None entries stay None.  A norm that is not finite, or that float32 does not hold, makes every
    result NaN (the reference's framework does the same: a broken step is seen, not applied).  The results carry no graph: tensors that require grad are refused outside
    torch.no_grad().  out: contiguous tensors of the same sizes and types to write to;
    `out=tensors` clips in place."""
    clip_norm = float(clip_norm)
    if not clip_norm > 0.0:
        raise ValueError("clip_norm must be positive")
    given, tensors = tensors, list(tensors)
    out = None if out is None else (tensors if out is given else list(out))
    if out is not None and len(out) != len(tensors):
        raise ValueError("out must hold one tensor per gradient (%d), got %d" % (len(tensors), len(out)))
    try:
        whole = bool(tensors) and all(map(_T.is_contiguous, tensors))
    except TypeError:                                      # (a None entry)
        whole = False
    if whole:
        ts = tensors
        _no_graph(ts)
    else:
        at = [i for i, t in enumerate(tensors) if t is not None]
        if not at:
            raise ValueError("no tensors")
        whole = len(at) == len(tensors)
        ts = [tensors[i] for i in at]
        _no_graph(ts)
        ts = [t.contiguous() for t in ts]
    of_ts = _looked_over(ts)
    if out is None:
        os_ = [torch.empty_like(t) for t in ts]
    else:
        os_ = out if whole else [out[i] for i in at]
        if any(o is None for o in os_):
            raise ValueError("out must hold a tensor for every gradient")
        if os_ is not ts:                                  # (in place: the tensors that were looked at above)
            _no_graph(os_)
            if not all(map(_T.is_contiguous, os_)) or _looked_over(os_) != of_ts:
                raise ValueError("out must hold contiguous tensors of the gradients' sizes, types and device")
    norm = _clip(ts, clip_norm, os_, of_ts)
    if out is None:
        if whole:
            return os_, norm
        out = list(tensors)
        for i, o in zip(at, os_):
            out[i] = o
        return out, norm
    torch.autograd.graph.increment_version(os_)            # (written behind torch's back: a saved copy of them is stale)
    return out, norm


class GradBucket(object):
    """ONE flat fp32 bucket behind the `.grad` fields of a list of parameters -- every SGC layer's [weight | bias | M_L | alpha
    (| beta)], the dense tail, the task heads (140 821 floats = 563 KB for SimpleAGCN + DenseMol + 12 heads) -- so
    that a whole-network step needs ONE collective.  Each parameter's `.grad` is a view into the bucket; autograd accumulates
    into the views in place, `zero()` (one memset) starts a step, `all_reduce()` (one RCCL all-reduce, SUM: the reference's
    loss divides by the GLOBAL batch size, multitask_classifier.py:207-208) ends it.  Works inside `engine.GraphedStep`:

        bucket = dist.GradBucket(params)
        def step():
            bucket.zero()
            loss(model(batch)).backward()
            bucket.all_reduce()            # captured into the HIP graph behind the last backward kernel (RCCL), or leave it
        gs = GraphedStep(step, dev)        # out of `step` and call bucket.all_reduce() after gs.replay() (same stream)

    Parameters that get no gradient (M_L in reference mode) keep a zero section."""

    def __init__(self, params):
        self.params = [p for p in params if p is not None and p.requires_grad]
        if not self.params:
            raise ValueError("no trainable parameters")
        dev = self.params[0].device
        total = sum(p.numel() for p in self.params)
        self.flat = torch.zeros(total, dtype=torch.float32, device=dev)
        self.views, o = [], 0
        for p in self.params:
            if p.dtype != torch.float32 or p.device != dev:
                raise ValueError("GradBucket holds fp32 parameters of one device")
            self.views.append(self.flat[o:o + p.numel()].view_as(p))
            o += p.numel()
        self.attach()

    def attach(self):
        """(Re)points every parameter's .grad at its section of the bucket (after something set it to None)."""
        for p, v in zip(self.params, self.views):
            if p.grad is not v:
                p.grad = v

    def zero(self):
        self.attach()
        self.flat.zero_()

    def all_reduce(self, group=None):
        return allreduce_bucket(self.flat, group)

    def clip(self, clip_norm):
        """Clips the whole bucket by its global norm, in place (after `all_reduce`: the norm of the SUMMED gradients, the same on
        every rank, without another collective).  Returns the norm before clipping (a 0-dim device tensor: no synchronisation)."""
        return clip_by_global_norm([self.flat], clip_norm, out=[self.flat])[1]

    def nbytes(self):
        return self.flat.numel() * 4
