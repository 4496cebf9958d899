"""Host-side mirror of the MegRay interface for the virtual-rank backend.

Names, argument meaning and error behaviour follow the reference's C++ API
(include/megray/common.h, include/megray/communicator.h): ``DType`` / ``ReduceOp`` / ``Status``
carry the same numeric values, lengths are element counts, contract violations raise
``MegRayError`` where the reference throws ``MegRay::Exception``.

The flat functions here take the buffers of all N virtual ranks at once (device pointers as ints,
or anything with ``data_ptr()``); they are thin wrappers over the C ABI.
"""
import ctypes
import enum

from . import _lib


class Status(enum.IntEnum):
    OK = 0
    SYS_ERROR = 1
    CUDA_ERR = 2
    NCCL_ERR = 3
    UCX_ERR = 4
    ENV_ERROR = 5
    INVALID_ARGUMENT = 6
    INVALID_USAGE = 7
    UNEXPECTED_ERR = 8
    NOT_IMPLEMENTED = 9
    HIP_ERR = 10
    RCCL_ERR = 11


class Backend(enum.IntEnum):
    NCCL = 0
    UCX = 1
    RCCL = 2
    SHM = 3
    VRANK = 4


class DType(enum.IntEnum):
    INT8 = 0
    UINT8 = 1
    INT32 = 2
    UINT32 = 3
    INT64 = 4
    UINT64 = 5
    FLOAT16 = 6
    FLOAT32 = 7
    FLOAT64 = 8
    CHAR = 9
    # element types of the folds with an epilogue (RmsNormPlan ... AdamWPlan) alone; every other call refuses them
    BFLOAT16 = 32
    FLOAT8_E4M3 = 33


class ReduceOp(enum.IntEnum):
    SUM = 0
    MAX = 1
    MIN = 2


class FoldOrder(enum.IntEnum):
    UCX = 0
    SHM = 1
    RANK0 = 2


class Schedule(enum.IntEnum):
    FUSED = 0
    TWO_PHASE = 1
    RING = 2


class Collective(enum.IntEnum):
    ALL_REDUCE = 0
    REDUCE_SCATTER = 1
    ALL_GATHER = 2
    ALL_TO_ALL = 3
    SCATTER = 4
    GATHER = 5
    BROADCAST = 6
    REDUCE2 = 7
    REDUCE = 8


MAX_RANKS = 16


class MegRayError(RuntimeError):
    """Raised where the reference throws MegRay::Exception or returns a non-OK Status."""

    def __init__(self, status, message):
        super().__init__(f"[{Status(status).name}] {message}")
        self.status = Status(status)
        self.message = message


def _check(status):
    if status != 0:
        raise MegRayError(status, _lib.load().mrv_last_error().decode())


def _ptr(buf):
    if buf is None:
        return None
    if hasattr(buf, "data_ptr"):
        return buf.data_ptr()
    return int(buf)


def _ptr_array(bufs):
    arr = (ctypes.c_void_p * len(bufs))()
    for i, b in enumerate(bufs):
        arr[i] = _ptr(b)
    return arr


def _rank_arrays(sendbuffs, recvbuffs, nranks=None):
    """The two per-rank pointer arrays of a flat call, both `nranks` long (the library indexes both up to
    nranks): lists of different lengths are rejected here, like any other invalid argument; a shorter list is
    allowed only where `nranks` says that its missing ranks are not used (root-only forms pad with None)."""
    n = nranks if nranks is not None else len(sendbuffs)
    if nranks is None and len(recvbuffs) != len(sendbuffs):
        raise MegRayError(Status.INVALID_ARGUMENT,
                          f"{len(sendbuffs)} send buffers but {len(recvbuffs)} receive buffers: one of each per rank")
    if len(sendbuffs) > n or len(recvbuffs) > n:
        raise MegRayError(Status.INVALID_ARGUMENT, f"more buffers than ranks ({n})")
    pad = lambda bufs: list(bufs) + [None] * (n - len(bufs))  # noqa: E731
    return _ptr_array(pad(sendbuffs)), _ptr_array(pad(recvbuffs)), n


def _stream(stream):
    if stream is None:
        return None
    if hasattr(stream, "cuda_stream"):
        return stream.cuda_stream
    return int(stream)


def get_dtype_size(dtype):
    """MegRay::get_dtype_size (src/core/common.cpp:19-38); raises 'unknown dtype'."""
    size = _lib.load().mrv_dtype_size(int(dtype))
    if size == 0:
        raise MegRayError(Status.INVALID_ARGUMENT, _lib.load().mrv_last_error().decode())
    return size


def reduce(i0, i1, o, length, dtype, op, stream=None):
    """o = i0 OP i1 (MegRay::reduce, src/ucx/utils.h:21-22)."""
    _check(_lib.load().mrv_reduce(_ptr(i0), _ptr(i1), _ptr(o), length, int(dtype), int(op), _stream(stream)))


def all_reduce(sendbuffs, recvbuffs, length, dtype, op, order=FoldOrder.UCX, schedule=Schedule.FUSED,
               stream=None):
    send, recv, nranks = _rank_arrays(sendbuffs, recvbuffs)
    _check(_lib.load().mrv_all_reduce(send, recv, nranks, length,
                                      int(dtype), int(op), int(order), int(schedule), _stream(stream)))


def reduce_scatter(sendbuffs, recvbuffs, recvlen, dtype, op, order=FoldOrder.UCX, stream=None):
    send, recv, nranks = _rank_arrays(sendbuffs, recvbuffs)
    _check(_lib.load().mrv_reduce_scatter(send, recv, nranks, recvlen,
                                          int(dtype), int(op), int(order), _stream(stream)))


def all_gather(sendbuffs, recvbuffs, sendlen, dtype, stream=None):
    send, recv, nranks = _rank_arrays(sendbuffs, recvbuffs)
    _check(_lib.load().mrv_all_gather(send, recv, nranks, sendlen,
                                      int(dtype), _stream(stream)))


def all_to_all(sendbuffs, recvbuffs, length, dtype, stream=None):
    send, recv, nranks = _rank_arrays(sendbuffs, recvbuffs)
    _check(_lib.load().mrv_all_to_all(send, recv, nranks, length,
                                      int(dtype), _stream(stream)))


def scatter(sendbuff_root, recvbuffs, recvlen, dtype, root, stream=None):
    _check(_lib.load().mrv_scatter(_ptr(sendbuff_root), _ptr_array(recvbuffs), len(recvbuffs), recvlen,
                                   int(dtype), root, _stream(stream)))


def gather(sendbuffs, recvbuff_root, sendlen, dtype, root, stream=None):
    _check(_lib.load().mrv_gather(_ptr_array(sendbuffs), _ptr(recvbuff_root), len(sendbuffs), sendlen,
                                  int(dtype), root, _stream(stream)))


def broadcast(sendbuff_root, recvbuffs, length, dtype, root, stream=None):
    _check(_lib.load().mrv_broadcast(_ptr(sendbuff_root), _ptr_array(recvbuffs), len(recvbuffs), length,
                                     int(dtype), root, _stream(stream)))


def reduce_to_root(sendbuffs, recvbuff_root, length, dtype, op, root, order=FoldOrder.UCX, stream=None):
    _check(_lib.load().mrv_reduce_to_root(_ptr_array(sendbuffs), _ptr(recvbuff_root), len(sendbuffs), length,
                                          int(dtype), int(op), int(order), root, _stream(stream)))


def probe_bounded_wait(limit_us, stream=None):
    """Launch one cross-stream wait that nothing will ever satisfy, with a time limit of `limit_us`; returns how
    many waits gave up (1).  mrv_probe_bounded_wait."""
    gave_up = ctypes.c_uint64(0)
    _check(_lib.load().mrv_probe_bounded_wait(int(limit_us), _stream(stream), ctypes.byref(gave_up)))
    return gave_up.value


def _written_array(written, count):
    if written is None:
        return None
    if len(written) != count:
        raise MegRayError(Status.INVALID_ARGUMENT, f"{count} buffers but {len(written)} written flags")
    return (ctypes.c_ubyte * max(count, 1))(*[1 if w else 0 for w in written])


def rank_buffers_layout(sizes, collective=None, written=None):
    """-> (offsets, total): where buffers of `sizes` bytes go inside one allocation so that a collective over them is
    served well by the memory system (buffers of 8 MiB and more an odd multiple of 128 MiB apart; with
    `collective` ALL_GATHER the buffers flagged in `written` a multiple of 128 MiB plus 32 MiB apart).
    mrv_rank_buffers_layout / mrv_rank_buffers_layout_for; needs no GPU."""
    count = len(sizes)
    arr = (ctypes.c_size_t * max(count, 1))(*[int(b) for b in sizes])
    offs = (ctypes.c_size_t * max(count, 1))()
    total = ctypes.c_size_t(0)
    if collective is None:
        _check(_lib.load().mrv_rank_buffers_layout(count, arr, offs, ctypes.byref(total)))
    else:
        _check(_lib.load().mrv_rank_buffers_layout_for(int(collective), count, arr, _written_array(written, count), offs,
                                                       ctypes.byref(total)))
    return list(offs)[:count], total.value


class RankBuffers:
    """Buffers of `sizes` bytes in one device allocation, placed by mrv_rank_buffers_alloc; `.ptrs` are their
    addresses.  free() (or the end of a with block) releases the allocation."""

    def __init__(self, sizes, collective=None, written=None):
        count = len(sizes)
        arr = (ctypes.c_size_t * max(count, 1))(*[int(b) for b in sizes])
        ptrs = (ctypes.c_void_p * max(count, 1))()
        base = ctypes.c_void_p(None)
        if collective is None:
            _check(_lib.load().mrv_rank_buffers_alloc(count, arr, ptrs, ctypes.byref(base)))
        else:
            _check(_lib.load().mrv_rank_buffers_alloc_for(int(collective), count, arr, _written_array(written, count),
                                                          ptrs, ctypes.byref(base)))
        self.ptrs = [int(p or 0) for p in ptrs][:count]
        self.sizes = [int(b) for b in sizes]
        self._base = base

    def free(self):
        if self._base is not None and self._base.value:
            _check(_lib.load().mrv_rank_buffers_free(self._base))
        self._base = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.free()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def place_tensors(torch, specs, device="cuda", collective=None, written=None):
    """Tensors of the given (numel, dtype) pairs as views into ONE torch allocation, placed by rank_buffers_layout:
    the way to hand torch-owned memory to a collective in the placement the library recommends (`collective` and
    `written` as for rank_buffers_layout).  The views keep the allocation alive."""
    sizes = [int(numel) * torch.empty((), dtype=dtype).element_size() for numel, dtype in specs]
    offsets, total = rank_buffers_layout(sizes, collective, written)
    align = 2 << 20
    arena = torch.empty(total + align, dtype=torch.uint8, device=device)
    skew = (-arena.data_ptr()) % align
    return [arena[skew + off:skew + off + size].view(dtype) for off, size, (_, dtype) in zip(offsets, sizes, specs)]


def chunk_partition(length, nchunks):
    sizes = (ctypes.c_size_t * nchunks)()
    offs = (ctypes.c_size_t * nchunks)()
    _check(_lib.load().mrv_chunk_partition(length, nchunks, sizes, offs))
    return list(sizes), list(offs)


def fold_order(collective, order, nranks, chunk):
    """-> (ranks, new_wins_ties, nchunks, owner)"""
    ranks = (ctypes.c_uint32 * max(nranks, 1))()
    new_wins = ctypes.c_int(0)
    nchunks = ctypes.c_uint32(0)
    owner = ctypes.c_uint32(0)
    _check(_lib.load().mrv_fold_order(int(collective), int(order), nranks, chunk, ranks, ctypes.byref(new_wins),
                                      ctypes.byref(nchunks), ctypes.byref(owner)))
    return list(ranks)[:nranks], bool(new_wins.value), nchunks.value, owner.value


def describe(collective, sendptrs, recvptrs, count, dtype, order=FoldOrder.UCX, schedule=Schedule.FUSED,
             root=0, nranks=None):
    """Plan a collective on the host only.  -> (list of run dicts, bytes_read, bytes_written)"""
    nranks = nranks if nranks is not None else max(len(sendptrs), len(recvptrs))
    send, recv, nranks = _rank_arrays(sendptrs, recvptrs, nranks)
    cap = 4096
    runs = (_lib.PlanRun * cap)()
    n = ctypes.c_size_t(0)
    br = ctypes.c_uint64(0)
    bw = ctypes.c_uint64(0)
    _check(_lib.load().mrv_describe(int(collective), send, recv, nranks, count,
                                    int(dtype), int(order), int(schedule), root, runs, cap, ctypes.byref(n),
                                    ctypes.byref(br), ctypes.byref(bw)))
    out = []
    for i in range(min(n.value, cap)):
        r = runs[i]
        out.append({name: getattr(r, name) for name, _ in _lib.PlanRun._fields_})
    return out, br.value, bw.value


class CollectivePlan:
    """A collective planned once and launched many times (mrv_plan_*).  `graph=True` instantiates
    the launches of a multi-launch plan as one HIP graph.  The buffers must outlive the plan."""

    def __init__(self, collective, sendbuffs, recvbuffs, count, dtype, op=ReduceOp.SUM, order=FoldOrder.UCX,
                 schedule=Schedule.FUSED, root=0, graph=False, nranks=None):
        self._h = ctypes.c_void_p()
        self._keep = (sendbuffs, recvbuffs)
        nranks = nranks if nranks is not None else max(len(sendbuffs), len(recvbuffs))
        send, recv, nranks = _rank_arrays(sendbuffs, recvbuffs, nranks)
        _check(_lib.load().mrv_plan_create(int(collective), send, recv, nranks,
                                           count, int(dtype), int(op), int(order), int(schedule), root,
                                           1 if graph else 0, ctypes.byref(self._h)))
        self._launch = _lib.load().mrv_plan_launch

    @property
    def launch_count(self):
        return _lib.load().mrv_plan_launch_count(self._h)

    def launch(self, stream=None):
        status = self._launch(self._h, _stream(stream))
        if status:
            _check(status)

    def close(self):
        if self._h:
            _lib.load().mrv_plan_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # at interpreter shutdown the modules this needs may be gone already
            pass


# ---------------------------------------------------------------------------------------------
# folds with an epilogue: what a tensor- or data-parallel model does with a sum right behind its reduction

def _optional_array(bufs, n, what):
    if bufs is None:
        return None
    if len(bufs) != n:
        raise MegRayError(Status.INVALID_ARGUMENT, f"{len(bufs)} {what}, {n} expected")
    return _ptr_array(bufs)


def _copies(collective, nranks):
    """How many copies of a residual a call reads: it is replicated behind an all_reduce, every rank's own behind a
    reduce_scatter."""
    return 1 if int(collective) == Collective.ALL_REDUCE else nranks


def _rms_norm_call(collective, sendbuffs, outs, weight, rows, cols, dtype, eps, residuals=None, residual_outs=None,
                   scales=None, residual_dtype=None, weight_dtype=None, out_dtype=None, send_stride=0, residual_stride=0,
                   residual_out_stride=0, out_stride=0):
    n = len(sendbuffs)
    pick = lambda t: int(dtype if t is None else t)  # noqa: E731
    return _lib.RmsNormCall(
        sendbuffs=_ptr_array(sendbuffs), residuals=_optional_array(residuals, _copies(collective, n), "residuals"),
        weight=_ptr(weight), residual_outs=_optional_array(residual_outs, n, "residual outputs"),
        outs=_optional_array(outs, n, "outputs"), scales=_optional_array(scales, n, "scale buffers"), rows=rows, cols=cols,
        send_stride=send_stride, residual_stride=residual_stride, residual_out_stride=residual_out_stride,
        out_stride=out_stride, nranks=n, dtype=int(dtype), residual_dtype=pick(residual_dtype),
        weight_dtype=pick(weight_dtype), out_dtype=pick(out_dtype), eps=eps)


def _rms_norm_backward_call(collective, sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps,
                            residual_grads=None, send_grads=None, weight_grads=None, workspace=None, workspace_bytes=None,
                            residual_dtype=None, weight_dtype=None, send_stride=0, hidden_stride=0, residual_grad_stride=0,
                            residual_out_grad_stride=0, send_grad_stride=0):
    n = len(sendbuffs)
    pick = lambda t: int(dtype if t is None else t)  # noqa: E731
    if workspace_bytes is None:
        workspace_bytes = workspace.numel() * workspace.element_size() if hasattr(workspace, "numel") else 0
    return _lib.RmsNormBackwardCall(
        sendbuffs=_ptr_array(sendbuffs), hiddens=_optional_array(hiddens, _copies(collective, n), "hidden states"),
        residual_grads=_optional_array(residual_grads, _copies(collective, n), "residual gradients"), weight=_ptr(weight),
        residual_out_grads=_optional_array(residual_out_grads, n, "residual gradient outputs"),
        send_grads=_optional_array(send_grads, n, "send gradients"),
        weight_grads=_optional_array(weight_grads, n, "weight gradients"), workspace=_ptr(workspace),
        workspace_bytes=workspace_bytes, rows=rows, cols=cols, send_stride=send_stride, hidden_stride=hidden_stride,
        residual_grad_stride=residual_grad_stride, residual_out_grad_stride=residual_out_grad_stride,
        send_grad_stride=send_grad_stride, nranks=n, dtype=int(dtype), residual_dtype=pick(residual_dtype),
        weight_dtype=pick(weight_dtype), eps=eps)


def all_reduce_rms_norm(sendbuffs, outs, weight, rows, cols, dtype, eps, stream=None, **more):
    """h = residual + sum of sendbuffs, outs = h / sqrt(mean(h * h) + eps) * weight, both to every rank (mrv_rms_norm).

    Optional: residuals=[one copy], residual_outs (h, one per rank), scales (one per rank, with out_dtype INT8 or
    FLOAT8_E4M3), residual_dtype, weight_dtype, out_dtype (default: dtype), and the strides from row to row in elements:
    send_stride, residual_stride, residual_out_stride, out_stride."""
    call = _rms_norm_call(Collective.ALL_REDUCE, sendbuffs, outs, weight, rows, cols, dtype, eps, **more)
    _check(_lib.load().mrv_rms_norm(int(Collective.ALL_REDUCE), call, _stream(stream)))


def reduce_scatter_rms_norm(sendbuffs, outs, weight, rows, cols, dtype, eps, stream=None, **more):
    """The same behind a reduce_scatter: rank r gets `rows` rows, r * rows and following, of the fold; residuals, residual_outs,
    outs and scales are each rank's own (mrv_rms_norm)."""
    call = _rms_norm_call(Collective.REDUCE_SCATTER, sendbuffs, outs, weight, rows, cols, dtype, eps, **more)
    _check(_lib.load().mrv_rms_norm(int(Collective.REDUCE_SCATTER), call, _stream(stream)))


def all_reduce_rms_norm_backward(sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps, stream=None, **more):
    """Backward of all_reduce_rms_norm: sendbuffs hold the ranks' partial gradients of its outs, hiddens=[one copy of h]
    (mrv_rms_norm_backward).  residual_out_grads (or None) get the gradient of the residual and of every forward send buffer.

    Optional: residual_grads=[one copy] (the gradient that arrives at h from elsewhere), send_grads (the same gradient
    in `dtype`), weight_grads (cols floats per rank; they need workspace=, of rms_norm_backward_workspace() bytes), residual_dtype, weight_dtype, and the
    strides send_stride, hidden_stride, residual_grad_stride, residual_out_grad_stride, send_grad_stride."""
    call = _rms_norm_backward_call(Collective.ALL_REDUCE, sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps, **more)
    _check(_lib.load().mrv_rms_norm_backward(int(Collective.ALL_REDUCE), call, _stream(stream)))


def reduce_scatter_rms_norm_backward(sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps, stream=None, **more):
    """Backward of reduce_scatter_rms_norm: hiddens, residual_grads and all outputs are each rank's own rows; weight_grads
    are sums over the rank's rows (mrv_rms_norm_backward)."""
    call = _rms_norm_backward_call(Collective.REDUCE_SCATTER, sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps, **more)
    _check(_lib.load().mrv_rms_norm_backward(int(Collective.REDUCE_SCATTER), call, _stream(stream)))


def rms_norm_backward_workspace(collective, nranks, rows, cols):
    """Bytes of workspace a backward with weight gradients needs (mrv_rms_norm_backward_workspace)."""
    size = ctypes.c_size_t(0)
    _check(_lib.load().mrv_rms_norm_backward_workspace(int(collective), nranks, rows, cols, ctypes.byref(size)))
    return size.value


class _NormPlan:
    def __init__(self, create, collective, call, keep):
        self._h = ctypes.c_void_p()
        self._keep = keep  # the buffers must outlive the plan
        _check(create(int(collective), call, ctypes.byref(self._h)))
        self._launch = _lib.load().mrv_norm_plan_launch

    @property
    def launch_count(self):
        return _lib.load().mrv_norm_plan_launch_count(self._h)

    def launch(self, stream=None):
        status = self._launch(self._h, _stream(stream))
        if status:
            _check(status)

    def close(self):
        if self._h:
            _lib.load().mrv_norm_plan_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # at interpreter shutdown the modules this needs may be gone already
            pass


class RmsNormPlan(_NormPlan):
    """all_reduce_rms_norm / reduce_scatter_rms_norm planned once and launched many times (mrv_rms_norm_plan_create): the same
    arguments behind `collective`."""

    def __init__(self, collective, sendbuffs, outs, weight, rows, cols, dtype, eps, **more):
        call = _rms_norm_call(collective, sendbuffs, outs, weight, rows, cols, dtype, eps, **more)
        super().__init__(_lib.load().mrv_rms_norm_plan_create, collective, call, (sendbuffs, outs, weight, more))


class RmsNormBackwardPlan(_NormPlan):
    """The backward calls planned once and launched many times (mrv_rms_norm_backward_plan_create)."""

    def __init__(self, collective, sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps, **more):
        call = _rms_norm_backward_call(collective, sendbuffs, hiddens, weight, residual_out_grads, rows, cols, dtype, eps, **more)
        super().__init__(_lib.load().mrv_rms_norm_backward_plan_create, collective, call,
                         (sendbuffs, hiddens, weight, residual_out_grads, more))


class AdamWPlan:
    """AdamW over many tensors whose gradients are still apart on the ranks (mrv_adamw_*).

    grads[r][t]: rank r's gradient of tensor t, lengths[t] elements of grad_dtype; params[r][t] likewise, written by step().
    masters[t]: the 32-bit parameters (None with FLOAT32 params: rank 0's are the masters).  exp_avgs, exp_avg_sqs: floats, or
    with state_dtype FLOAT8_E4M3 codes with a float for each 256 elements in exp_avg_scales[t], exp_avg_sq_scales[t].
    Without params a plan has grad_norm() alone.  The tensors must outlive the plan, and stay where they are.  The plan owns a
    table in device memory that its launches read: keep the plan as long as any graph into which its calls were captured; close(), and
    the end of the last reference, free the table."""

    def __init__(self, grads, lengths, grad_dtype, params=None, param_dtype=None, masters=None, exp_avgs=None, exp_avg_sqs=None,
                 state_dtype=DType.FLOAT32, exp_avg_scales=None, exp_avg_sq_scales=None, weight_decays=None):
        self._h = ctypes.c_void_p()
        self._keep = (grads, params, masters, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales)
        n = len(lengths)

        def ranks(lists, what):
            if lists is None:
                return None
            if any(len(x) != n for x in lists):
                raise MegRayError(Status.INVALID_ARGUMENT, f"every rank has {n} {what}")
            return _ptr_array([t for x in lists for t in x])

        if weight_decays is not None and len(weight_decays) != n:
            raise MegRayError(Status.INVALID_ARGUMENT, f"{len(weight_decays)} weight decays for {n} tensors")
        call = _lib.AdamwTensors(
            ntensors=n, lens=(ctypes.c_size_t * max(n, 1))(*lengths), grads=ranks(grads, "gradients"), params=ranks(params, "parameters"),
            masters=_optional_array(masters, n, "masters"), exp_avgs=_optional_array(exp_avgs, n, "running means"),
            exp_avg_sqs=_optional_array(exp_avg_sqs, n, "running means of squares"),
            exp_avg_scales=_optional_array(exp_avg_scales, n, "scale buffers"),
            exp_avg_sq_scales=_optional_array(exp_avg_sq_scales, n, "scale buffers"),
            weight_decays=None if weight_decays is None else (ctypes.c_float * max(n, 1))(*weight_decays),
            grad_ranks=len(grads), param_ranks=0 if params is None else len(params), grad_dtype=int(grad_dtype),
            param_dtype=int(grad_dtype if param_dtype is None else param_dtype), state_dtype=int(state_dtype))
        _check(_lib.load().mrv_adamw_create(call, ctypes.byref(self._h)))
        self._norm_bytes = 4 * _lib.load().mrv_adamw_norm_floats(self._h)
        self._step = _lib.load().mrv_adamw_step
        self._norm = _lib.load().mrv_adamw_grad_norm

    @property
    def norm_floats(self):
        """Floats that grad_norm()'s `out` has to hold."""
        return self._norm_bytes // 4

    def grad_norm(self, out, grad_scale=1.0, max_norm=float("inf"), stream=None):
        """out[0] = the norm of grad_scale * the folded gradients, out[1] = min(1, max_norm / (norm + 1e-6)), NaN where the norm is
        not finite; what follows is scratch (mrv_adamw_grad_norm)."""
        if hasattr(out, "numel") and out.numel() * out.element_size() < self._norm_bytes:
            raise MegRayError(Status.INVALID_ARGUMENT, f"out has to hold {self.norm_floats} floats")
        status = self._norm(self._h, grad_scale, max_norm, _ptr(out), _stream(stream))
        if status:
            _check(status)

    def step(self, lr, step, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, clip=None, stream=None):
        """One AdamW step, number `step` (from 1 on), on grad_scale * clip * the folded gradients; clip: a float in device
        memory (grad_norm()'s out[1:], say).  A step whose clip is not finite changes nothing (mrv_adamw_step)."""
        if step < 1:
            raise MegRayError(Status.INVALID_ARGUMENT, "step counts from 1")
        args = _lib.AdamwStepArgs(lr=lr, beta1=beta1, beta2=beta2, eps=eps, grad_scale=grad_scale, step=step, clip=_ptr(clip))
        status = self._step(self._h, args, _stream(stream))
        if status:
            _check(status)

    def close(self):
        if self._h:
            _lib.load().mrv_adamw_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # at interpreter shutdown the modules this needs may be gone already
            pass


# ---------------------------------------------------------------------------------------------
# the Communicator API, one object per rank (include/megray/communicator.h:32-123)

def get_free_port():
    """MegRay::get_free_port (include/megray/server.h:21)."""
    port = _lib.load().mrv_get_free_port()
    if port <= 0:
        raise MegRayError(Status.SYS_ERROR, _lib.load().mrv_last_error().decode())
    return port


def create_server(nranks, port):
    """MegRay::create_server (include/megray/server.h:24)."""
    _check(_lib.load().mrv_create_server(nranks, port))


class Client:
    """MegRay::Client (include/megray/client.h:24-49): host-side barrier / broadcast / allgather."""

    def __init__(self, nranks, rank):
        self._h = ctypes.c_void_p()
        self.nranks = nranks
        _check(_lib.load().mrv_client_create(nranks, rank, ctypes.byref(self._h)))

    def connect(self, master_ip, port):
        _check(_lib.load().mrv_client_connect(self._h, master_ip.encode(), port))

    def barrier(self):
        _check(_lib.load().mrv_client_barrier(self._h))

    def broadcast(self, data, root, is_root):
        """data: bytes on the root (any bytes-like of the same length elsewhere) -> bytes"""
        out = ctypes.create_string_buffer(len(data))
        src = ctypes.create_string_buffer(bytes(data), len(data)) if is_root else None
        _check(_lib.load().mrv_client_broadcast(self._h, src, out, len(data), root))
        return out.raw

    def allgather(self, data):
        out = ctypes.create_string_buffer(len(data) * self.nranks)
        src = ctypes.create_string_buffer(bytes(data), len(data))
        _check(_lib.load().mrv_client_allgather(self._h, src, out, len(data)))
        return out.raw

    def close(self):
        if self._h:
            _lib.load().mrv_client_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # at interpreter shutdown the modules this needs may be gone already
            pass


class Communicator:
    """One rank's communicator, as returned by MegRay::get_communicator (include/megray.h:33-34).

    Every method takes the device pointers of THIS rank and an optional stream, and must be called
    from this rank's own thread; it returns when all ranks of the group have made the same call
    and the work is enqueued.
    """

    def __init__(self, nranks, rank, backend=Backend.VRANK):
        self._h = ctypes.c_void_p()
        self.nranks, self.rank = nranks, rank
        _check(_lib.load().mrv_comm_create(nranks, rank, int(backend), ctypes.byref(self._h)))

    def init(self, master_ip, port):
        _check(_lib.load().mrv_comm_init(self._h, master_ip.encode(), port))

    def init_callback(self, broadcast):
        """Communicator::init(BcastCallback) (include/megray/communicator.h:49): form the group through the
        caller's own broadcast instead of the bootstrap server.  `broadcast(data: bytearray) -> bytes-like` is
        called once on this rank's thread with this rank's bytes (meaningful on rank 0 only) and returns rank 0's."""
        def trampoline(data, length, _user):
            mine = ctypes.string_at(data, length)
            got = bytes(broadcast(bytearray(mine)))
            if len(got) != length:
                raise ValueError(f"the broadcast returned {len(got)} bytes, {length} were handed in")
            ctypes.memmove(data, got, length)
        fn = _lib.BCAST_FN(trampoline)
        _check(_lib.load().mrv_comm_init_callback(self._h, fn, None))

    def check(self, stream=None):
        """Raises if a stream wait of this rank's group has given up (mrv_comm_check; synchronous)."""
        _check(_lib.load().mrv_comm_check(self._h, _stream(stream)))

    def stats(self):
        """{"collectives", "plans_built", "sleeps"} of this rank's group since it was formed (mrv_comm_stats)."""
        c, p, s = ctypes.c_uint64(0), ctypes.c_uint64(0), ctypes.c_uint64(0)
        _check(_lib.load().mrv_comm_stats(self._h, ctypes.byref(c), ctypes.byref(p), ctypes.byref(s)))
        return {"collectives": c.value, "plans_built": p.value, "sleeps": s.value}

    def configure(self, order=FoldOrder.UCX, schedule=Schedule.FUSED):
        _check(_lib.load().mrv_comm_configure(self._h, int(order), int(schedule)))

    def send(self, sendbuff, length, dtype, rank, stream=None):
        _check(_lib.load().mrv_comm_send(self._h, _ptr(sendbuff), length, int(dtype), rank, _stream(stream)))

    def recv(self, recvbuff, length, dtype, rank, stream=None):
        _check(_lib.load().mrv_comm_recv(self._h, _ptr(recvbuff), length, int(dtype), rank, _stream(stream)))

    def scatter(self, sendbuff, recvbuff, recvlen, dtype, root, stream=None):
        _check(_lib.load().mrv_comm_scatter(self._h, _ptr(sendbuff), _ptr(recvbuff), recvlen, int(dtype), root,
                                            _stream(stream)))

    def gather(self, sendbuff, recvbuff, sendlen, dtype, root, stream=None):
        _check(_lib.load().mrv_comm_gather(self._h, _ptr(sendbuff), _ptr(recvbuff), sendlen, int(dtype), root,
                                           _stream(stream)))

    def all_to_all(self, sendbuff, recvbuff, length, dtype, stream=None):
        _check(_lib.load().mrv_comm_all_to_all(self._h, _ptr(sendbuff), _ptr(recvbuff), length, int(dtype),
                                               _stream(stream)))

    def all_gather(self, sendbuff, recvbuff, sendlen, dtype, stream=None):
        _check(_lib.load().mrv_comm_all_gather(self._h, _ptr(sendbuff), _ptr(recvbuff), sendlen, int(dtype),
                                               _stream(stream)))

    def all_reduce(self, sendbuff, recvbuff, length, dtype, op, stream=None):
        _check(_lib.load().mrv_comm_all_reduce(self._h, _ptr(sendbuff), _ptr(recvbuff), length, int(dtype),
                                               int(op), _stream(stream)))

    def all_reduce_no_alloc(self, sendbuff, recvbuff, length, dtype, op, stream=None):
        """all_reduce for callers that may not allocate device memory: the counters that order the ranks'
        streams are a block of the library's static device array (mrv_comm_all_reduce_no_alloc)."""
        _check(_lib.load().mrv_comm_all_reduce_no_alloc(self._h, _ptr(sendbuff), _ptr(recvbuff), length, int(dtype),
                                                        int(op), _stream(stream)))

    def reduce_scatter(self, sendbuff, recvbuff, recvlen, dtype, op, stream=None):
        _check(_lib.load().mrv_comm_reduce_scatter(self._h, _ptr(sendbuff), _ptr(recvbuff), recvlen, int(dtype),
                                                   int(op), _stream(stream)))

    def broadcast(self, sendbuff, recvbuff, length, dtype, root, stream=None):
        _check(_lib.load().mrv_comm_broadcast(self._h, _ptr(sendbuff), _ptr(recvbuff), length, int(dtype), root,
                                              _stream(stream)))

    def reduce(self, sendbuff, recvbuff, length, dtype, op, root, stream=None):
        _check(_lib.load().mrv_comm_reduce(self._h, _ptr(sendbuff), _ptr(recvbuff), length, int(dtype), int(op),
                                           root, _stream(stream)))

    def group_start(self):
        _check(_lib.load().mrv_comm_group_start(self._h))

    def group_end(self):
        _check(_lib.load().mrv_comm_group_end(self._h))

    def close(self):
        if self._h:
            _lib.load().mrv_comm_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # at interpreter shutdown the modules this needs may be gone already
            pass


def get_communicator(nranks, rank, backend=Backend.VRANK):
    """MegRay::get_communicator (include/megray.h:33-34); raises 'unknown backend' like src/megray.cpp:56-57."""
    return Communicator(nranks, rank, backend)
