"""Rows in groups: products, joins and gradients over rows that an index sorts into groups, with the groups' sizes known
on the device only (tfh_row_groups and the calls that take it, include/tenferro_hip.h).  No counterpart in the
reference; beside HipBackend.plan_grouped, whose groups' extents are fixed when the plan is made.

    groups = RowGroups.from_ids(expert_of, n_experts)              # [tokens, fan] indices, on the GPU
    h = ragged_gemm(x, w_up, groups, gather=True)                  # [tokens * fan, N], group by group
    y = combine_rows(ragged_gemm(act(h), w_down, groups), groups, gates)      # [tokens, K]

Operands are torch CUDA tensors or GpuMemory Tensors of bf16, f16, f32 or f64, with any strides (scales: contiguous); a result is of the
first operand's kind.  Work is enqueued on `stream` (default: torch's current stream of the operands' device), never
waited for, and allocates through torch only, so the calls can be captured into a graph: on the current stream, and behind
no event from before the capture (when the graph runs is the caller's to order).  On a stream other than the current one the
caller orders the operands' earlier and the results' later use, as with any torch tensor.

The calls record nothing for torch's autograd: gradients are calls of their own (*_backward), for a torch.autograd.Function to
make.  So that none goes missing, an operand that requires grad is taken under torch.no_grad() (or in such a Function) only, and a
forward-mode dual is not taken.
"""
import ctypes as C
import struct

from . import (BF16, F16, F32, F64, CompletionEvent, CrossMemorySpaceOperation, GpuMemory, InvalidArgument,
               NoCompatibleComputeDevice, RankMismatch, ShapeMismatch, Tensor, _check, _hold, lib, tfh_view)

GATHER_A, SCATTER_C, ZERO_REST = 1, 2, 4      # TFH_ROWS_*
_MOST = 0x7fffffff      # what the C structure's 32-bit fields hold (ctypes would cut off the rest without a word)


class tfh_row_groups(C.Structure):
    _fields_ = [("offsets", C.c_void_p), ("order", C.c_void_p), ("positions", C.c_void_p), ("n_rows", C.c_int64),
                ("n_groups", C.c_int32), ("fan", C.c_int32)]


_CODES, _TYPES = {}, {}
_stream_of = None       # device index -> the handle of torch's current stream
_torch = None


def _codes():
    global _stream_of, _torch
    if not _CODES:
        import torch
        import torch.autograd.forward_ad
        _torch = torch
        # (the call behind torch.cuda.current_stream, without the object: 1 us of the 10 that a call takes)
        _stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
        _CODES.update({torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.float64: F64})
        _TYPES.update({c: t for t, c in _CODES.items()})
    return _CODES


_VIEW_BYTES = C.c_char * C.sizeof(tfh_view)
_PACKERS = [struct.Struct("<Qiiq%dq%dx%dq" % (r, tfh_view.strides.offset - tfh_view.dims.offset - 8 * r, r)).pack_into for r in range(5)]


def _view(t):
    """The tfh_view of a torch tensor or a Tensor, None for None."""
    if t is None:
        return None
    if isinstance(t, Tensor):
        return C.byref(t._view())
    rank = t.dim()
    if rank > 4:
        raise RankMismatch(f"rank mismatch: expected at most 3, got {rank}", 3, rank)
    v = _VIEW_BYTES()
    _PACKERS[rank](v, 0, t.data_ptr(), rank, 0, 0, *t.shape, *t.stride())
    return v


def _device(t):
    if isinstance(t, Tensor):
        if t.logical_memory_space_.kind == 0:
            raise NoCompatibleComputeDevice("no compatible compute device for this operation on MainMemory")
        return t.logical_memory_space_.space_id
    if not t.is_cuda:
        raise NoCompatibleComputeDevice("no compatible compute device for this operation on MainMemory")
    if t.is_neg():
        raise InvalidArgument("invalid argument: a tensor with torch's negative bit holds its values with the other sign: resolve_neg() it first")
    return t.get_device()


def _code(t):
    if isinstance(t, Tensor):
        dt = t.dtype
    else:
        dt = _codes().get(t.dtype, -1)
        if t.requires_grad and _torch.is_grad_enabled():
            raise InvalidArgument("invalid argument: an operand requires grad, which the call records nothing for: detach() it, or call under torch.no_grad()")
        if getattr(_torch.autograd.forward_ad, "_current_level", 0) >= 0 and _torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise InvalidArgument("invalid argument: an operand is a forward-mode dual, whose tangent the call knows nothing of")
    if dt not in (BF16, F16, F32, F64):
        raise InvalidArgument(f"invalid argument: operations on rows in groups take bf16, f16, f32 and f64; got {t.dtype}")
    return dt


def _shape(t):
    return t._dims if isinstance(t, Tensor) else t.shape


def _capturing():
    import torch
    return torch.cuda.is_current_stream_capturing()


def _stream(stream, current):
    if stream is None or stream == current:
        return current
    if _capturing():    # its events would have to be kept, and none asked, until the capture ends
        raise InvalidArgument("invalid argument: while a graph is captured, calls go to the current stream: make that the other one")
    return stream


def _hold_all(event, tensors):
    _hold(event, [getattr(t, "_buf", t) for t in tensors])


class _Call:
    """What every call does around its launches: one device for all operands, one element type, the stream and the
    events of Tensors, and buffers kept alive while another stream than torch's uses them."""

    def __init__(self, like, operands, groups, stream, sums=()):
        import torch
        self.torch, self.like = torch, like
        _CODES or _codes()
        self.device = _device(like)
        self.dtype = _code(like)
        wide = F64 if self.dtype == F64 else F32
        self.used = [like]
        for sort, wanted, why in ((operands, self.dtype, "operands of different element types"),
                                  (sums, wide, "weights and scales are f32 (f64 beside f64 operands)")):
            for t in sort:
                if t is None:
                    continue
                if _device(t) != self.device:
                    raise CrossMemorySpaceOperation(f"cross-memory-space operation between {GpuMemory(self.device)!r} and {GpuMemory(_device(t))!r}",
                                                    GpuMemory(self.device), GpuMemory(_device(t)))
                if _code(t) != wanted:
                    raise InvalidArgument("invalid argument: " + why)
                self.used.append(t)
        if groups is not None:
            if groups.device != self.device:
                raise CrossMemorySpaceOperation(f"cross-memory-space operation between {GpuMemory(self.device)!r} and {GpuMemory(groups.device)!r}",
                                                GpuMemory(self.device), GpuMemory(groups.device))
            self.used.append(groups)
        self.current = _stream_of(self.device)
        self.stream = _stream(stream, self.current)
        self.guard = None
        if torch.cuda.current_device() != self.device:
            self.guard = torch.cuda.device(self.device)
        self.ordered = False

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        pending = [t for t in self.used if isinstance(t, (Tensor, RowGroups)) and t.event is not None]
        if pending and not _capturing():
            for t in pending:
                _check(lib().tfh_stream_wait_event(self.stream, t.event._h))
        return self

    def __exit__(self, *error):
        try:
            if error[0] is not None and self.stream != self.current:
                _hold_all(CompletionEvent(self.stream), self.used)   # an earlier launch of the call may be using them
        finally:
            if self.guard is not None:
                self.guard.__exit__(*error)

    def empty(self, dims, dtype=None, like=None):
        """A new buffer from torch's allocator.  Its memory may still be read by earlier work of the current stream: another
        stream waits for that first."""
        torch = self.torch
        if self.stream != self.current and not self.ordered:
            _check(lib().tfh_stream_wait_event(self.stream, CompletionEvent(self.current)._h))
            self.ordered = True
        dtype = self.dtype if dtype is None else dtype
        if isinstance(like, Tensor):   # (torch has no negative strides)
            ordered = min(like._strides, default=0) >= 0 and 0 not in like._dims
            like = torch.as_strided(like._buf, like._dims, like._strides, like._buf.storage_offset() + like._offset) if ordered else None
        if like is not None:
            t = torch.empty_like(like)
        else:
            tdt = dtype if isinstance(dtype, torch.dtype) else _TYPES[dtype]
            if isinstance(self.like, Tensor):
                t = torch.empty(dims, dtype=tdt, device=torch.device("cuda", self.device))
            elif dtype == self.dtype:
                t = self.like.new_empty(dims)
            else:
                t = self.like.new_empty(dims, dtype=tdt)
        self.used.append(t)
        return t

    def result(self, t):
        """`t` as the first operand's kind."""
        return Tensor.from_torch(t) if isinstance(self.like, Tensor) else t

    def done(self, *outputs):
        other = self.stream != self.current
        tensors = [t for t in outputs if isinstance(t, Tensor)]
        if other or tensors:
            ev = None if _capturing() else CompletionEvent(self.stream)
            for t in tensors:
                t.event = ev
            if other:
                _hold_all(ev, self.used + list(outputs))


class RowGroups:
    """tfh_row_groups: rows listed group by group.

    offsets    int32 [n_groups + 1]: group g is p = offsets[g] .. offsets[g + 1]; the rows behind belong to no group
    order      int32 [n_rows], place p holds row order[p]; None: the rows lie in that order already
    positions  int32 [n_rows], where row i stands, -1 for a row of no group; None if nothing is joined by it
    fan        rows per source row: row i = t * fan + j is choice j of token t"""

    __slots__ = ("offsets", "order", "positions", "n_rows", "n_groups", "fan", "device", "event", "_c")

    def __init__(self, offsets, order=None, positions=None, n_rows=None, fan=1):
        import torch
        self.device = _device(offsets)
        for name, t in (("offsets", offsets), ("order", order), ("positions", positions)):
            if t is None:
                continue
            if isinstance(t, Tensor) or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise InvalidArgument(f"invalid argument: {name} has to be a contiguous int32 vector")
            if _device(t) != self.device:
                raise CrossMemorySpaceOperation(f"cross-memory-space operation between {GpuMemory(self.device)!r} and {GpuMemory(_device(t))!r}",
                                                GpuMemory(self.device), GpuMemory(_device(t)))
        if n_rows is None:
            if order is None:
                raise InvalidArgument("invalid argument: row groups without an order need n_rows")
            n_rows = order.numel()
        for name, t in (("order", order), ("positions", positions)):
            if t is not None and t.numel() != n_rows:
                raise InvalidArgument(f"invalid argument: {name} has {t.numel()} entries for {n_rows} rows")
        self.offsets, self.order, self.positions, self.n_rows, self.fan = offsets, order, positions, int(n_rows), int(fan)
        self.n_groups = offsets.numel() - 1
        self.event = None
        if max(self.n_rows, self.n_groups, self.fan) > _MOST:
            raise InvalidArgument(f"invalid argument: {self.n_groups} groups of {self.n_rows} rows with a fan of {self.fan} are out of range")
        self._c = tfh_row_groups(offsets.data_ptr(), order.data_ptr() if order is not None else None,
                                 positions.data_ptr() if positions is not None else None, self.n_rows, self.n_groups, self.fan)
        if self.n_groups < 1 or self.n_rows < 0 or self.fan < 1 or self.n_rows % self.fan:
            raise InvalidArgument(f"invalid argument: {self.n_groups} groups of {self.n_rows} rows with a fan of {self.fan}")

    @classmethod
    def from_ids(cls, ids, n_groups, stream=None):
        """Groups the rows by ids (int32 or int64, [n_rows] or [tokens, fan]); an index outside 0 .. n_groups puts its row
        into no group.  Stable: a group's rows keep their order."""
        import torch
        device = _device(ids)
        bits = {torch.int32: 32, torch.int64: 64}.get(ids.dtype) if not isinstance(ids, Tensor) else None
        if bits is None:
            raise InvalidArgument("invalid argument: ids have to be an int32 or int64 tensor")
        if ids.dim() not in (1, 2):
            raise RankMismatch(f"rank mismatch: expected 1, got {ids.dim()}", 1, ids.dim())
        n_groups, n = int(n_groups), ids.numel()
        if n_groups < 1 or max(n, n_groups) > _MOST:
            raise InvalidArgument(f"invalid argument: {n_groups} groups of {n} rows are out of range")
        fan = ids.shape[1] if ids.dim() == 2 else 1
        _CODES or _codes()
        current = _stream_of(device)
        st = _stream(stream, current)
        need = lib().tfh_group_rows_workspace(n, n_groups)
        # one buffer for all: [order | positions | offsets | scratch], each 16-byte aligned
        at_p, at_o = (n + 3) & ~3, 2 * ((n + 3) & ~3)
        at_w = at_o + ((n_groups + 4) & ~3)
        buf = torch.empty(at_w + (need + 3) // 4, dtype=torch.int32, device=ids.device)
        guard = torch.cuda.device(device) if torch.cuda.current_device() != device else None
        if guard is not None:
            guard.__enter__()
        try:
            if st != current:
                _check(lib().tfh_stream_wait_event(st, CompletionEvent(current)._h))
            p = buf.data_ptr()
            _check(lib().tfh_group_rows(bits, _view(ids), n_groups, p + 4 * at_o, p, p + 4 * at_p, p + 4 * at_w, need, st))
            g = cls.__new__(cls)
            g.offsets, g.order, g.positions = buf[at_o:at_o + n_groups + 1], buf[:n], buf[at_p:at_p + n]
            g.n_rows, g.n_groups, g.fan, g.device, g.event = n, n_groups, max(1, fan), device, None
            g._c = tfh_row_groups(p + 4 * at_o, p, p + 4 * at_p, n, n_groups, g.fan)
            if st != current:
                g.event = CompletionEvent(st)
        finally:
            if st != current:
                _hold(CompletionEvent(st), [buf, ids])
            if guard is not None:
                guard.__exit__(None, None, None)
        return g

    def _need(self, what):
        if getattr(self, what) is None:
            raise InvalidArgument(f"invalid argument: row groups without {what}")


def _groups(groups):
    if not isinstance(groups, RowGroups):
        raise InvalidArgument("invalid argument: groups have to be RowGroups")
    return C.byref(groups._c)


def _dims(t, dims):
    """What a call of several launches asks of an operand, before the first of them."""
    got = list(_shape(t))
    if len(got) != len(dims):
        raise RankMismatch(f"rank mismatch: expected {len(dims)}, got {len(got)}", len(dims), len(got))
    if got != list(dims):
        raise ShapeMismatch(f"shape mismatch: expected {list(dims)}, got {got}", list(dims), got)


def _rank(what, t, rank):
    got = len(_shape(t))
    if got != rank:
        raise RankMismatch(f"rank mismatch: expected {rank}, got {got}", rank, got)


def ragged_gemm_into(a, b, groups, alpha, beta, c, gather=False, scatter=False, stream=None):
    """c[p] = alpha * a[src(p)] @ b[g(p)] + beta * c[p] for every row p of a group g(p); the rows of no group are left as
    they are.  gather: src(p) = order[p] // fan, a [n_rows / fan, K]; else src(p) = p.  scatter: the result of p is row
    order[p] of c.  beta = 0 overwrites without reading."""
    _groups(groups)
    with _Call(a, (a, b, c), groups, stream) as k:
        flags = (GATHER_A if gather else 0) | (SCATTER_C if scatter else 0)
        _check(lib().tfh_ragged_gemm(k.dtype, _groups(groups), flags, alpha, _view(a), _view(b), beta, _view(c), k.stream))
        k.done(c)


def ragged_gemm(a, b, groups, gather=False, stream=None):
    """A matrix product for each group: [n_rows, N], row p = a[src(p)] @ b[g(p)], zeros for the rows of no group.
    a [n_rows, K] in the groups' order, or with gather=True [n_rows / fan, K] read through it; b [n_groups, K, N]."""
    _groups(groups)
    _rank("a", a, 2), _rank("b", b, 3)
    with _Call(a, (a, b), groups, stream) as k:
        c = k.empty((groups.n_rows, _shape(b)[2]))
        _check(lib().tfh_ragged_gemm(k.dtype, _groups(groups), ZERO_REST | (GATHER_A if gather else 0), 1.0, _view(a), _view(b),
                                     0.0, _view(c), k.stream))
        c = k.result(c)
        k.done(c)
    return c


def ragged_gemm_grad_into(a, dc, groups, alpha, beta, db, gather=False, stream=None):
    """db[g] = alpha * sum over p in g of a[src(p)]^T dc[p] + beta * db[g]; zeros (beta * db[g]) for a group without rows."""
    _groups(groups)
    with _Call(a, (a, dc, db), groups, stream) as k:
        _check(lib().tfh_ragged_gemm_grad(k.dtype, _groups(groups), GATHER_A if gather else 0, alpha, _view(a), _view(dc), beta,
                                          _view(db), k.stream))
        k.done(db)


def ragged_gemm_backward(a, b, dc, groups, gather=False, stream=None):
    """The gradients of ragged_gemm(a, b, groups, gather): (da, db), db laid out like b.  With gather a row's choices are
    added up in 32 bits (64 for f64) and rounded once; for a fan above 1 positions are needed."""
    _groups(groups)
    _rank("b", b, 3), _rank("dc", dc, 2)
    _dims(a, (groups.n_rows // groups.fan if gather else groups.n_rows, _shape(b)[1]))
    _dims(b, (groups.n_groups, _shape(b)[1], _shape(dc)[1]))
    _dims(dc, (groups.n_rows, _shape(b)[2]))
    if gather:
        groups._need("order")
    if gather and groups.fan > 1:
        groups._need("positions")
    with _Call(a, (a, b, dc), groups, stream) as k:
        K, flags = _shape(b)[1], GATHER_A if gather else 0
        da, db = k.empty((groups.n_rows // groups.fan if gather else groups.n_rows, K)), k.empty(_shape(b), like=b)
        need = lib().tfh_ragged_gemm_grad_a_workspace(k.dtype, groups.n_rows, K, groups.fan, flags)
        ws = k.empty((need,), k.torch.uint8).data_ptr() if need else None
        _check(lib().tfh_ragged_gemm_grad_a(k.dtype, _groups(groups), flags, 1.0, _view(dc), _view(b), _view(da), ws, need, k.stream))
        _check(lib().tfh_ragged_gemm_grad(k.dtype, _groups(groups), flags, 1.0, _view(a), _view(dc), 0.0, _view(db), k.stream))
        da, db = k.result(da), k.result(db)
        k.done(da, db)
    return da, db


def combine_rows_into(x, groups, weights, y, stream=None):
    """y[t] = sum_j weights[t, j] * x[positions[t * fan + j]]; weights None: ones."""
    _groups(groups)
    with _Call(x, (x, y), groups, stream, (weights,)) as k:
        _check(lib().tfh_combine_rows(k.dtype, _groups(groups), _view(x), _view(weights), _view(y), k.stream))
        k.done(y)


def combine_rows(x, groups, weights=None, stream=None):
    """The rows of a token joined again: [n_rows / fan, N], sum_j weights[t, j] * x[positions[t * fan + j]].  x [n_rows, N] in
    the groups' order; a choice of no group adds nothing.  weights f32 (f64 beside f64) [n_rows / fan, fan] or None: ones."""
    _groups(groups)
    _rank("x", x, 2)
    with _Call(x, (x,), groups, stream, (weights,)) as k:
        y = k.empty((groups.n_rows // groups.fan, _shape(x)[1]))
        _check(lib().tfh_combine_rows(k.dtype, _groups(groups), _view(x), _view(weights), _view(y), k.stream))
        y = k.result(y)
        k.done(y)
    return y


def combine_rows_backward(x, weights, dy, groups, stream=None):
    """The gradients of combine_rows(x, groups, weights): (dx, dweights); dweights is None where weights is."""
    _groups(groups)
    _rank("x", x, 2)
    with _Call(x, (x, dy), groups, stream, (weights,)) as k:
        dx = k.empty(_shape(x))
        dw = None if weights is None else k.empty((groups.n_rows // groups.fan, groups.fan), F64 if k.dtype == F64 else F32)
        _check(lib().tfh_combine_rows_grad(k.dtype, _groups(groups), _view(x), _view(weights), _view(dy), _view(dx), _view(dw), k.stream))
        dx, dw = k.result(dx), None if dw is None else k.result(dw)
        k.done(dx, dw)
    return dx, dw


def _workspace(k, groups, rank, gradient):
    need = lib().tfh_adapter_workspace(k.dtype, groups.n_rows, rank, gradient)
    return k.empty((max(need, 1),), k.torch.uint8).data_ptr(), need


def adapter_gemm_into(x, w, a, b, groups, y, scales=None, stream=None):
    """adapter_gemm with a given output."""
    _groups(groups)
    _rank("a", a, 3)
    with _Call(x, (x, w, a, b, y), groups, stream, (scales,)) as k:
        ws, need = _workspace(k, groups, _shape(a)[2], 0)
        _check(lib().tfh_adapter_gemm(k.dtype, _groups(groups), _view(x), _view(w), _view(a), _view(b), _view(scales), _view(y), ws, need,
                                      k.stream))
        k.done(y)


def adapter_gemm(x, w, a, b, groups, scales=None, stream=None):
    """x @ w + scales[g] * (x @ a[g]) @ b[g], row by row with the row's group g; x @ w alone for a row of none.
    x [n_rows, K] in its own order, w [K, N], a [n_groups, K, R], b [n_groups, R, N], scales f32 (f64 beside f64)
    [n_groups], contiguous, or None: ones.  groups with fan 1."""
    _groups(groups)
    _rank("w", w, 2), _rank("a", a, 3)
    with _Call(x, (x, w, a, b), groups, stream, (scales,)) as k:
        y = k.empty((groups.n_rows, _shape(w)[1]))
        ws, need = _workspace(k, groups, _shape(a)[2], 0)
        _check(lib().tfh_adapter_gemm(k.dtype, _groups(groups), _view(x), _view(w), _view(a), _view(b), _view(scales), _view(y), ws, need,
                                      k.stream))
        y = k.result(y)
        k.done(y)
    return y


def adapter_gemm_backward(x, w, a, b, dy, groups, scales=None, stream=None):
    """The gradients of adapter_gemm for a w that stays as it is: (dx, da, db), da and db laid out like a and b, zeros for
    a group without rows."""
    _groups(groups)
    _rank("w", w, 2), _rank("a", a, 3)
    with _Call(x, (x, w, a, b, dy), groups, stream, (scales,)) as k:
        dx, da, db = k.empty((groups.n_rows, _shape(w)[0])), k.empty(_shape(a), like=a), k.empty(_shape(b), like=b)
        ws, need = _workspace(k, groups, _shape(a)[2], 1)
        _check(lib().tfh_adapter_gemm_grad(k.dtype, _groups(groups), _view(x), _view(w), _view(a), _view(b), _view(scales), _view(dy),
                                           _view(dx), _view(da), _view(db), ws, need, k.stream))
        dx, da, db = k.result(dx), k.result(da), k.result(db)
        k.done(dx, da, db)
    return dx, da, db
