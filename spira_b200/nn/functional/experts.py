"""Expert feed-forward blocks over voxel rows: routing, row exchange and ragged products, with their gradients.

    routing = expert_route(logits, top_k)                      # logits [N, E]
    rows = expert_dispatch(feats, routing)                     # [N * top_k, C], in expert order
    rows = grouped_linear(rows, weights, routing.offsets)      # weights [E, C, C_out]
    feats = expert_combine(rows, routing)                      # [N, C_out]

No reference counterpart (the reference stops at convolutions, BatchNorm and ReLU).  All calls run on the current stream
of their tensors' device, never synchronise, and may be captured into a CUDA graph (``grouped_linear`` after one call outside
of it: the device's status word has to exist).  Results do not depend on scheduling:
the same inputs give the same bits.  Gradients once and in reverse mode only; anything else is refused.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from spira_b200 import _lib
from spira_b200.nn.functional import _C

__all__ = ["ExpertRouting", "expert_route", "expert_dispatch", "expert_combine", "grouped_linear"]

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 512, 32, 1024
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _launch(index: int, name: str, *args) -> None:
    """One library call whose last argument is the current stream of device ``index``."""
    if index == _current_device():
        _lib.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _raw_stream(index))


def _query(index: int, name: str, *args) -> None:
    """A library call without a stream that depends on the device (scratch sizes)."""
    if index == _current_device():
        _lib.call(name, *args)
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args)


def _fail(message: str):
    raise RuntimeError("[spira_b200] " + message)


def _no_tangents(*tensors) -> None:
    """Refuses tensors with a forward-mode tangent: kernels read the values alone, a result would say that it is constant."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _fail("the expert and norm operators have no forward-mode derivatives (an input has a tangent)")


def _device_of(*tensors) -> int:
    """The device index all given tensors share; refuses CPU tensors and mixtures."""
    _no_tangents(*tensors)
    index = -1
    for t in tensors:
        if t is None:
            continue
        i = t.get_device() if t.is_cuda else -1
        if i < 0:
            raise NotImplementedError("spira_b200 runs on CUDA tensors only")
        if index < 0:
            index = i
        elif i != index:
            _fail("tensors on different devices")
    return index


def _dense(like: torch.Tensor, rows: int, columns: int) -> torch.Tensor:
    """An uninitialised dense matrix of the type and device of ``like`` (the cheapest of torch's allocating calls)."""
    return like.new_empty_strided((rows, columns), (columns, 1))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself if its columns are neighbours (rows may lie any distance apart), else a dense copy."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _addr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _once(*grads) -> None:
    """In a backward function: refuses to be recorded itself (``create_graph=True``), and gradients with tangents."""
    _no_tangents(*grads)
    if torch.is_grad_enabled():
        _fail("the expert and norm operators can be differentiated once only (create_graph=True was asked for)")


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class ExpertRouting(NamedTuple):
    """Result of :func:`expert_route` for ``N`` rows, ``k`` experts per row and ``E`` experts."""
    weights: torch.Tensor    # [N, k] fp32, differentiable
    experts: torch.Tensor    # [N, k] int32, -1: none
    slots: torch.Tensor      # [N, k] int32: place of the pair in expert order, -1: none
    order: torch.Tensor      # [N * k] int32: row * k + j of every place, -1 behind the last
    offsets: torch.Tensor    # [E + 1] int32: first place of every expert


# ------------------------------------------------------------------------------------------------ routing
def _route(logits: torch.Tensor, top_k: int, renormalize: bool) -> ExpertRouting:
    n, experts = logits.shape
    weights = logits.new_empty_strided((n, top_k), (top_k, 1), dtype=torch.float32)
    chosen = torch.empty_like(weights, dtype=torch.int32)
    slots = torch.empty_like(chosen)
    order = chosen.new_empty(n * top_k)
    offsets = chosen.new_empty(experts + 1)
    index = logits.get_device()
    need, workspace = C.c_size_t(), None
    if n * top_k > 4096:          # (a few rows need no scratch: one CTA routes them)
        _query(index, "spira_b200_expert_route_workspace", n, experts, top_k, C.byref(need))
        workspace = chosen.new_empty((need.value + 3) // 4)
    _launch(index, "spira_b200_expert_route", logits.data_ptr(), _DTYPES[logits.dtype], n, logits.stride(0), experts, top_k,
            1 if renormalize else 0, weights.data_ptr(), chosen.data_ptr(), slots.data_ptr(), order.data_ptr(), offsets.data_ptr(),
            None if workspace is None else workspace.data_ptr(), need.value)
    return ExpertRouting(weights, chosen, slots, order, offsets)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize):
        r = _route(logits, top_k, renormalize)
        ctx.renormalize = renormalize
        ctx.save_for_backward(logits, r.weights, r.experts)
        ctx.mark_non_differentiable(r.experts, r.slots, r.order, r.offsets)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    def backward(ctx, dweights, *_):
        _once(dweights)
        if dweights is None:
            return None, None, None
        logits, weights, chosen = ctx.saved_tensors
        n, experts = logits.shape
        dweights = dweights.float()
        dlogits = _dense(logits, n, experts)
        _launch(logits.get_device(), "spira_b200_expert_route_backward", logits.data_ptr(), _DTYPES[logits.dtype], n, logits.stride(0),
                experts, weights.shape[1], 1 if ctx.renormalize else 0, weights.data_ptr(), chosen.data_ptr(), dweights.data_ptr(),
                dweights.stride(0), dweights.stride(1), dlogits.data_ptr())
        return dlogits, None, None


def expert_route(logits: torch.Tensor, top_k: int, renormalize: bool = True) -> ExpertRouting:
    """The ``top_k`` experts of every row of ``logits [N, E]`` (fp16, bf16 or fp32).

    The largest logits win, equal ones by the lower index; an expert whose logit is ``-inf`` is never chosen, so a row may
    get fewer than ``top_k`` experts or none (``experts`` and ``slots`` are -1 there, the weight 0).  ``weights`` is the
    softmax over the chosen experts, or over all of them with ``renormalize=False``.  A NaN counts as the largest logit
    and makes the weights of its row NaN."""
    index = _device_of(logits)
    if logits.dim() != 2 or logits.dtype not in _DTYPES:
        _fail(f"Tensor logits is expected to be a float16, bfloat16 or float32 matrix [N, E], got {logits.dtype} {tuple(logits.shape)}")
    top_k = int(top_k)
    n, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS:
        _fail(f"expert_route takes 1 to {MAX_EXPERTS} experts, got {experts}")
    if not 1 <= top_k <= min(experts, MAX_TOP_K):
        _fail(f"top_k must be 1 to min(experts, {MAX_TOP_K}), got {top_k}")
    if n * top_k >= 1 << 31:
        _fail(f"{n} rows x {top_k} experts are out of range")
    logits = _rows(logits) if n and logits.stride(0) >= experts else logits.contiguous()
    if _needs_grad(logits):
        return ExpertRouting(*_Route.apply(logits, top_k, bool(renormalize)))
    return _route(logits, top_k, renormalize)


# ------------------------------------------------------------------------------------------------ rows to experts and back
def _check_routing(routing: ExpertRouting):
    slots, offsets = routing.slots, routing.offsets
    if slots.dim() != 2 or slots.dtype != torch.int32 or offsets.dim() != 1 or offsets.dtype != torch.int32 or offsets.shape[0] < 2:
        _fail("routing.slots is expected to be int32 [N, k] and routing.offsets int32 [E + 1]")
    if not 1 <= slots.shape[1] <= MAX_TOP_K:
        _fail(f"a routing holds 1 to {MAX_TOP_K} experts per row, got {slots.shape[1]}")
    return slots if slots.is_contiguous() else slots.contiguous(), offsets if offsets.is_contiguous() else offsets.contiguous()


def _check_rows(t: torch.Tensor, name: str, rows: int) -> torch.Tensor:
    if t.dim() != 2 or t.dtype not in _DTYPES or t.shape[1] < 1:
        _fail(f"Tensor {name} is expected to be a float16, bfloat16 or float32 matrix, got {t.dtype} {tuple(t.shape)}")
    if t.shape[0] != rows:
        _fail(f"The dimension 0 of Tensor {name} is expected to be {rows} but found {t.shape[0]}")
    return _rows(t)


def _order_hint(routing: ExpertRouting, slots: torch.Tensor) -> Optional[torch.Tensor]:
    """``routing.order`` where it can tell the kernels which places are taken.  They check what it says: places that no slot names
    are cleared whatever it holds (a caller may have taken slots out of a routing), a right one only spares them the rest."""
    o = routing.order
    if isinstance(o, torch.Tensor) and o.dtype is torch.int32 and o.shape == (slots.numel(),) and o.is_contiguous() \
            and o.get_device() == slots.get_device():
        return o
    return None


def _dispatch(feats, slots, order):
    n, k = slots.shape
    channels = feats.shape[1]
    rows = _dense(feats, n * k, channels)
    _launch(feats.get_device(), "spira_b200_expert_dispatch_cleared", feats.data_ptr(), _DTYPES[feats.dtype], n, feats.stride(0), channels,
            slots.data_ptr(), _addr(order), k, rows.data_ptr())
    return rows


def _combine(rows, weights, slots):
    n, k = slots.shape
    channels = rows.shape[1]
    out = _dense(rows, n, channels)
    _launch(rows.get_device(), "spira_b200_expert_combine", rows.data_ptr(), _DTYPES[rows.dtype], n, rows.stride(0), channels,
            None if weights is None else weights.data_ptr(), 0 if weights is None else weights.stride(0),
            0 if weights is None else weights.stride(1), slots.data_ptr(), k, out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feats, slots, order):
        ctx.save_for_backward(slots)
        return _dispatch(feats, slots, order)

    @staticmethod
    def backward(ctx, drows):
        _once(drows)
        return _combine(_rows(drows), None, ctx.saved_tensors[0]), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slots, order):
        ctx.save_for_backward(rows, weights, slots, order)
        return _combine(rows, weights, slots)

    @staticmethod
    def backward(ctx, dout):
        _once(dout)
        rows, weights, slots, order = ctx.saved_tensors
        dout = _rows(dout)
        (n, k), channels = slots.shape, rows.shape[1]
        drows = _dense(rows, n * k, channels) if ctx.needs_input_grad[0] else None
        dweights = _dense(weights, n, k) if ctx.needs_input_grad[1] else None
        _launch(rows.get_device(), "spira_b200_expert_combine_backward_cleared", rows.data_ptr(), dout.data_ptr(), _DTYPES[rows.dtype], n,
                rows.stride(0), dout.stride(0), channels, weights.data_ptr(), weights.stride(0), weights.stride(1), slots.data_ptr(),
                _addr(order), k, None if drows is None else drows.data_ptr(), None if dweights is None else dweights.data_ptr())
        return drows, dweights, None, None


def expert_dispatch(feats: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    """``feats [N, C]`` -> ``[N * k, C]`` in the expert order of ``routing`` (a row appears once per expert it goes to); rows of
    places that no slot names are zero (those behind ``routing.offsets[E]``, and those of pairs that were taken out of the
    routing by setting their slot to -1).  Slots are distinct; a place that two of them name holds one of the two rows."""
    slots, offsets = _check_routing(routing)
    _device_of(feats, slots, offsets)
    feats = _check_rows(feats, "feats", slots.shape[0])
    order = _order_hint(routing, slots)
    if _needs_grad(feats):
        return _Dispatch.apply(feats, slots, order)
    return _dispatch(feats, slots, order)


def expert_combine(rows: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    """``rows [N * k, C]`` in expert order -> ``[N, C]``: every voxel's rows, weighted with ``routing.weights`` and added in
    the order of its experts (fp32, one rounding).  Voxels without an expert are zero, and so is the gradient of rows that no
    slot names."""
    slots, offsets = _check_routing(routing)
    weights = routing.weights
    _device_of(rows, slots, offsets, weights)
    if weights.dtype != torch.float32 or weights.shape != slots.shape:
        _fail(f"routing.weights is expected to be float32 {tuple(slots.shape)}, got {weights.dtype} {tuple(weights.shape)}")
    rows = _check_rows(rows, "rows", slots.shape[0] * slots.shape[1])
    if _needs_grad(rows, weights):
        return _Combine.apply(rows, weights, slots, _order_hint(routing, slots))
    return _combine(rows, weights, slots)


# ------------------------------------------------------------------------------------------------ ragged products
def _status(index: int) -> int:
    """Address of the status word the tensor-core kernels raise; it must exist before a capture (it outlives the graph)."""
    t = _C._status.get(index)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            _fail("make one grouped_linear call before capturing a graph (the device's status word does not exist yet)")
        t = _C.status_word(torch.device("cuda", index))
    return t.data_ptr()


def _grouped_desc(n, weights, offsets, relu, x=None, bias=None, dy=None, y=None, mask=None, dx=None, dweight=None, dbias=None) -> bytes:
    """``spira_b200_grouped_desc`` (fields as in ``_lib.GroupedDesc``)."""
    experts, c_in, c_out = weights.shape
    return _lib.GROUPED_PACK.pack(_DTYPES[weights.dtype], experts, c_in, c_out, relu, 0, n, 0 if x is None else x.stride(0),
                                  0 if dy is None else dy.stride(0), offsets.data_ptr(), 0 if x is None else x.data_ptr(), weights.data_ptr(),
                                  _addr(bias), _addr(dy), _addr(y), _addr(mask), _addr(dx), _addr(dweight), _addr(dbias))


def _grouped(x, weights, offsets, bias, relu, want_mask=False):
    """The product and, for a backward pass, what its ReLU let through: the bit mask the kernel writes (None without a ReLU or rows).
    It is the sign of the unrounded values: a positive one that rounds to zero lets its gradient through."""
    index, n = x.get_device(), x.shape[0]
    y = _dense(x, n, weights.shape[2])
    mask, workspace, room = None, 0, 0
    want_mask = want_mask and relu
    relu = 1 if relu else 0
    # channels, strides or addresses off the 16-byte boundaries may need scratch, and so may rows that overlap
    stride = x.stride(0)
    off = ((x.shape[1] | y.shape[1] | stride) & 7) | ((x.data_ptr() | weights.data_ptr()) & 15) or stride < x.shape[1]
    if want_mask or off:
        need, mask_bytes = C.c_size_t(), C.c_size_t()
        _query(index, "spira_b200_grouped_linear_workspace", _grouped_desc(n, weights, offsets, relu, x, bias, y=y), C.byref(need), C.byref(mask_bytes))
        if want_mask and mask_bytes.value:
            mask = x.new_empty(mask_bytes.value, dtype=torch.uint8)
        room = need.value
        if room:
            scratch = x.new_empty(room, dtype=torch.uint8)
            workspace = scratch.data_ptr()
    _launch(index, "spira_b200_grouped_linear", _grouped_desc(n, weights, offsets, relu, x, bias, y=y, mask=mask), workspace, room, _status(index))
    return y, mask


def _with_workspace(index, like, name, desc, *rest):
    need = C.c_size_t()
    _query(index, name + "_workspace", desc, C.byref(need))
    workspace = like.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _launch(index, name, desc, None if workspace is None else workspace.data_ptr(), need.value, *rest)


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, offsets, bias, relu):
        y, mask = _grouped(x, weights, offsets, bias, relu, want_mask=True)
        ctx.relu, ctx.has_bias = relu, bias is not None
        ctx.save_for_backward(x, weights, offsets, mask)
        return y

    @staticmethod
    def backward(ctx, dy):
        _once(dy)
        x, weights, offsets, mask = ctx.saved_tensors
        dy = _rows(dy)
        need = ctx.needs_input_grad
        index, n = x.get_device(), x.shape[0]
        dx = _dense(dy, n, x.shape[1]) if need[0] else None
        dw = torch.empty_like(weights) if need[1] else None            # (dense: the call made it so)
        db = _dense(weights, weights.shape[0], weights.shape[2]) if ctx.has_bias and need[3] else None
        _with_workspace(index, dy, "spira_b200_grouped_linear_backward",
                        _grouped_desc(n, weights, offsets, 1 if ctx.relu else 0, x, None, dy, None, mask, dx, dw, db), _status(index))
        return dx, dw, None, db, None


def grouped_linear(feats: torch.Tensor, weights: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   relu: bool = False) -> torch.Tensor:
    """``relu?(feats[r] @ weights[e] + bias[e])`` for the rows ``offsets[e] <= r < offsets[e + 1]`` of every expert ``e``.

    ``feats [N, C_in]`` and ``weights [E, C_in, C_out]`` are fp16 or bf16 (sums in fp32, one rounding), ``offsets [E + 1]``
    is int32 on the device and is never read by the host; ``bias`` is ``[E, C_out]``; ``E <= 1024``, channels up to 65 536.  Groups may be empty; rows outside
    every group are zero in the result and have no gradient.  A kernel that gives up on an internal wait raises the device's
    status word, which ``_C.check_status()`` reports (it synchronises)."""
    index = _device_of(feats, weights, offsets, bias)
    if feats.dim() != 2 or weights.dim() != 3:
        _fail(f"feats is expected to be [N, C_in] and weights [E, C_in, C_out], got {tuple(feats.shape)} and {tuple(weights.shape)}")
    if feats.dtype != weights.dtype or feats.dtype not in (torch.float16, torch.bfloat16):
        _fail(f"feats and weights must both be float16 or both bfloat16 (fp32 accumulation), got {feats.dtype} and {weights.dtype}")
    experts, c_in, c_out = weights.shape
    if feats.shape[1] != c_in:
        _fail(f"The dimension 1 of Tensor feats is expected to be {c_in} but found {feats.shape[1]}")
    if not 1 <= experts <= MAX_GROUPS or c_in < 1 or c_out < 1:
        _fail(f"grouped_linear takes 1 to {MAX_GROUPS} experts with at least one channel, got weights {tuple(weights.shape)}")
    if offsets.dim() != 1 or offsets.shape[0] != experts + 1 or offsets.dtype != torch.int32:
        _fail(f"offsets is expected to be int32 [{experts + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    if bias is not None and (bias.dtype != feats.dtype or bias.shape != (experts, c_out)):
        _fail(f"bias is expected to be {feats.dtype} [{experts}, {c_out}], got {bias.dtype} {tuple(bias.shape)}")
    feats = _rows(feats)
    weights, offsets = weights.contiguous(), offsets.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if _needs_grad(feats, weights, bias):
        return _Grouped.apply(feats, weights, offsets, bias, bool(relu))
    return _grouped(feats, weights, offsets, bias, relu)[0]
