"""Norms around a block, fused with the block's gate and the residual, with their gradients.

    stream, normed = residual_norm(feats, block, weight=w, ...)

No reference counterpart: the reference normalises with BatchNorm as a pass of its own (spira/nn/normalizations.py:8-10)
and adds residuals as another (spira/tensors.py:47-53).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from spira_b200 import _lib
from spira_b200.nn.functional.experts import _addr, _dense, _device_of, _DTYPES, _fail, _launch, _needs_grad, _once, _rows, _with_workspace

__all__ = ["residual_norm"]

MAX_CHANNELS = 8192
GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_FULL = 0, 1, 2, 3


class _Spec(NamedTuple):
    """What stays the same between the forward and the backward call."""
    params_f32: bool
    layer: bool
    pre: bool
    post: bool
    gate_kind: int
    residual_scale: float
    block_scale: float
    eps: float


def _desc(spec, x, params, stream=None, normed=None, stats=None, dstream=None, dnormed=None, grads=(None,) * 7) -> bytes:
    """``spira_b200_norm_desc`` (fields as in ``_lib.NormDesc``); ``params`` = block, gate, weight, bias, post_weight, post_bias,
    ``grads`` = the places for the gradients of x and of these."""
    block, gate, weight, bias, post_weight, post_bias = params
    dx, dblock, dgate, dweight, dbias, dpost_weight, dpost_bias = grads
    return _lib.NORM_PACK.pack(
        _DTYPES[x.dtype], spec.params_f32, x.shape[1], spec.layer, spec.pre, spec.post, spec.gate_kind, 0,
        spec.residual_scale, spec.block_scale, spec.eps, 0.0,
        x.shape[0], x.stride(0), 0 if block is None else block.stride(0), 0 if gate is None else gate.stride(0),
        0 if dstream is None else dstream.stride(0), 0 if dnormed is None else dnormed.stride(0),
        x.data_ptr(), _addr(block), _addr(gate), _addr(weight), _addr(bias), _addr(post_weight), _addr(post_bias), _addr(stream), _addr(normed),
        _addr(stats), _addr(dstream), _addr(dnormed), _addr(dx), _addr(dblock), _addr(dgate), _addr(dweight), _addr(dbias), _addr(dpost_weight),
        _addr(dpost_bias))


def _forward(spec, x, params, stats):
    n, channels = x.shape
    stream = _dense(x, n, channels) if params[0] is not None else None
    normed = _dense(x, n, channels) if spec.pre else None
    _launch(x.get_device(), "spira_b200_residual_norm", _desc(spec, x, params, stream, normed, stats))
    return stream, normed


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, spec, x, *params):
        stats = x.new_empty_strided((x.shape[0], 4), (4, 1), dtype=torch.float32)
        stream, normed = _forward(spec, x, params, stats)
        ctx.spec = spec
        ctx.save_for_backward(x, *params, stats)
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    def backward(ctx, dstream, dnormed):
        _once(dstream, dnormed)
        x, *params, stats = ctx.saved_tensors
        spec = ctx.spec
        if dstream is None and dnormed is None:
            return (None,) * 8
        if spec.pre and dnormed is None:
            dnormed = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        dstream = None if dstream is None else _rows(dstream)
        dnormed = None if dnormed is None else _rows(dnormed)
        grads = [None if t is None or not wanted else torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)
                 for t, wanted in zip((x, *params), ctx.needs_input_grad[1:])]
        desc = _desc(spec, x, params, None, None, stats, dstream, dnormed, grads)
        if grads[3] is not None or grads[4] is not None or grads[5] is not None or grads[6] is not None \
                or (grads[2] is not None and spec.gate_kind == GATE_CHANNEL):
            _with_workspace(x.get_device(), x, "spira_b200_residual_norm_backward", desc)
        else:
            _launch(x.get_device(), "spira_b200_residual_norm_backward", desc, None, 0)
        return (None, *grads)


def residual_norm(feats: torch.Tensor, block: Optional[torch.Tensor] = None, *, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, pre: bool = True, post: bool = False, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, kind: str = "rms",
                  residual_scale: float = 1.0, block_scale: float = 1.0, eps: float = 1e-6
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(stream, normed)`` with

    ``stream = residual_scale * feats + block_scale * gate * p``, ``p = norm(block) * post_weight + post_bias`` if ``post``
    else ``block`` (without a block the stream is ``feats`` itself), and ``normed = norm(stream) * weight + bias`` (``None``
    with ``pre=False``).

    ``norm`` is ``v / sqrt(mean(v^2) + eps)`` for ``kind="rms"``, ``(v - mean) / sqrt(var + eps)`` for ``kind="layer"``, in
    fp32 on the unrounded stream.  ``feats`` and ``block`` are ``[N, C]`` in fp16, bf16 or fp32, ``C <= 8192`` (rows
    less than 2^31 elements apart); ``gate`` is a parameter ``[C]``, or ``[N, 1]`` or ``[N, C]`` in the type of ``feats``.
    Parameters are all fp32 or all of the type of ``feats``; a missing one counts as ones (weights) or zeros (biases).  The two
    scales are constants."""
    _device_of(feats, block, weight, bias, post_weight, post_bias, gate)
    if feats.dim() != 2 or feats.dtype not in _DTYPES:
        _fail(f"Tensor feats is expected to be a float16, bfloat16 or float32 matrix [N, C], got {feats.dtype} {tuple(feats.shape)}")
    n, channels = feats.shape
    if not 1 <= channels <= MAX_CHANNELS:
        _fail(f"residual_norm takes 1 to {MAX_CHANNELS} channels, got {channels}")
    if kind not in ("rms", "layer"):
        _fail(f"kind must be 'rms' or 'layer', got {kind!r}")
    if not eps > 0:
        _fail(f"eps must be positive, got {eps}")
    if block is None:
        if post or gate is not None or post_weight is not None or post_bias is not None or residual_scale != 1.0 or block_scale != 1.0:
            _fail("a gate, a scale or a norm after the block needs a block")
        if not pre:
            _fail("neither a block nor a norm: nothing to compute")
    elif block.shape != feats.shape or block.dtype != feats.dtype:
        _fail(f"block is expected to be {feats.dtype} {tuple(feats.shape)}, got {block.dtype} {tuple(block.shape)}")
    if not pre and (weight is not None or bias is not None):
        _fail("weight and bias belong to the norm that pre=False leaves out")
    if not post and (post_weight is not None or post_bias is not None):
        _fail("post_weight and post_bias need post=True")
    gate_kind, channel_gate = GATE_NONE, None
    if gate is not None:
        if gate.dim() == 1:
            gate_kind, channel_gate = GATE_CHANNEL, gate
            gate = gate.contiguous()
        elif gate.shape == (n, 1) or gate.shape == (n, channels):
            gate_kind = GATE_ROW if gate.shape[1] == 1 else GATE_FULL
            if gate.dtype != feats.dtype:
                _fail(f"a gate per row or element has the type of feats, {feats.dtype}, got {gate.dtype}")
            gate = _rows(gate)
        else:
            _fail(f"gate is expected to be [{channels}], [{n}, 1] or [{n}, {channels}], got {tuple(gate.shape)}")
    dtype, dense = None, True
    for p in (weight, bias, post_weight, post_bias, channel_gate):
        if p is not None:
            if p.shape != (channels,) or (p.dtype != feats.dtype and p.dtype != torch.float32):
                _fail(f"parameters (and a gate per channel) are expected to be {feats.dtype} or float32 [{channels}], got {p.dtype} {tuple(p.shape)}")
            if dtype is not None and p.dtype != dtype:
                _fail("parameters of one call must have one type")
            dtype = p.dtype
            dense = dense and p.is_contiguous()
    params = (weight, bias, post_weight, post_bias) if dense else tuple(p if p is None else p.contiguous() for p in (weight, bias, post_weight, post_bias))
    feats_rows = _rows(feats)
    block = None if block is None else _rows(block)
    spec = _Spec(dtype is torch.float32, kind == "layer", bool(pre), bool(post), gate_kind, float(residual_scale), float(block_scale), float(eps))
    if _needs_grad(feats, block, gate, *params):
        stream, normed = _ResidualNorm.apply(spec, feats_rows, block, gate, *params)
    else:
        stream, normed = _forward(spec, feats_rows, (block, gate, *params), None)
    return feats if block is None else stream, normed
