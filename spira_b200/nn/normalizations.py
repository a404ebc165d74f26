"""Norms over SparseTensor features: BatchNorm (reference: spira/nn/normalizations.py:8-10) and the norms around a block
with its gate and residual in one pass (no reference counterpart)."""
__all__ = ['BatchNorm', 'ResidualNorm']

from typing import Optional

import torch

from spira_b200.nn.functional.norms import residual_norm
from spira_b200.utils.apply import fapply


class BatchNorm(torch.nn.BatchNorm1d):
    def forward(self, input):
        return fapply(input, super().forward)


class ResidualNorm(torch.nn.Module):
    """``stream, normed = module(inputs, block)`` over the voxels of SparseTensors:

    ``stream = residual_scale * inputs + block_scale * gate * p`` with ``p = norm(block)`` if ``post`` else ``block``, and
    ``normed = norm(stream)``.  ``kind`` is ``"rms"`` or ``"layer"`` (then with biases); ``gate=True`` learns one factor per
    channel (initial value ``gate_init``).  Without a block (the first norm of a network) the stream is ``inputs`` itself;
    ``post``, gate and scales then have nothing to act on and are left out.  ``compile_model`` replays a network that holds this
    module operator by operator (the library's tape executor takes convolutions only)."""

    def __init__(self, channels: int, kind: str = "rms", post: bool = False, gate: bool = False, gate_init: float = 1.0,
                 residual_scale: float = 1.0, block_scale: float = 1.0, eps: float = 1e-6):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
        self.channels, self.kind, self.post, self.eps = channels, kind, post, eps
        self.residual_scale, self.block_scale = residual_scale, block_scale
        one = lambda wanted, value: torch.nn.Parameter(torch.full((channels,), float(value))) if wanted else None  # noqa: E731
        self.register_parameter('weight', one(True, 1))
        self.register_parameter('bias', one(kind == "layer", 0))
        self.register_parameter('post_weight', one(post, 1))
        self.register_parameter('post_bias', one(post and kind == "layer", 0))
        self.register_parameter('gate', one(gate, gate_init))

    def _alone(self, feats: torch.Tensor):
        return residual_norm(feats, weight=self.weight, bias=self.bias, kind=self.kind, eps=self.eps)[1]

    def _around(self, feats: torch.Tensor, block: torch.Tensor):
        return residual_norm(feats, block, weight=self.weight, bias=self.bias, post=self.post, post_weight=self.post_weight,
                             post_bias=self.post_bias, gate=self.gate, kind=self.kind, residual_scale=self.residual_scale,
                             block_scale=self.block_scale, eps=self.eps)

    def forward(self, inputs, block: Optional["SparseTensor"] = None):  # noqa: F821
        if block is None:
            return inputs, fapply(inputs, self._alone)
        from spira_b200.tensors import SparseTensor
        from spira_b200 import compile as _compile
        outputs = tuple(SparseTensor(coordinates=inputs._coordinates, features=f, stride=inputs._stride)
                        for f in self._around(inputs._features, block._features))
        if _compile._recorder is not None:
            _compile._recorder.call(self._around, (inputs, block), outputs)
        return outputs
