"""``SparseExperts``: a feed-forward layer of routed experts over the voxels of a SparseTensor.

No reference counterpart; it stands beside the 1x1x1 ``SparseConv`` (one weight matrix for all voxels) as the layer with
one pair of weight matrices per expert and ``top_k`` experts per voxel.
"""
__all__ = ['SparseExperts']

import math
from typing import Optional

import torch
from torch.nn import Module

from spira_b200.nn.functional import _C
from spira_b200.nn.functional.experts import expert_combine, expert_dispatch, expert_route, grouped_linear
from spira_b200.utils.apply import fapply


class SparseExperts(Module):
    """``out = sum over the voxel's experts e of weight_e * (relu(x W1[e] + b1[e]) W2[e] + b2[e])``, experts and weights from
    ``expert_route(x @ router, top_k)``.  ``forward(inputs, mask)``: voxels where the boolean ``mask [N]`` is False go to no
    expert and come out as zeros; what they hold (also NaN) shows nowhere.  Weights are laid out like ``SparseConv.kernel``: ``[E, c_in, c_out]``.

    Runs in float16 or bfloat16, module and features alike (``module.cuda().half()``).  The router's logits have that type too;
    for logits of another precision call ``expert_route`` and the functions behind it.  ``compile_model`` replays a network
    that holds this module operator by operator (the library's tape executor takes convolutions only)."""

    def __init__(self, in_channels: int, hidden_channels: int, num_experts: int, top_k: int = 2, out_channels: Optional[int] = None,
                 bias: bool = True, renormalize: bool = True):
        super().__init__()
        if not 1 <= top_k <= num_experts:
            raise ValueError(f"top_k must be 1 to num_experts, got {top_k} of {num_experts}")
        self.in_channels, self.hidden_channels, self.num_experts, self.top_k = in_channels, hidden_channels, num_experts, top_k
        self.out_channels = in_channels if out_channels is None else out_channels
        self.renormalize = renormalize
        self.router = torch.nn.Parameter(torch.empty(in_channels, num_experts))
        self.kernel1 = torch.nn.Parameter(torch.empty(num_experts, in_channels, hidden_channels))
        self.kernel2 = torch.nn.Parameter(torch.empty(num_experts, hidden_channels, self.out_channels))
        if bias:
            self.bias1 = torch.nn.Parameter(torch.empty(num_experts, hidden_channels))
            self.bias2 = torch.nn.Parameter(torch.empty(num_experts, self.out_channels))
        else:
            self.register_parameter('bias1', None)
            self.register_parameter('bias2', None)
        self.reset_parameters()

    def reset_parameters(self):
        for p, fan_in in ((self.router, self.in_channels), (self.kernel1, self.in_channels), (self.bias1, self.in_channels),
                          (self.kernel2, self.hidden_channels), (self.bias2, self.hidden_channels)):
            if p is not None:
                p.data.uniform_(-1. / math.sqrt(fan_in), 1. / math.sqrt(fan_in))

    def logits(self, feats: torch.Tensor) -> torch.Tensor:
        """Router logits ``[N, E]``: a 1x1x1 layer, on the kernel such layers run on where it takes the shape."""
        pointwise = getattr(_C, "pointwise", None)
        if pointwise is not None and not torch.is_grad_enabled():
            y = pointwise(feats, self.router, None)
            if y is not None:
                return y
        return torch.mm(feats, self.router)

    def _run(self, feats: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        for p in (self.router, self.kernel1, self.kernel2):
            if feats.dtype not in (torch.float16, torch.bfloat16) or p.dtype != feats.dtype:
                raise RuntimeError(f"[spira_b200] SparseExperts runs in float16 or bfloat16, module and features alike (module.cuda().half()), "
                                   f"got features {feats.dtype} and weights {p.dtype}")
        if mask is not None and torch.is_grad_enabled():      # (0 * NaN would reach the router's gradient)
            feats = feats.masked_fill(~mask[:, None], 0)
        logits = self.logits(feats)
        if mask is not None:
            logits = logits.masked_fill(~mask[:, None], float("-inf"))
        routing = expert_route(logits, self.top_k, renormalize=self.renormalize)
        rows = expert_dispatch(feats, routing)
        rows = grouped_linear(rows, self.kernel1, routing.offsets, self.bias1, relu=True)
        rows = grouped_linear(rows, self.kernel2, routing.offsets, self.bias2)
        return expert_combine(rows, routing)

    def forward(self, inputs, mask: Optional[torch.Tensor] = None):
        if mask is not None and (mask.dtype != torch.bool or mask.shape != (inputs._features.shape[0],)):
            raise ValueError(f"mask is expected to be bool [{inputs._features.shape[0]}], got {mask.dtype} {tuple(mask.shape)}")
        if mask is not None:
            from spira_b200 import compile as _compile
            if _compile._recorder is not None:
                raise RuntimeError("[spira_b200] compile_model cannot record a mask (it belongs to one scene); call SparseExperts eagerly")
            return fapply(inputs, self._run, mask)
        return fapply(inputs, self._run)
