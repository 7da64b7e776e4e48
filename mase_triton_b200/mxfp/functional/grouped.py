"""``mxfp_grouped_linear``: quantised linears grouped by expert (no counterpart in the reference)."""

from __future__ import annotations

import torch
from torch import Tensor

from .. import grouped as _grouped
from ..meta import MXFPMeta, MXFPTensorMeta


def expert_shape(w_tensor_meta: MXFPTensorMeta) -> tuple[int, int, int]:
    """``(groups, out_features, in_features)`` of a quantised expert weight; its blocks run along ``in_features``."""
    shape = tuple(w_tensor_meta.shape)
    if len(shape) != 3 or w_tensor_meta.block_dim not in (2, -1):
        raise ValueError(f"the weight has to be quantised as [groups, out_features, in_features] with block_dim=-1: got {shape}, block_dim={w_tensor_meta.block_dim}")
    return shape


@torch.no_grad()
def mxfp_grouped_linear(
    x: Tensor,
    x_meta: MXFPMeta,
    w_scales: Tensor,
    w_elements: Tensor,
    w_tensor_meta: MXFPTensorMeta,
    offsets: Tensor,
    bias: Tensor | None = None,
    activation: str | None = None,
    multiplier: Tensor | None = None,
    residual: Tensor | None = None,
    row_index: Tensor | None = None,
    out: Tensor | None = None,
) -> Tensor:
    """Row ``i`` of the result, for ``offsets[g] <= i < offsets[g + 1]``, is
    ``act(Q(x[row_index[i]]) @ W[g]^T + bias[g]) * multiplier[i]`` or ``... + residual[i]``.

    ``x [tokens, in_features]`` is quantised as ``x_meta`` says, the weights are
    ``extract_mxfp_components(weight, -1, meta)`` of a ``[groups, out_features, in_features]`` tensor.  ``offsets``
    (int32 or int64, ``groups + 1`` entries, rising) is read on the GPU: nothing is copied to the host, and the call can be
    captured in a CUDA graph and replayed with other offsets.  Entries are clamped to the rows there are.
    ``row_index`` (int32 or int64) names the row of ``x`` for each row of the result, e.g. the token of each (token, expert)
    pair; without it row ``i`` is ``x[i]``, and an index outside ``x`` stands for a row of zeros.  ``activation``: ``"relu"``, ``"gelu"``,
    ``"gelu_tanh"``, ``"silu"`` or ``None``.  Bias, ``multiplier`` and ``residual`` have ``x``'s dtype; everything behind the
    product is computed in fp32 and rounded once.  With ``out`` the rows outside every group keep what they hold
    (``out`` may be the residual itself); without it they are zero.

    The weights are packed for the tensor cores in every call; ``MXFPGroupedLinearPTQ`` keeps them packed."""
    groups, n, k = expert_shape(w_tensor_meta)
    w = _grouped.pack_experts(w_scales, w_elements, groups, n, k, w_tensor_meta.meta, x_meta)
    return _grouped.grouped_linear(x, x_meta, w, offsets, bias, activation, multiplier, residual, row_index, out)
