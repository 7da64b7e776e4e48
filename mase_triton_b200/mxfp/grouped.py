"""Host side of the products with an epilogue (``csrc/mxq_grouped.cu``): one quantised weight for all rows of an
activation, or one for each group of rows (experts).  The reference has neither (its linears are
``src/mase_triton/mxfp/functional/linear.py:10-210``: a product and a bias)."""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch import Tensor

from .. import _lib
from .gemm import _raise_if_failed, fp4_pair, is_e2m1, status_word, supported
from .meta import MXFPMeta

EXTRA_NONE, EXTRA_MULTIPLY, EXTRA_ADD = 0, 1, 2
_INDEX_DTYPES = (torch.int32, torch.int64)


@dataclass
class PackedExperts:
    """Weights ``[groups, N, K]`` as the kernel reads them: hardware codes (bytes, or nibbles when ``hw_format`` is 5)
    and scale chunks of every group."""

    codes: Tensor
    sf: Tensor
    hw_format: int
    groups: int
    N: int
    K: int


def check_formats(x_meta: MXFPMeta | None, w_meta: MXFPMeta | None, K: int) -> None:
    if not (supported(x_meta) and supported(w_meta)):
        raise ValueError("activation and weight have to be MXFP with 32-element blocks and is_finite elements: "
                         f"got x_meta={x_meta}, w_meta={w_meta}")
    if K <= 0 or K % 32 != 0:
        raise ValueError(f"in_features has to be a positive multiple of 32: got {K}")


def pack_experts(w_scales: Tensor, w_elements: Tensor, groups: int, N: int, K: int, w_meta: MXFPMeta, x_meta: MXFPMeta) -> PackedExperts:
    """Reference ``(scales, elements)`` of a ``[groups, N, K]`` weight with blocks along K, for activations of ``x_meta``
    (an MXFP4 pair with K a multiple of 256 keeps packed nibbles and runs on the 4-bit x 4-bit tensor-core kind)."""
    _lib.require_cuda(w_elements, "pack_experts")
    check_formats(x_meta, w_meta, K)
    if w_elements.dtype != torch.uint8 or w_scales.dtype != torch.uint8:
        raise ValueError(f"weight codes and scales have to be uint8: got {w_elements.dtype} and {w_scales.dtype}")
    if w_elements.numel() != groups * N * K or w_scales.numel() != groups * N * K // 32:
        raise ValueError(f"{w_elements.numel()} codes and {w_scales.numel()} scales are not a weight of shape [{groups}, {N}, {K}]")
    if w_scales.device != w_elements.device:
        raise ValueError(f"weight codes are on {w_elements.device}, scales on {w_scales.device}")
    L, dev = _lib.load(), w_elements.device
    if groups > L.mxq_mx_max_groups():
        raise ValueError(f"{groups} groups: {L.mxq_mx_max_groups()} at most")
    nibbles = fp4_pair(x_meta, w_meta, K)
    w_scales, w_elements = w_scales.contiguous(), w_elements.contiguous()
    if w_elements.data_ptr() % 16 != 0:
        w_elements = w_elements.clone()
    codes = torch.empty((groups, N, K // 2 if nibbles else K), dtype=torch.uint8, device=dev)
    sf = torch.empty((groups * L.mxq_mx_sf_bytes(N, K, 0, 0),), dtype=torch.uint8, device=dev)
    fmt = ctypes.c_int(0)
    with torch.cuda.device(dev):
        rc = L.mxq_mx_pack_experts(w_scales.data_ptr(), w_elements.data_ptr(), groups, N, K, w_meta.element_exp_bits, w_meta.element_frac_bits,
                                   int(nibbles), codes.data_ptr(), sf.data_ptr(), ctypes.addressof(fmt), _lib.stream_ptr(dev))
    _lib.check(rc, "mxq_mx_pack_experts")
    return PackedExperts(codes, sf, fmt.value, groups, N, K)


def epilogue_operand(multiplier: Tensor | None, residual: Tensor | None) -> tuple[Tensor | None, int]:
    """The second operand of an epilogue and what is done with it."""
    if multiplier is not None and residual is not None:
        raise ValueError("an epilogue takes a multiplier or a residual, not both")
    if multiplier is not None:
        return multiplier, EXTRA_MULTIPLY
    return (None, EXTRA_NONE) if residual is None else (residual, EXTRA_ADD)


def check_activation(activation: str | None) -> int:
    try:
        return _lib.ACTIVATION_ID[activation]
    except KeyError:
        raise ValueError(f"activation {activation!r}: one of {[a for a in _lib.ACTIVATION_ID if a]} or None") from None


def _index(t: Tensor, name: str, n: int | None, dev: torch.device) -> Tensor:
    if t.dtype not in _INDEX_DTYPES or t.ndim != 1 or (n is not None and t.numel() != n):
        raise ValueError(f"{name} has to be a 1-D int32 or int64 tensor{'' if n is None else f' of {n} entries'}: got {t.dtype} {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the input on {dev}")
    return t.contiguous()


def grouped_linear(x: Tensor, x_meta: MXFPMeta, w: PackedExperts, offsets: Tensor | None, bias: Tensor | None = None,
                   activation: str | None = None, multiplier: Tensor | None = None, residual: Tensor | None = None,
                   row_index: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """``act(Q(x[row_index]) @ W_g^T + bias_g) (* multiplier | + residual)`` for ``x [tokens, K]``; the rows of group ``g`` are
    ``offsets[g] .. offsets[g + 1]`` (``offsets=None``: one group of all rows).  Returns ``[rows, N]`` of ``x``'s dtype."""
    _lib.require_cuda(x, "grouped_linear")
    act = check_activation(activation)
    extra, extra_mode = epilogue_operand(multiplier, residual)
    if x.dtype not in _lib.DTYPE_ID:
        raise ValueError(f"input dtype {x.dtype}: one of {[str(d) for d in _lib.DTYPE_ID]}")
    if x.ndim != 2 or x.shape[1] != w.K:
        raise ValueError(f"input of shape {tuple(x.shape)}: expected [tokens, {w.K}]")
    if not supported(x_meta) or (w.hw_format == 5 and not is_e2m1(x_meta)):
        raise ValueError(f"the weight was packed for another activation format than {x_meta}")
    dev, tokens, N = x.device, x.shape[0], w.N
    if w.codes.device != dev:
        raise ValueError(f"the weight is on {w.codes.device}, the input on {dev}")
    x = x.contiguous()
    if offsets is not None:
        offsets = _index(offsets, "offsets", w.groups + 1, dev)
    elif w.groups != 1:
        raise ValueError("offsets are missing")
    rows = tokens
    if row_index is not None:
        row_index = _index(row_index, "row_index", None, dev)
        rows = row_index.numel()
    for name, t, shape in (("bias", bias, (w.groups, N)), ("multiplier" if multiplier is not None else "residual", extra, (rows, N)), ("out", out, (rows, N))):
        if t is not None and (t.device != dev or t.dtype != x.dtype or tuple(t.shape) != shape):
            raise ValueError(f"{name} has to be {x.dtype} {shape} on {dev}: got {t.dtype} {tuple(t.shape)} on {t.device}")
    if out is not None and not out.is_contiguous():
        raise ValueError("out has to be contiguous")
    bias = None if bias is None else bias.contiguous()
    extra = None if extra is None else extra.contiguous()
    zero_rest = out is None and offsets is not None
    if out is None:
        out = torch.empty((rows, N), dtype=x.dtype, device=dev)
    if rows == 0:
        return out
    _raise_if_failed(dev)
    L = _lib.load()
    nbytes = L.mxq_mx_grouped_scratch_bytes(tokens, rows, w.K)
    # of this call alone: two captured graphs, or two streams, never share it
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = L.mxq_mx_grouped_linear(
            x.data_ptr(), _lib.DTYPE_ID[x.dtype], tokens, rows, w.K, x_meta.element_exp_bits, x_meta.element_frac_bits, _lib.ROUND_ID[x_meta.round_mode],
            None if row_index is None else row_index.data_ptr(), int(row_index is not None and row_index.dtype == torch.int64),
            w.codes.data_ptr(), w.sf.data_ptr(), w.hw_format, w.groups, N,
            None if offsets is None else offsets.data_ptr(), int(offsets is not None and offsets.dtype == torch.int64),
            out.data_ptr(), None if bias is None else bias.data_ptr(), act, None if extra is None else extra.data_ptr(), extra_mode, int(zero_rest),
            scratch.data_ptr(), nbytes, status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "mxq_mx_grouped_linear")
    return out
