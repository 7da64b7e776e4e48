"""Host side of the products with an epilogue (``csrc/mxq_grouped.cu``): one quantised weight for all rows of an
activation, or one for each group of rows (experts).  The reference has neither (its linears are
``src/mase_triton/mxfp/functional/linear.py:10-210``: a product and a bias)."""

from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass

import torch
from torch import Tensor

from .. import _lib
from .gemm import fp4_pair, is_e2m1, status_address, supported
from .meta import MXFPMeta

EXTRA_NONE, EXTRA_MULTIPLY, EXTRA_ADD = 0, 1, 2
_INDEX_DTYPES = (torch.int32, torch.int64)
# mxq_grouped_linear_args: one packed argument costs the host 1 us, 26 separate ones cost it 2.5
_ARGS = struct.Struct("@10P6q10i")


@dataclass
class PackedExperts:
    """Weights ``[groups, N, K]`` as the kernels read them: blocks of 128 features and 128 elements of K (256 for packed
    4-bit codes, ``hw_format`` 5), the codes of a block and its scales one after the other."""

    blocks: Tensor
    hw_format: int
    groups: int
    N: int
    K: int

    def __post_init__(self):
        self.device_index, self.pointer = self.blocks.get_device(), self.blocks.data_ptr()
        self._row_format: tuple[MXFPMeta | None, tuple[int, int, int]] = (None, (0, 0, 0))
        self._scratch_bytes: dict[tuple[int, int, int, bool], int] = {}

    def row_format(self, x_meta: MXFPMeta) -> tuple[int, int, int]:
        """Exponent bits, fraction bits and rounding mode of an activation format that goes with these weights."""
        known, row_format = self._row_format
        if known is not x_meta:
            if not supported(x_meta) or (self.hw_format == 5 and not is_e2m1(x_meta)):
                raise ValueError(f"the weight was packed for another activation format than {x_meta}")
            row_format = (x_meta.element_exp_bits, x_meta.element_frac_bits, _lib.ROUND_ID[x_meta.round_mode])
            self._row_format = (x_meta, row_format)
        return row_format

    def scratch_bytes(self, x_ptr: int, round_id: int, tokens: int, rows: int) -> int:
        """Workspace of a call (asked of the library once per size)."""
        key = (tokens, rows, round_id, x_ptr % 16 == 0)
        known = self._scratch_bytes.get(key)
        if known is None:
            with torch.cuda.device(self.device_index):
                known = _lib.load().mxq_mx_grouped_scratch_bytes(x_ptr, round_id, tokens, rows, self.K, self.groups, self.N)
            if len(self._scratch_bytes) >= 4096:
                self._scratch_bytes.clear()
            self._scratch_bytes[key] = known
        return known


def check_formats(x_meta: MXFPMeta | None, w_meta: MXFPMeta | None, K: int) -> None:
    if not (supported(x_meta) and supported(w_meta)):
        raise ValueError("activation and weight have to be MXFP with 32-element blocks and is_finite elements: "
                         f"got x_meta={x_meta}, w_meta={w_meta}")
    if K <= 0 or K % 32 != 0:
        raise ValueError(f"in_features has to be a positive multiple of 32: got {K}")


def pack_experts(w_scales: Tensor, w_elements: Tensor, groups: int, N: int, K: int, w_meta: MXFPMeta, x_meta: MXFPMeta,
                 into: PackedExperts | None = None) -> PackedExperts:
    """Reference ``(scales, elements)`` of a ``[groups, N, K]`` weight with blocks along K, for activations of ``x_meta``
    (an MXFP4 pair with K a multiple of 256 keeps packed nibbles and runs on the 4-bit x 4-bit tensor-core kind).
    ``into``: an earlier result whose memory is taken again where it fits."""
    _lib.require_cuda(w_elements, "pack_experts")
    check_formats(x_meta, w_meta, K)
    if groups <= 0 or N <= 0:
        raise ValueError(f"a weight of shape [{groups}, {N}, {K}] has no entries")
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
    nbytes = L.mxq_mx_packed_experts_bytes(groups, N, K, int(nibbles))
    blocks = into.blocks if into is not None and into.blocks.numel() == nbytes and into.blocks.device == dev else \
        torch.empty(nbytes, dtype=torch.uint8, device=dev)
    fmt = ctypes.c_int(0)
    with torch.cuda.device(dev):
        rc = L.mxq_mx_pack_experts(w_scales.data_ptr(), w_elements.data_ptr(), groups, N, K, w_meta.element_exp_bits, w_meta.element_frac_bits,
                                   int(nibbles), blocks.data_ptr(), ctypes.addressof(fmt), _lib.stream_ptr(dev))
    _lib.check(rc, "mxq_mx_pack_experts")
    return PackedExperts(blocks, fmt.value, groups, N, K)


def kept_weight(layer, groups: int, N: int, K: int) -> PackedExperts:
    """The packed weight of a layer (``w_scales``, ``w_elements``, ``w_tensor_meta``, ``x_mxfp_meta``), kept with it until its code tensors
    are written, replaced or moved.  It is packed anew into the same memory, so that a captured graph finds it there, once nothing
    on the device reads that memory any more (a replay on any stream may), and before this returns it is complete for every
    stream.  While a graph is captured nothing is kept: packing is then part of the graph."""
    params, kept = layer._parameters, layer._row_weight
    if "w_elements" in params:
        w_scales, w_elements = params["w_scales"], params["w_elements"]
    else:                                                            # a replica of nn.DataParallel: plain attributes
        w_scales, w_elements = layer.w_scales, layer.w_elements
    try:
        state = (w_elements._version, w_scales._version, w_elements.data_ptr(), w_scales.data_ptr())
    except RuntimeError:                                             # inference tensors count no versions: packed in every call
        return pack_experts(w_scales.data, w_elements.data, groups, N, K, layer.w_tensor_meta.meta, layer.x_mxfp_meta)
    if kept is not None and kept[0] is w_elements and kept[1] is w_scales and kept[2] is layer.w_tensor_meta and kept[3] is layer.x_mxfp_meta and kept[4] == state:
        return kept[5]
    _lib.require_cuda(w_elements, "pack_experts")
    with torch.cuda.device(w_elements.device):
        capturing = torch.cuda.is_current_stream_capturing()
        if kept is not None and not capturing:
            torch.cuda.synchronize()
        packed = pack_experts(w_scales.data, w_elements.data, groups, N, K, layer.w_tensor_meta.meta, layer.x_mxfp_meta,
                              None if kept is None or capturing else kept[5])
        if not capturing:
            torch.cuda.current_stream().synchronize()
            layer._row_weight = (w_elements, w_scales, layer.w_tensor_meta, layer.x_mxfp_meta, state, packed)
    return packed


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


def _bad_index(t: Tensor, name: str, n: int | None, dev: int) -> bool:
    return t.dtype not in _INDEX_DTYPES or t.ndim != 1 or (n is not None and t.shape[0] != n) or t.get_device() != dev


def _index_error(t: Tensor, name: str, n: int | None, x: Tensor) -> ValueError:
    return ValueError(f"{name} has to be a 1-D int32 or int64 tensor{'' if n is None else f' of {n} entries'} on {x.device}: "
                      f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _operand_error(t: Tensor, name: str, shape: tuple, x: Tensor) -> ValueError:
    return ValueError(f"{name} has to be {x.dtype} {shape} on {x.device}: got {t.dtype} {tuple(t.shape)} on {t.device}")


def grouped_linear(x: Tensor, x_meta: MXFPMeta, w: PackedExperts, offsets: Tensor | None, bias: Tensor | None = None,
                   activation: str | None = None, multiplier: Tensor | None = None, residual: Tensor | None = None,
                   row_index: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """``act(Q(x[row_index]) @ W_g^T + bias_g) (* multiplier | + residual)`` for ``x [tokens, K]``; the rows of group ``g`` are
    ``offsets[g] .. offsets[g + 1]`` (``offsets=None``: one group of all rows).  Returns ``[rows, N]`` of ``x``'s dtype.

    A decoding step makes hundreds of these calls of a few microseconds each on the GPU, so the checks here are kept
    to a few attribute reads each."""
    if not x.is_cuda:
        _lib.require_cuda(x, "grouped_linear")
    act = check_activation(activation)
    extra, extra_mode = epilogue_operand(multiplier, residual)
    dtype, dev, N, K, groups = x.dtype, x.get_device(), w.N, w.K, w.groups
    dtype_id = _lib.DTYPE_ID.get(dtype)
    if dtype_id is None:
        raise ValueError(f"input dtype {dtype}: one of {[str(d) for d in _lib.DTYPE_ID]}")
    if x.ndim != 2 or x.shape[1] != K:
        raise ValueError(f"input of shape {tuple(x.shape)}: expected [tokens, {K}]")
    exp_bits, frac_bits, round_id = w.row_format(x_meta)
    if w.device_index != dev:
        raise ValueError(f"the weight is on {w.blocks.device}, the input on {x.device}")
    x = x.contiguous()
    tokens = rows = x.shape[0]
    offsets_ptr = index_ptr = bias_ptr = extra_ptr = offsets64 = index64 = 0
    if offsets is not None:
        if _bad_index(offsets, "offsets", groups + 1, dev):
            raise _index_error(offsets, "offsets", groups + 1, x)
        offsets = offsets.contiguous()
        offsets_ptr, offsets64 = offsets.data_ptr(), int(offsets.dtype == torch.int64)
    elif groups != 1:
        raise ValueError("offsets are missing")
    if row_index is not None:
        if _bad_index(row_index, "row_index", None, dev):
            raise _index_error(row_index, "row_index", None, x)
        row_index = row_index.contiguous()
        rows = row_index.shape[0]
        index_ptr, index64 = row_index.data_ptr(), int(row_index.dtype == torch.int64)
    if bias is not None:
        if bias.dtype != dtype or bias.get_device() != dev or (bias.shape != (groups, N) and (offsets is not None or bias.shape != (N,))):
            raise _operand_error(bias, "bias", (groups, N), x)
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if extra is not None:
        if extra.dtype != dtype or extra.shape != (rows, N) or extra.get_device() != dev:
            raise _operand_error(extra, "residual" if multiplier is None else "multiplier", (rows, N), x)
        extra = extra.contiguous()
        extra_ptr = extra.data_ptr()
    zero_rest = 0
    if out is None:
        zero_rest = int(offsets is not None)
        out = x.new_empty(rows, N)
    else:
        if out.dtype != dtype or out.shape != (rows, N) or out.get_device() != dev:
            raise _operand_error(out, "out", (rows, N), x)
        if not out.is_contiguous():
            raise ValueError("out has to be contiguous")
        begin, end = out.data_ptr(), out.data_ptr() + out.nbytes
        for t, name in ((x, "input"), (offsets, "offsets"), (row_index, "row_index"), (bias, "bias"), (extra, "multiplier or residual")):
            if t is not None and t.data_ptr() < end and begin < t.data_ptr() + t.nbytes and not (t is extra and t.data_ptr() == begin):
                raise ValueError(f"out overlaps the {name}, which other rows of the result are still computed from")
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)
    if rows == 0:
        return out
    status = status_address(dev)
    x_ptr = x.data_ptr()
    nbytes = w.scratch_bytes(x_ptr, round_id, tokens, rows)
    # of this call alone: two captured graphs, or two streams, never share it
    scratch = None if nbytes == 0 else x.new_empty(nbytes // x.element_size())           # (a multiple of 256 bytes)
    args = _ARGS.pack(x_ptr, index_ptr, w.pointer, offsets_ptr, out.data_ptr(), bias_ptr, extra_ptr, 0 if scratch is None else scratch.data_ptr(), status,
                      _lib.raw_stream(dev), tokens, rows, K, groups, N, nbytes, dtype_id, exp_bits, frac_bits, round_id, index64, offsets64, w.hw_format, act,
                      extra_mode, zero_rest)
    run = _lib.load().mxq_mx_grouped_linear
    if _lib.current_device() == dev:
        rc = run(args)
    else:
        with torch.cuda.device(dev):
            rc = run(args)
    if rc != 0:
        _lib.check(rc, "mxq_mx_grouped_linear")
    return out
