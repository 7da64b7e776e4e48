"""Behaviour shared by ``MXFPLinearPTQ`` and ``MinifloatLinearPTQ``.

Both layers keep integer code tensors as ``nn.Parameter``s (so they travel with
``state_dict``) next to plain-Python tensor metas (which do not).  Moving the module
must never re-type a code tensor, and must refresh the device recorded in the metas
because ``compose_*`` dispatches on the meta's device string
(reference: ``src/mase_triton/mxfp/layers.py:100-121``, ``src/mase_triton/minifloat/layers.py:89-108``).
"""

from __future__ import annotations

import torch
from torch import nn

from .utils.qlayer import ChangeDtypeError


class PTQLinearBase(nn.Module):
    # names of the integer code tensors, and for each tensor meta the code tensor whose device it follows
    _code_tensors: tuple[str, ...] = ()
    _meta_follows: dict[str, str] = {}

    in_features: int
    out_features: int

    # the quantised weight as the products with an epilogue read it, and what it was built from (mxfp.grouped.kept_weight)
    _row_weight = None

    def __getstate__(self):
        return self.__dict__ | {"_row_weight": None}          # a copy counts its tensors' versions anew

    def _replicate_for_data_parallel(self):
        replica = super()._replicate_for_data_parallel()
        replica._row_weight = None                            # packing the replica's tensors must not write to this layer's memory
        return replica

    def _apply(self, fn, recurse=True):
        def where():
            kept = {name: getattr(self, name) for name in self._code_tensors if getattr(self, name) is not None}
            return {name: (t.dtype, t.device, None if self._row_weight is None else t.data_ptr()) for name, t in kept.items()}

        before = where()
        result = super()._apply(fn, recurse)
        after = where()
        if any(after[name][1] != device for name, (_, device, _) in before.items()):
            self._row_weight = None
        elif self._row_weight is not None and after != before:
            # other storage on the same device, which counts no version: packed anew, into the memory that captured graphs point at
            self._row_weight = (None, *self._row_weight[1:])
        for name, (dtype, _, _) in before.items():
            now = after[name][0]
            if now != dtype:
                raise ChangeDtypeError(f"Changing dtype of {name} from {dtype} to {now} is not allowed.")
        for meta_name, tensor_name in self._meta_follows.items():
            meta, tensor = getattr(self, meta_name), getattr(self, tensor_name)
            if meta is not None and tensor is not None:
                moved = meta.create(device=tensor.device)
                if moved != meta:
                    setattr(self, meta_name, moved)
        return result

    @staticmethod
    def _frozen(t):
        if t.is_inference():
            # what a layer lays out once is rebuilt when a tensor's version changes, which inference tensors do not count
            with torch.inference_mode(False):
                t = t.clone()
        return nn.Parameter(t, requires_grad=False)
