"""What a layer keeps of its packed weight, and when it lays it out anew: the host's part, with the packing itself replaced."""

from __future__ import annotations

import contextlib

import pytest
import torch

from mase_triton_b200 import _lib
from mase_triton_b200.mxfp import grouped as GR
from mase_triton_b200.mxfp.layers import MXFPGroupedLinearPTQ, MXFPLinearPTQ
from mase_triton_b200.mxfp.meta import MXFPTensorMeta, MXFP8_E4M3_fn

E, N, K = 3, 8, 64


def a_layer():
    tm = MXFPTensorMeta("cpu", "bfloat16", (E, N, K), -1, MXFP8_E4M3_fn)
    codes = torch.arange(E * N * K, dtype=torch.int64).to(torch.uint8).reshape(-1, 32)
    return MXFPGroupedLinearPTQ(torch.full((E * N * K // 32, 1), 127, dtype=torch.uint8), codes, tm, None, MXFP8_E4M3_fn)


def a_linear():
    tm = MXFPTensorMeta("cpu", "bfloat16", (N, K), -1, MXFP8_E4M3_fn)
    codes = torch.zeros(N * K // 32, 32, dtype=torch.uint8)
    return MXFPLinearPTQ.from_quantized(torch.full((N * K // 32, 1), 127, dtype=torch.uint8), codes, tm, None, None, None, None, MXFP8_E4M3_fn, "XqWqB", "fused")


@pytest.fixture
def log(monkeypatch):
    """The calls in their order: "wait for the device", "wait for the stream", ("pack", memory it was given)."""
    calls = []

    class Stream:
        def synchronize(self):
            calls.append("wait for the stream")

    def pack(w_scales, w_elements, groups, n, k, w_meta, x_meta, into=None):
        blocks = into.blocks if into is not None else torch.empty(w_elements.numel(), dtype=torch.uint8)
        calls.append(("pack", None if into is None else into.blocks.data_ptr()))
        blocks.copy_(w_elements.reshape(-1))
        return GR.PackedExperts(blocks, 0, groups, n, k)

    monkeypatch.setattr(GR, "pack_experts", pack)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: calls.append("wait for the device"))
    return calls


def packs(log):
    return [c for c in log if isinstance(c, tuple)]


@pytest.mark.parametrize("make", [a_layer, a_linear])
@pytest.mark.parametrize("move", [lambda m: m.to("cpu"), lambda m: m.to(torch.bfloat16), lambda m: m.cpu(), lambda m: torch.nn.Sequential(m).to("cpu")[0], lambda m: m.float()])
def test_a_move_that_moves_nothing_keeps_the_packed_weight(log, make, move):
    """A captured graph holds the address of the blocks only."""
    layer = make()
    packed = layer.row_weight()
    move(layer)
    assert layer.row_weight() is packed and len(packs(log)) == 1


def test_a_move_to_another_device_gives_the_packed_weight_up(log):
    layer = a_layer()
    layer.row_weight()
    layer.to("meta")
    assert layer._row_weight is None and layer.w_tensor_meta.device == "meta"


def test_codes_with_new_storage_are_packed_into_the_same_memory(log):
    """``_apply`` may give a Parameter other storage without counting a version, and after two such turns the first address again."""
    layer = a_layer()
    first = layer.row_weight().pointer
    address = layer.w_elements.data_ptr()
    held = [layer.w_elements.data]
    layer._apply(lambda t: t.clone())
    assert layer.w_elements.data_ptr() != address

    def back(t):
        return held[0].add_(1) if t.shape == held[0].shape else t

    layer._apply(back)
    assert layer.w_elements.data_ptr() == address
    again = layer.row_weight()
    assert again.pointer == first and len(packs(log)) == 2
    assert torch.equal(again.blocks, layer.w_elements.reshape(-1))


@pytest.mark.parametrize("change", ["written", "replaced", "loaded", "assigned", "functional_call"])
def test_readers_on_every_stream_are_done_before_the_memory_is_written_again(log, change):
    """A product that another stream, or a graph there, still runs reads the blocks; whoever replaces a Parameter writes to nothing
    that it was given, and has no reason to wait for it."""
    layer = a_layer()
    first = layer.row_weight()
    log.clear()
    other = {"w_elements": layer.w_elements.data + 1, "w_scales": layer.w_scales.data.clone()}
    if change == "written":
        layer.w_elements.add_(1)
    elif change == "replaced":
        layer.w_elements = torch.nn.Parameter(other["w_elements"], requires_grad=False)
    elif change == "functional_call":
        layer.forward = lambda: layer.row_weight()
        packed = torch.func.functional_call(layer, other, ())
    else:
        layer.load_state_dict(other, assign=change == "assigned")
    if change != "functional_call":
        packed = layer.row_weight()
    assert packed.pointer == first.pointer and torch.equal(packed.blocks, other["w_elements"].reshape(-1))
    assert log == ["wait for the device", ("pack", first.pointer), "wait for the stream"]


def test_the_first_packing_waits_for_no_reader(log):
    a_layer().row_weight()
    assert log == [("pack", None), "wait for the stream"]


@pytest.mark.parametrize("make", [a_layer, a_linear])
def test_replicas_pack_their_own_copy(log, make):
    """A replica of ``nn.DataParallel`` holds its tensors as plain attributes; its blocks are not those of the module it was made from."""
    layer = make()
    packed = layer.row_weight()
    replica = layer._replicate_for_data_parallel()
    replica.w_scales, replica.w_elements = layer.w_scales.data.clone(), layer.w_elements.data + 1
    theirs = replica.row_weight()
    assert theirs.pointer != packed.pointer and torch.equal(theirs.blocks, replica.w_elements.reshape(-1))
    assert replica.row_weight() is theirs and layer.row_weight() is packed
    assert torch.equal(packed.blocks, layer.w_elements.reshape(-1))
