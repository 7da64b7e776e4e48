"""Packed weights of layers under captured graphs and beside other streams."""

from __future__ import annotations

import pytest
import torch
from test_gpu_grouped import DEV, grouped_case, linear_layer, offsets_of, rand

from mase_triton_b200.mxfp.layers import MXFPGroupedLinearPTQ
from mase_triton_b200.mxfp.meta import MXFP8_E4M3_fn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("move", [lambda m: m.to(DEV), lambda m: m.cuda(), lambda m: m.to(torch.bfloat16)])
def test_a_captured_graph_keeps_its_weights_through_a_move_that_moves_nothing(lib, move):
    counts = [5, 6]
    off = offsets_of(counts)
    layer, _, _, x = grouped_case(counts, 256, 512, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    linear, _, _ = linear_layer(256, 512, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=True)
    want, want_lin = layer(x, off), linear(x, activation="silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_lin = layer(x, off), linear(x, activation="silu")
    held = [m.row_weight().pointer for m in (layer, linear)]
    move(layer), move(linear)
    assert [m.row_weight().pointer for m in (layer, linear)] == held
    # memory that had been given back would be handed out here
    filled = [torch.full((m.row_weight().blocks.numel(),), 0x38, dtype=torch.uint8, device=DEV) for m in (layer, linear) for _ in range(4)]
    got.zero_(), got_lin.zero_()
    graph.replay()
    assert torch.equal(got, want) and torch.equal(got_lin, want_lin) and len(filled) == 8
    assert torch.equal(layer(x, off), want)


@pytest.mark.parametrize("how", ["call", "replay"])
def test_a_product_still_queued_elsewhere_has_the_weights_of_its_call(lib, how):
    """A code tensor that is replaced leaves what a running call was given as it is; so does packing the new one."""
    counts = [5, 200]
    off = offsets_of(counts)
    layer, _, _, x = grouped_case(counts, 512, 1024, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    other = MXFPGroupedLinearPTQ.from_weight(rand(2, 512, 1024, seed=31), layer.bias, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    old, new = layer(x, off), other(x, off)
    assert not torch.equal(old, new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = layer(x, off)
    big = torch.ones(1 << 28, device=DEV)
    busy = torch.cuda.Stream()
    busy.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(busy):
        for _ in range(20):
            big.mul_(1.0)
        if how == "call":
            queued = layer(x, off)
        else:
            graph.replay()
    layer.load_state_dict(other.state_dict(), assign=True)
    now = layer(x, off)
    torch.cuda.synchronize()
    assert torch.equal(queued if how == "call" else replayed, old) and torch.equal(now, new)
    graph.replay()
    assert torch.equal(replayed, new)
