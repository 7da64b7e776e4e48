"""What the grouped products and the epilogues refuse, and the parts of them that need no GPU."""

from __future__ import annotations

import math

import pytest
import torch

from mase_triton_b200 import _lib
from mase_triton_b200._linear_common import activate
from mase_triton_b200.mxfp import functional as MX
from mase_triton_b200.mxfp import grouped as GR
from mase_triton_b200.mxfp.functional.linear import _separate_epilogue
from mase_triton_b200.mxfp.layers import MXFPGroupedLinearPTQ, MXFPLinearPTQ
from mase_triton_b200.mxfp.meta import MXFPMeta, MXFPTensorMeta, MXFP8_E4M3_fn, OCP_MXFP4_E2M1

E, N, K = 3, 8, 64


def codes(shape=(E, N, K)):
    n = math.prod(shape)
    return torch.zeros(n // 32, 1, dtype=torch.uint8), torch.zeros(n // 32, 32, dtype=torch.uint8), MXFPTensorMeta("cpu", "bfloat16", shape, -1, MXFP8_E4M3_fn)


def test_activations_in_plain_torch():
    z = torch.linspace(-9, 9, 41)
    w = z.double()
    for name, want in (("relu", w.clamp(min=0)), ("gelu", 0.5 * w * (1 + torch.erf(w / math.sqrt(2)))), ("silu", w / (1 + torch.exp(-w))),
                       ("gelu_tanh", 0.5 * w * (1 + torch.tanh(math.sqrt(2 / math.pi) * (w + 0.044715 * w**3)))), (None, w)):
        # a few fp32 roundings of values up to |z|, each 2^-24
        assert bool(((activate(z, name).double() - want).abs() <= 8 * 2.0**-24 * (1 + w.abs())).all()), name
    with pytest.raises(ValueError):
        activate(z, "swish")


def test_separate_epilogue():
    y = torch.tensor([[-1.0, 2.0]], dtype=torch.bfloat16)
    m = torch.tensor([[3.0, 0.5]], dtype=torch.bfloat16)
    assert torch.equal(_separate_epilogue(y, "relu", m, None), torch.tensor([[0.0, 1.0]], dtype=torch.bfloat16))
    assert torch.equal(_separate_epilogue(y, None, None, m), torch.tensor([[2.0, 2.5]], dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="not both"):
        _separate_epilogue(y, None, m, m)
    with pytest.raises(ValueError, match="residual"):
        _separate_epilogue(y, None, None, m[0])
    with pytest.raises(ValueError, match="multiplier"):
        _separate_epilogue(y, None, m.float(), None)


def test_linear_refusals():
    x, w = torch.randn(2, K), torch.randn(N, K)
    args = (x, None, w, None, None, None, None, None, None, None, "XWB")
    y = MX.mxfp_linear(*args, "separate", activation="silu", residual=torch.ones(2, N))
    assert torch.allclose(y, torch.nn.functional.silu(x @ w.t()) + 1, atol=1e-5)
    with pytest.raises(ValueError, match="activation"):
        MX.mxfp_linear(*args, "separate", activation="tanh")
    with pytest.raises(ValueError, match="not both"):
        MX.mxfp_linear(*args, "separate", multiplier=y, residual=y)
    for backend_args in (args, (x, MXFP8_E4M3_fn, *args[2:10], "XqWB")):
        with pytest.raises(NotImplementedError, match="separate"):
            MX.mxfp_linear(*backend_args, "fused", activation="relu")
    layer = MXFPLinearPTQ(w, None, None, None, None, "XWB", "separate")
    assert torch.equal(layer(x, activation="silu", residual=torch.ones(2, N)), y)


def test_layer_refusals():
    s, e, tm = codes()
    with pytest.raises(ValueError, match="groups, out_features, in_features"):
        MXFPGroupedLinearPTQ(*codes((N, K)), None, MXFP8_E4M3_fn)
    with pytest.raises(ValueError, match="block_dim"):
        MXFPGroupedLinearPTQ(s, e, tm.create(block_dim=1), None, MXFP8_E4M3_fn)
    with pytest.raises(ValueError, match="bias"):
        MXFPGroupedLinearPTQ(s, e, tm, torch.zeros(N), MXFP8_E4M3_fn)
    with pytest.raises(ValueError, match="32-element"):
        MXFPGroupedLinearPTQ(s, e, tm, None, MXFPMeta(16, 8, 4, 3, True, "rn"))
    with pytest.raises(ValueError, match="is_finite"):
        MXFPGroupedLinearPTQ(s, e, tm, None, MXFPMeta(32, 8, 4, 3, False, "rn"))
    with pytest.raises(ValueError, match="multiple of 32"):
        GR.check_formats(MXFP8_E4M3_fn, MXFP8_E4M3_fn, 48)
    with pytest.raises(ValueError, match="groups"):
        MXFPGroupedLinearPTQ.from_weight(torch.zeros(N, K), None, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    lin = [torch.nn.Linear(K, N), torch.nn.Linear(K, N, bias=False)]
    with pytest.raises(ValueError, match="bias"):
        MXFPGroupedLinearPTQ.from_linears(lin, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    layer = MXFPGroupedLinearPTQ(s, e, tm, None, MXFP8_E4M3_fn)
    assert "groups=3" in repr(layer) and set(layer.state_dict()) == {"w_scales", "w_elements"}
    with pytest.raises(_lib.MXQError, match="CUDA"):
        layer(torch.zeros(2, K), torch.zeros(E + 1, dtype=torch.int32))


class FakeCuda(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks of arguments run on it, nothing is launched."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(FakeCuda)


@pytest.mark.parametrize("change,match", [
    (dict(activation="tanh"), "activation"),
    (dict(x=fake(2, K, dtype=torch.float64)), "dtype"),
    (dict(x=fake(2, K + 32)), "expected"),
    (dict(x=fake(K)), "expected"),
    (dict(offsets=None), "offsets"),
    (dict(offsets=torch.zeros(E, dtype=torch.int32)), "offsets"),
    (dict(offsets=torch.zeros(E + 1)), "offsets"),
    (dict(offsets=torch.zeros(1, E + 1, dtype=torch.int32)), "offsets"),
    (dict(row_index=torch.zeros(2, 1, dtype=torch.int32)), "row_index"),
    (dict(row_index=torch.zeros(2, dtype=torch.int16)), "row_index"),
    (dict(bias=torch.zeros(N, dtype=torch.bfloat16)), "bias"),
    (dict(bias=torch.zeros(E, N)), "bias"),
    (dict(multiplier=torch.zeros(2, N)), "multiplier"),
    (dict(multiplier=torch.zeros(3, N, dtype=torch.bfloat16)), "multiplier"),
    (dict(residual=torch.zeros(2, N + 1, dtype=torch.bfloat16)), "residual"),
    (dict(residual=torch.zeros(2, N, dtype=torch.bfloat16), multiplier=torch.zeros(2, N, dtype=torch.bfloat16)), "not both"),
    (dict(out=torch.zeros(2, N)), "out"),
    (dict(out=torch.zeros(N, 2, dtype=torch.bfloat16).t()), "contiguous"),
    (dict(row_index=torch.zeros(5, dtype=torch.int32), out=torch.zeros(2, N, dtype=torch.bfloat16)), "out"),
    (dict(x_meta=MXFPMeta(16, 8, 4, 3, True, "rn")), "format"),
    (dict(w=GR.PackedExperts(torch.zeros(1), 5, E, N, K)), "format"),
])
def test_grouped_refusals(change, match):
    w = GR.PackedExperts(torch.zeros(1, dtype=torch.uint8), 0, E, N, K)
    call = dict(x=fake(2, K), x_meta=MXFP8_E4M3_fn, w=w, offsets=torch.zeros(E + 1, dtype=torch.int32)) | change
    with pytest.raises(ValueError, match=match):
        GR.grouped_linear(**call)


@pytest.mark.parametrize("name", ["x", "multiplier", "residual", "row_index", "bias", "offsets"])
def test_out_may_not_overlap_what_is_read(name):
    """``out`` shares its last row with an operand; only the residual or multiplier itself may be ``out``."""
    room = torch.zeros(4096, dtype=torch.bfloat16)
    out = room[:2 * N].view(2, N)
    at = room[N:]
    operand = {"x": lambda: at[:2 * K].view(2, K).as_subclass(FakeCuda), "row_index": lambda: at[:4].view(torch.int32),
               "offsets": lambda: at[:2 * (E + 1)].view(torch.int32), "bias": lambda: at[:E * N].view(E, N)}.get(name, lambda: at[:2 * N].view(2, N))()
    w = GR.PackedExperts(torch.zeros(1, dtype=torch.uint8), 0, E, N, K)
    call = dict(x=fake(2, K), x_meta=MXFP8_E4M3_fn, w=w, offsets=torch.zeros(E + 1, dtype=torch.int32), out=out) | {name: operand}
    with pytest.raises(ValueError, match="overlaps the .*" + ("input" if name == "x" else name)):
        GR.grouped_linear(**call)


def test_pack_refusals():
    s, e, _ = codes()
    e = e.as_subclass(FakeCuda)
    for bad in (dict(groups=2), dict(K=K * 2), dict(w_elements=e.to(torch.int8)), dict(w_scales=s.int()), dict(w_scales=s[:-1]),
                dict(groups=0, w_scales=s[:0], w_elements=e[:0]), dict(N=0, w_scales=s[:0], w_elements=e[:0])):
        with pytest.raises(ValueError):
            GR.pack_experts(**(dict(w_scales=s, w_elements=e, groups=E, N=N, K=K, w_meta=MXFP8_E4M3_fn, x_meta=MXFP8_E4M3_fn) | bad))
    with pytest.raises(_lib.MXQError, match="CUDA"):
        GR.pack_experts(s, torch.zeros(E * N * K, dtype=torch.uint8), E, N, K, MXFP8_E4M3_fn, OCP_MXFP4_E2M1)


def test_c_entry_refuses_before_it_launches():
    """Status codes of the C entry for arguments that no kernel may see (nothing here touches a GPU)."""
    L = _lib.load()
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    p = (buf.data_ptr() + 255) // 256 * 256
    good = dict(x=p, row_index=0, w=p, offsets=0, out=p, bias=0, extra=0, scratch=p, status=0, stream=0, rows_in=2, rows=2, K=64, groups=1, N=8, nbytes=1 << 16,
                x_dtype=1, eb=4, fb=3, rm=0, index64=0, offsets64=0, fmt=0, act=0, mode=0, zero=0)

    def entry(**change):
        return L.mxq_mx_grouped_linear(GR._ARGS.pack(*(good | change).values()))

    assert entry(rows=0, rows_in=0) == 0 and L.mxq_mx_grouped_linear(None) == -1
    for bad in (dict(K=48), dict(K=0), dict(N=0), dict(groups=0), dict(groups=2), dict(rows=3), dict(rows=-1), dict(x_dtype=3), dict(act=5), dict(act=-1), dict(mode=3),
                dict(mode=1), dict(x=0), dict(w=0), dict(w=p + 8), dict(out=0), dict(scratch=0, rm=1), dict(scratch=p + 16), dict(fmt=3), dict(fmt=5),
                dict(eb=3, fb=3)):
        assert entry(**bad) == -1, bad
    for bad in (dict(groups=L.mxq_mx_max_groups() + 1, offsets=p), dict(nbytes=64, rm=1), dict(rows=1 << 31, rows_in=1 << 31)):
        assert entry(**bad) == -3, bad
    assert L.mxq_mx_grouped_scratch_bytes(p, 0, 2, 2, 48, 1, 8) == -1 and L.mxq_mx_grouped_scratch_bytes(p, 0, 2, 2, 64, 1, 8) == 0
    assert L.mxq_mx_grouped_scratch_bytes(p + 2, 0, 2, 2, 64, 1, 8) > 0 and L.mxq_mx_grouped_scratch_bytes(p, 1, 2, 2, 64, 1, 8) > 0
    assert L.mxq_mx_grouped_scratch_bytes(p, 0, 500, 500, 64, 1, 8) > 0
