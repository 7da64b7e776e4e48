"""Products with an epilogue and products grouped by expert, against the formula in 64 bits on the operands that the
extract / compose kernels give (those are compared with the oracle bit for bit elsewhere)."""

from __future__ import annotations

import math

import pytest
import torch

from mase_triton_b200.mxfp import functional as MX
from mase_triton_b200.mxfp import gemm as G
from mase_triton_b200.mxfp import kernels as mxk
from mase_triton_b200.mxfp.layers import MXFPGroupedLinearPTQ, MXFPLinearPTQ
from mase_triton_b200.mxfp.meta import MXFPMeta, MXFP8_E4M3_fn, MXFP8_E5M2_fn, OCP_MXFP4_E2M1, OCP_MXFP6_E2M3, OCP_MXFP6_E3M2

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
ALL = [MXFP8_E4M3_fn, MXFP8_E5M2_fn, OCP_MXFP6_E2M3, OCP_MXFP6_E3M2, OCP_MXFP4_E2M1]
ACTIVATIONS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def dequant(x, meta):
    s, e = mxk.extract_mxfp_components(x.contiguous().reshape(-1), meta)
    return mxk.compose_mxfp_tensor(s, e, meta, torch.float32).reshape(x.shape).double()


def act64(z, activation):
    if activation == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if activation == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    return z


def expected(xq, wq, bias, activation, multiplier, residual, dtype):
    """(y, tolerance) for dequantised operands in 64 bits.

    Sum: an instruction adds the products of 32 elements (64 for E2M1 pairs) to a 32-bit accumulator, one step of which is at
    most 2^-23 of the largest partial sum, itself at most s = |x| |w|^T; aligning the 32 products and adding lose at
    most two steps each: (K / 32) 2^-22 s.  The operand format loses half a step of elements 2^14 times smaller than
    their block's largest where that one is 480: 2^-18 s.  The activations' slopes are at most 1.13; their own arithmetic (a few roundings
    and an exponential of 2^-21 relative error for |z| < 20) is within 2^-18 of |z|.  A product or sum with the second
    operand adds 2^-24 relative; the rounding to the output's type half a step."""
    z = xq @ wq.t()
    s = xq.abs() @ wq.abs().t()
    if bias is not None:
        z = z + bias.double()
    y = act64(z, activation)
    tol = 1.13 * ((xq.shape[1] + 31) // 32 * 2.0**-22 + 2.0**-18) * s + 2.0**-18 * z.abs()
    if multiplier is not None:
        y, tol = y * multiplier.double(), tol * multiplier.double().abs()
    if residual is not None:
        y = y + residual.double()
    tol = tol + 2.0**-22 * y.abs()
    return y, tol + torch.finfo(dtype).eps / 2 * (y.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def check(got, want, tol, what=""):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - tol
    assert not got.isnan().any() and bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} of {off.numel()} outside, worst by {off.max().item():.3g}"


def rand(*shape, dtype=torch.bfloat16, by=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g, device=DEV) * by).to(dtype)


def linear_layer(N, K, x_meta, w_meta, dtype=torch.bfloat16, bias=False, backend="fused"):
    w = rand(N, K, dtype=dtype, by=0.5 / math.sqrt(K), seed=7)
    b = rand(N, dtype=dtype, seed=8) if bias else None
    layer = MXFPLinearPTQ(w, b, x_meta, w_meta, None, "XqWqB", backend)
    return layer, dequant(w, w_meta), b


def offsets_of(counts, dtype=torch.int32, start=0):
    return torch.tensor([start + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=dtype, device=DEV)


# ------------------------------------------------------------------------------------------------
# linear with an epilogue
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 64, 65, 128, 129, 240, 241, 257, 500])
@pytest.mark.parametrize("N,K", [(1, 32), (130, 96), (257, 1184), (520, 128), (512, 4096)])
def test_linear_epilogue_sizes(lib, M, N, K):
    layer, wq, b = linear_layer(N, K, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=True)
    x, r = rand(M, K), rand(M, N, seed=1)
    check(layer(x, activation="silu", residual=r), *expected(dequant(x, MXFP8_E4M3_fn), wq, b, "silu", None, r, torch.bfloat16))
    G.check_status(DEV)


@pytest.mark.parametrize("x_meta", ALL, ids=lambda m: m.tag)
@pytest.mark.parametrize("w_meta", ALL, ids=lambda m: m.tag)
@pytest.mark.parametrize("M,K", [(9, 1184), (9, 768), (300, 512), (300, 160)])
def test_linear_epilogue_formats(lib, x_meta, w_meta, M, K):
    layer, wq, b = linear_layer(200, K, x_meta, w_meta, bias=True)
    x, m = rand(M, K, by=3.0), rand(M, 200, seed=1)
    check(layer(x, activation="gelu", multiplier=m), *expected(dequant(x, x_meta), wq, b, "gelu", m, None, torch.bfloat16))
    G.check_status(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("extra", [None, "multiplier", "residual"])
@pytest.mark.parametrize("M", [3, 200])
def test_linear_epilogue_kinds(lib, dtype, activation, extra, M):
    if activation is None and extra is None:
        return                                           # no epilogue: another kernel
    layer, wq, b = linear_layer(136, 256, MXFP8_E4M3_fn, OCP_MXFP6_E3M2, dtype, bias=True)
    x, e = rand(M, 256, dtype=dtype), rand(M, 136, dtype=dtype, seed=1)
    kw = {} if extra is None else {extra: e}
    check(layer(x, activation=activation, **kw), *expected(dequant(x, MXFP8_E4M3_fn), wq, b, activation, kw.get("multiplier"), kw.get("residual"), dtype))
    y3 = layer(x.reshape(1, M, 256), activation=activation, **{k: v.reshape(1, M, 136) for k, v in kw.items()})
    assert y3.shape == (1, M, 136) and torch.equal(y3[0], layer(x, activation=activation, **kw))


@pytest.mark.parametrize("mode", ["rn", "ru", "rd", "rz"])
def test_round_modes_of_the_activation(lib, mode):
    meta = MXFPMeta(32, 8, 4, 3, True, mode)
    layer, wq, _ = linear_layer(96, 128, meta, OCP_MXFP4_E2M1)
    x, r = rand(33, 128), rand(33, 96, seed=1)
    check(layer(x, residual=r), *expected(dequant(x, meta), wq, None, None, None, r, torch.bfloat16))


def test_functional_equals_layer_and_separate_is_close(lib):
    layer, wq, b = linear_layer(264, 512, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=True)
    x, m = rand(70, 512), rand(70, 264, seed=1)
    args = (x, layer.x_mxfp_meta, None, layer.w_scales, layer.w_elements, layer.w_tensor_meta, b, None, None, None, "XqWqB")
    fused = MX.mxfp_linear(*args, "fused", activation="gelu_tanh", multiplier=m)
    assert torch.equal(fused, layer(x, activation="gelu_tanh", multiplier=m))
    sep = MX.mxfp_linear(*args, "separate", activation="gelu_tanh", multiplier=m)
    y, tol = expected(dequant(x, MXFP8_E4M3_fn), wq, b, "gelu_tanh", m, None, torch.bfloat16)
    # bf16 operands are rounded once more than MXFP8 values need (exact), the linear's result once: half a step before the slope of 1.13
    check(sep, y, tol + 1.13 * 2.0**-8 * (dequant(x, MXFP8_E4M3_fn) @ wq.t() + b.double()).abs() * m.double().abs())


def test_layers_without_epilogue_keep_their_result(lib):
    layer, _, _ = linear_layer(264, 512, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=True)
    x = rand(70, 512)
    before = layer(x)
    layer(x, activation="relu")
    assert torch.equal(before, layer(x))


# ------------------------------------------------------------------------------------------------
# grouped
# ------------------------------------------------------------------------------------------------
def grouped_case(counts, N, K, x_meta, w_meta, dtype=torch.bfloat16, bias=True, tokens=None):
    E = len(counts)
    w = rand(E, N, K, dtype=dtype, by=0.5 / math.sqrt(K), seed=3)
    b = rand(E, N, dtype=dtype, seed=4) if bias else None
    layer = MXFPGroupedLinearPTQ.from_weight(w, b, x_meta, w_meta)
    x = rand(sum(counts) if tokens is None else tokens, K, dtype=dtype, seed=5)
    return layer, torch.stack([dequant(w[e], w_meta) for e in range(E)]), b, x


def grouped_expected(xq, wq, b, first, counts, activation, multiplier, residual, dtype, base):
    y, tol = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64, device=DEV)
    for e, n in enumerate(counts):
        rows = slice(first[e], first[e] + n)
        if n:
            y[rows], tol[rows] = expected(xq[rows], wq[e], None if b is None else b[e], activation, None if multiplier is None else multiplier[rows],
                                          None if residual is None else residual[rows], dtype)
    return y, tol


COUNTS = [
    [1],
    [0, 1, 0, 2, 0],
    [3, 0, 16, 17, 1, 0, 0, 33],
    [0, 15, 129, 240, 241, 0, 500, 1],
    [700, 5],
]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("N,K", [(8, 32), (130, 160), (257, 1184), (520, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_grouped_sizes(lib, counts, N, K, dtype):
    layer, wq, b, x = grouped_case(counts, N, K, MXFP8_E4M3_fn, OCP_MXFP6_E2M3, dtype)
    r = rand(sum(counts), N, dtype=dtype, seed=6)
    got = layer(x, offsets_of(counts), activation="gelu", residual=r)
    G.check_status(DEV)
    first = [sum(counts[:i]) for i in range(len(counts))]
    check(got, *grouped_expected(dequant(x, MXFP8_E4M3_fn), wq, b, first, counts, "gelu", None, r, dtype, torch.zeros_like(r)))


@pytest.mark.parametrize("counts", COUNTS[1:], ids=str)
@pytest.mark.parametrize("pair", [(OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, 256), (OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, 1280), (OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, 128),
                                  (MXFP8_E5M2_fn, MXFP8_E4M3_fn, 640), (OCP_MXFP6_E3M2, MXFP8_E5M2_fn, 96)], ids=lambda p: f"{p[0].tag}-{p[1].tag}-{p[2]}")
def test_grouped_formats(lib, counts, pair):
    x_meta, w_meta, K = pair
    layer, wq, b, x = grouped_case(counts, 300, K, x_meta, w_meta)
    m = rand(sum(counts), 300, seed=6)
    got = layer(x, offsets_of(counts, torch.int64), activation="silu", multiplier=m)
    G.check_status(DEV)
    first = [sum(counts[:i]) for i in range(len(counts))]
    check(got, *grouped_expected(dequant(x, x_meta), wq, b, first, counts, "silu", m, None, torch.bfloat16, torch.zeros_like(m)))


@pytest.mark.parametrize("pair", [(MXFP8_E4M3_fn, OCP_MXFP6_E2M3, 160), (MXFP8_E5M2_fn, MXFP8_E4M3_fn, 640), (OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, 1280)],
                         ids=lambda p: f"{p[0].tag}-{p[1].tag}-{p[2]}")
@pytest.mark.parametrize("N", [8192, 7873])
def test_many_tiles(lib, pair, N):
    """Sizes with several rounds of tiles on every SM: the widest tiles, and those of pairs of CTAs, whole and with the last of
    the features and rows missing; a row's result is that of the kernel for few rows within what their orders of summation differ."""
    x_meta, w_meta, K = pair
    layer, wq, b = linear_layer(N, K, x_meta, w_meta, bias=True)
    x, m = rand(2500, K), rand(2500, N, seed=1)
    y = layer(x, activation="silu", multiplier=m)
    check(y, *expected(dequant(x, x_meta), wq, b, "silu", m, None, torch.bfloat16))
    counts = [1200, 0, 1, 2000, 700, 16]
    grouped, wq, b, x = grouped_case(counts, N // 4, K, x_meta, w_meta)
    r = rand(sum(counts), N // 4, seed=2)
    first = [sum(counts[:i]) for i in range(len(counts))]
    check(grouped(x, offsets_of(counts), residual=r), *grouped_expected(dequant(x, x_meta), wq, b, first, counts, None, None, r, torch.bfloat16, torch.zeros_like(r)))
    G.check_status(DEV)


@pytest.mark.parametrize("M,N,K", [(300, 1024, 1024), (1000, 2048, 512), (2000, 640, 2080)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_middle_sizes(lib, M, N, K, dtype):
    layer, wq, b = linear_layer(N, K, MXFP8_E4M3_fn, MXFP8_E4M3_fn, dtype, bias=True)
    x, r = rand(M, K, dtype=dtype), rand(M, N, dtype=dtype, seed=1)
    check(layer(x, activation="gelu_tanh", residual=r), *expected(dequant(x, MXFP8_E4M3_fn), wq, b, "gelu_tanh", None, r, dtype))


@pytest.mark.parametrize("start,pad", [(0, 37), (5, 0), (300, 131)])
def test_rows_outside_the_groups(lib, start, pad):
    counts = [20, 0, 150, 3]
    layer, wq, b, _ = grouped_case(counts, 96, 128, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    rows = start + sum(counts) + pad
    x = rand(rows, 128, seed=11)
    x[:start] = float("nan")
    x[rows - pad:] = float("inf")
    held = rand(rows, 96, seed=12)
    first = [start + sum(counts[:i]) for i in range(4)]
    xq = dequant(x, MXFP8_E4M3_fn)
    out = held.clone()
    got = layer(x, offsets_of(counts, start=start), out=out)
    assert got.data_ptr() == out.data_ptr()
    y, tol = grouped_expected(xq, wq, b, first, counts, None, None, None, torch.bfloat16, held)
    check(got, y, tol)
    assert torch.equal(got[:start], held[:start]) and torch.equal(got[rows - pad:], held[rows - pad:])
    fresh = layer(x, offsets_of(counts, start=start))
    assert torch.equal(fresh[start:rows - pad], got[start:rows - pad])
    assert not fresh[:start].any() and not fresh[rows - pad:].any()


def test_every_group_empty(lib):
    layer, _, _, x = grouped_case([4, 4], 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert not layer(x, off).any()
    held = rand(8, 64, seed=2)
    assert torch.equal(layer(x, off, out=held.clone()), held)
    assert layer(x[:0], off).shape == (0, 64)


def test_offsets_out_of_order_or_range_stay_inside(lib):
    """Offsets beyond the rows are clamped, one below an earlier one counts as that one."""
    layer, wq, b, x = grouped_case([10, 10, 10, 10], 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    for given, meant in (([-5, 12, 7, 90, 2**31 - 1], [0, 12, 12, 40, 40]), ([40, 3, 1, 0, 0], [40] * 5), ([0, 0, 50, 0, 60], [0, 0, 40, 40, 40])):
        want = torch.zeros(40, 64, dtype=torch.bfloat16, device=DEV)
        counts = [meant[i + 1] - meant[i] for i in range(4)]
        y, tol = grouped_expected(dequant(x, MXFP8_E4M3_fn), wq, b, meant, counts, None, None, None, torch.bfloat16, want)
        for dtype in (torch.int32, torch.int64):
            check(layer(x, torch.tensor(given, dtype=dtype, device=DEV)), y, tol, str(given))
    y64 = layer(x, torch.tensor([0, 10, 20, 30, 2**40], dtype=torch.int64, device=DEV))
    assert torch.equal(y64, layer(x, offsets_of([10, 10, 10, 10])))


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_row_index(lib, index_dtype):
    counts = [7, 0, 25, 180]
    layer, wq, b, x = grouped_case(counts, 72, 96, MXFP8_E4M3_fn, MXFP8_E4M3_fn, tokens=50)
    g = torch.Generator(device=DEV).manual_seed(1)
    idx = torch.randint(0, 50, (212,), generator=g, device=DEV).to(index_dtype)
    idx[3] = idx[4] = 11                                 # the same row twice in one group
    got = layer(x, offsets_of(counts), activation="silu", row_index=idx)
    assert torch.equal(got, layer(x[idx.long()].contiguous(), offsets_of(counts), activation="silu"))
    idx[0], idx[40], idx[211] = -1, 50, 2**31 - 1        # outside x: rows of zeros
    got = layer(x, offsets_of(counts), activation="silu", row_index=idx)
    rows = x[idx.long().clamp(0, 49)].clone()
    rows[[0, 40, 211]] = 0
    assert torch.equal(got, layer(rows, offsets_of(counts), activation="silu"))
    bias_only = act64(b[3].double(), "silu")
    check(got[211], bias_only, 2.0**-8 * bias_only.abs() + 2.0**-18)


def test_nonfinite_rows_and_operands_stay_where_they_are(lib):
    counts = [30, 40]
    layer, wq, b, x = grouped_case(counts, 64, 128, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    m = rand(70, 64, seed=1)
    want = layer(x, offsets_of(counts), multiplier=m)
    x2, m2 = x.clone(), m.clone()
    x2[29, 5], x2[30, 127] = float("nan"), float("inf")
    m2[31, 3], m2[0, 0] = float("inf"), float("nan")
    got = layer(x2, offsets_of(counts), multiplier=m2)
    assert got[29].isnan().all() and got[30].isnan().all() and got[31, 3].isinf() and got[0, 0].isnan()
    same = torch.ones(70, 64, dtype=torch.bool, device=DEV)
    same[29] = same[30] = False
    same[31, 3] = same[0, 0] = False
    assert torch.equal(got[same], want[same])
    neg = layer(x2, offsets_of(counts), activation="relu")
    assert neg[29].isnan().all()


def test_strides_alignment_and_output_in_place(lib):
    counts = [30, 2, 150]
    layer, wq, b, x = grouped_case(counts, 100, 96, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    r = rand(182, 100, seed=1)
    want = layer(x, offsets_of(counts), residual=r)
    wide = torch.zeros(182, 200, dtype=torch.bfloat16, device=DEV)
    wide[:, 7:103] = x
    assert torch.equal(layer(wide[:, 7:103], offsets_of(counts), residual=r), want)
    assert torch.equal(layer(x.t().contiguous().t(), offsets_of(counts), residual=r.t().contiguous().t()), want)
    off_by_one = torch.empty(182 * 96 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(182, 96)
    off_by_one.copy_(x)
    odd_out = torch.empty(182 * 100 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(182, 100)
    odd_r = torch.empty(182 * 100 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(182, 100)
    odd_r.copy_(r)
    assert torch.equal(layer(off_by_one, offsets_of(counts), residual=odd_r, out=odd_out), want)
    acc = r.clone()
    assert torch.equal(layer(x, offsets_of(counts), residual=acc, out=acc), want)


@pytest.mark.parametrize("meta", ALL, ids=lambda m: m.tag)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [96, 256, 4160])
def test_one_pass_quantiser_equals_extract_and_pack(lib, meta, dtype, K):
    """Rows that lie on 16 bytes are quantised in one pass, others by the extract kernel (bit-exact to the oracle) and a
    table: the same operand, so the same bits, whatever the values."""
    layer, _, _ = linear_layer(128, K, meta, MXFP8_E4M3_fn if meta.element_exp_bits > 2 else meta, dtype)
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(40, K, generator=g, device=DEV) * torch.exp2(torch.randint(-30, 12, (40, K), generator=g, device=DEV).float())
    x[0], x[1], x[2, ::2], x[3] = 0.0, -0.0, 0.0, 1.0
    x[4, :64] = torch.tensor([479.0, 480.0, 448.0, 465.0, 0.9, -3.0, 2.0**-20, -(2.0**-24)] * 8, device=DEV)
    x[5, :32] = torch.tensor([57344.0, 65000.0, 61440.0, -1e-7] * 8, device=DEV)
    x[6] = torch.nextafter(torch.full((K,), 2.0**9, device=DEV), torch.zeros((), device=DEV))
    if dtype == torch.float32:
        x[7], x[8, :8] = 1e-40, 2.0**-126
        x[9, 3], x[10, 40] = float("inf"), float("nan")
    x = x.to(dtype)
    aside = torch.empty(40 * K + 1, dtype=dtype, device=DEV)[1:].view(40, K)
    aside.copy_(x)
    a, b = layer(x, activation="relu"), layer(aside, activation="relu")
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    idx = torch.randint(-1, 41, (90,), generator=g, device=DEV)
    one = MX.grouped._grouped.grouped_linear(x, meta, layer.row_weight(), None, row_index=idx)
    two = MX.grouped._grouped.grouped_linear(aside, meta, layer.row_weight(), None, row_index=idx)
    assert torch.equal(one.isnan(), two.isnan()) and torch.equal(one.nan_to_num(), two.nan_to_num())


def test_inference_mode_and_copies(lib):
    import copy

    with torch.inference_mode():
        layer, _, _, x = grouped_case([5, 6], 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
        first = layer(x, offsets_of([5, 6]))
        assert torch.equal(layer(x, offsets_of([5, 6]), out=torch.zeros_like(first)), first)
    layer.w_elements.zero_()
    twin = copy.deepcopy(layer)
    for one in (layer, twin):
        assert torch.equal(one(x, offsets_of([5, 6]))[:5], one.bias[0].expand(5, 64))
    a = torch.ones(11, 64, dtype=torch.bfloat16, device=DEV)
    before = a._version
    layer(torch.zeros(11, 64, dtype=torch.bfloat16, device=DEV), offsets_of([5, 6]), out=a)
    assert a._version > before


def test_buffers_around_the_output_are_untouched(lib):
    counts = [17, 0, 130]
    layer, _, _, x = grouped_case(counts, 33, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    big = torch.full((147 * 33 + 4096,), 77.0, dtype=torch.bfloat16, device=DEV)
    out = big[2048:2048 + 147 * 33].view(147, 33)
    layer(x, offsets_of(counts), out=out)
    assert bool((big[:2048] == 77).all()) and bool((big[2048 + 147 * 33:] == 77).all())


def test_repeated_calls_give_the_same_bits(lib):
    counts = [300, 1, 77, 0, 900]
    layer, _, _, x = grouped_case(counts, 520, 1184, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    a = layer(x, offsets_of(counts), activation="gelu")
    for _ in range(5):
        assert torch.equal(a, layer(x, offsets_of(counts), activation="gelu"))
    lin, _, _ = linear_layer(512, 4096, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    y = rand(3, 4096)
    a = lin(y, activation="silu")
    for _ in range(5):
        assert torch.equal(a, lin(y, activation="silu"))
    # a row's result does not depend on the rows beside it in the same tile
    assert torch.equal(lin(y[:1], activation="silu"), a[:1])


def test_streams_and_graphs(lib):
    counts = [20, 0, 60, 140]
    layer, _, _, x = grouped_case(counts, 200, 256, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    other = [100, 100, 0, 20]
    x2 = rand(220, 256, seed=21)
    want, want2 = layer(x, offsets_of(counts), activation="silu"), layer(x2, offsets_of(other), activation="silu")
    lin, _, _ = linear_layer(640, 512, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    z = rand(2, 512, seed=9)
    want_lin = lin(z, activation="relu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layer(x, offsets_of(counts), activation="silu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    # two graphs, replayed side by side on two streams, each with inputs of its own
    state = []
    for seed in range(2):
        xin, off, zin = torch.zeros_like(x), torch.zeros(5, dtype=torch.int32, device=DEV), torch.zeros_like(z)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = layer(xin, off, activation="silu")
            c = lin(zin, activation="relu")
        state.append((graph, xin, off, zin, a, c))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for k in range(2):
            pick = (turn + k) % 2
            graph, xin, off, zin, a, c = state[k]
            streams[k].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[k]):
                xin.copy_((x, x2)[pick])
                off.copy_(offsets_of((counts, other)[pick]))
                zin.copy_(z)
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(state[k][4], (want, want2)[(turn + k) % 2])
            assert torch.equal(state[k][5], want_lin)
    G.check_status(DEV)


def test_many_groups(lib):
    E = 1024
    counts = [(i * 7) % 3 for i in range(E)]
    layer, wq, b, x = grouped_case(counts, 40, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    first = [sum(counts[:i]) for i in range(E)]
    got = layer(x, offsets_of(counts))
    check(got, *grouped_expected(dequant(x, MXFP8_E4M3_fn), wq, b, first, counts, None, None, None, torch.bfloat16, torch.zeros_like(got)))


# ------------------------------------------------------------------------------------------------
# together, as a model uses them
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 9, 300])
def test_gated_experts_in_a_row(lib, tokens):
    """Routed tokens through up, gate and down projections of their experts, then a dense gated layer and its residual;
    each step against the formula on the step's own inputs."""
    E, top, K, H = 6, 2, 256, 384
    meta = MXFP8_E4M3_fn
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = rand(tokens, K, seed=31)
    expert = torch.rand(tokens, E, generator=g, device=DEV).topk(top, dim=1).indices.reshape(-1)
    order = torch.argsort(expert, stable=True)
    row_index = (order // top).to(torch.int32)
    counts = torch.bincount(expert, minlength=E)
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    first, counts = off.tolist(), counts.tolist()
    weights = [rand(E, *s, by=0.06, seed=40 + i) for i, s in enumerate(((H, K), (H, K), (K, H)))]
    up, gate, down = (MXFPGroupedLinearPTQ.from_weight(w, None, meta, meta) for w in weights)
    wq = [torch.stack([dequant(w[e], meta) for e in range(E)]) for w in weights]
    base = torch.zeros(tokens * top, H, dtype=torch.bfloat16, device=DEV)
    xq = dequant(x, meta)[row_index.long()]
    u = up(x, off, row_index=row_index)
    check(u, *grouped_expected(xq, wq[0], None, first, counts, None, None, None, torch.bfloat16, base))
    h = gate(x, off, activation="silu", multiplier=u, row_index=row_index)
    check(h, *grouped_expected(xq, wq[1], None, first, counts, "silu", u, None, torch.bfloat16, base))
    d = down(h, off)
    check(d, *grouped_expected(dequant(h, meta), wq[2], None, first, counts, None, None, None, torch.bfloat16, torch.zeros_like(d)))
    y = torch.zeros_like(x).index_add_(0, row_index.long(), d)
    lin, lq, b = linear_layer(K, K, meta, OCP_MXFP6_E3M2, bias=True)
    z = lin(y, residual=x)
    check(z, *expected(dequant(y, meta), lq, b, None, None, x, torch.bfloat16))
    G.check_status(DEV)


def test_layer_follows_its_codes(lib):
    counts = [5, 6]
    layer, _, _, x = grouped_case(counts, 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=False)
    twin, _, _, _ = grouped_case(counts, 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=False)
    first = layer(x, offsets_of(counts))
    with torch.no_grad():
        layer.w_elements.zero_()
    assert not layer(x, offsets_of(counts)).any()
    layer.load_state_dict(twin.state_dict())
    assert torch.equal(layer(x, offsets_of(counts)), first)
    assert set(layer.state_dict()) == {"w_scales", "w_elements"}
    moved = layer.to("cpu").to(DEV)
    assert torch.equal(moved(x, offsets_of(counts)), first)
    fun = MX.mxfp_grouped_linear(x, MXFP8_E4M3_fn, layer.w_scales, layer.w_elements, layer.w_tensor_meta, offsets_of(counts))
    assert torch.equal(fun, first)
    linears = [torch.nn.Linear(64, 32, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    stacked = MXFPGroupedLinearPTQ.from_linears(linears, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    one = MXFPLinearPTQ.from_linear(linears[1], MXFP8_E4M3_fn, MXFP8_E4M3_fn, None, "XqWqB", "fused")
    r = rand(11, 32, seed=2)
    assert torch.equal(stacked(x, offsets_of(counts), residual=r)[5:], one(x[5:], residual=r[5:]))


def test_replaced_code_tensors(lib):
    """A new Parameter counts its versions anew: what the layer has packed is told apart by more than those."""
    counts = [5, 6]
    off = offsets_of(counts)
    layer, _, _, x = grouped_case(counts, 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=False)
    other = MXFPGroupedLinearPTQ.from_weight(rand(2, 64, 64, seed=31), None, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    want = other(x, off)
    assert not torch.equal(layer(x, off), want)
    layer.load_state_dict(other.state_dict(), assign=True)
    assert torch.equal(layer(x, off), want)
    layer.w_elements = torch.nn.Parameter(torch.zeros_like(other.w_elements), requires_grad=False)
    assert not layer(x, off).any()
    layer.w_elements.data = other.w_elements.data.clone()
    assert torch.equal(layer(x, off), want)


def test_code_tensors_made_in_inference_mode(lib):
    """Such tensors count no versions; what a layer computes follows them all the same."""
    off = offsets_of([5, 6])
    layer, _, _, x = grouped_case([5, 6], 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=False)
    with torch.inference_mode():
        want = layer(x, off)
        layer.load_state_dict({k: v.clone() for k, v in layer.state_dict().items()}, assign=True)
        assert torch.equal(layer(x, off), want)
        layer.w_elements.zero_()
        assert not layer(x, off).any()


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("mode", ["rn", "rz"])
def test_no_tokens_at_all(lib, rows, mode):
    """Every row index lies outside an empty x: rows of zeros, the bias is left."""
    meta = MXFPMeta(32, 8, 4, 3, True, mode)
    layer, _, b, _ = grouped_case([rows], 72, 96, meta, MXFP8_E4M3_fn)
    got = layer(torch.empty(0, 96, dtype=torch.bfloat16, device=DEV), offsets_of([rows]), activation="relu",
                row_index=torch.zeros(rows, dtype=torch.int32, device=DEV))
    assert torch.equal(got, torch.relu(b).expand(rows, 72))


def test_first_call_on_another_stream(lib):
    """What a layer packs in its first call is complete for every stream, whatever the first one is busy with."""
    layer, _, _, x = grouped_case([5, 200], 256, 512, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    off = offsets_of([5, 200])
    want = layer(x, off)
    layer._row_weight = None
    busy = torch.cuda.Stream()
    busy.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(busy):
        big = torch.ones(1 << 28, device=DEV)
        for _ in range(20):
            big.mul_(1.0)
        one = layer(x, off)
    two = layer(x, off)
    torch.cuda.synchronize()
    assert torch.equal(one, want) and torch.equal(two, want)


def test_first_call_inside_a_capture(lib):
    """A graph that packs the weight does so in every replay; the layer keeps nothing that only a replay fills."""
    counts = [5, 6]
    off = offsets_of(counts)
    layer, _, _, x = grouped_case(counts, 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=False)
    want = MX.mxfp_grouped_linear(x, MXFP8_E4M3_fn, layer.w_scales, layer.w_elements, layer.w_tensor_meta, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x, off)
    assert torch.equal(layer(x, off), want)
    graph.replay()
    assert torch.equal(got, want)
    with torch.no_grad():
        layer.w_elements.zero_()
    graph.replay()
    assert not got.any()


def test_a_captured_graph_finds_the_weights_packed_anew(lib):
    counts = [5, 6]
    off = offsets_of(counts)
    layer, _, _, x = grouped_case(counts, 64, 64, MXFP8_E4M3_fn, MXFP8_E4M3_fn, bias=False)
    other = MXFPGroupedLinearPTQ.from_weight(rand(2, 64, 64, seed=31), None, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    layer(x, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x, off)
    layer.load_state_dict(other.state_dict())
    want = layer(x, off)
    assert torch.equal(want, other(x, off))
    graph.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("M", [3, 200])
def test_calls_in_a_row_read_what_the_one_before_wrote(lib, M):
    """Kernels that may start before the one in front of them has ended: each call's input is the last one's output, in place and
    through an odd width (no wide accesses), many times over."""
    square, wq, _ = linear_layer(256, 256, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    x = rand(M, 256, seed=4)
    want, got = x.clone(), x.clone()
    for _ in range(30):
        want = square(want, residual=want)
        torch.cuda.synchronize()
        want = want / 4
    for _ in range(30):
        got = square(got, residual=got).div_(4)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    y = x.clone()
    square(y, activation="relu")
    with torch.cuda.graph(graph):
        z = y
        for _ in range(12):
            z = square(z, activation="silu", residual=z)
    graph.replay()
    v = x.clone()
    for _ in range(12):
        v = square(v, activation="silu", residual=v)
        torch.cuda.synchronize()
    assert torch.equal(z, v)


def test_long_axis_and_many_rows(lib):
    """More row tiles than CTAs, offsets of the output past 2^31 bytes, a long K."""
    layer, wq, b, x = grouped_case([9000, 0, 20000, 1], 40, 2048, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    got = layer(x, offsets_of([9000, 0, 20000, 1]), activation="relu")
    check(got, *grouped_expected(dequant(x, MXFP8_E4M3_fn), wq, b, [0, 9000, 9000, 29000], [9000, 0, 20000, 1], "relu", None, None, torch.bfloat16, torch.zeros_like(got)))
    lin, lq, _ = linear_layer(32, 32768, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    y, r = rand(5, 32768, seed=3), rand(5, 32, seed=4)
    check(lin(y, residual=r), *expected(dequant(y, MXFP8_E4M3_fn), lq, None, None, None, r, torch.bfloat16))
    # 70000 x 32768 16-bit results: 4.6 GB
    lin, lq, _ = linear_layer(32768, 32, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    y = rand(70000, 32, seed=3)
    got = lin(y, activation="relu")
    for rows in (slice(0, 3), slice(32767, 32770), slice(69990, 70000)):
        check(got[rows], *expected(dequant(y[rows], MXFP8_E4M3_fn), lq, None, "relu", None, None, torch.bfloat16))
    G.check_status(DEV)
