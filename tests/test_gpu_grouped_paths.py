"""Kernels and their variants that only certain sizes reach: pairs of CTAs over ragged groups, few rows in four bits over a cluster,
values at the border through the quantiser on the chip, calls in place and through odd widths behind one another."""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_grouped import ALL, DEV, check, dequant, expected, grouped_case, grouped_expected, linear_layer, offsets_of, rand

from mase_triton_b200.mxfp import gemm as G
from mase_triton_b200.mxfp import grouped as GR
from mase_triton_b200.mxfp.meta import MXFP8_E4M3_fn, MXFP8_E5M2_fn, OCP_MXFP4_E2M1, OCP_MXFP6_E2M3

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pair", [(MXFP8_E4M3_fn, OCP_MXFP6_E2M3, 160), (MXFP8_E5M2_fn, MXFP8_E4M3_fn, 1056), (OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, 512)],
                         ids=lambda p: f"{p[0].tag}-{p[1].tag}-{p[2]}")
@pytest.mark.parametrize("N", [6016, 5889])
@pytest.mark.parametrize("start", [0, 3])
def test_pairs_of_ctas_over_ragged_groups(lib, pair, N, start):
    """Units for several rounds of pairs (six groups of 653 rows on average, 24 pairs of feature tiles, the last of them half empty): group
    starts of any remainder, an empty group, groups of 1 and 8 rows, rows named by an index."""
    x_meta, w_meta, K = pair
    counts = [1203, 0, 1, 2000, 705, 8]
    rows = start + sum(counts) + 5
    layer, wq, b, x = grouped_case(counts, N, K, x_meta, w_meta, tokens=1000)
    g = torch.Generator(device=DEV).manual_seed(3)
    idx = torch.randint(0, 1000, (rows,), generator=g, device=DEV)
    m = rand(rows, N, seed=2)
    first = [start + sum(counts[:i]) for i in range(len(counts))]
    got = layer(x, offsets_of(counts, start=start), activation="silu", multiplier=m, row_index=idx)
    G.check_status(DEV)
    check(got, *grouped_expected(dequant(x, x_meta)[idx], wq, b, first, counts, "silu", m, None, torch.bfloat16, torch.zeros_like(m)))
    for _ in range(3):
        assert torch.equal(got, layer(x, offsets_of(counts, start=start), activation="silu", multiplier=m, row_index=idx))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [2048, 4096])
@pytest.mark.parametrize("M", [1, 7, 12, 16])
def test_few_rows_in_four_bits_over_a_cluster(lib, dtype, K, M):
    layer, wq, b = linear_layer(520, K, OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, dtype, bias=True)
    x, r = rand(M, K, dtype=dtype), rand(M, 520, dtype=dtype, seed=1)
    got = layer(x, activation="gelu", residual=r)
    G.check_status(DEV)
    check(got, *expected(dequant(x, OCP_MXFP4_E2M1), wq, b, "gelu", None, r, dtype))
    counts = [3, 0, M, 1]
    layer, wq, b, x = grouped_case(counts, 264, K, OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, dtype)
    got = layer(x, offsets_of(counts), activation="relu")
    first = [sum(counts[:i]) for i in range(4)]
    check(got, *grouped_expected(dequant(x, OCP_MXFP4_E2M1), wq, b, first, counts, "relu", None, None, dtype, torch.zeros_like(got)))


def border_rows(K, dtype, scale):
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(32, K, generator=g, device=DEV) * torch.exp2(torch.randint(-30, 4, (32, K), generator=g, device=DEV).float())
    x[0], x[1], x[2, ::2], x[3] = 0.0, -0.0, 0.0, 1.0
    x[4, :64] = torch.tensor([479.0, 480.0, 448.0, 465.0, 0.9, -3.0, 2.0**-20, -(2.0**-24)] * 8, device=DEV) * scale
    x[5, :32] = torch.tensor([57344.0, 65000.0, 61440.0, -1e-7] * 8, device=DEV) * scale
    x[6] = torch.nextafter(torch.full((K,), 2.0**9, device=DEV), torch.zeros((), device=DEV)) * scale
    x[7, 3], x[8, K - 1], x[9, 33] = float("inf"), float("nan"), -float("inf")
    if dtype == torch.float32:
        x[10], x[11, :8] = 1e-40, 2.0**-126
    return x.to(dtype)


def lost_by_halving(xq, wq):
    """What blocks that hold a code the tensor cores read as Inf / NaN may lose, per output.

    Such a block is stored as (scale + 1, elements / 2).  E4M3: the code is that of 480 times the block's scale 2^S; an element below
    2^-5 2^S has a subnormal half, on a grid of 2^-9 2^S, and is off by at most half of that, twice (the scale is doubled): 2^-9 2^S, which
    is 2^-9 / 480 of the block's largest.  Larger elements are halved exactly.  E5M2: 2^-16 2^S beside a largest of 2^16 2^S or more,
    far less.  An element that is off counts with the magnitude of its partner, in either operand."""
    def blocks(t):
        t = t.abs().unflatten(-1, (-1, 32))
        return t.amax(-1), t.sum(-1)

    (x_max, x_sum), (w_max, w_sum) = blocks(xq), blocks(wq)
    return 2.0**-9 / 480 * (x_max @ w_sum.t() + x_sum @ w_max.t())


@pytest.mark.parametrize("meta", ALL, ids=lambda m: m.tag)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [96, 256, 4096])
def test_borders_through_the_quantiser_on_the_chip(lib, meta, dtype, K):
    """Zeros, elements that round up to what the tensor cores read as Inf / NaN, subnormals, values just below a power of two, Inf and NaN:
    calls of at most 16 rows (one kernel) against the formula, and their NaN against those of rows that lie off 16 bytes (extract kernel
    and table)."""
    layer, wq, _ = linear_layer(136, K, meta, MXFP8_E4M3_fn if meta.element_exp_bits > 2 else meta, dtype)
    x = border_rows(K, dtype, 2.0**-6)
    aside = torch.empty(32 * K + 1, dtype=dtype, device=DEV)[1:].view(32, K)
    aside.copy_(x)
    bad = torch.zeros(32, dtype=torch.bool, device=DEV)
    bad[7:10] = True
    xq = torch.where(bad[:, None], torch.zeros((), dtype=torch.float64, device=DEV), dequant(x, meta))
    y, tol = expected(xq, wq, None, "relu", None, None, dtype)
    tol = tol + (1 + torch.finfo(dtype).eps) * lost_by_halving(xq, wq)
    off = layer(aside, activation="relu")
    assert torch.equal(off.isnan(), bad[:, None].expand_as(off))
    for rows in (slice(0, 16), slice(16, 32), slice(0, 11), slice(11, 22), slice(22, 32), slice(4, 5), slice(8, 9)):
        got = layer(x[rows], activation="relu")
        assert torch.equal(got.isnan(), off[rows].isnan())
        check(torch.where(bad[rows, None], torch.zeros_like(got), got), y[rows], tol[rows], str(rows))
        check(torch.where(bad[rows, None], torch.zeros_like(got), off[rows]), y[rows], tol[rows], "off 16 bytes, " + str(rows))
    G.check_status(DEV)


@pytest.mark.parametrize("rows", [12, 300])
@pytest.mark.parametrize("width", [256, 257])
def test_calls_behind_one_another_in_place(lib, rows, width):
    """Each call's residual is the last one's result and its own output, through rows that take wide accesses and through odd ones."""
    counts = [rows // 2, 0, rows - rows // 2]
    layer, _, _, x = grouped_case(counts, width, 128, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    off = offsets_of(counts)
    want, got = rand(rows, width, seed=9), rand(rows, width, seed=9)
    layer(x, off)
    for _ in range(30):
        want = layer(x, off, activation="silu", residual=want)
        torch.cuda.synchronize()
    for _ in range(30):
        assert layer(x, off, activation="silu", residual=got, out=got) is got
    assert torch.equal(got, want)
    held = got.clone()
    for _ in range(10):
        layer(x, off, activation="gelu", multiplier=got, out=got)
        held = layer(x, off, activation="gelu", multiplier=held)
        torch.cuda.synchronize()
    assert torch.equal(got, held)


def test_a_row_of_a_tall_tile_and_alone(lib):
    """The same row in a call of 2500 rows and in calls of at most 16: each within the bound of the formula, so no further apart than twice that."""
    layer, wq, b = linear_layer(8192, 640, MXFP8_E5M2_fn, MXFP8_E4M3_fn, bias=True)
    x, m = rand(2500, 640), rand(2500, 8192, seed=1)
    many = layer(x, activation="silu", multiplier=m)
    for rows in (slice(0, 16), slice(1247, 1252), slice(2499, 2500)):
        few = layer(x[rows].contiguous(), activation="silu", multiplier=m[rows].contiguous())
        y, tol = expected(dequant(x[rows], MXFP8_E5M2_fn), wq, b, "silu", m[rows], None, torch.bfloat16)
        check(few, y, tol)
        check(many[rows], few.double(), 2 * tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [3, 200])
def test_product_and_bias_alone(lib, dtype, M):
    layer, wq, b = linear_layer(136, 256, MXFP8_E4M3_fn, MXFP8_E4M3_fn, dtype, bias=True)
    x = rand(M, 256, dtype=dtype)
    y, tol = expected(dequant(x, MXFP8_E4M3_fn), wq, b, None, None, None, dtype)
    alone = GR.grouped_linear(x, layer.x_mxfp_meta, layer.row_weight(), None, b)
    check(alone, y, tol)
    check(layer(x), y, tol, "without an epilogue")
    assert math.isfinite(alone.double().abs().max().item())


@pytest.mark.parametrize("groups", [351, 352, 1024])
@pytest.mark.parametrize("K,few", [(1024, False), (1024, True), (160, False)])
def test_many_groups_beside_the_ring(lib, groups, K, few):
    """Group tables around the size where they and a cluster's exchange no longer fit twice beside the ring; ``few``: rows in two groups only,
    so that clusters share units."""
    counts = [(i * 5) % 3 for i in range(groups)] if not few else [0] * 7 + [3] + [0] * (groups - 9) + [16]
    layer, wq, b, x = grouped_case(counts, 136, K, MXFP8_E4M3_fn, MXFP8_E4M3_fn)
    first = [sum(counts[:i]) for i in range(groups)]
    got = layer(x, offsets_of(counts), activation="silu")
    G.check_status(DEV)
    check(got, *grouped_expected(dequant(x, MXFP8_E4M3_fn), wq, b, first, counts, "silu", None, None, torch.bfloat16, torch.zeros_like(got)))


@pytest.mark.parametrize("pair", [(MXFP8_E4M3_fn, OCP_MXFP6_E2M3, 1184), (MXFP8_E5M2_fn, MXFP8_E4M3_fn, 64), (OCP_MXFP4_E2M1, OCP_MXFP4_E2M1, 512)],
                         ids=lambda p: f"{p[0].tag}-{p[1].tag}-{p[2]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [264, 129])
def test_popular_groups_among_idle_ones(lib, pair, dtype, N):
    """Few rows a group on average (one kernel), but groups of several tiles of 16 rows, the last one whole, of one row or of 15."""
    x_meta, w_meta, K = pair
    counts = [0, 32, 0, 0, 17, 1, 0, 47] + [0] * 60 + [16, 33] + [0] * 7
    layer, wq, b, x = grouped_case(counts, N, K, x_meta, w_meta, dtype)
    r = rand(sum(counts), N, dtype=dtype, seed=6)
    got = layer(x, offsets_of(counts), activation="gelu", residual=r)
    G.check_status(DEV)
    first = [sum(counts[:i]) for i in range(len(counts))]
    check(got, *grouped_expected(dequant(x, x_meta), wq, b, first, counts, "gelu", None, r, dtype, torch.zeros_like(r)))


@pytest.mark.parametrize("meta", [MXFP8_E4M3_fn, OCP_MXFP4_E2M1], ids=lambda m: m.tag)
@pytest.mark.parametrize("N,K", [(512, 256), (9600, 256), (9600, 4096), (4096, 8192)])
def test_rows_around_the_choice_of_kernel(lib, meta, N, K):
    """Row counts on both sides of where the choice falls, by the sizes and the operands' bits."""
    layer, wq, b = linear_layer(N, K, meta, meta, bias=True)
    x, r = rand(18, K), rand(18, N, seed=1)
    y, tol = expected(dequant(x, meta), wq, b, "silu", None, r, torch.bfloat16)
    for M in (4, 5, 6, 8, 9, 12, 13, 16, 17):
        check(layer(x[:M], activation="silu", residual=r[:M]), y[:M], tol[:M], str(M))
    G.check_status(DEV)
