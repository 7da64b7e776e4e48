"""Kernels and their variants that only certain sizes reach: pairs of CTAs over ragged groups."""

from __future__ import annotations

import pytest
import torch
from test_gpu_grouped import DEV, check, dequant, grouped_case, grouped_expected, offsets_of, rand

from mase_triton_b200.mxfp import gemm as G
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
