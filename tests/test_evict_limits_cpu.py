"""Decode attention with accumulated weights at the ends of its range, on the CPU."""

import math

import paged_oracle as O
import pytest
import torch

from infera_b200.ops import evict

SCALE = 1 / math.sqrt(128)


@pytest.mark.parametrize("big", [0, 300])
def test_infinite_values_whatever_their_weight(big):
    table, pool = O.page_table([40], 1)
    k, v = O.caches(pool, 1)
    slot = lambda p: int(table[0, p // 16]) * 16 + p % 16  # noqa: E731
    q = torch.randn(1, 256, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    q[:, ::128] = 8
    k[slot(39), 0] = big  # 0: ordinary scores; 300: 300 above the others in log2
    for p, d, x in ((3, 5, float("inf")), (4, 6, float("-inf")), (5, 7, float("inf")), (6, 7, float("-inf")), (39, 8, float("inf"))):
        v[slot(p), d] = x
    mass = torch.zeros(1, 1, 48)
    out = evict.attn_decode(q, k, v, table, torch.tensor([40], dtype=torch.int32), 2, 1, SCALE, mass)
    kk, vv = (O.rows_of(x, table[0], 40, 1) for x in (k, v))
    want, bound, _, _ = O.attend(q, kk, vv, torch.ones(1, 40, dtype=torch.bool), 2, 1, SCALE, 0.0)
    O.close(out, want, bound)
