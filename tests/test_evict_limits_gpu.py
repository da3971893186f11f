"""Decode attention with accumulated weights and moves of rows at the ends of their ranges on the GPU."""

import math

import paged_oracle as O
import pytest
import torch
from test_evict_gpu import W_STEP, batch, check, i32, status

from infera_b200.ops import evict
from infera_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


@pytest.mark.parametrize("hq", [1, 4, 8])
def test_values_near_the_largest(hq):
    """Sums of weighted values stay in range, however far the maximum lags and in however many shares a sequence is cut."""
    lens = [1500, 40]
    q, k, v, table, mass = batch(lens, hq, 1, 3)
    for s, n in enumerate(lens):
        for p in range(n):  # scores that grow by some 6 in log2 from tile to tile, under the lag
            at = int(table[s, p // 16]) * 16 + p % 16
            k[at, 0] = p / 128
            v[at, 20] = 3.3e38
            v[at, 21] = -3.3e38 if p % 3 else 3.3e38
            v[at, 22] = 3.3e38 if p % 50 == 7 else 1.0
    for h in range(hq):
        q[:, 128 * h] = 48
    for splits, tps in ((1, 0), (2, 0), (12, 1)):
        got = mass.cuda()
        out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, 1, SCALE, got, splits,
                                tiles_per_split=tps)
        check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, 1)
    assert status()["code"] == 0
