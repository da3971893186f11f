"""The 8-bit paged KV cache on CPU at the ends of its ranges, and the calls that
it refuses there."""

import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import kv8
from test_kv8_cpu import random_cache

D = 128


@pytest.mark.parametrize("e", [253, 254, 255])
def test_largest_scales(e):
    """Exponents end at 253, and 254 and 255 count as it: a row that joins such a page keeps its values."""
    hkv = 2
    kc, vc = [kv8.KV8Cache(random_cache(32, hkv, s).q, torch.full((2, hkv), e, dtype=torch.uint8)) for s in (1, 2)]
    old = vc.q.float()
    assert bool((vc.dequant()[16:] == (old * 2.0 ** 126)[16:]).all())  # (infinite above 2)
    qkv = torch.full((1, 8 * D), 2.0 ** 120, dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32)
    kv8.rope_kvwrite(qkv, zero, zero + 21, K.rope_cos_sin(2, D, 1e4), 4, hkv, D, kc, vc)
    for c in (kc, vc):
        assert bool((c.dequant()[21] == 2.0 ** 120).all()) and bool((c.sf[1] == 253).all())
    rest = [16 + o for o in range(16) if o != 5]
    assert torch.equal(vc.q.float()[rest], old[rest]) and torch.equal(vc.q.float()[:16], old[:16])
