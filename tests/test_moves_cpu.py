"""Moves of rows within sequences' pages, on the CPU: which sequences of a batch move."""

import paged_oracle as O
import torch

from infera_b200.ops import kernels as K


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_a_row_named_twice_moves_by_the_first_alone_even_if_that_one_is_refused():
    table, pool = O.page_table([40, 40], 4)
    k, v = O.caches(pool, 1, 5)
    kc, vc = k.clone(), v.clone()
    K.kv_compact(kc, vc, table, i32([[5], [7], [9]]), i32([1, 1, 1]), start=i32([-1, 0, 0]), bt_rows=i32([0, 0, 1]))
    assert torch.equal(kc, O.moved(k, table[1], [9], 0, 128, 0)) and torch.equal(vc, O.moved(v, table[1], [9], 0, 128, 0))
