"""GPU tests of what the three bf16 terms of a float32 operand leave out, in the attention of trees and over an int8 pool.

The terms are cut off, not rounded: the second is up to 2^-7 of the operand, the third 2^-15.  A product of two such
operands keeps six of its nine parts and leaves out 2 * 2^-22 + 2^-30 of itself, 2^-21, towards zero, where the lower bits of
both operands are ones.  A score s then is off by 2^-21 |s|: 3e-6 for the largest here (|s| < 6), which a weight is off by too,
and an output by that times what the values differ by, at most 1.2 of a token's largest output (60 rows and more, 256 columns);
the values' products add 2^-21 of themselves, 5e-7, and the sums' roundings 1e-6: 6e-6 in all.  The bar is the other tests'.
"""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from _served import SCALE, Served, far, masks_of, signed

pytestmark = pytest.mark.gpu

BAR = 1e-5


def _attend(s: Served) -> torch.Tensor:
    """Chunks as chains of a tree, over either pool."""
    import uocr_moe as u

    on = lambda x, dtype=torch.int32: torch.tensor(x, dtype=dtype, device=DEV)  # noqa: E731
    visible = on([signed(b) for c in s.chunks for b in masks_of([j - 1 for j in range(c)])], torch.int64)
    kv = u.PagedChunk(kv_blocks=s.pool.to(DEV), lookup_table=s.table.to(DEV), cache_lengths=on(s.cached),
                      chunk_offsets=s.offsets.to(DEV), attend_max=s.attend_max, visible=visible)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    return u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE).cpu()


def _want(s: Served) -> torch.Tensor:
    q, k, v = s.qkv.unbind(1)
    return s.want(s.stored(1, k, v), 1, q)


@pytest.mark.parametrize("cached", [60, 300])
@pytest.mark.parametrize("seed", range(3))
def test_operands_whose_lower_bits_are_ones(seed, cached) -> None:
    s = Served(seed, [20], [cached], int8=False, heads=2)
    ones = lambda x: (x.contiguous().view(torch.int32) | 0xffff).view(torch.float32)  # noqa: E731
    s.pool, s.qkv = ones(s.pool), ones(s.qkv)
    assert far(_attend(s), _want(s)) <= BAR


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -60, 2.0 ** 100])
def test_values_of_any_usual_size(int8, size) -> None:
    """bf16 ends at 2^-133, which the third terms are off by at most: of an int8 row's weight times its scale, times 127 and 80
    rows, 2^-119.7 or 2.4e-6 of outputs near 2^-101; of a float32 row's values 2^-32 of them."""
    s = Served(7, [20], [60], int8=int8, heads=2)
    s.qkv[:, 2] *= size
    if int8:
        scales = s.pool[:, 1, ..., 256:264].contiguous().view(torch.float32)
        s.pool[:, 1, ..., 256:264] = (scales * size).view(torch.int8)
    else:
        s.pool[:, 1] *= size
    assert far(_attend(s), _want(s)) <= BAR
