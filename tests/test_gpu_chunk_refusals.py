"""GPU tests of what the chunk attention's wrapper refuses: by its text, and without memory taken first."""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from test_gpu_chunk import SCALE, Setup, _uocr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("attend_max", [2 ** 31 - 1, 2 ** 26, 513, 0, -1])
def test_an_attend_max_that_the_table_does_not_address(attend_max) -> None:
    """The workspace of 2^31 - 1 rows would be 1.1 GB here."""
    u = _uocr()
    s = Setup(1, [4], [300])
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    good = s.kv()
    assert good.lookup_table.shape[1] * s.page_size == 512
    kv = u.PagedChunk(good.kv_blocks, good.lookup_table, good.cache_lengths, good.chunk_offsets, attend_max)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(u.UocrError, match=f"attend_max {attend_max} is not in"):
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
