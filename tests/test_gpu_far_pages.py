"""GPU tests of the served operators on pages whose bytes lie past 32-bit offsets: the results and rows have the bits of the same
pages in a small pool.

Pools of 5 GiB (each operator's offsets are a page's, a layer's and a row's together), the pages in use the last ones.
"""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from _served import SCALE, Served, masks_of, signed

pytestmark = pytest.mark.gpu

BYTES = 5 << 30


def _uocr():
    import uocr_moe

    return uocr_moe


def _on(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _far(s: Served) -> tuple[torch.Tensor, int]:
    """A pool of 5 GiB whose last pages are s's, and the shift of their numbers."""
    page = s.pool[0].numel() * s.pool.element_size()
    pages = BYTES // page
    shift = pages - s.pool.shape[0]
    assert shift * page > 1 << 32
    pool = torch.zeros(pages, *s.pool.shape[1:], dtype=s.pool.dtype, device=DEV)
    pool[shift:] = s.pool.to(DEV)
    return pool, shift


def _same(far: torch.Tensor, shift: int, near: torch.Tensor) -> None:
    assert torch.equal(far[shift:].view(torch.uint8), near.view(torch.uint8))
    assert not bool(far[:4].any()) and not bool(far[shift - 4:shift].any())


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
def test_attention_and_acceptance(int8) -> None:
    u = _uocr()
    s = Served(1, [21, 9, 40], [700, 0, 130], int8=int8)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    parents = [j - 1 if j % 3 else max(j - 3, -1) for c in s.chunks for j in range(c)]
    bits = [signed(b) for i, c in enumerate(s.chunks)
            for b in masks_of(parents[int(s.offsets[i]):int(s.offsets[i]) + c])]
    g = torch.Generator().manual_seed(2)
    drafted = torch.randint(0, 2, (s.tokens,), generator=g, dtype=torch.int32).to(DEV)
    answers = torch.randint(0, 2, (s.tokens,), generator=g, dtype=torch.int32).to(DEV)
    results = []
    for far in (False, True):
        pool, shift = _far(s) if far else (s.pool.to(DEV), 0)
        table = (s.table + shift).to(DEV)
        kv = u.PagedChunk(kv_blocks=pool, lookup_table=table, cache_lengths=_on(s.cached), chunk_offsets=s.offsets.to(DEV),
                          attend_max=s.attend_max, visible=_on(bits, torch.int64))
        got = [u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE)]
        if int8:
            chunk = type(kv)(**{**vars(kv), "visible": None})
            got.append(u.paged_chunk_attention(q, k, v, kv=chunk, layer_idx=0, scale=SCALE))
            step = u.PagedKv(kv_blocks=pool, lookup_table=table, attend_lengths=_on([600, 3, 100]), attend_max=641,
                             write_index=_on([600, 3, 20]))
            got.append(u.paged_decode_attention(q[:3], k[:3], v[:3], kv=step, layer_idx=0, scale=SCALE))
        got += list(u.accept_drafts(kv, _on(parents), drafted, answers))
        results.append((got, pool, shift))
    (near, pool, _), (far, large, shift) = results
    for a, b in zip(near, far):
        assert torch.equal(a, b)
    _same(large, shift, pool)


def test_tiles() -> None:
    u = _uocr()
    s = Served(2, [600], [5000], heads=3)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    results = []
    for far in (False, True):
        pool, shift = _far(s) if far else (s.pool.to(DEV), 0)
        kv = u.PagedChunk(kv_blocks=pool, lookup_table=(s.table + shift).to(DEV), cache_lengths=_on(s.cached),
                          chunk_offsets=s.offsets.to(DEV), attend_max=s.attend_max)
        results.append((u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE), pool, shift))
    assert torch.equal(results[0][0], results[1][0])
    _same(results[1][1], results[1][2], results[0][1])


def test_conversions() -> None:
    u = _uocr()
    wide, narrow = Served(3, [1], [600], int8=False), Served(4, [1], [600])
    far_wide, w = _far(wide)
    far_narrow, m = _far(narrow)
    near_wide, near_narrow = wide.pool.to(DEV), narrow.pool.to(DEV)
    src, dst, rows = [0, 3, 1], [2, 0, 2], [128, 17, 50]
    u.quantize_pages(near_wide, _on(src), near_narrow, _on(dst), rows=_on(rows))
    u.quantize_pages(far_wide, _on([x + w for x in src]), far_narrow, _on([x + m for x in dst]), rows=_on(rows))
    _same(far_narrow, m, near_narrow)
    u.dequantize_pages(near_narrow, _on(src), near_wide, _on(dst), rows=_on(rows))
    u.dequantize_pages(far_narrow, _on([x + m for x in src]), far_wide, _on([x + w for x in dst]), rows=_on(rows))
    _same(far_wide, w, near_wide)


def test_slots_of_many_heads() -> None:
    """64 heads of a row (8448 bytes) and a last page's last rows."""
    u = _uocr()
    s = Served(5, [2, 1], [126, 255], heads=64, layers=1)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    results = []
    for far in (False, True):
        pool, shift = _far(s) if far else (s.pool.to(DEV), 0)
        kv = u.PagedChunk(kv_blocks=pool, lookup_table=(s.table + shift).to(DEV), cache_lengths=_on(s.cached),
                          chunk_offsets=s.offsets.to(DEV), attend_max=s.attend_max)
        results.append((u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE), pool, shift))
    assert torch.equal(results[0][0], results[1][0])
    _same(results[1][1], results[1][2], results[0][1])
    stored = s.stored(0, *s.qkv.unbind(1)[1:])
    assert torch.equal(results[0][1].cpu(), stored)
