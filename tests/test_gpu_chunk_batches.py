"""GPU tests of the chunk attention's plan for batches: more requests than a wave counts the pieces of, in several splits,
and one long chunk among short and empty ones."""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from test_gpu_chunk import BAR, SCALE, Setup, _far, _same_bits, _uocr

pytestmark = pytest.mark.gpu


def _check(s, splits) -> None:
    u = _uocr()
    assert (u._lib.load().uocr_paged_chunk_workspace_bytes(s.tokens, len(s.chunks), s.heads, s.attend_max) > 0) == splits
    q, k, v = s.qkv.unbind(1)
    pool = s.pool.to(DEV)
    out = torch.full((s.tokens, s.heads, 128), 3.0, device=DEV)
    u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(pool), layer_idx=1, scale=SCALE, out=out)
    assert _same_bits(pool.cpu(), s.stored(1, k, v))
    used = s.covered()
    assert _far(out[used].cpu(), s.want(1, q, k, v)[used]) <= BAR
    assert (out[used.stop:] == 3.0).all()


@pytest.mark.parametrize("requests", [65, 85])
@pytest.mark.parametrize("tail", [0, 9100])
def test_many_requests_of_unlike_lengths(requests, tail) -> None:
    """Tiles of 32 queries, or, with so many token rows, of 256; from one split of a tile to all of them, and empty
    chunks, whose pieces are left out."""
    chunks = [(3 * i) % 5 for i in range(requests)]
    cached = [0 if i % 7 == 0 else (311 * i) % 1201 for i in range(requests)]
    cached[40] = 1300
    _check(Setup(requests, chunks, cached, heads=1, tail=tail), True)


def test_many_chunks_of_several_tiles() -> None:
    """66 chunks of up to 300 tokens: tiles of 256 that begin anywhere in the token rows."""
    chunks = [70 + (37 * i) % 41 for i in range(66)]
    chunks[30], chunks[65] = 300, 257
    cached = [(97 * i) % 700 for i in range(66)]
    cached[30] = 1024
    _check(Setup(66, chunks, cached, heads=1), True)


@pytest.mark.parametrize(("chunks", "cached"), [
    ([1] * 15 + [600] + [1] * 16, [(53 * i) % 900 for i in range(32)]),
    ([0] * 7 + [4], [0] * 7 + [3000]),
    ([0, 0, 700, 0], [900, 0, 1100, 5]),
    ([1] * 50 + [520] + [1] * 20, [17] * 71),
])
def test_one_long_chunk_among_short_and_empty_ones(chunks, cached) -> None:
    _check(Setup(sum(chunks), chunks, cached, heads=2), True)
