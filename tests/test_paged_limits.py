"""Limits of the chunk attention's plan, checked on the host before anything is enqueued (no GPU)."""

from __future__ import annotations

from test_paged_refusals import _err

TB = 1 << 40  # addresses that are never dereferenced


def test_calls_of_more_pieces_than_a_wave_counts() -> None:
    """The pieces of up to 64 requests are counted in 32 bits whatever the offsets say, if need be all of them for each:
    64 times 78 tiles of 65535 heads in 64 splits pass that."""
    assert "invalid argument" in _err(
        "uocr_paged_chunk_attention", TB, 2 * TB, 3 * TB, 4 * TB, 512, 65535, 128, 65535 * 128, 16 * TB, 3, 2, 128, 0, 8 * TB,
        64, 1 << 16, 8 * TB, 8 * TB, 1 << 19, 1.0, 32 * TB, 8 * TB, None)
