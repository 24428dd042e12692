"""Outputs of the chunk attention and of the page operators that overlap what other workgroups of the same call still
read: refused on the host before anything is enqueued (no GPU)."""

from __future__ import annotations

import pytest

from test_paged_refusals import _err

MB = 1 << 20  # addresses that are never dereferenced
ROW = 2 * 128 * 4  # bytes of a row of two heads
POOL = 3 * 2 * 2 * 128 * ROW


def _chunk(**at):
    """Four tokens, two heads, a pool of three pages and two layers."""
    t = {"out": MB, "q": 2 * MB, "k": 3 * MB, "v": 4 * MB, "pool": 16 * MB, "meta": 32 * MB} | at
    return _err("uocr_paged_chunk_attention", t["out"], t["q"], t["k"], t["v"], 4, 2, 128, 256, t["pool"], 3, 2, 128, 0,
                t["meta"], 1, 2, t["meta"], t["meta"], 4, 1.0, 8, 0, None)


def test_chunk_attention_refuses_a_pool_that_holds_its_other_tensors() -> None:
    assert _chunk().endswith("workspace must be 16-byte aligned")  # all apart: the next check speaks
    for place in (16 * MB - 4 * ROW + 16, 16 * MB, 16 * MB + POOL - 16):
        assert _chunk(out=place) == "paged_chunk_attention: out must not overlap kv_blocks"
        for name in "qkv":
            assert _chunk(**{name: place}) == "paged_chunk_attention: the inputs must not overlap kv_blocks"
    for place in (16 * MB - 4 * ROW, 16 * MB + POOL):
        for name in ("out", "q", "k", "v"):
            assert _chunk(**{name: place}).endswith("workspace must be 16-byte aligned")


def test_chunk_attention_qkv_refuses_a_pool_that_holds_its_rows() -> None:
    def call(qkv, out):
        return _err("uocr_paged_chunk_attention_qkv", out, qkv, 4, 2, 128, 768, 32 * MB, 33 * MB, 33 * MB, 16, 128, 16 * MB,
                    3, 2, 128, 0, 32 * MB, 1, 2, 32 * MB, 32 * MB, 4, 1.0, 8, 0, None)

    op = "paged_chunk_attention_qkv: "
    assert call(2 * MB, MB) == op + "workspace must be 16-byte aligned"
    assert call(16 * MB - 16, MB) == op + "the inputs must not overlap kv_blocks"
    assert call(2 * MB, 16 * MB + 16) == op + "out must not overlap kv_blocks"


def test_a_pool_past_the_address_space_is_refused() -> None:
    assert _err("uocr_paged_chunk_attention", MB, 2 * MB, 3 * MB, 4 * MB, 4, 2, 128, 256, 16 * MB, (1 << 31) - 1,
                (1 << 31) - 1, 128, 0, 32 * MB, 1, 2, 32 * MB, 32 * MB, 4, 1.0, 8, 0, None) == \
        "paged_chunk_attention: the pool is too large"


# counts of nine pages at 1 and 2 MB, tables of three rows of four at 3 and 4 MB
INPUTS, OUTPUTS = [MB, MB + 32, 3 * MB, 3 * MB + 44], [2 * MB, 2 * MB + 32, 4 * MB, 4 * MB + 44]


@pytest.mark.parametrize(("in_place", "missing"),
                         [(True, x) for x in INPUTS] + [(False, x) for x in INPUTS + OUTPUTS])
def test_missing_apart_from_the_tables(in_place, missing) -> None:
    args = (MB, MB, 3 * MB, 3 * MB, 3, 4) if in_place else (2 * MB, MB, 4 * MB, 3 * MB, 3, 4)
    assert _err("uocr_fork_pages", 16 * MB, 9, 2, 128, 2, 128, *args, *[8 * MB] * 4, 2, missing, 6 * MB, MB, None) == \
        "fork_pages: missing must not overlap the tables"
    assert _err("uocr_resize_pages", args[0], MB, 9, 128, args[2], 3 * MB, 3, 4, 8 * MB, missing, None, 0, None) == \
        "resize_pages: missing must not overlap the tables"
