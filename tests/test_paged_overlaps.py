"""Outputs of the chunk attention that overlap what other workgroups of the same call still
read: refused on the host before anything is enqueued (no GPU)."""

from __future__ import annotations

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
