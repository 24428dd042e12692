"""The host checks of the chunk attention and of the page operators, before anything is enqueued (no GPU)."""

from __future__ import annotations

import pytest

FAKE = 1 << 20  # an address that is never dereferenced: the calls are refused on the host


def _err(name: str, *args) -> str:
    from uocr_moe import _lib

    with pytest.raises(_lib.UocrError) as info:
        _lib.call(name, *args)
    return str(info.value)


def _chunk(tokens=4, heads=10, head_dim=128, stride=1280, pages=3, layers=2, page_size=128, layer=0, requests=1, cols=2,
           attend_max=4, out=None, q=None, k=None, v=None, pool=None, table=None, ws=None, ws_bytes=0, scale=1.0):
    return _err("uocr_paged_chunk_attention", out, q, k, v, tokens, heads, head_dim, stride, pool, pages, layers, page_size,
                layer, table, requests, cols, table, table, attend_max, scale, ws, ws_bytes, None)


@pytest.mark.parametrize(("kwargs", "message"), [
    ({"head_dim": 64}, "head_dim must be 128, got 64"),
    ({"page_size": 64}, "page_size must be a positive multiple of 128"),
    ({"page_size": 192}, "page_size must be a positive multiple of 128"),
    ({"layer": 2}, "layer 2 is not in the pool's 2 layers"),
    ({"layer": -1}, "layer -1 is not in the pool's 2 layers"),
    ({"pages": 1 << 31}, "more than 2^31 pages"),
    ({"heads": 0}, "heads must be in [1, 65535]"),
    ({"tokens": -1}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"tokens": (1 << 25) // 10 + 1}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"tokens": (1 << 63) - 1}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"requests": 65536}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"cols": 0}, "bad lookup table width 0"),
    ({"cols": 1 << 24}, "bad lookup table width 16777216"),
    ({"attend_max": 257}, "attend_max 257 is not in [1, 256], the rows the lookup table addresses"),
    ({"attend_max": 0}, "attend_max 0 is not in [1, 256], the rows the lookup table addresses"),
    ({"scale": float("inf")}, "scale must be finite"),
    ({"scale": float("nan")}, "scale must be finite"),
    ({"stride": 1279}, "input rows 1279 floats apart overlap rows of 1280"),
    ({}, "a tensor is missing"),
])
def test_chunk_attention_refusals(kwargs, message) -> None:
    assert _chunk(**kwargs) == "paged_chunk_attention: " + message


def test_chunk_attention_refuses_unaligned_and_overlapping_tensors() -> None:
    far = {"q": FAKE, "k": 2 * FAKE, "v": 3 * FAKE, "pool": 5 * FAKE, "table": 6 * FAKE}
    aligned = "paged_chunk_attention: q, k_new, v_new, out and kv_blocks must be 16-byte aligned"
    assert _chunk(out=4 * FAKE + 4, **far) == aligned
    assert _chunk(out=4 * FAKE, stride=1282, **far) == aligned
    # the last byte of k_new's last row, and the first of v_new
    assert _chunk(out=2 * FAKE + 4 * 1280 * 4 - 16, **far) == "paged_chunk_attention: out must not overlap the inputs"
    assert _chunk(out=3 * FAKE - 4 * 1280 * 4 + 16, **far) == "paged_chunk_attention: out must not overlap the inputs"
    assert _chunk(out=4 * FAKE, stride=1 << 25, **far) == \
        "paged_chunk_attention: input rows must be less than 2^25 floats apart"
    assert _chunk(out=4 * FAKE, ws=8, **far) == "paged_chunk_attention: workspace must be 16-byte aligned"


def test_chunk_attention_qkv_refusals() -> None:
    def call(stride=3840, table_rows=16, table_dim=128, heads=10, qkv=None, rest=None, out=None, cos=None, sin=None):
        return _err("uocr_paged_chunk_attention_qkv", out, qkv, 4, heads, 128, stride, rest, cos or rest, sin or rest,
                    table_rows, table_dim, rest, 3, 2, 128, 0, rest, 1, 2, rest, rest, 4, 1.0, None, 0, None)

    op = "paged_chunk_attention_qkv: "
    assert call(table_dim=64) == op + "the cos/sin tables are 64 wide, not head_dim 128"
    assert call(table_rows=0) == op + "bad cos/sin table"
    assert call(heads=0) == op + "heads must be in [1, 65535]"
    assert call(stride=3839) == op + "qkv rows 3839 floats apart overlap rows of 3840"
    assert call() == op + "a tensor is missing"
    for tables in ({"cos": 4 * FAKE + 4}, {"sin": 4 * FAKE + 8}):
        assert call(qkv=FAKE, rest=2 * FAKE, out=3 * FAKE, **tables) == \
            op + "the cos/sin tables must be 16-byte aligned"
    # out within qkv's rows
    assert call(qkv=FAKE, rest=2 * FAKE, out=FAKE + 3 * 3840 * 4) == op + "out must not overlap the inputs"


def _copy(pages=3, layers=2, page_size=128, heads=10, head_dim=128, pool=None, count=1):
    return _err("uocr_copy_pages", pool, pages, layers, page_size, heads, head_dim, None, None, None, count, None)


@pytest.mark.parametrize(("kwargs", "message"), [
    ({"pages": 0}, "bad pool [0, 2, 2, 128, 10, 128]"),
    ({"layers": 0}, "bad pool [3, 2, 0, 128, 10, 128]"),
    ({"page_size": 0}, "bad pool [3, 2, 2, 0, 10, 128]"),
    ({"heads": 1 << 30}, "bad pool [3, 2, 2, 128, 1073741824, 128]"),
    ({"pages": 1 << 30, "page_size": 1 << 30}, "bad pool [1073741824, 2, 2, 1073741824, 10, 128]"),
    ({"heads": 1, "head_dim": 6}, "heads * head_dim must be a multiple of 4"),
    ({"pool": FAKE + 4}, "kv_blocks must be 16-byte aligned"),
    ({"count": -1}, "bad number of pairs -1"),
    ({}, "a tensor is missing"),
])
def test_copy_pages_refusals(kwargs, message) -> None:
    assert _copy(**kwargs) == "copy_pages: " + message


def test_table_operators_refuse_bad_tables() -> None:
    def resize(counts_out=FAKE, counts=FAKE, lookup_out=2 * FAKE, lookup=2 * FAKE, pages=9, page_size=128, requests=3,
               cols=4, lengths=3 * FAKE, missing=4 * FAKE, ws=None, ws_bytes=0):
        return _err("uocr_resize_pages", counts_out, counts, pages, page_size, lookup_out, lookup, requests, cols,
                    lengths, missing, ws, ws_bytes, None)

    op = "resize_pages: "
    assert resize(pages=0) == op + "bad pool of 0 pages of 128 rows"
    assert resize(page_size=0) == op + "bad pool of 9 pages of 0 rows"
    assert resize(cols=0) == op + "bad lookup table [3, 0]"
    assert resize(requests=1 << 30) == op + "bad lookup table [1073741824, 4]"
    assert resize(counts=None) == op + "a tensor is missing"
    assert resize(lengths=None) == op + "a tensor is missing"
    overlapping = op + "an output must be its input or not overlap an input"
    assert resize(counts_out=FAKE + 4) == overlapping
    assert resize(lookup_out=2 * FAKE + 44) == overlapping
    assert resize(lookup_out=FAKE + 32) == overlapping
    assert resize(ws=8) == op + "workspace must be 16-byte aligned"
    assert resize(pages=20000, lookup_out=4 * FAKE, lookup=4 * FAKE, ws=16, ws_bytes=79999) == \
        op + "workspace of 79999 bytes is smaller than the 80000 needed"

    def fork(pool=5 * FAKE, count=2, lists=3 * FAKE, missing=4 * FAKE, ws=16, ws_bytes=0):
        return _err("uocr_fork_pages", pool, 9, 2, 128, 10, 128, FAKE, FAKE, 2 * FAKE, 2 * FAKE, 3, 4, lists, lists, lists,
                    lists, count, missing, ws, ws_bytes, None)

    assert fork(pool=None) == "fork_pages: a tensor is missing"
    assert fork(lists=None) == "fork_pages: a tensor is missing"
    assert fork(count=1 << 30) == "fork_pages: bad number of pairs 1073741824"
    assert "fork_pages: workspace of 0 bytes is smaller than" in fork()
    lib = __import__("uocr_moe")._lib.load()
    assert lib.uocr_fork_pages_workspace_bytes(9, 3, 4, 2, 0) == 0  # one launch, which keeps its state in LDS
    assert lib.uocr_fork_pages_workspace_bytes(9, 3, 4, 2, 1) > 0
    assert lib.uocr_fork_pages_workspace_bytes(2049, 3, 4, 2, 0) > 0
    assert lib.uocr_compact_pages_workspace_bytes(2048, 0) == 0
    assert min(lib.uocr_compact_pages_workspace_bytes(2048, 1), lib.uocr_compact_pages_workspace_bytes(2049, 0)) > 0
    apart = "an output must not overlap a list"
    for lists in (FAKE + 32, 2 * FAKE + 44, 4 * FAKE - 4):
        assert fork(lists=lists) == "fork_pages: " + apart
    for lengths in (FAKE + 32, 2 * FAKE + 44, 4 * FAKE - 8):
        assert resize(lengths=lengths) == op + apart
    for remap in (FAKE - 32, 2 * FAKE + 44):
        assert _err("uocr_compact_pages", 5 * FAKE, 9, 2, 128, 10, 128, FAKE, FAKE, 2 * FAKE, 2 * FAKE, 3, 4, remap, None,
                    0, None) == "compact_pages: remap must not overlap the tables"
    assert _err("uocr_compact_pages", 5 * FAKE, 9, 2, 128, 10, 128, FAKE, FAKE, 2 * FAKE, 2 * FAKE, 3, 4, None, None, 0,
                None) == "compact_pages: a tensor is missing"


def test_workspace_sizes_of_bad_shapes_are_zero() -> None:
    from uocr_moe import _lib

    lib = _lib.load()
    assert lib.uocr_paged_chunk_workspace_bytes(-1, 1, 10, 5) == 0
    assert lib.uocr_paged_chunk_workspace_bytes(4, 1, 10, 0) == 0
    assert lib.uocr_fork_pages_workspace_bytes(9, 3, 0, 2, 1) == 0
    assert lib.uocr_resize_pages_workspace_bytes(0) == 0
    assert lib.uocr_resize_pages_workspace_bytes(9) == 0  # in LDS
    assert lib.uocr_resize_pages_workspace_bytes(20000) == 80000
    assert lib.uocr_compact_pages_workspace_bytes(-1, 1) == 0


def test_the_wrappers_refuse_cpu_tensors_and_other_types() -> None:
    import torch

    import uocr_moe

    pool = torch.zeros(3, 2, 1, 128, 1, 128)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="copy_pages: kv_blocks must be a contiguous f32"):
        uocr_moe.copy_pages(pool, ints, ints)
    with pytest.raises(ValueError, match="fork_pages: kv_blocks must be a contiguous f32"):
        uocr_moe.fork_pages(pool, ints, ints.view(1, 2), ints, ints, ints, ints)
    with pytest.raises(ValueError, match="resize_pages: ref_counts must be on the GPU"):
        uocr_moe.resize_pages(ints, ints.view(1, 2), ints, page_size=128)
    with pytest.raises(TypeError, match="resize_pages: ref_counts must be torch.int32"):
        uocr_moe.resize_pages(ints.long(), ints.view(1, 2), ints, page_size=128)
    with pytest.raises(ValueError, match="compact_pages: kv_blocks must be a contiguous f32"):
        uocr_moe.compact_pages(pool, ints, ints.view(1, 2))
    q = torch.zeros(1, 1, 128)
    kv = uocr_moe.PagedChunk(pool, ints.view(1, 2), ints[:1], ints, 1)
    with pytest.raises(ValueError, match="paged_chunk_attention: q must be an fp32"):
        uocr_moe.paged_chunk_attention(q, q, q, kv=kv, layer_idx=0, scale=1.0)
    with pytest.raises(ValueError, match="paged_chunk_attention_qkv: qkv must be an fp32"):
        uocr_moe.paged_chunk_attention_qkv(q.view(1, 128), ints, pool, pool, heads=1, kv=kv, layer_idx=0, scale=1.0)
