"""The host checks of the int8 pool's operators, of trees' and of beams', before anything is enqueued (no GPU)."""

from __future__ import annotations

import pytest

FAKE = 1 << 24  # an address that is never dereferenced: the calls are refused on the host
SLOT = 1408     # ten heads


def _err(name: str, *args) -> str:
    from uocr_moe import _lib

    with pytest.raises(_lib.UocrError) as info:
        _lib.call(name, *args)
    return str(info.value)


def _nothing(name: str, *args) -> None:
    from uocr_moe import _lib

    _lib.call(name, *args)


DEFAULTS = dict(out=None, q=None, k=None, v=None, tokens=4, heads=10, head_dim=128, stride=1280, positions=None, cos=None,
                sin=None, table_rows=0, pool=None, pages=3, layers=2, page_size=128, slot=SLOT, layer=0, lookup=None, requests=1,
                cols=2, lengths=None, other=None, attend_max=4, visible=None, scale=1.0, ws=None, ws_bytes=0)
GIVEN = dict(out=2 * FAKE, q=3 * FAKE, k=4 * FAKE, v=5 * FAKE, pool=8 * FAKE, lookup=11 * FAKE, lengths=12 * FAKE,
             other=13 * FAKE, visible=14 * FAKE)


def _args(entry: str, **kw) -> tuple:
    a = {**DEFAULTS, **kw}
    head = [a[x] for x in ("out", "q", "k", "v", "tokens", "heads", "head_dim", "stride", "positions", "cos", "sin", "table_rows",
                           "pool", "pages", "layers", "page_size")]
    if entry == "paged_decode_attention_int8":
        tail = ("slot", "layer", "lookup", "cols", "lengths", "attend_max", "other", "scale", "ws", "ws_bytes")
    elif entry == "paged_chunk_attention_int8":
        tail = ("slot", "layer", "lookup", "requests", "cols", "lengths", "other", "attend_max", "visible", "scale", "ws",
                "ws_bytes")
    else:
        tail = ("layer", "lookup", "requests", "cols", "lengths", "other", "attend_max", "visible", "scale", "ws", "ws_bytes")
    return ("uocr_" + entry, *head, *(a[x] for x in tail), None)


ENTRIES = ["paged_decode_attention_int8", "paged_chunk_attention_int8", "paged_tree_attention"]


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize(("kwargs", "message"), [
    ({"head_dim": 64}, "head_dim must be 128, got 64"),
    ({"heads": 0}, "heads must be in [1, 65535]"),
    ({"heads": 65536}, "heads must be in [1, 65535]"),
    ({"pages": 0}, "bad pool of 0 pages, 2 layers, 128 rows a page"),
    ({"pages": 1 << 31}, "bad pool of 2147483648 pages, 2 layers, 128 rows a page"),
    ({"layers": 32768}, "bad pool of 3 pages, 32768 layers, 128 rows a page"),
    ({"page_size": 0}, "bad pool of 3 pages, 2 layers, 0 rows a page"),
    ({"pages": (1 << 31) - 1, "layers": 32767, "page_size": 128 << 23}, "the pool is too large"),
    ({"pool": FAKE + 8}, "the pool must be 16-byte aligned"),
    ({"page_size": 64}, "page_size must be a positive multiple of 128"),
    ({"page_size": 192}, "page_size must be a positive multiple of 128"),
    ({"layer": 2}, "layer 2 is not in the pool's 2 layers"),
    ({"layer": -1}, "layer -1 is not in the pool's 2 layers"),
    ({"tokens": -1}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"tokens": (1 << 25) // 10 + 1, "requests": 1}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"requests": 65536, "tokens": 65536}, "requests must be in [0, 65535] and tokens * heads in [0, 2^25]"),
    ({"cols": 0}, "bad lookup table width 0"),
    ({"cols": 1 << 24}, "bad lookup table width 16777216"),
    ({"attend_max": 257}, "attend_max 257 is not in [1, 256], the rows the lookup table addresses"),
    ({"attend_max": 0}, "attend_max 0 is not in [1, 256], the rows the lookup table addresses"),
    ({"scale": float("inf")}, "scale must be finite"),
    ({"scale": float("nan")}, "scale must be finite"),
    ({"stride": 1276}, "input rows must be a multiple of 4 floats apart, at least 1280 and less than 2^25, got 1276"),
    ({"stride": 1282}, "input rows must be a multiple of 4 floats apart, at least 1280 and less than 2^25, got 1282"),
    ({"stride": 1 << 25}, "input rows must be a multiple of 4 floats apart, at least 1280 and less than 2^25, got 33554432"),
    ({"positions": FAKE}, "bad cos/sin table"),
    ({"positions": FAKE, "cos": FAKE, "sin": FAKE, "table_rows": 0}, "bad cos/sin table"),
    ({"positions": FAKE, "cos": FAKE, "table_rows": 9}, "bad cos/sin table"),
    ({}, "a tensor is missing"),
])
def test_attention_refusals(entry, kwargs, message) -> None:
    assert _err(*_args(entry, **kwargs)) == f"{entry}: {message}"


@pytest.mark.parametrize("entry", ENTRIES[:2])
@pytest.mark.parametrize("slot", [0, 1312, 1320, 1412, (1 << 26) + 16])
def test_slots_that_do_not_hold_the_heads(entry, slot) -> None:
    assert _err(*_args(entry, slot=slot)) == \
        f"{entry}: a slot of {slot} bytes does not hold 10 heads of 128 values and a scale in pieces of 16"


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("name", ["out", "q", "k", "v", "pool", "lookup", "lengths", "other"])
def test_each_tensor_that_is_missing(entry, name) -> None:
    assert _err(*_args(entry, **{**GIVEN, name: None})) == f"{entry}: a tensor is missing"


def test_a_tree_needs_masks_over_float32() -> None:
    assert _err(*_args("paged_tree_attention", **{**GIVEN, "visible": None})) == "paged_tree_attention: a tensor is missing"


@pytest.mark.parametrize("entry", ENTRIES)
def test_attention_refuses_unaligned_and_overlapping_tensors(entry) -> None:
    def said(**kw):
        return _err(*_args(entry, **{**GIVEN, **kw}))

    for name in ("out", "q", "k", "v"):
        assert said(**{name: GIVEN[name] + 4}) == f"{entry}: q, k_new, v_new and out must be 16-byte aligned"
    rope = dict(positions=FAKE, cos=FAKE, sin=FAKE, table_rows=4)
    for name in ("cos", "sin"):
        assert said(**{**rope, name: FAKE + 8}) == f"{entry}: the cos/sin tables must be 16-byte aligned"
    rows = 4 * 1280 * 4
    pool = 3 * 2 * 2 * 128 * (5120 if entry == "paged_tree_attention" else SLOT)
    for at in (GIVEN["pool"] - rows + 16, GIVEN["pool"] + pool - 16):
        assert said(out=at) == f"{entry}: out must not overlap the pool"
        for name in ("q", "k", "v"):
            assert said(**{name: at}) == f"{entry}: the inputs must not overlap the pool"
    for name in ("q", "k", "v"):
        assert said(out=GIVEN[name] + rows - 16) == f"{entry}: out must not overlap the inputs"
        assert said(out=GIVEN[name] - rows + 16) == f"{entry}: out must not overlap the inputs"


@pytest.mark.parametrize("entry", ENTRIES)
def test_attention_refuses_small_and_unaligned_workspaces(entry) -> None:
    from uocr_moe import _lib

    kw = {**GIVEN, "attend_max": 6000, "cols": 47, "requests": 4}
    form = ENTRIES.index(entry)
    need = _lib.load().uocr_paged_pool_workspace_bytes(4, 4, 10, 6000, form)
    assert need > 0
    assert _err(*_args(entry, **{**kw, "ws": 16 * FAKE, "ws_bytes": need - 1})) == \
        f"{entry}: workspace of {need - 1} bytes is smaller than the {need} needed"
    assert _err(*_args(entry, **{**kw, "ws": 16 * FAKE + 8, "ws_bytes": need})) == \
        f"{entry}: workspace must be 16-byte aligned"


@pytest.mark.parametrize("entry", ENTRIES)
def test_attention_of_nothing(entry) -> None:
    _nothing(*_args(entry, tokens=0))
    if entry != "paged_decode_attention_int8":
        _nothing(*_args(entry, requests=0))


def test_workspace_bytes() -> None:
    from uocr_moe import _lib

    size = _lib.load().uocr_paged_pool_workspace_bytes
    for bad in ((-1, 1, 1, 1, 0), (1, -1, 1, 1, 0), (1, 1, 0, 1, 0), (1, 1, 65536, 1, 0), (1, 1, 1, 0, 0), (1, 1, 1, 1, -1),
                (1, 1, 1, 1, 3), (1 << 31, 1, 1, 1, 0), (1, 1 << 31, 1, 1, 1), (1, 1, 1, 1 << 31, 1)):
        assert size(*bad) == 0
    for form in (0, 1, 2):
        assert size(0, 0, 10, 4000, form) == 0 and size(1, 1, 10, 500, form) == 0
        # a split has 130 floats of a token and a head
        assert (size(1, 1, 10, 9000, form) - 4) % (130 * 4 * 10) == 0
    # rows enough of themselves
    assert size(4096, 1, 10, 4096, 1) < 4096 * 10 * 130 * 4 * 8


def _pages(kind, *, wide=2 * FAKE, narrow=4 * FAKE, wide_pages=3, narrow_pages=5, layers=2, page_size=128, heads=10, slot=SLOT,
           src=6 * FAKE, dst=7 * FAKE, rows=None, count=2):
    pools = (wide, wide_pages, narrow, narrow_pages) if kind == "quantize_pages" else (narrow, narrow_pages, wide, wide_pages)
    return ("uocr_" + kind, *pools, layers, page_size, heads, slot, src, dst, rows, count, None)


@pytest.mark.parametrize("kind", ["quantize_pages", "dequantize_pages"])
@pytest.mark.parametrize(("kwargs", "message"), [
    ({"heads": 0}, "heads must be in [1, 65535]"),
    ({"wide_pages": 0}, "bad pool of 0 pages, 2 layers, 128 rows a page"),
    ({"narrow_pages": 0}, "bad pool of 0 pages, 2 layers, 128 rows a page"),
    ({"layers": 0}, "bad pool of 3 pages, 0 layers, 128 rows a page"),
    ({"slot": 1316}, "a slot of 1316 bytes does not hold 10 heads of 128 values and a scale in pieces of 16"),
    ({"wide": 2 * FAKE + 4}, "the pool must be 16-byte aligned"),
    ({"narrow": 4 * FAKE + 4}, "the pool must be 16-byte aligned"),
    ({"count": -1}, "bad number of pairs -1"),
    ({"count": 1 << 31}, "bad number of pairs 2147483648"),
    ({"page_size": (1 << 20) + 1}, "more than 2^20 rows a page"),
    ({"wide": None}, "a tensor is missing"),
    ({"narrow": None}, "a tensor is missing"),
    ({"src": None}, "a tensor is missing"),
    ({"dst": None}, "a tensor is missing"),
    ({"narrow": 2 * FAKE + 3 * 4 * 128 * 5120 - 16}, "the pools must not overlap"),
    ({"src": 2 * FAKE}, "a list must not overlap a pool"),
    ({"dst": 4 * FAKE - 4}, "a list must not overlap a pool"),
    ({"rows": 4 * FAKE + 5 * 4 * 128 * SLOT - 4}, "a list must not overlap a pool"),
])
def test_page_conversions_refusals(kind, kwargs, message) -> None:
    assert _err(*_pages(kind, **kwargs)) == f"{kind}: {message}"


def test_no_pages_to_convert() -> None:
    _nothing(*_pages("quantize_pages", count=0, wide=None, narrow=None, src=None, dst=None))


@pytest.mark.parametrize(("args", "message"), [
    ((FAKE, 2 * FAKE, -1, 3 * FAKE, 1), "requests must be in [0, 65535] and tokens in [0, 2^25]"),
    ((FAKE, 2 * FAKE, (1 << 25) + 1, 3 * FAKE, 1), "requests must be in [0, 65535] and tokens in [0, 2^25]"),
    ((FAKE, 2 * FAKE, 4, 3 * FAKE, 65536), "requests must be in [0, 65535] and tokens in [0, 2^25]"),
    ((None, 2 * FAKE, 4, 3 * FAKE, 1), "a tensor is missing"),
    ((FAKE, None, 4, 3 * FAKE, 1), "a tensor is missing"),
    ((FAKE, 2 * FAKE, 4, None, 1), "a tensor is missing"),
    ((FAKE, FAKE + 28, 4, 3 * FAKE, 1), "the masks must not overlap the inputs"),
    ((FAKE, 2 * FAKE, 4, FAKE - 4, 1), "the masks must not overlap the inputs"),
])
def test_draft_masks_refusals(args, message) -> None:
    assert _err("uocr_draft_masks", *args, None) == "draft_masks: " + message


ACCEPT = dict(pool=2 * FAKE, pages=3, layers=2, page_size=128, slot=SLOT, lookup=4 * FAKE, requests=2, cols=2, lengths=5 * FAKE,
              offsets=6 * FAKE, parents=7 * FAKE, drafted=8 * FAKE, answers=9 * FAKE, tokens=6, counts=10 * FAKE,
              path=11 * FAKE, following=12 * FAKE, lengths_out=13 * FAKE)


def _accept(**kw) -> tuple:
    return ("uocr_accept_drafts", *{**ACCEPT, **kw}.values(), None)


@pytest.mark.parametrize(("kwargs", "message"), [
    ({"pages": 0}, "bad pool of 0 pages, 2 layers, 128 rows a page"),
    ({"slot": 100}, "a slot of 100 bytes does not hold 1 heads of 128 values and a scale in pieces of 16"),
    ({"pool": 2 * FAKE + 8}, "the pool must be 16-byte aligned"),
    ({"tokens": -1}, "requests must be in [0, 65535] and tokens in [0, 2^25]"),
    ({"requests": 65536}, "requests must be in [0, 65535] and tokens in [0, 2^25]"),
    ({"cols": 0}, "bad lookup table width 0"),
    ({"cols": 1 << 24}, "bad lookup table width 16777216"),
    *(({name: None}, "a tensor is missing") for name in ("pool", "lookup", "lengths", "offsets", "parents", "drafted", "answers",
                                                         "counts", "path", "following", "lengths_out")),
    ({"counts": 5 * FAKE + 4}, "an output must not overlap an input"),
    ({"path": 8 * FAKE + 20}, "an output must not overlap an input"),
    ({"lengths_out": 5 * FAKE}, "an output must not overlap an input"),
    ({"lookup": 2 * FAKE + 64}, "an output must not overlap an input"),
    ({"following": 10 * FAKE + 4}, "the outputs must not overlap one another"),
    ({"path": 2 * FAKE + 3 * 4 * 128 * SLOT - 4}, "the outputs must not overlap one another"),
])
def test_accept_drafts_refusals(kwargs, message) -> None:
    assert _err(*_accept(**kwargs)) == "accept_drafts: " + message


def test_accepting_for_no_requests() -> None:
    _nothing(*_accept(requests=0))


BEAM = dict(tokens=FAKE, parents=2 * FAKE, scores_out=3 * FAKE, ended_out=4 * FAKE, lengths_out=None, history_out=None,
            logits=5 * FAKE, rows=8, vocab=1000, beams=4, scores=6 * FAKE, eos=1, ended=7 * FAKE, lengths=None, alpha=0.0,
            history=None, width=0, ws=None, ws_bytes=0)
SIZES = "are not at most 65535 beams in groups of"


def _beam(**kw) -> tuple:
    return ("uocr_beam_select", *{**BEAM, **kw}.values(), None)


@pytest.mark.parametrize(("kwargs", "message"), [
    ({"beams": 0}, f"8 rows of 1000 logits {SIZES} 0 (1 to 32, at most the vocabulary)"),
    ({"beams": 33, "rows": 33}, f"33 rows of 1000 logits {SIZES} 33 (1 to 32, at most the vocabulary)"),
    ({"beams": 3}, f"8 rows of 1000 logits {SIZES} 3 (1 to 32, at most the vocabulary)"),
    ({"vocab": 3, "eos": 0}, f"8 rows of 3 logits {SIZES} 4 (1 to 32, at most the vocabulary)"),
    ({"rows": 65536}, f"65536 rows of 1000 logits {SIZES} 4 (1 to 32, at most the vocabulary)"),
    ({"rows": -4}, f"-4 rows of 1000 logits {SIZES} 4 (1 to 32, at most the vocabulary)"),
    ({"eos": -1}, "eos -1 is not in the vocabulary"),
    ({"eos": 1000}, "eos 1000 is not in the vocabulary"),
    ({"alpha": float("nan")}, "alpha must be finite"),
    ({"alpha": float("inf")}, "alpha must be finite"),
    ({"lengths": 8 * FAKE}, "lengths and history need an output each, and only then"),
    ({"lengths_out": 8 * FAKE}, "lengths and history need an output each, and only then"),
    ({"history": 8 * FAKE, "width": 4}, "lengths and history need an output each, and only then"),
    ({"history": 8 * FAKE, "history_out": 9 * FAKE, "width": -1}, "lengths and history need an output each, and only then"),
    *(({name: None}, "a tensor is missing") for name in ("tokens", "parents", "scores_out", "ended_out", "logits", "scores")),
    ({"tokens": 6 * FAKE + 28}, "an output must not overlap an input"),
    ({"ended_out": 7 * FAKE}, "an output must not overlap an input"),
    ({"scores_out": 5 * FAKE + 8 * 4000 - 4}, "an output must not overlap an input"),
    ({"history": 8 * FAKE, "history_out": 8 * FAKE + 124, "width": 4}, "an output must not overlap an input"),
    ({"parents": FAKE + 4}, "the outputs must not overlap one another"),
    ({"ws": 9 * FAKE + 8, "ws_bytes": 1 << 30}, "workspace must be 16-byte aligned"),
])
def test_beam_select_refusals(kwargs, message) -> None:
    assert _err(*_beam(**kwargs)) == "beam_select: " + message


def test_beam_select_refuses_a_small_workspace() -> None:
    from uocr_moe import _lib

    need = _lib.load().uocr_beam_select_workspace_bytes(8, 1000, 4)
    assert need > 0
    assert _err(*_beam(ws=9 * FAKE, ws_bytes=need - 1)) == \
        f"beam_select: workspace of {need - 1} bytes is smaller than the {need} needed"
    for bad in ((8, 1000, 0), (8, 1000, 33), (7, 1000, 4), (8, 3, 4), (65540, 1000, 4)):
        assert _lib.load().uocr_beam_select_workspace_bytes(*bad) == 0


def test_no_beams() -> None:
    _nothing(*_beam(rows=0))
