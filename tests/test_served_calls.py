"""What the wrappers of the served cache's operators check and hand to the library's entries (no GPU: the tensors are the
CPU's, which say that they are on one, and the entry's call is taken down instead of made)."""

from __future__ import annotations

import pytest
import torch

HEADS, D, SLOT = 2, 128, 384


class OnGpu(torch.Tensor):
    """A CPU tensor that passes the wrappers' checks."""

    is_cuda = property(lambda self: True)


def _on(t: torch.Tensor) -> torch.Tensor:
    return t.as_subclass(OnGpu)


@pytest.fixture
def calls(monkeypatch):
    """The entries' calls: (name, arguments)."""
    from uocr_moe import ops

    made: list = []
    monkeypatch.setattr(ops, "_on_device", lambda op, name, *args, tensors: made.append((name, args)))
    return made


def _pool(int8: bool) -> torch.Tensor:
    return _on(torch.zeros(3, 2, 1, 128, SLOT, dtype=torch.int8) if int8 else torch.zeros(3, 2, 1, 128, HEADS, D))


def _i32(*values) -> torch.Tensor:
    return _on(torch.tensor(values, dtype=torch.int32))


def _attend(form: str, qkv: torch.Tensor, table_width: int = D):
    """The fused call over one request: of a decode step, of a chunk over the int8 pool, or of a tree over either."""
    import uocr_moe as u

    tokens = qkv.shape[0]
    tables = [_on(torch.zeros(8, table_width)) for _ in range(2)]
    positions = _i32(*range(tokens))
    if form == "decode":
        kv = u.PagedKv(kv_blocks=_pool(True), lookup_table=_i32([0]), attend_lengths=_i32(0), attend_max=1,
                       write_index=_i32(0))
        call = u.paged_decode_attention_qkv
    else:
        visible = _on(torch.ones(tokens, dtype=torch.int64)) if "tree" in form else None
        kv = u.PagedChunk(kv_blocks=_pool("int8" in form), lookup_table=_i32([0]), cache_lengths=_i32(0),
                          chunk_offsets=_i32(0, tokens), attend_max=tokens, visible=visible)
        call = u.paged_chunk_attention_qkv
    return call(qkv, positions, *tables, heads=HEADS, kv=kv, layer_idx=0, scale=1.0)


FORMS = ["decode", "int8 chunk", "int8 tree", "float32 tree"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("width", [64, 127, 129, 256])
def test_tables_of_another_width_are_refused(calls, form, width) -> None:
    """The kernels read rows of 128 from the tables, past the end of narrower ones."""
    qkv = _on(torch.zeros(1, 3 * HEADS * D))
    with pytest.raises(ValueError, match=f"the cos/sin tables are {width} wide, not head_dim 128"):
        _attend(form, qkv, width)
    assert calls == []
    _attend(form, qkv)
    assert len(calls) == 1


@pytest.mark.parametrize("form", [*FORMS, "float32 chunk"])
@pytest.mark.parametrize("stride", [0, 1, 3 * HEADS * D + 2, (1 << 25) + 1])
def test_one_row_of_any_stride(calls, form, stride) -> None:
    """A single row is contiguous whatever its stride is, and goes to the entries as one that is packed."""
    width = 3 * HEADS * D
    qkv = _on(torch.zeros(width).as_strided((1, width), (stride, 1)))
    assert qkv.is_contiguous() and qkv.stride(0) == stride
    _attend(form, qkv)
    (name, args), = calls
    passed = args[5 if name == "uocr_paged_chunk_attention_qkv" else 7]  # row_stride
    assert passed >= (width if "qkv" in name else HEADS * D) and passed % 4 == 0 and passed < 1 << 25


def test_accepting_for_no_requests_leaves_no_word_unset(calls, monkeypatch) -> None:
    """Tokens of no chunk have -1 in the path, where there is no request at all too."""
    import uocr_moe as u

    allocate = torch.Tensor.new_empty
    monkeypatch.setattr(OnGpu, "new_empty", lambda self, *a, **kw: allocate(self, *a, **kw).fill_(77))
    kv = u.PagedChunk(kv_blocks=_pool(True), lookup_table=_on(torch.zeros(0, 1, dtype=torch.int32)), cache_lengths=_i32(),
                      chunk_offsets=_i32(0), attend_max=1)
    counts, path, following, lengths = u.accept_drafts(kv, _i32(-1, 0, 1), _i32(5, 6, 7), _i32(6, 7, 8))
    assert path.tolist() == [-1, -1, -1]
    assert counts.shape == following.shape == lengths.shape == (0,)
