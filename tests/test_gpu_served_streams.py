"""GPU tests of the served operators on two streams at once with the library's own workspaces, one for each stream, which grow
from call to call, and of a batch that mixes a long prompt's piece with single tokens.

The bar is the other ops' (1e-5 of a token's largest output); calls on either stream have the bits of a call alone.
"""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from _served import D, SCALE, Served, far, masks_of, quantized, signed

pytestmark = pytest.mark.gpu

BAR = 1e-5


def _uocr():
    import uocr_moe

    return uocr_moe


def _on(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _calls() -> list:
    """Calls in splits, of every form, and a beam step, by the workspaces that they need: (bytes, call of a fresh pool)."""
    u = _uocr()
    size = u._lib.load().uocr_paged_pool_workspace_bytes
    calls = []
    for seed, chunks, cached, form in ((1, [1, 1], [4100, 3000], 0), (2, [30, 4], [2500, 900], 2), (3, [9] * 5, [1700] * 5, 1),
                                       (4, [64, 50], [4000, 3500], 2), (5, [530], [6000], 1)):
        s = Served(seed, chunks, cached, heads=3)
        q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
        table, lengths = s.table.to(DEV), _on(s.cached)
        visible = None if form != 2 else _on([signed(b) for c in chunks for b in masks_of([j - 1 for j in range(c)])],
                                             torch.int64)

        def call(s=s, q=q, k=k, v=v, table=table, lengths=lengths, form=form, visible=visible, offsets=s.offsets.to(DEV),
                 start=s.pool.to(DEV)):
            pool = start.clone()
            if form == 0:
                kv = u.PagedKv(kv_blocks=pool, lookup_table=table, attend_lengths=lengths, attend_max=s.attend_max,
                               write_index=lengths)
                return u.paged_decode_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE), pool
            kv = u.PagedChunk(kv_blocks=pool, lookup_table=table, cache_lengths=lengths, chunk_offsets=offsets,
                              attend_max=s.attend_max, visible=visible)
            return u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE), pool

        need = size(s.tokens, len(chunks), 3, s.attend_max, form)
        assert need > 0, "cut into splits"
        calls.append((need, call))
    logits = torch.randn(64, 20000, generator=torch.Generator().manual_seed(6)).to(DEV)
    scores = torch.zeros(64, device=DEV)
    need = u._lib.load().uocr_beam_select_workspace_bytes(64, 20000, 8)
    calls.append((need, lambda: u.beam_select(logits, scores, beams=8, eos=0)[:4]))
    calls.sort(key=lambda x: x[0])
    assert calls[-1][0] > 1 << 20, "more than a workspace begins with"
    return [call for _, call in calls]


def test_two_streams_with_the_librarys_workspaces(monkeypatch) -> None:
    """Small calls first on one stream, large ones first on the other, three times over, nothing waited for between them."""
    from uocr_moe import ops

    calls = _calls()
    want = [call() for call in calls]
    monkeypatch.setattr(ops, "_workspace", lambda *a: None)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for i in range(len(calls)):
            for stream, at in zip(streams, (i, len(calls) - 1 - i)):
                with torch.cuda.stream(stream):
                    got.append((at, calls[at]()))
    torch.cuda.synchronize()
    for at, results in got:
        assert all(torch.equal(a, b) for a, b in zip(results, want[at]))


def test_a_prompts_piece_beside_single_tokens() -> None:
    """A chunk of 700 tokens over 5000 rows and thirty-one single tokens, the served decoder's ten heads, over the int8 pool."""
    u = _uocr()
    chunks = [1] * 11 + [700] + [1] * 20
    s = Served(8, chunks, [5000 if c > 1 else 40 + 61 * i for i, c in enumerate(chunks)], heads=10, layers=1)
    q, k, v = s.qkv.unbind(1)
    pool = s.pool.to(DEV)
    kv = u.PagedChunk(kv_blocks=pool, lookup_table=s.table.to(DEV), cache_lengths=_on(s.cached),
                      chunk_offsets=s.offsets.to(DEV), attend_max=s.attend_max)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=0, scale=SCALE).cpu()
    stored = s.pool.clone()
    new = quantized(torch.stack([k, v], 1), s.slot)[..., :132 * 10]
    for i, t, j in s.each():
        page, slot = s.place(i, s.cached[i] + j)
        stored[page, :, 0, slot, :132 * 10] = new[t]
    assert torch.equal(pool.cpu(), stored)
    for i, c in enumerate(chunks):
        first, rows = int(s.offsets[i]), s.cached[i] + c
        keys, vals = s.rows_of(stored, i, rows, 0)
        for j in range(0, c, 50):  # every fiftieth token of the long chunk
            t, n = first + j, s.cached[i] + j + 1
            weight = torch.softmax(torch.einsum("hd,rhd->hr", q[t].double(), keys[:n]) * SCALE, dim=1)
            assert far(got[t:t + 1], torch.einsum("hr,rhd->hd", weight, vals[:n])[None]) <= BAR
    assert got.shape == (s.tokens, 10, D)
