"""GPU tests of how calls over an int8 pool, and of trees, are cut into workgroups: tiles of 256 queries and of 32, a head or
two a wave, splits that the device counts from the lengths, joins of few and many, more requests than lanes.

The bar is the float32 ops' (1e-5 of a token's largest output).  Of the arithmetic, the sums over the rows are what grows
here: at 9100 rows in three terms each sqrt(27300) 2^-25 = 5e-6 of the result, a split's and a join's roundings (2^-24 each)
beside it; the scores' 6e-7 stay.
"""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from _served import D, SCALE, Served, far, masks_of, signed

pytestmark = pytest.mark.gpu

BAR = 1e-5


def _uocr():
    import uocr_moe

    return uocr_moe


def _on(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _chunk(s: Served, pool, visible=None, cached=None, attend_max=None):
    return _uocr().PagedChunk(kv_blocks=pool, lookup_table=s.table.to(DEV), cache_lengths=_on(cached or s.cached),
                              chunk_offsets=s.offsets.to(DEV), attend_max=attend_max or s.attend_max, visible=visible)


def _want(s: Served, pool, q, layer=1) -> torch.Tensor:
    """As Served.want, a chunk at a time."""
    out = torch.zeros(s.tokens, s.heads, D, dtype=torch.float64)
    for i, c in enumerate(s.chunks):
        if c == 0:
            continue
        first = int(s.offsets[i])
        keys, vals = s.rows_of(pool, i, s.cached[i] + c, layer)
        x = q[first:first + c].double().permute(1, 0, 2) @ keys.permute(1, 2, 0) * SCALE
        later = torch.arange(s.cached[i] + c)[None, :] > s.cached[i] + torch.arange(c)[:, None]
        out[first:first + c] = (torch.softmax(x.masked_fill(later, -torch.inf), dim=2) @ vals.permute(1, 0, 2)).permute(1, 0, 2)
    return out


def _run(s: Served, pool=None, **kw):
    pool = s.pool.to(DEV) if pool is None else pool
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    return _uocr().paged_chunk_attention(q, k, v, kv=_chunk(s, pool), layer_idx=1, scale=SCALE, **kw), pool


# Tiles of 256 queries: 256 tokens a request on average, tokens * attend_max >= 3 * 2^20.
TILES = [
    ([530], [6000], 2), ([700, 0, 300, 257], [2800, 0, 0, 517], 3), ([256], [12300], 1), ([1025], [2100], 1),
    ([2000], [0], 2), ([3, 900, 1, 1200], [40, 1500, 3100, 0], 2), ([1100] * 3, [0, 130, 77], 10), ([260] * 65, [0] * 65, 1),
    ([256] * 65, [0, 300, 600, 7, 128] * 13, 1),
]


@pytest.mark.parametrize(("chunks", "cached", "heads"), TILES, ids=lambda v: "-".join(map(str, v[:4])) if isinstance(v, list) else str(v))
def test_tiles(chunks, cached, heads) -> None:
    s = Served(len(chunks) + sum(chunks) + sum(cached), chunks, cached, heads=heads)
    assert s.tokens // len(chunks) >= 256 and s.tokens * s.attend_max >= 3 << 20
    got, pool = _run(s)
    q, k, v = s.qkv.unbind(1)
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu(), want)
    assert far(got.cpu(), _want(s, want, q)) <= BAR


@pytest.mark.parametrize(("chunks", "cached"), [
    ([256], [12031]), ([256], [12032]), ([255, 256], [6000, 5900]), ([256, 256], [5888, 5800]),
], ids=lambda v: "-".join(map(str, v)))
def test_either_side_of_the_tiles(chunks, cached) -> None:
    s = Served(sum(cached), chunks, cached, heads=1)
    got, pool = _run(s)
    q, k, v = s.qkv.unbind(1)
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu(), want)
    assert far(got.cpu(), _want(s, want, q)) <= BAR


def test_tiles_of_a_projection_before_rope_with_rows_of_no_chunk() -> None:
    u = _uocr()
    s = Served(3, [600, 290], [3000, 3500], heads=3, lead=2, tail=5)
    cos, sin = (torch.from_numpy(x).to(DEV) for x in u.rope_tables(head_dim=D, seq_len=s.attend_max, theta=10000.0))
    pos = s.positions().to(DEV)
    pool, out = s.pool.to(DEV), torch.full((s.tokens, 3, D), 7.0, device=DEV)
    u.paged_chunk_attention_qkv(s.qkv.view(s.tokens, -1).to(DEV), pos, cos, sin, heads=3, kv=_chunk(s, pool), layer_idx=1,
                                scale=SCALE, out=out)
    q, k, v = s.qkv.unbind(1)
    q, k, _ = (None if x is None else x.cpu() for x in u.rope(q.to(DEV), k.to(DEV), pos, cos, sin))
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu(), want)
    chunk = slice(2, 2 + 890)
    assert far(out[chunk].cpu(), _want(s, want, q)[chunk]) <= BAR
    assert bool((out[:2] == 7).all()) and bool((out[-5:] == 7).all())


def test_what_tiles_do_not_attend_leaves_nothing() -> None:
    """NaN behind the last row, in pages of nobody and, among the new rows, for the tokens before it."""
    s = Served(4, [600], [5000], heads=2)
    clean, _ = _run(s)
    pool = s.pool.clone()
    bad = torch.full((), float("nan")).repeat(2).view(torch.int8)
    own = set(s.table[0, :-(-5600 // 128)].tolist())
    for p in range(pool.shape[0]):
        if p not in own:
            pool[p, :, :, :, 256:264] = bad
    page, at = s.place(0, 5599)
    pool[page, :, :, at + 1:, 256:264] = bad
    got, _ = _run(s, pool.to(DEV))
    assert torch.equal(got, clean)
    for what in (float("nan"), float("inf")):
        s.qkv[333, 2, 1, 50] = what  # a value
        got, _ = _run(s)
        assert torch.equal(got[:333], clean[:333]) and torch.equal(got[:, 0], clean[:, 0])
        assert bool(got[333:, 1].isnan().all())
        s.qkv[333, 2, 1, 50] = 0.5


# Few new tokens: cut once or twice over, joined by a wave or by four, counted by the lanes or (65 on) by slots.
CUTS = [
    ([8], [9000], 10), ([1], [2047], 1), ([33], [4000], 10), ([2] * 24, list(range(300, 2700, 100)), 10),
    ([40] * 8, [1900, 30, 700, 0, 1400, 1, 513, 250], 3), ([3] * 70, [0, 1500, 64, 700, 1023] * 14, 1),
    ([5, 0] * 33, [1200, 9] * 33, 2), ([70] * 20, [900, 0, 100, 1700] * 5, 10), ([1] * 64, [513] * 64, 3),
]


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
@pytest.mark.parametrize(("chunks", "cached", "heads"), CUTS, ids=lambda v: "-".join(map(str, v[:4])) if isinstance(v, list) else str(v))
def test_cuts(chunks, cached, heads, int8) -> None:
    """As chunks over the int8 pool, and as chains of a tree over either."""
    u = _uocr()
    s = Served(len(chunks) + sum(chunks) + sum(cached), chunks, cached, heads=heads, int8=int8)
    q, k, v = s.qkv.unbind(1)
    stored = s.stored(1, k, v)
    want = _want(s, stored, q)
    if int8:
        got, pool = _run(s)
        assert torch.equal(pool.cpu(), stored)
        assert far(got.cpu(), want) <= BAR
    if max(chunks) <= 64:
        visible = u.draft_masks(_on([j - 1 for c in chunks for j in range(c)]), s.offsets.to(DEV))
        pool = s.pool.to(DEV)
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_chunk(s, pool, visible), layer_idx=1, scale=SCALE)
        assert torch.equal(pool.cpu(), stored)
        assert far(got.cpu(), want) <= BAR


@pytest.mark.parametrize(("n", "heads", "longest"), [(43, 3, 1000), (30, 5, 2900), (129, 1, 900), (16, 9, 5000), (1, 3, 6000),
                                                     (12, 10, 1500), (13, 10, 1500), (2, 64, 1409)])
def test_decode_cuts(n, heads, longest) -> None:
    """A head a wave or two, an odd last one alone; whole rows and splits, short requests beside long ones."""
    u = _uocr()
    attend = [max(1, longest * (i + 1) // n - 37 * (i % 3)) for i in range(n)]
    s = Served(n * heads + longest, [1] * n, [a - 1 for a in attend], heads=heads)
    q, k, v = s.qkv.unbind(1)
    where = [(a - 1) // (1 + i % 2) for i, a in enumerate(attend)]
    pool = s.pool.to(DEV)
    kv = u.PagedKv(kv_blocks=pool, lookup_table=s.table.to(DEV), attend_lengths=_on([a - 1 for a in attend]),
                   attend_max=max(attend), write_index=_on(where))
    got = u.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=1, scale=SCALE)
    stored = s.stored(1, k, v, where)
    assert torch.equal(pool.cpu(), stored)
    assert far(got.cpu(), _want(s, stored, q)) <= BAR


@pytest.mark.parametrize("big", [False, True], ids=["queries-32", "queries-256"])
def test_replays_cut_by_the_lengths_they_find(big) -> None:
    """A captured call whose lengths and chunks change between replays."""
    u = _uocr()
    s = Served(6, [600, 500] if big else [20, 11, 9], [3200, 1500] if big else [2500, 1100, 30], heads=4)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    pool, out = s.pool.to(DEV), torch.zeros_like(s.qkv[:, 0], device=DEV)
    kv = _chunk(s, pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE, out=out)
    for change in range(4):
        lengths = [max(0, c - 311 * change) for c in s.cached]
        bounds = s.offsets.clone()
        bounds[1] -= 3 * change
        kv.cache_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        kv.chunk_offsets.copy_(bounds)
        pool.copy_(s.pool)
        eager_pool = s.pool.to(DEV)
        eager = u.paged_chunk_attention(q, k, v, kv=type(kv)(**{**vars(kv), "kv_blocks": eager_pool}), layer_idx=1, scale=SCALE)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(pool, eager_pool)
        t = Served(6, [int(b - a) for a, b in zip(bounds, bounds[1:])], lengths, heads=4)
        t.table, t.pool = s.table, s.pool
        stored = t.stored(1, *s.qkv.unbind(1)[1:])
        assert torch.equal(pool.cpu(), stored)
        assert far(out.cpu(), _want(t, stored, s.qkv[:, 0])) <= BAR


def test_two_calls_at_once() -> None:
    """Calls of every form on two streams, each with a workspace that the library finds, twice over."""
    u = _uocr()
    work = []
    for seed, chunks, cached, masked in ((1, [530], [6000], False), (2, [30, 4], [2500, 900], True), (3, [9] * 5, [1700] * 5, False)):
        s = Served(seed, chunks, cached, heads=3)
        visible = None
        if masked:
            visible = _on([signed(b) for c in chunks for b in masks_of([j - 1 for j in range(c)])], torch.int64)
        work.append((s, visible, [x.to(DEV) for x in s.qkv.unbind(1)], [s.pool.to(DEV) for _ in range(4)]))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for turn in range(2):
        for at, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for s, visible, (q, k, v), pools in (work if at == 0 else work[::-1]):
                    pool = pools[2 * turn + at]
                    got.append((s, pool, u.paged_chunk_attention(q, k, v, kv=_chunk(s, pool, visible), layer_idx=1, scale=SCALE)))
    torch.cuda.synchronize()
    for s, pool, out in got:
        q, k, v = s.qkv.unbind(1)
        stored = s.stored(1, k, v)
        assert torch.equal(pool.cpu(), stored)
        assert far(out.cpu(), _want(s, stored, q)) <= BAR


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
@pytest.mark.parametrize("chunks", [[16] * 8, [17] + [16] * 7, [32] * 4, [33] * 3, [128] + [0] * 3, [97] + [1] * 31, [1] * 128],
                         ids=lambda v: f"{sum(v)}-{len(v)}")
def test_either_side_of_rows_stored_by_their_readers(chunks, int8) -> None:
    """Up to 128 tokens, 32 a request on average; one request may have most of them."""
    u = _uocr()
    s = Served(len(chunks), chunks, [(37 * i) % 150 for i in range(len(chunks))], heads=3, int8=int8, lead=1, tail=2)
    q, k, v = s.qkv.unbind(1)
    stored = s.stored(1, k, v)
    bits = [signed((b & (1 << 64) - 1)) for c in chunks for b in masks_of([j - 1 for j in range(c)])]
    visible = _on([0] + bits + [0, 0], torch.int64)
    pool, out = s.pool.to(DEV), torch.full((s.tokens, 3, D), 7.0, device=DEV)
    u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_chunk(s, pool, None if int8 else visible), layer_idx=1,
                            scale=SCALE, out=out)
    assert torch.equal(pool.cpu(), stored)
    assert bool((out[:1] == 7).all()) and bool((out[-2:] == 7).all())
    want = _want(s, stored, q)
    if not int8:  # a tree's tokens past the first 64 see the first 64 alone
        seen = [min(j, 63) for c in chunks for j in range(c)]
        keep = torch.tensor([True] + [x == j for x, j in zip(seen, (j for c in chunks for j in range(c)))] + [True] * 2)
        want, out = want[keep], out[keep.to(DEV)]
    assert far(out[1:-2].cpu(), want[1:-2]) <= BAR


@pytest.mark.parametrize("chunk", [7, 40, 130])
def test_rows_past_what_is_attended_are_stored(chunk) -> None:
    """An attend_max below the last rows: all new rows are stored, those below it are attended."""
    u = _uocr()
    s = Served(chunk, [chunk], [300], heads=3)
    q, k, v = s.qkv.unbind(1)
    stored = s.stored(1, k, v)
    for most in (302, 300, 128):
        pool = s.pool.to(DEV)
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_chunk(s, pool, attend_max=most), layer_idx=1, scale=SCALE)
        assert torch.equal(pool.cpu(), stored)
        want = s.want(stored, 1, q, seen=lambda i, j: list(range(min(300 + j + 1, most))))
        assert far(got.cpu(), want) <= BAR
