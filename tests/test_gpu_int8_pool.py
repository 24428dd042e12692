"""GPU tests of the attention over an int8 pool, and of the pages' conversions, against the formulas in 64 bits.

What is stored has the bits of the format's definition (each of its steps is IEEE's), so pools are compared exactly.

The attention's bar is the float32 ops' (1e-5 of a token's largest output).  What the arithmetic gives, for operands of
unit variance: the products are exact (24 bits by 8 in three), so a score has the roundings of its sum alone, 384 terms in
32 bits: about sqrt(384) 2^-25 of partial sums near 11, 6e-6, times the scale 128^-0.5: 6e-7 on a score and so on a
weight, whose own roundings are 2^-23.  The sums over the rows (at most 3000 here) add sqrt(9000) 2^-25 = 3e-6.  So 1e-5
leaves a factor of two and a half of what all at once would be, and a lost term of an operand (2^-8, 2^-16 of every
weight), a row too many or too few, or a wrong scale is outside it; the third term of an operand (2^-16) has a test of its own.
"""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV
from _served import D, SCALE, Served, far, quantized, values

pytestmark = pytest.mark.gpu

BAR = 1e-5


def _uocr():
    import uocr_moe

    return uocr_moe


def _tables(rows):
    cos, sin = _uocr().rope_tables(head_dim=D, seq_len=rows, theta=10000.0)
    return torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV)


def _chunk(s: Served, pool, visible=None):
    return _uocr().PagedChunk(kv_blocks=pool, lookup_table=s.table.to(DEV),
                              cache_lengths=torch.tensor(s.cached, dtype=torch.int32, device=DEV),
                              chunk_offsets=s.offsets.to(DEV), attend_max=s.attend_max, visible=visible)


def _run(s: Served, form: str, layer: int = 1, out=None, **kw):
    """(result, pool after it, the q, k and v that were attended and stored)."""
    u = _uocr()
    pool = s.pool.to(DEV)
    q, k, v = s.qkv.unbind(1)
    if form == "qkv":
        cos, sin = _tables(s.attend_max)
        pos = s.positions().to(DEV)
        got = u.paged_chunk_attention_qkv(s.qkv.view(s.tokens, -1).to(DEV), pos, cos, sin, heads=s.heads,
                                          kv=_chunk(s, pool), layer_idx=layer, scale=SCALE, out=out, **kw)
        q, k, _ = (None if x is None else x.cpu() for x in u.rope(q.to(DEV), k.to(DEV), pos, cos, sin))
    else:
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_chunk(s, pool), layer_idx=layer, scale=SCALE,
                                      out=out, **kw)
    return got, pool, (q, k, v)


SHAPES = [
    ([1], [0]), ([1], [1]), ([2], [127]), ([1], [128]), ([5], [123]), ([31], [1]), ([32], [0]), ([33], [95]),
    ([64], [64]), ([65], [0]), ([127], [300]), ([129], [129]), ([291], [0]), ([300], [517]), ([7], [2900]),
    ([1, 1, 1], [0, 5, 640]), ([4, 0, 9, 1], [300, 0, 0, 128]), ([0, 3], [0, 0]), ([513, 1, 70], [0, 999, 57]),
    ([3, 2, 1, 0] * 20, [0, 130, 64, 7] * 20),
]


@pytest.mark.parametrize(("chunks", "cached"), SHAPES, ids=lambda v: "-".join(map(str, v[:4])))
@pytest.mark.parametrize("form", ["plain", "qkv"])
def test_chunks_match_the_formula(chunks, cached, form) -> None:
    s = Served(len(chunks) + sum(chunks) + sum(cached), chunks, cached)
    got, pool, (q, k, v) = _run(s, form)
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu(), want), "the pool's rows"
    assert far(got.cpu(), s.want(want, 1, q)) <= BAR


@pytest.mark.parametrize(("heads", "page_size", "layers", "layer"), [(1, 128, 1, 0), (3, 256, 3, 2), (10, 384, 1, 0),
                                                                     (32, 128, 1, 0), (33, 128, 2, 1)])
def test_head_counts_page_sizes_and_layers(heads, page_size, layers, layer) -> None:
    s = Served(heads, [40, 3], [200, 400], heads=heads, page_size=page_size, layers=layers)
    got, pool, (q, k, v) = _run(s, "plain", layer)
    want = s.stored(layer, k, v)
    assert torch.equal(pool.cpu(), want)
    assert far(got.cpu(), s.want(want, layer, q)) <= BAR


def test_slots_of_another_width() -> None:
    for heads, slot in ((2, 272), (3, 1024)):
        s = Served(slot, [9], [150], heads=heads, slot=slot)
        got, pool, (q, k, v) = _run(s, "plain")
        want = s.stored(1, k, v)
        assert torch.equal(pool.cpu(), want)
        assert far(got.cpu(), s.want(want, 1, q)) <= BAR


def test_token_rows_of_no_chunk_keep_what_they_held() -> None:
    s = Served(3, [5, 0, 40], [10, 0, 200], lead=3, tail=2)
    out = torch.full((s.tokens, s.heads, D), 7.0, device=DEV)
    got, pool, (q, k, v) = _run(s, "plain", out=out)
    assert got is out
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu(), want)
    mine = slice(3, 48)
    assert far(out[mine].cpu(), s.want(want, 1, q)[mine]) <= BAR
    assert bool((out[:3] == 7).all()) and bool((out[48:] == 7).all())


@pytest.mark.parametrize("form", ["plain", "qkv"])
@pytest.mark.parametrize(("attend", "where"), [
    ([1], [0]), ([2], [0]), ([128], [127]), ([129], [128]), ([640], [200]), ([1, 640, 33, 129], [0, 639, 5, 128]),
    ([3000], [1]), ([700, 1, 2] * 30, [0, 0, 1] * 30), ([4, 4], [6, 300]),
], ids=lambda v: "-".join(map(str, v[:4])))
def test_decode_matches_the_formula(attend, where, form) -> None:
    """A new row anywhere: at the end, over an old one (a ring's), or behind what is attended."""
    u = _uocr()
    n = len(attend)
    s = Served(sum(attend) + n, [1] * n, [max(a, w + 1) - 1 for a, w in zip(attend, where)])
    pool = s.pool.to(DEV)
    kv = u.PagedKv(kv_blocks=pool, lookup_table=s.table.to(DEV),
                   attend_lengths=torch.tensor([a - 1 for a in attend], dtype=torch.int32, device=DEV),
                   attend_max=max(attend), write_index=torch.tensor(where, dtype=torch.int32, device=DEV))
    q, k, v = s.qkv.unbind(1)
    if form == "qkv":
        cos, sin = _tables(max(attend))
        pos = torch.tensor([a - 1 for a in attend], dtype=torch.int32, device=DEV)
        got = u.paged_decode_attention_qkv(s.qkv.view(n, -1).to(DEV), pos, cos, sin, heads=2, kv=kv, layer_idx=1,
                                           scale=SCALE)
        q, k, _ = (None if x is None else x.cpu() for x in u.rope(q.to(DEV), k.to(DEV), pos, cos, sin))
    else:
        got = u.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=1, scale=SCALE)
    want = s.stored(1, k, v, where)
    assert torch.equal(pool.cpu(), want)
    assert far(got.cpu(), s.want(want, 1, q, seen=lambda i, j: list(range(attend[i])))) <= BAR


def test_a_decode_step_is_a_chunk_of_one() -> None:
    """Both read what the pool holds: a prompt cut anywhere gives the rows that it gives in one piece."""
    u = _uocr()
    whole = Served(11, [150], [0], heads=3)
    got, pool, _ = _run(whole, "plain")
    pieces = Served(11, [150], [0], heads=3)
    again = pieces.pool.to(DEV)
    q, k, v = (x.to(DEV) for x in pieces.qkv.unbind(1))
    at = 0
    for size in (1, 31, 64, 53, 1):
        rows = slice(at, at + size)
        lengths = torch.tensor([at], dtype=torch.int32, device=DEV)
        if size == 1:
            kv = u.PagedKv(kv_blocks=again, lookup_table=pieces.table.to(DEV), attend_lengths=lengths, attend_max=at + 1,
                           write_index=lengths)
            out = u.paged_decode_attention(q[rows], k[rows], v[rows], kv=kv, layer_idx=1, scale=SCALE)
        else:
            kv = u.PagedChunk(kv_blocks=again, lookup_table=pieces.table.to(DEV), cache_lengths=lengths,
                              chunk_offsets=torch.tensor([0, size], dtype=torch.int32, device=DEV), attend_max=at + size)
            out = u.paged_chunk_attention(q[rows], k[rows], v[rows], kv=kv, layer_idx=1, scale=SCALE)
        assert far(out.cpu(), got[rows].double().cpu()) <= 2 * BAR
        at += size
    assert torch.equal(again, pool)


def test_every_term_of_the_operands_counts() -> None:
    """Two rows of 127 s with signs, of scores near 16384 and nearly equal: the weight of the first (its values are 1, the
    other's 0) is off by a quarter of what the scores are.  The sum's roundings leave 16384 sqrt(384) 2^-25 = 0.0096 of
    each, so 0.25 sqrt(2) 0.0096 = 0.0034; a lost third term of the query (2^-17 of an element) 16384 2^-17 = 0.125, so
    0.044.  The bar, of eight heads' mean square, is between."""
    heads = 8
    g = torch.Generator().manual_seed(5)
    s = Served(5, [1], [1], heads=heads, layers=1)
    q = torch.randn(heads, D, generator=g) * 16384
    keys = torch.empty(2, heads, D)
    for h in range(heads):
        signs = torch.randint(0, 2, (4000, D), generator=g).double() * 2 - 1
        scores, order = torch.sort((signs @ q[h].double()) * SCALE)
        near = int((scores[1:] - scores[:-1]).argmin())
        assert float(scores[near + 1] - scores[near]) < 0.5
        keys[:, h] = signs[order[near:near + 2]].float()
    vals = torch.stack([torch.ones(heads, D), torch.zeros(heads, D)])
    page = int(s.table[0, 0])
    s.pool[page, 0, 0, 0] = quantized(keys[0], s.slot)
    s.pool[page, 1, 0, 0] = quantized(vals[0], s.slot)
    s.qkv = torch.stack([q, keys[1], vals[1]])[None]
    got, pool, (q, k, v) = _run(s, "plain", 0)
    want = s.want(s.stored(0, k, v), 0, q)
    assert float((want[0, :, 0] - 0.5).abs().max()) < 0.2, "the weights are near a half"
    assert float((got.cpu().double() - want)[0, :, 0].square().mean().sqrt()) <= 0.01


def test_what_is_not_attended_leaves_nothing() -> None:
    """Rows past a token's, of other requests' pages and of the null page hold NaN and infinities."""
    s = Served(8, [37, 2], [90, 128])
    rows = torch.full((s.heads, D), 3.0)
    dead = quantized(rows, s.slot)
    dead[128 * s.heads:132 * s.heads] = torch.tensor([float("nan"), float("inf")]).view(torch.int8)
    used = {s.place(i, r) for i in (0, 1) for r in range(s.cached[i])}
    for p in range(s.pool.shape[0]):
        for r in range(s.page_size):
            if (p, r) not in used:
                s.pool[p, :, :, r] = dead
    got, pool, (q, k, v) = _run(s, "plain")
    assert far(got.cpu(), s.want(s.stored(1, k, v), 1, q)) <= BAR


def test_a_row_that_is_not_finite_reaches_those_that_attend_it() -> None:
    s = Served(9, [40], [20])
    s.qkv[11, 1, 0, 5] = float("inf")   # a key of head 0
    s.qkv[30, 2, 1, 100] = float("nan")  # a value of head 1
    got, pool, (q, k, v) = _run(s, "plain")
    want = s.want(s.stored(1, k, v), 1, q)
    assert torch.equal(got.cpu().isnan(), want.isnan())
    assert bool(got[11:, 0].isnan().all()) and bool(got[30:, 1].isnan().all())
    assert bool(got[:11].isfinite().all()) and bool(got[:30, 1].isfinite().all())
    fine = want.isfinite()
    assert float((got.cpu().double() - want)[fine].abs().max()) <= BAR * float(want[fine].abs().max())


def test_rows_of_zeros_and_of_extreme_sizes_are_stored_as_defined() -> None:
    s = Served(10, [8], [0])
    k = s.qkv[:, 1]
    k[0] = 0.0
    k[1] *= 1e-44
    k[2] *= 1e-38
    k[3] *= 1e30
    k[4, 0] = 127.0
    k[4, 0, 1:4] = torch.tensor([0.5, 1.5, -2.5])  # ties go to even
    k[5] = torch.finfo(torch.float32).max
    got, pool, (q, k, v) = _run(s, "plain")
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu(), want)
    assert pool[s.place(0, 4)[0], 0, 1, 4, :4].tolist() == [127, 0, 2, -2]


def test_strided_rows_other_outputs_and_workspaces() -> None:
    u = _uocr()
    s = Served(12, [5, 70], [260, 31], heads=3)
    got, pool, (q, k, v) = _run(s, "plain")
    wide = torch.zeros(s.tokens, 3, 5, D, device=DEV)
    wide[:, :, 1:4] = s.qkv.to(DEV)
    again = s.pool.to(DEV)
    need = u._lib.load().uocr_paged_pool_workspace_bytes(s.tokens, 2, 3, s.attend_max, 1)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    out = u.paged_chunk_attention(*(wide[:, j, 1:4] for j in range(3)), kv=_chunk(s, again), layer_idx=1, scale=SCALE,
                                  workspace=ws)
    assert torch.equal(out, got) and torch.equal(again, pool)
    assert bool((ws[need:] == 0xFF).all())
    unsigned = _chunk(s, s.pool.to(DEV))
    unsigned = type(unsigned)(**{**vars(unsigned), "lookup_table": unsigned.lookup_table.view(torch.uint32),
                                 "cache_lengths": unsigned.cache_lengths.view(torch.uint32)})
    out = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=unsigned, layer_idx=1, scale=SCALE)
    assert torch.equal(out, got)


def test_a_negative_scale_and_none() -> None:
    s = Served(13, [33], [100])
    u = _uocr()
    q, k, v = s.qkv.unbind(1)
    for scale in (-0.3, 0.0):
        pool = s.pool.to(DEV)
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_chunk(s, pool), layer_idx=1, scale=scale)
        # scores are 3.4 times those of 128^-0.5, and so are their errors
        assert far(got.cpu(), s.want(s.stored(1, k, v), 1, q, scale=scale)) <= 4 * BAR


def test_tables_cut_short_and_lengths_that_lie() -> None:
    """Lengths past the table are clamped to it, and pages past the pool to the null page: nothing is read or written
    outside."""
    u = _uocr()
    s = Served(14, [3], [200])
    pool = s.pool.to(DEV)
    before = pool.clone()
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    table = s.table.clone()
    table[0, 1] = 1 << 30
    kv = u.PagedChunk(kv_blocks=pool, lookup_table=table.to(DEV),
                      cache_lengths=torch.tensor([1 << 30], dtype=torch.int32, device=DEV),
                      chunk_offsets=torch.tensor([0, 1 << 20], dtype=torch.int32, device=DEV), attend_max=250)
    out = u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE)
    assert out.shape == q.shape
    assert torch.equal(pool, before)  # the rows lie past the table


def test_no_tokens_and_no_requests() -> None:
    u = _uocr()
    s = Served(15, [0, 0], [5, 0])
    got, pool, _ = _run(s, "plain")
    assert got.shape == (0, 2, D) and torch.equal(pool.cpu(), s.pool)
    kv = u.PagedKv(kv_blocks=pool, lookup_table=s.table[:0].to(DEV), attend_lengths=s.offsets[:0].to(DEV), attend_max=1,
                   write_index=s.offsets[:0].to(DEV))
    none = torch.empty(0, 2, D, device=DEV)
    assert u.paged_decode_attention(none, none, none, kv=kv, layer_idx=0, scale=1.0).shape == (0, 2, D)


def test_captured_and_replayed_on_another_stream() -> None:
    """Replays with other lengths, eager calls between them."""
    u = _uocr()
    s = Served(16, [6, 2], [700, 0], heads=10)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    pool = s.pool.to(DEV)
    kv = _chunk(s, pool)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.graph(graph, stream=stream):
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE, out=out)
    for first, lengths in (([0, 6, 8], [700, 0]), ([0, 1, 8], [300, 130]), ([0, 8, 8], [690, 0]), ([0, 6, 8], [700, 0])):
        kv.chunk_offsets.copy_(torch.tensor(first, dtype=torch.int32))
        kv.cache_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        pool.copy_(s.pool)
        eager_pool = s.pool.to(DEV)
        eager = u.paged_chunk_attention(q, k, v, kv=type(kv)(**{**vars(kv), "kv_blocks": eager_pool}), layer_idx=1,
                                        scale=SCALE)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(pool, eager_pool)


# ------------------------------------------------------------------------------------------ pages


@pytest.mark.parametrize(("heads", "page_size", "layers"), [(10, 128, 2), (1, 128, 1), (3, 256, 3), (33, 128, 1), (2, 5, 2)])
@pytest.mark.parametrize("partial", [False, True])
def test_pages_converted(heads, page_size, layers, partial) -> None:
    u = _uocr()
    g = torch.Generator().manual_seed(heads + page_size)
    wide = torch.randn(5, 2, layers, page_size, heads, D, generator=g)
    wide[1, 0, 0, 0] = 0.0
    wide[2, 1, 0, 1, 0, 3] = float("nan")
    narrow = u.int8_kv_blocks(6, layers, page_size, heads, device="cpu")
    narrow.copy_(torch.randint(-127, 128, narrow.shape, generator=g, dtype=torch.int8))
    slot = narrow.shape[-1]
    narrow[..., 128 * heads:132 * heads] = torch.rand(6, 2, layers, page_size, heads, generator=g).view(torch.int8)
    src, dst = [1, 2, 4, 9, 0, 3], [5, 0, 5, 1, -1, 3]  # a page twice; pairs outside a pool
    rows = [page_size, 3, 2, page_size, page_size, page_size - 1] if partial else [page_size] * 6
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    want = narrow.clone()
    for a, b, r in zip(src, dst, rows):
        if 0 <= a < 5 and 0 <= b < 6:
            want[b, :, :, :r, :132 * heads] = quantized(wide[a, :, :, :r], slot)[..., :132 * heads]
    got = narrow.to(DEV)
    assert u.quantize_pages(wide.to(DEV), on(src), got, on(dst), rows=on(rows) if partial else None) is got
    assert torch.equal(got.cpu(), want)
    want = wide.clone()
    back = [5, 0, 5, -1, 9, 2]
    to = [1, 0, 1, 2, 3, 4]
    for a, b, r in zip(back, to, rows):
        if 0 <= a < 6:
            want[b, :, :, :r] = values(narrow[a, :, :, :r], heads).float()
    got = wide.to(DEV)
    assert u.dequantize_pages(narrow.to(DEV), on(back), got, on(to), rows=on(rows) if partial else None) is got
    assert torch.equal(got.cpu().view(torch.int32), want.view(torch.int32))


def test_no_pages_converted() -> None:
    u = _uocr()
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    wide, narrow = torch.ones(1, 2, 1, 128, 1, D, device=DEV), u.int8_kv_blocks(1, 1, 128, 1, device=DEV)
    u.quantize_pages(wide, none, narrow, none)
    u.dequantize_pages(narrow, none, wide, none)
    assert bool((narrow == 0).all()) and bool((wide == 1).all())


def test_page_operators_take_an_int8_pool() -> None:
    """Copies, forks and compactions of an int8 pool move the bytes that they move of a float32 one."""
    u = _uocr()
    g = torch.Generator().manual_seed(4)
    pool = u.int8_kv_blocks(9, 2, 128, 3, device="cpu")
    pool.copy_(torch.randint(-128, 128, pool.shape, generator=g, dtype=torch.int8))  # NaN patterns among the scales
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = pool.to(DEV)
    assert u.copy_pages(got, on([0, 1]), on([1, 2]), rows=on([128, 40])) is got
    want = pool.clone()
    want[1] = want[0]
    want[2, :, :, :40] = want[1, :, :, :40]
    assert torch.equal(got.cpu(), want)
    got = pool.to(DEV)
    table, counts, missing = u.fork_pages(got, on([1, 1, 0, 0, 0, 0, 0, 0, 0]), on([[0, 1], [8, 8]]), on([0]), on([1]),
                                          on([200]), on([128]))
    assert table.tolist() == [[0, 1], [0, 2]] and counts.tolist()[:3] == [2, 1, 1] and int(missing) == 0
    want = pool.clone()
    want[2, :, :, :72] = want[1, :, :, :72]
    assert torch.equal(got.cpu(), want)
    got = pool.to(DEV)
    table, counts, remap = u.compact_pages(got, on([0, 0, 0, 1, 0, 1, 0, 0, 0]), on([[5, 3]]))
    assert table.tolist() == [[1, 0]]
    want = pool.clone()
    want[0], want[1] = pool[3], pool[5]
    assert torch.equal(got.cpu(), want)
