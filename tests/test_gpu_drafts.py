"""GPU tests of trees of drafted tokens (masks, attention over either pool, acceptance) against plain walks and the
formula in 64 bits.

The attention's bar is the other ops' (1e-5 of a token's largest output), and the int8 pool's arithmetic that of its
other entries.  Over the float32 pool a product of two operands of 24 bits leaves out 2^-24 of itself in its six terms,
less than the roundings of its sum (768 terms in 32 bits: sqrt(768) 2^-25 of partial sums near 11, 9e-6, times the
scale: 8e-7 on a score); the values' sums over 3000 rows add sqrt(18000) 2^-25 = 4e-6.
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


def _tree(g: torch.Generator, nodes: int) -> list[int]:
    """Parents: the root's -1, the others' an earlier node."""
    return [-1] + [int(torch.randint(max(0, i - 6), i, (1,), generator=g)) for i in range(1, nodes)] if nodes else []


def _kv(s: Served, pool, visible=None):
    return _uocr().PagedChunk(kv_blocks=pool, lookup_table=s.table.to(DEV), cache_lengths=_on(s.cached),
                              chunk_offsets=s.offsets.to(DEV), attend_max=s.attend_max, visible=visible)


def _seen(s: Served, bits: list[list[int]]):
    return lambda i, j: list(range(s.cached[i])) + [s.cached[i] + b for b in range(min(64, s.chunks[i]))
                                                    if bits[i][j] >> b & 1]


# ------------------------------------------------------------------------------------------ masks


@pytest.mark.parametrize("sizes", [[1], [2], [15], [61], [64], [3, 0, 64, 1, 17], [65], [130, 2], list(range(70))])
def test_masks(sizes) -> None:
    u = _uocr()
    g = torch.Generator().manual_seed(sum(sizes))
    trees = [_tree(g, n) for n in sizes]
    want = []
    for p in trees:
        first = masks_of(p[:64])
        more = [first[x] if 0 <= x < 64 else 0 for x in p[64:]]
        want += [signed(b) for b in first + more]
    offsets = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    got = u.draft_masks(_on([x for p in trees for x in p]), _on(offsets))
    assert got.dtype == torch.int64 and got.tolist() == want


def test_masks_of_chains_and_of_parents_that_are_none() -> None:
    u = _uocr()
    assert u.draft_masks(_on(list(range(-1, 63))), _on([0, 64])).tolist() == \
        [signed((1 << i + 1) - 1) for i in range(64)]
    # a root with a parent, nodes whose parent is themselves, behind them, or no place at all
    assert u.draft_masks(_on([3, 1, 5, -7, 2, 1 << 30]), _on([0, 6])).tolist() == [1, 2, 4, 8, 4 | 16, 32]
    out = torch.full((4,), 9, dtype=torch.int64, device=DEV)
    assert u.draft_masks(_on([5, -1, 0, 5]), _on([1, 3]), out=out) is out
    assert out.tolist() == [9, 1, 3, 9]
    assert u.draft_masks(_on([]), _on([0, 0])).shape == (0,)


# ------------------------------------------------------------------------------------------ attention


SHAPES = [
    ([1], [0]), ([1], [1]), ([2], [127]), ([5], [123]), ([15], [300]), ([31], [1]), ([32], [96]), ([33], [95]),
    ([61], [0]), ([64], [64]), ([63], [70]), ([64], [2900]), ([4, 0, 9, 1], [300, 0, 0, 128]),
    ([61, 1, 40], [0, 999, 57]), ([3, 2, 1, 0] * 20, [0, 130, 64, 7] * 20),
]


@pytest.mark.parametrize(("chunks", "cached"), SHAPES, ids=lambda v: "-".join(map(str, v[:4])))
@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
@pytest.mark.parametrize("form", ["plain", "qkv"])
def test_trees_match_the_formula(chunks, cached, int8, form) -> None:
    u = _uocr()
    s = Served(len(chunks) + sum(chunks) + sum(cached), chunks, cached, int8=int8, heads=2)
    trees = [_tree(s.g, n) for n in chunks]
    bits = [masks_of(p) for p in trees]
    visible = u.draft_masks(_on([x for p in trees for x in p]), s.offsets.to(DEV))
    pool = s.pool.to(DEV)
    q, k, v = s.qkv.unbind(1)
    if form == "qkv":
        cos, sin = (torch.from_numpy(x).to(DEV) for x in u.rope_tables(head_dim=D, seq_len=s.attend_max, theta=10000.0))
        pos = [0] * s.tokens
        for i, t, j in s.each():  # a node's position is its depth
            pos[t] = s.cached[i] + bin(bits[i][j]).count("1") - 1
        got = u.paged_chunk_attention_qkv(s.qkv.view(s.tokens, -1).to(DEV), _on(pos), cos, sin, heads=2,
                                          kv=_kv(s, pool, visible), layer_idx=1, scale=SCALE)
        q, k, _ = (None if x is None else x.cpu() for x in u.rope(q.to(DEV), k.to(DEV), _on(pos), cos, sin))
    else:
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_kv(s, pool, visible), layer_idx=1, scale=SCALE)
    want = s.stored(1, k, v)
    assert torch.equal(pool.cpu().view(torch.int8), want.view(torch.int8)), "the pool's rows"
    assert far(got.cpu(), s.want(want, 1, q, seen=_seen(s, bits))) <= BAR


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
@pytest.mark.parametrize("heads", [1, 3, 10])
def test_any_masks(int8, heads) -> None:
    """Masks that no tree has: bits at random, of later tokens too, none at all (a row of zeros where nothing is cached),
    bits past the chunk (there is nothing), and a chunk of more than 64 tokens."""
    u = _uocr()
    chunks, cached = [40, 3, 90, 2], [0, 200, 33, 0]
    s = Served(heads, chunks, cached, int8=int8, heads=heads, lead=1, tail=2)
    bits = [[int(torch.randint(0, 1 << 62, (1,), generator=s.g)) << 2 | int(torch.randint(0, 4, (1,), generator=s.g))
             for _ in range(c)] for c in chunks]
    bits[0][3] = bits[0][39] = bits[1][1] = bits[2][70] = 0
    bits[3] = [0, 0]
    words = [0] + [signed(b) for row in bits for b in row] + [0, 0]
    pool = s.pool.to(DEV)
    q, k, v = s.qkv.unbind(1)
    out = torch.full((s.tokens, heads, D), 5.0, device=DEV)
    u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_kv(s, pool, _on(words, torch.int64)), layer_idx=0,
                            scale=SCALE, out=out)
    want = s.stored(0, k, v)
    assert torch.equal(pool.cpu().view(torch.int8), want.view(torch.int8))
    mine = slice(1, s.tokens - 2)
    assert far(out[mine].cpu(), s.want(want, 0, q, seen=_seen(s, bits))[mine]) <= BAR
    assert bool((out[0] == 5).all()) and bool((out[-2:] == 5).all())
    assert bool((out[1 + 3] == 0).all()) and bool((out[-4:-2] == 0).all())


def test_a_chain_is_a_chunk() -> None:
    u = _uocr()
    s = Served(21, [50, 7], [300, 129], int8=False, heads=10)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    pools = s.pool.to(DEV), s.pool.to(DEV)
    visible = u.draft_masks(_on(list(range(-1, 49)) + list(range(-1, 6))), s.offsets.to(DEV))
    a = u.paged_chunk_attention(q, k, v, kv=_kv(s, pools[0], visible), layer_idx=1, scale=SCALE)
    b = u.paged_chunk_attention(q, k, v, kv=_kv(s, pools[1]), layer_idx=1, scale=SCALE)
    assert torch.equal(*pools) and far(a.cpu(), b.double().cpu()) <= 2 * BAR


def test_a_chain_is_a_chunk_over_int8() -> None:
    u = _uocr()
    s = Served(22, [50, 7], [300, 129], heads=10)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    pools = s.pool.to(DEV), s.pool.to(DEV)
    visible = u.draft_masks(_on(list(range(-1, 49)) + list(range(-1, 6))), s.offsets.to(DEV))
    a = u.paged_chunk_attention(q, k, v, kv=_kv(s, pools[0], visible), layer_idx=1, scale=SCALE)
    b = u.paged_chunk_attention(q, k, v, kv=_kv(s, pools[1]), layer_idx=1, scale=SCALE)
    assert torch.equal(*pools) and far(a.cpu(), b.double().cpu()) <= 2 * BAR


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
def test_other_branches_and_unused_rows_leave_nothing(int8) -> None:
    """A branch of NaN and infinities, and such rows behind the chunk and in other pages, change nothing of the others;
    what attends them is NaN."""
    u = _uocr()
    s = Served(23, [40], [100], int8=int8, heads=2)
    parents = [-1] + [0 if i % 2 else max(0, i - 2) for i in range(1, 40)]
    bad = [i for i in range(40) if masks_of(parents)[i] >> 6 & 1]  # below node 6
    for i in bad:
        s.qkv[i, 1] = float("inf")
        s.qkv[i, 2, :, ::2] = float("nan")
    if not int8:
        used = {s.place(0, r) for r in range(140)}
        for p in range(s.pool.shape[0]):
            for r in range(128):
                if (p, r) not in used:
                    s.pool[p, :, :, r] = float("nan")
    bits = [masks_of(parents)]
    pool = s.pool.to(DEV)
    q, k, v = s.qkv.unbind(1)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=_kv(s, pool, _on([signed(b) for b in bits[0]],
                                                                                      torch.int64)),
                                  layer_idx=1, scale=SCALE).cpu()
    fine = [i for i in range(40) if i not in bad]
    clean = Served(23, [40], [100], int8=int8, heads=2)
    clean.qkv[bad] = 0.0
    _, ck, cv = clean.qkv.unbind(1)
    want = clean.want(clean.stored(1, ck, cv), 1, q, seen=_seen(clean, bits))
    assert far(got[fine], want[fine]) <= BAR
    assert len(bad) > 2 and bool(got[bad].isnan().all())


def test_values_of_very_different_sizes() -> None:
    """Rows whose keys and values are 2^40 times the others': float32's range, and nothing shared between elements."""
    u = _uocr()
    s = Served(24, [20], [150], int8=False, heads=2)
    s.pool[int(s.table[0, 0]), 1, 1, 7] *= 2.0 ** 40  # a value that every token attends: outputs are about its size
    s.qkv[5, 2] *= 2.0 ** -40
    s.qkv[6, 0, :, 3] = 2.0 ** 20  # a query element beside which the others count: the keys' are zero there
    s.pool[:, 0, :, :, :, 3] = 0.0
    s.qkv[:, 1, :, 3] = 0.0
    bits = [masks_of([-1] + list(range(19)))]
    pool = s.pool.to(DEV)
    q, k, v = s.qkv.unbind(1)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV),
                                  kv=_kv(s, pool, _on([signed(b) for b in bits[0]], torch.int64)), layer_idx=1, scale=SCALE)
    assert far(got.cpu(), s.want(s.stored(1, k, v), 1, q, seen=_seen(s, bits))) <= BAR


def test_captured_and_replayed() -> None:
    u = _uocr()
    s = Served(25, [30, 9], [500, 3], int8=False, heads=4)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    pool, parents = s.pool.to(DEV), _on([-1] + [i // 2 for i in range(29)] + [-1] + [0] * 8)
    kv = _kv(s, pool, torch.empty(s.tokens, dtype=torch.int64, device=DEV))
    out = torch.empty_like(q)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        u.draft_masks(parents, kv.chunk_offsets, out=kv.visible)
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE, out=out)
    for first, lengths in (([0, 30, 39], [500, 3]), ([0, 39, 39], [490, 0]), ([0, 30, 39], [500, 3])):
        kv.chunk_offsets.copy_(torch.tensor(first, dtype=torch.int32))
        kv.cache_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        pool.copy_(s.pool)
        eager_pool = s.pool.to(DEV)
        masks = u.draft_masks(parents, kv.chunk_offsets)
        eager = u.paged_chunk_attention(q, k, v, kv=type(kv)(**{**vars(kv), "kv_blocks": eager_pool, "visible": masks}),
                                        layer_idx=0, scale=SCALE)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kv.visible, masks) and torch.equal(out, eager) and torch.equal(pool, eager_pool)


# ------------------------------------------------------------------------------------------ acceptance


def _walk(parents, tokens, answers) -> list[int]:
    if not parents:
        return []
    path = [0]
    while True:
        nxt = next((i for i in range(path[-1] + 1, min(64, len(parents)))
                    if parents[i] == path[-1] and tokens[i] == answers[path[-1]]), None)
        if nxt is None:
            return path
        path.append(nxt)


def _accept(s: Served, parents, tokens, answers, pool):
    """What accept_drafts gives, by walking: (counts, path, next, lengths, pool)."""
    pool = pool.clone()
    counts, following, path = [], [], [-1] * s.tokens
    for i, c in enumerate(s.chunks):
        at = int(s.offsets[i])
        p = _walk(parents[at:at + c], tokens[at:at + c], answers[at:at + c])
        counts.append(len(p))
        following.append(answers[at + p[-1]] if p else -1)
        for j, node in enumerate(p):
            path[at + j] = node
            (a, ra), (b, rb) = s.place(i, s.cached[i] + node), s.place(i, s.cached[i] + j)
            pool[b, :, :, rb] = pool[a, :, :, ra]
    return counts, path, following, [k + c for k, c in zip(s.cached, counts)], pool


@pytest.mark.parametrize(("chunks", "cached"), [
    ([1], [0]), ([2], [127]), ([15], [300]), ([64], [120]), ([0], [5]), ([61, 0, 1, 33], [0, 9, 128, 250]),
    ([90, 3], [60, 126]), ([5] * 70, list(range(100, 170))),
], ids=lambda v: "-".join(map(str, v[:4])))
@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
def test_accepted_paths(chunks, cached, int8) -> None:
    u = _uocr()
    s = Served(sum(chunks), chunks, cached, int8=int8, heads=3, layers=3, lead=2, tail=1)
    parents, tokens, answers = [7, 7], [1, 1], [1, 1]
    for n in chunks:
        p = _tree(s.g, n)
        tok = torch.randint(0, 5, (n,), generator=s.g).tolist()  # twins among the siblings
        ans = torch.randint(0, 5, (n,), generator=s.g).tolist()
        for i in range(1, n):
            if i % 4:
                ans[p[i]] = tok[i]
        parents, tokens, answers = parents + p, tokens + tok, answers + ans
    parents, tokens, answers = parents + [0], tokens + [1], answers + [1]
    want = _accept(s, parents, tokens, answers, s.pool)
    pool = s.pool.to(DEV)
    kv = _kv(s, pool)
    got = u.accept_drafts(kv, _on(parents), _on(tokens), _on(answers))
    for x, y in zip(got, want):
        assert x.tolist() == y
    assert torch.equal(pool.cpu().view(torch.int8), want[4].view(torch.int8))
    assert kv.cache_lengths.tolist() == s.cached


def test_long_paths_and_rejections() -> None:
    """A whole chain of 64, every second node of a chain, and a root whose answer nobody drafted; rows that move across
    pages."""
    u = _uocr()
    s = Served(31, [64, 64, 64], [100, 100, 127], heads=1, layers=2, int8=False)
    chain = list(range(-1, 63))
    comb = [-1, 0] + [i - 2 for i in range(2, 64)]  # 0 <- 2 <- 4 ..., 1 <- 3 <- 5 ...
    parents = chain + comb + chain
    tokens = list(range(64)) + [i % 2 for i in range(64)] + [3] * 64
    answers = [i + 1 for i in range(64)] + [0] * 64 + [4] * 64
    want = _accept(s, parents, tokens, answers, s.pool)
    assert want[0] == [64, 32, 1]
    pool = s.pool.to(DEV)
    got = u.accept_drafts(_kv(s, pool), _on(parents), _on(tokens), _on(answers))
    for x, y in zip(got, want):
        assert x.tolist() == y
    assert torch.equal(pool.cpu(), want[4])


def test_rows_past_the_table_do_not_move() -> None:
    u = _uocr()
    s = Served(32, [3], [254], heads=1, layers=1, int8=False)
    s.table = s.table[:, :2].contiguous()  # rows 254 and 255 exist, 256 does not
    pool = s.pool.to(DEV)
    counts, path, nxt, lengths = u.accept_drafts(_kv(s, pool), _on([-1, 0, 0]), _on([0, 1, 2]), _on([2, 9, 7]))
    assert (counts.tolist(), path.tolist(), nxt.tolist(), lengths.tolist()) == ([2], [0, 2, -1], [7], [256])
    assert torch.equal(pool.cpu(), s.pool)


def test_unsigned_tables_and_no_tokens() -> None:
    u = _uocr()
    s = Served(33, [4], [10], heads=1)
    kv = _kv(s, s.pool.to(DEV))
    kv = type(kv)(**{**vars(kv), "cache_lengths": kv.cache_lengths.view(torch.uint32),
                     "lookup_table": kv.lookup_table.view(torch.uint32)})
    *_, lengths = u.accept_drafts(kv, _on([-1, 0, 1, 2]), _on([0, 1, 2, 3]), _on([1, 2, 9, 9]))
    assert lengths.dtype == torch.uint32 and lengths.view(torch.int32).tolist() == [13]
    s = Served(34, [0, 0], [10, 0], heads=1)
    counts, path, nxt, lengths = u.accept_drafts(_kv(s, s.pool.to(DEV)), _on([]), _on([]), _on([]))
    assert (counts.tolist(), path.tolist(), nxt.tolist(), lengths.tolist()) == ([0, 0], [], [-1, -1], [10, 0])
