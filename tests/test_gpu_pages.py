"""GPU tests of the page operators (``copy_pages``, ``fork_pages``, ``resize_pages``, ``compact_pages``) against the same
steps on lists, one page at a time.  Tables are whole numbers and rows are moved, not computed: everything is equal to
the bit."""

from __future__ import annotations

import random

import pytest
import torch

from _gpu import DEV

pytestmark = pytest.mark.gpu


def _uocr():
    import uocr_moe

    return uocr_moe


def _ints(values, shape=None):
    x = torch.tensor(values, dtype=torch.int32, device=DEV)
    return x if shape is None else x.view(shape)


def _same_bits(a, b) -> bool:
    return torch.equal(a.cpu().contiguous().view(torch.int32), b.cpu().contiguous().view(torch.int32))


def _pool(seed, pages, *, layers=2, page_size=8, heads=1, head_dim=4):
    g = torch.Generator().manual_seed(seed)
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (pages, 2, layers, page_size, heads, head_dim), generator=g,
                         dtype=torch.int64).to(torch.int32)
    return bits.view(torch.float32)  # any bits, NaN among them


# ------------------------------------------------------------------------------ the steps on lists


def _need(length, page_size, cols):
    return min(cols, max(0, -(-length // page_size)))


def copied(pool, src, dst, rows=None):
    pool = pool.view(torch.int32).clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        if 0 <= a < pool.shape[0] and 0 <= b < pool.shape[0]:
            k = pool.shape[3] if rows is None else max(0, min(pool.shape[3], rows[i]))
            pool[b, :, :, :k] = pool[a, :, :, :k].clone()
    return pool.view(torch.float32)


def resized(counts, table, lengths, page_size):
    counts, table = list(counts), [list(r) for r in table]
    null = len(counts) - 1
    for row, length in zip(table, lengths):
        for c, page in enumerate(row):
            if not 0 <= page < null:
                row[c] = null
            elif c >= _need(length, page_size, len(row)):
                counts[page] -= counts[page] > 0
                row[c] = null
    free, missing = [p for p in range(null) if counts[p] <= 0], 0
    for row, length in zip(table, lengths):
        for c in range(_need(length, page_size, len(row))):
            if row[c] == null:
                if free:
                    row[c] = free.pop(0)
                    counts[row[c]] = 1
                else:
                    missing += 1
    return table, counts, missing


def forked(pool, counts, table, parents, children, lengths, shared):
    null, page_size = len(counts) - 1, pool.shape[3]
    bits = pool.view(torch.int32).clone()
    new_counts, new_table = list(counts), [list(r) for r in table]
    free, missing = [p for p in range(null) if counts[p] <= 0], 0
    last = {c: i for i, c in enumerate(children)}
    pairs = [(i, p, c) for i, (p, c) in enumerate(zip(parents, children))
             if 0 <= p < len(table) and 0 <= c < len(table) and last[c] == i and p != c]
    for i, p, c in pairs:
        for col, page in enumerate(table[p]):
            new_table[c][col] = null
            if not 0 <= page < null or col >= _need(lengths[i], page_size, len(table[p])):
                continue
            if col < max(shared[i], 0) // page_size:
                new_table[c][col] = page
                new_counts[page] += 1
            elif free:
                fresh = free.pop(0)
                k = min(page_size, lengths[i] - col * page_size)
                bits[fresh, :, :, :k] = pool.view(torch.int32)[page, :, :, :k]
                new_table[c][col] = fresh
                new_counts[fresh] = 1
            else:
                missing += 1
    for i, p, c in pairs:
        for page in table[c]:
            if 0 <= page < null:
                new_counts[page] -= new_counts[page] > 0
    return bits.view(torch.float32), new_table, new_counts, missing


def compacted(pool, counts, table):
    null = len(counts) - 1
    bits = pool.view(torch.int32).clone()
    live = [p for p in range(null) if counts[p] > 0]
    holes = [p for p in range(len(live)) if counts[p] <= 0]
    remap = [p if counts[p] > 0 else -1 for p in range(null)] + [null]
    counts = list(counts)
    for p in live:
        if p >= len(live):
            remap[p] = holes.pop(0)
            bits[remap[p]] = bits[p]
            counts[remap[p]], counts[p] = counts[p], 0
    table = [[null if not 0 <= x < null or remap[x] < 0 else remap[x] for x in row] for row in table]
    return bits.view(torch.float32), table, counts, remap


def _scene(seed, requests, cols, pages, *, share=True):
    """Random tables that agree with their counts: rows with gaps, shared pages, free pages between."""
    r = random.Random(seed)
    null = pages - 1
    free = list(range(null))
    r.shuffle(free)
    counts, table = [0] * pages, []
    for _ in range(requests):
        row, held = [null] * cols, r.randint(0, cols)
        if share and table and r.random() < 0.4:
            for c, page in enumerate(r.choice(table)[:held]):
                if page != null:
                    row[c] = page
                    counts[page] += 1
        for c in range(held):
            if row[c] == null and free and r.random() < 0.9:
                row[c] = free.pop()
                counts[row[c]] += 1
        table.append(row)
    return table, counts


# ------------------------------------------------------------------------------ copies


@pytest.mark.parametrize(("layers", "page_size", "heads", "head_dim"), [(2, 8, 1, 4), (1, 1, 1, 4), (3, 128, 3, 20),
                                                                        (2, 128, 10, 128)])
@pytest.mark.parametrize("partial", [False, True])
def test_copy(layers, page_size, heads, head_dim, partial) -> None:
    u = _uocr()
    pool = _pool(layers, 11, layers=layers, page_size=page_size, heads=heads, head_dim=head_dim)
    src, dst = [3, 0, 10, 7], [5, 1, 2, 9]
    rows = [page_size, 1, page_size // 2, 0] if partial else None
    gpu = pool.to(DEV)
    got = u.copy_pages(gpu, _ints(src), _ints(dst), rows=None if rows is None else _ints(rows))
    assert got is gpu and _same_bits(gpu, copied(pool, src, dst, rows))


@pytest.mark.parametrize(("src", "dst"), [
    ([0, 1, 2, 3], [1, 2, 3, 4]),            # a chain: page 0 goes all the way
    ([4, 3, 2, 1], [5, 4, 3, 2]),            # a shift
    ([0, 1, 0, 2, 1], [3, 3, 3, 3, 3]),      # one destination again and again: the last counts
    ([0, 1, 9], [9, 0, 1]),                  # a swap by way of a third
    ([2, 2, 2, 2, 2, 2, 2], [2, 3, 4, 5, 6, 7, 8]),
    ([-1, 3, 11, 2, 2 ** 31 - 1, 4], [0, -5, 1, 11, 2, 5]),  # ids outside the pool are skipped
    ([1], [1]), ([], []),
    (list(range(10)) * 7, [(3 * i + i // 10) % 11 for i in range(70)]),
])
def test_copies_happen_in_order(src, dst) -> None:
    u = _uocr()
    pool = _pool(len(src), 11, layers=2, page_size=16, heads=2, head_dim=8)
    for rows in (None, [(5 * i) % 19 - 1 for i in range(len(src))]):
        gpu = pool.to(DEV)
        u.copy_pages(gpu, _ints(src), _ints(dst), rows=None if rows is None else _ints(rows))
        assert _same_bits(gpu, copied(pool, src, dst, rows)), rows


# ------------------------------------------------------------------------------ resizes


@pytest.mark.parametrize(("seed", "requests", "cols", "pages"), [
    (1, 1, 1, 2), (2, 1, 5, 9), (3, 7, 3, 40), (4, 64, 6, 200), (5, 200, 17, 3000), (6, 40, 40, 1100), (7, 5, 4, 1),
    (8, 3000, 2, 4000), (9, 5000, 1, 6000), (10, 300, 60, 16384), (11, 90, 190, 16385), (12, 4100, 5, 21000),
    (13, 128, 16, 2048), (14, 683, 3, 2048), (15, 50, 30, 2049)])
@pytest.mark.parametrize("in_place", [False, True])
def test_resize(seed, requests, cols, pages, in_place) -> None:
    u = _uocr()
    r = random.Random(seed)
    table, counts = _scene(seed, requests, cols, pages)
    lengths = [r.randint(-3, 8 * cols + 9) for _ in range(requests)]
    want_table, want_counts, want_missing = resized(counts, table, lengths, 8)
    gt, gc = _ints(table, (requests, cols)), _ints(counts)
    kept = gt.clone(), gc.clone()
    outs = {"out_lookup": gt, "out_ref_counts": gc} if in_place else {}
    new_table, new_counts, missing = u.resize_pages(gc, gt, _ints(lengths), page_size=8, **outs)
    assert new_table.tolist() == want_table and new_counts.tolist() == want_counts
    assert missing.tolist() == [want_missing]
    if in_place:
        assert new_table is gt and new_counts is gc
    else:
        assert torch.equal(gt, kept[0]) and torch.equal(gc, kept[1])


@pytest.mark.parametrize("output", ["out_lookup", "out_ref_counts"])
def test_one_table_in_place(output) -> None:
    u = _uocr()
    table, counts = _scene(3, 9, 4, 40)
    pool = _pool(3, 40)
    lists = [0, 1, 2], [5, 6, 7], [32, 9, 17], [8, 0, 16]
    lengths = [8 * (i % 5) for i in range(9)]
    for name in ("resize", "fork", "compact"):
        gpu, gt, gc = pool.to(DEV), _ints(table), _ints(counts)
        out = {output: gt if output == "out_lookup" else gc}
        if name == "resize":
            got, want = u.resize_pages(gc, gt, _ints(lengths), page_size=8, **out), resized(counts, table, lengths, 8)
        elif name == "fork":
            got = u.fork_pages(gpu, gc, gt, *map(_ints, lists), **out)
            want = forked(pool, counts, table, *lists)[1:]
        else:
            got, want = u.compact_pages(gpu, gc, gt, **out), compacted(pool, counts, table)[1:]
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1], name
        kept = (gc, counts) if output == "out_lookup" else (gt, table)
        assert kept[0].tolist() == kept[1], name


def test_tables_without_requests_and_forks_without_pairs() -> None:
    u = _uocr()
    none, counts = torch.zeros(0, 3, dtype=torch.int32, device=DEV), [0, 2, 0, 1, 0]
    pool = _pool(4, 5)
    lookup, got, missing = u.resize_pages(_ints(counts), none, none[:, 0].contiguous(), page_size=8)
    assert lookup.shape == (0, 3) and got.tolist() == counts and missing.tolist() == [0]
    gpu, table = pool.to(DEV), [[1, 3, 4]]
    empty = torch.zeros(0, dtype=torch.int32, device=DEV)
    lookup, got, missing = u.fork_pages(gpu, _ints(counts), _ints(table), empty, empty, empty, empty)
    assert lookup.tolist() == table and got.tolist() == counts and missing.tolist() == [0] and _same_bits(gpu, pool)
    lookup, got, remap = u.compact_pages(gpu, _ints(counts), none)
    assert got.tolist() == [1, 2, 0, 0, 0] and remap.tolist() == [-1, 1, -1, 0, 4]
    assert _same_bits(gpu[:2], pool[[3, 1]])


def test_resize_runs_out_and_recovers() -> None:
    """Too few free pages: the first entries in (request, column) order get them; released pages are free at once; the
    lowest page goes first."""
    u = _uocr()
    null = 6
    table, counts = _ints([[4, 1, null], [null, null, null], [2, null, null]]), _ints([0, 1, 1, 0, 1, 0, 9])
    t1, c1, m1 = u.resize_pages(counts, table, _ints([0, 24, 24]), page_size=8)
    assert t1.tolist() == [[6, 6, 6], [0, 1, 3], [2, 4, 5]] and m1.tolist() == [0]
    assert c1.tolist() == [1, 1, 1, 1, 1, 1, 9]
    t2, c2, m2 = u.resize_pages(c1, t1, _ints([17, 24, 24]), page_size=8)
    assert t2.tolist() == t1.tolist() and c2.tolist() == c1.tolist() and m2.tolist() == [3]
    t3, c3, m3 = u.resize_pages(c2, t2, _ints([9, 1, 24]), page_size=8)
    assert t3.tolist() == [[1, 3, 6], [0, 6, 6], [2, 4, 5]] and m3.tolist() == [0]


def test_entries_and_counts_that_no_call_would_write() -> None:
    """Entries outside the pool (negative, past it) are unset; counts below zero are free and never fall further."""
    u = _uocr()
    table, counts = [[-1, 3, 2 ** 31 - 1], [5, 0, 4]], [0, -7, 2, 1, 0, 3]
    for lengths in ([0, 0], [24, 8], [1, 24]):
        want = resized(counts, table, lengths, 8)
        got = u.resize_pages(_ints(counts), _ints(table), _ints(lengths), page_size=8)
        assert (got[0].tolist(), got[1].tolist(), got[2].item()) == want, lengths


# ------------------------------------------------------------------------------ forks


def _check_fork(pool, counts, table, parents, children, lengths, shared, in_place=False):
    u = _uocr()
    want_pool, want_table, want_counts, want_missing = forked(pool, counts, table, parents, children, lengths, shared)
    gpu, gt, gc = pool.to(DEV), _ints(table), _ints(counts)
    outs = {"out_lookup": gt, "out_ref_counts": gc} if in_place else {}
    got = u.fork_pages(gpu, gc, gt, *(_ints(x) for x in (parents, children, lengths, shared)), **outs)
    assert got[0].tolist() == want_table and got[1].tolist() == want_counts and got[2].item() == want_missing
    assert _same_bits(gpu, want_pool)
    if not in_place:
        assert gt.tolist() == table and gc.tolist() == counts


@pytest.mark.parametrize("seed", range(10))
@pytest.mark.parametrize("in_place", [False, True])
def test_fork(seed, in_place) -> None:
    r = random.Random(100 + seed)
    requests, cols = r.randint(1, 30), r.randint(1, 9)
    pages = r.randint(2, 2 * requests * cols + 2)
    table, counts = _scene(seed, requests, cols, pages)
    k = r.randint(1, requests)
    # rows outside the table, one child twice and a row with itself among them
    parents = [r.randint(-1, requests) for _ in range(k)]
    children = [r.randint(-1, requests) for _ in range(k)]
    lengths = [r.randint(-1, 8 * cols + 3) for _ in range(k)]
    shared = [r.randint(-9, 8 * cols) for _ in range(k)]
    _check_fork(_pool(seed, pages), counts, table, parents, children, lengths, shared, in_place)


@pytest.mark.parametrize(("requests", "cols", "pages"), [
    (4096, 2, 9000), (4097, 2, 9000), (70, 300, 16384), (60, 250, 16385), (90, 400, 30000), (64, 32, 2048), (65, 32, 2048)])
@pytest.mark.parametrize("in_place", [False, True])
def test_fork_of_many(requests, cols, pages, in_place) -> None:
    r = random.Random(requests + cols)
    table, counts = _scene(requests, requests, cols, pages)
    parents = [r.randrange(requests) for _ in range(requests)]
    children = [r.randrange(requests) for _ in range(requests)]
    lengths = [r.randint(0, 2 * cols) for _ in range(requests)]
    shared = [r.randint(0, 2 * cols) for _ in range(requests)]
    _check_fork(_pool(1, pages, layers=1, page_size=2), counts, table, parents, children, lengths, shared, in_place)


def test_fork_swaps_and_repeats() -> None:
    """A swap takes each parent's row as it was; the last of three pairs with one child counts; a row with itself stays
    (as the last pair, it undoes those before)."""
    table, counts = [[0, 1, 9], [2, 9, 9], [3, 4, 5]], [1, 1, 1, 1, 1, 1, 0, 0, 0, 4]
    pool = _pool(1, 10)
    _check_fork(pool, counts, table, [0, 1], [1, 0], [16, 8], [8, 0])
    _check_fork(pool, counts, table, [0, 1, 2], [1, 0, 1], [16, 8, 20], [8, 0, 16])
    _check_fork(pool, counts, table, [0, 1], [1, 1], [16, 8], [8, 0])
    _check_fork(pool, counts, table, [2, 2, 2], [0, 1, 2], [24, 24, 24], [24, 24, 24])
    _check_fork(pool, counts, table, [2, 2], [0, 1], [24, 24], [0, 0])  # three pages short
    _check_fork(pool, counts, table, [], [], [], [])


def test_fork_of_the_served_decoders_pages() -> None:
    """Pages of 128 rows, 10 heads of 128, 3 layers: one prompt of 291 rows continued three ways."""
    table, counts = [[5, 2, 7, 19], [19] * 4, [11, 19, 19, 19], [19] * 4], [0] * 20
    for p in (5, 2, 7, 11):
        counts[p] = 1
    pool = torch.randn(20, 2, 3, 128, 10, 128, generator=torch.Generator().manual_seed(3))
    _check_fork(pool, counts, table, [0, 0, 0], [1, 2, 3], [345, 291, 129], [291, 291, 291])


# ------------------------------------------------------------------------------ compaction


def _check_compact(pool, counts, table, in_place=False):
    u = _uocr()
    want_pool, want_table, want_counts, remap = compacted(pool, counts, table)
    gpu, gt, gc = pool.to(DEV), _ints(table).view(len(table), -1), _ints(counts)
    outs = {"out_lookup": gt, "out_ref_counts": gc} if in_place else {}
    got = u.compact_pages(gpu, gc, gt, **outs)
    assert got[0].tolist() == want_table and got[1].tolist() == want_counts and got[2].tolist() == remap
    live = sum(c > 0 for c in counts[:-1])
    assert _same_bits(gpu[:live], want_pool[:live]) and _same_bits(gpu, want_pool)


@pytest.mark.parametrize(("seed", "requests", "cols", "pages"), [
    (1, 1, 1, 2), (2, 3, 2, 9), (3, 8, 5, 100), (4, 60, 4, 1025), (5, 60, 20, 2600), (6, 2, 3, 5000), (7, 1, 1, 1), (8, 40, 400, 16384),
    (9, 500, 34, 16385), (10, 7, 5000, 40000),
    (11, 256, 8, 2048), (12, 64, 32, 2049)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(seed, requests, cols, pages, in_place) -> None:
    table, counts = _scene(seed, requests, cols, pages)
    _check_compact(_pool(seed, pages, layers=1, page_size=2), counts, table, in_place)


def test_compact_edges() -> None:
    """Nothing in use, everything in use, a table that names free pages or none of the pool's, the null page's count."""
    pool = _pool(2, 6)
    _check_compact(pool, [0, 0, 0, 0, 0, 3], [[5, 5], [1, -1]])
    _check_compact(pool, [1, 2, 1, 1, 1, 0], [[4, 1], [1, 0]])
    _check_compact(pool, [0, -2, 0, 1, 5, 7], [[3, 4], [0, 2 ** 31 - 1]])
    _check_compact(pool, [0, 0, 0, 0, 1, 0], [[4, 5]])


def test_compact_of_the_served_decoders_pages() -> None:
    pool = torch.randn(12, 2, 2, 128, 10, 128, generator=torch.Generator().manual_seed(4))
    _check_compact(pool, [0, 1, 0, 0, 2, 0, 0, 1, 0, 1, 1, 0], [[1, 4, 10], [7, 4, 9]])


# ------------------------------------------------------------------------------ all of them


def test_uint32_tables_views_and_refusals() -> None:
    u = _uocr()
    table, counts = _scene(9, 6, 4, 60)
    pool = _pool(9, 60)
    lengths = [31, 0, 9, 16, 1, 32]
    want = resized(counts, table, lengths, 8)
    wide = torch.zeros(6, 9, dtype=torch.int32, device=DEV)
    wide[:, 3:7] = _ints(table)
    got = u.resize_pages(_ints(counts), wide[:, 3:7], _ints(lengths), page_size=8)  # a strided view is packed
    assert got[0].tolist() == want[0]
    u32 = u.resize_pages(_ints(counts), _ints(table).view(torch.uint32), _ints(lengths), page_size=8)
    assert u32[0].dtype == torch.uint32 and u32[0].view(torch.int32).tolist() == want[0]
    with pytest.raises(ValueError, match="must be contiguous"):
        u.resize_pages(_ints(counts), wide[:, 3:7], _ints(lengths), page_size=8, out_lookup=wide[:, 3:7])
    with pytest.raises(ValueError, match="5 lengths for 6 requests"):
        u.resize_pages(_ints(counts), _ints(table), _ints(lengths[:5]), page_size=8)
    with pytest.raises(ValueError, match="ref_counts is for 59 pages, the pool has 60"):
        u.compact_pages(pool.to(DEV), _ints(counts[:59]), _ints(table))
    with pytest.raises(ValueError, match="must have one length"):
        u.fork_pages(pool.to(DEV), _ints(counts), _ints(table), _ints([0]), _ints([1, 2]), _ints([8]), _ints([0]))
    with pytest.raises(ValueError, match="must have one length"):
        u.copy_pages(pool.to(DEV), _ints([0]), _ints([1, 2]))
    flat = torch.zeros(60 + 24, dtype=torch.int32, device=DEV)
    with pytest.raises(u.UocrError, match="an output must be its input or not overlap an input"):
        u.resize_pages(flat[:60], _ints(table), _ints(lengths), page_size=8, out_ref_counts=flat[8:68])


def test_graphs_replay_the_tables_of_their_time() -> None:
    """A captured resize, fork and compaction over tables in place: each replay goes on from the last one's tables."""
    u = _uocr()
    pool = _pool(11, 40)
    table, counts = _scene(11, 6, 4, 40, share=False)
    lengths = [9, 20, 0, 32, 7, 12]
    parents, children, shared = [0, 1, 3], [2, 4, 5], [8, 0, 16]
    gt, gc, gpu = _ints(table), _ints(counts), pool.to(DEV)
    lists = [_ints(x) for x in (parents, children, [9, 20, 30], shared)]
    glen = _ints(lengths)

    def step():
        u.resize_pages(gc, gt, glen, page_size=8, out_ref_counts=gc, out_lookup=gt)
        u.fork_pages(gpu, gc, gt, *lists, out_ref_counts=gc, out_lookup=gt)
        u.compact_pages(gpu, gc, gt, out_ref_counts=gc, out_lookup=gt)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(4):
        table, counts, _ = resized(counts, table, lengths, 8)
        pool, table, counts, _ = forked(pool, counts, table, parents, children, [9, 20, 30], shared)
        pool, table, counts, _ = compacted(pool, counts, table)
        graph.replay() if i != 2 else step()
        torch.cuda.synchronize()
        assert gt.tolist() == table and gc.tolist() == counts, i
        live = sum(c > 0 for c in counts[:-1])
        assert _same_bits(gpu[:live], pool[:live]), i


def test_a_served_cache_from_prompts_to_the_last_answer() -> None:
    """The operators as a serving loop runs them, against each request's rows kept as plain lists: prompts, a fork into
    three samples, decode steps, a further chunk, a request that ends, compaction, a new prompt, decode again."""
    u = _uocr()
    heads, d, page, layers, cols, rows = 2, 128, 128, 2, 4, 5
    pages = 17
    g = torch.Generator(device=DEV).manual_seed(5)
    pool = torch.randn(pages, 2, layers, page, heads, d, generator=g, device=DEV)
    table = torch.full((rows, cols), pages - 1, dtype=torch.int32, device=DEV)
    counts = torch.zeros(pages, dtype=torch.int32, device=DEV)
    held = [torch.zeros(0, 2, layers, heads, d, device=DEV) for _ in range(rows)]

    def attend(q, row, layer, upto):
        k, v = held[row][:upto, 0, layer].double(), held[row][:upto, 1, layer].double()
        w = torch.softmax((q.double() * k).sum(-1).T * d ** -0.5, dim=1)  # [heads, upto]
        return (w.T[..., None] * v).sum(0)

    def chunk(lengths):
        """A chunk of lengths[r] new tokens of each request, all layers."""
        nonlocal table, counts
        before = [len(h) for h in held]
        total = sum(lengths)
        qkv = torch.randn(layers, total, 3, heads, d, generator=g, device=DEV)
        table, counts, missing = u.resize_pages(counts, table, _ints([b + n if n or b else 0
                                                                      for b, n in zip(before, lengths)]),
                                                page_size=page)
        assert missing.item() == 0
        offsets = [sum(lengths[:i]) for i in range(rows + 1)]
        for r in range(rows):
            part = qkv[:, offsets[r]:offsets[r + 1]]
            held[r] = torch.cat([held[r], part[:, :, 1:].permute(1, 2, 0, 3, 4)])
        kv = u.PagedChunk(pool, table, _ints(before), _ints(offsets), max(b + n for b, n in zip(before, lengths)))
        for layer in range(layers):
            q, k, v = qkv[layer].unbind(1)
            out = u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=layer, scale=d ** -0.5)
            for r in range(rows):
                for i in range(0, lengths[r], 7):
                    want = attend(q[offsets[r] + i], r, layer, before[r] + i + 1)
                    err = (out[offsets[r] + i].double() - want).abs().max() / want.abs().max()
                    assert err <= 1e-5, (r, i, layer, float(err))

    def decode(which):
        """One token of each of the requests `which`."""
        nonlocal table, counts
        lengths = [len(h) + (r in which) for r, h in enumerate(held)]
        table, counts, missing = u.resize_pages(counts, table, _ints(lengths), page_size=page)
        assert missing.item() == 0
        at = _ints([len(held[r]) for r in which])
        qkv = torch.randn(layers, len(which), 3, heads, d, generator=g, device=DEV)
        for i, r in enumerate(which):
            held[r] = torch.cat([held[r], qkv[:, i, 1:].transpose(0, 1)[None]])
        kv = u.PagedKv(pool, table[torch.tensor(which, device=DEV)], at, max(lengths[r] for r in which), at)
        for layer in range(layers):
            out = u.paged_decode_attention(*qkv[layer].unbind(1), kv=kv, layer_idx=layer, scale=d ** -0.5)
            for i, r in enumerate(which):
                want = attend(qkv[layer, i, 0], r, layer, len(held[r]))
                assert (out[i].double() - want).abs().max() <= 1e-5 * want.abs().max(), (r, layer)

    chunk([291, 0, 0, 40, 0])
    length = len(held[0])
    table, counts, missing = u.fork_pages(pool, counts, table, _ints([0, 0]), _ints([1, 2]), _ints([length] * 2),
                                          _ints([length] * 2))
    assert missing.item() == 0
    held[1], held[2] = held[0].clone(), held[0].clone()
    assert counts[table[0, :2].long()].tolist() == [3, 3]
    for _ in range(3):
        decode([0, 1, 2, 3])
    chunk([0, 100, 5, 0, 0])
    held[0] = held[0][:0]  # request 0 ends; its shared pages live on
    table, counts, _ = u.resize_pages(counts, table, _ints([len(h) for h in held]), page_size=page)
    table, counts, remap = u.compact_pages(pool, counts, table)
    live = int((counts[:-1] > 0).sum())
    assert (counts[:live] > 0).all() and (remap >= 0).sum() == live + 1
    pool[live:] = float("nan")  # what is past the pages in use is nobody's
    decode([1, 2, 3])
    chunk([30, 0, 0, 0, 130])
    decode([0, 1, 2, 3, 4])
    assert int(counts[:-1].sum()) == int((table < pages - 1).sum())
