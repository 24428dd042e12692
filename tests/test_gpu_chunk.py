"""GPU tests of ``paged_chunk_attention`` / ``paged_chunk_attention_qkv`` against the formula in 64 bits.

The bar is the decode op's (1e-5 of a token's largest output, unlimited_ocr_max tests/test_kv_cache.py:427-433).
What the arithmetic gives, for operands of unit variance: a score sums 128 products; an operand held to 22 bits is
off by 2^-23 at most and a dropped product of two remainders by 2^-22, so the 128 independent errors leave about
sqrt(128) 2^-23 = 1.3e-6, and the sum's own roundings (2^-25 of partial sums near 11) as much, times the scale
128^-0.5: 2e-7 on a score and so on a weight.  The sums over the rows (at most 3000 here, running sums in 32 bits) add
sqrt(3000) 2^-25 = 1.6e-6.  So 1e-5 leaves a factor of five, and a lost term of a product (2^-11), a row too many or
too few (1 / rows) or a wrong page is far outside it.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from _gpu import DEV, n, t

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
BAR = 1e-5


def _uocr():
    import uocr_moe

    return uocr_moe


class Setup:
    """Requests with rows in a shuffled pool, and a chunk of new tokens of each (float32, on the CPU)."""

    def __init__(self, seed, chunks, cached, *, heads=2, page_size=128, layers=2, spare=2, lead=0, tail=0) -> None:
        g = torch.Generator().manual_seed(seed)
        self.chunks, self.cached, self.heads, self.page_size, self.layers = chunks, cached, heads, page_size, layers
        self.lead = lead  # token rows before the first chunk, and behind the last
        per = [-(-(c + k) // page_size) for c, k in zip(chunks, cached)]
        pages = sum(per) + spare + 1
        order = torch.randperm(pages - 1, generator=g).tolist()
        cols = max(max(per), 1) + 1
        self.table = torch.full((len(chunks), cols), pages - 1, dtype=torch.int32)
        for i, k in enumerate(per):
            self.table[i, :k] = torch.tensor(order[:k], dtype=torch.int32)
            order = order[k:]
        self.pool = torch.randn(pages, 2, layers, page_size, heads, D, generator=g)
        self.offsets = torch.tensor([lead + sum(chunks[:i]) for i in range(len(chunks) + 1)], dtype=torch.int32)
        self.tokens = lead + sum(chunks) + tail
        self.qkv = torch.randn(self.tokens, 3, heads, D, generator=g)
        self.attend_max = max(1, max(c + k for c, k in zip(chunks, cached)))

    def kv(self, pool=None):
        u = _uocr()
        return u.PagedChunk(kv_blocks=self.pool.to(DEV) if pool is None else pool, lookup_table=self.table.to(DEV),
                            cache_lengths=torch.tensor(self.cached, dtype=torch.int32, device=DEV),
                            chunk_offsets=self.offsets.to(DEV), attend_max=self.attend_max)

    def positions(self):
        p = torch.zeros(self.tokens, dtype=torch.int32)
        for i, (c, k) in enumerate(zip(self.chunks, self.cached)):
            at = int(self.offsets[i])
            p[at:at + c] = torch.arange(k, k + c, dtype=torch.int32)
        return p

    def covered(self) -> slice:
        return slice(self.lead, self.lead + sum(self.chunks))

    def history(self, i, layer, k_new, v_new):
        """Request i's keys and values [rows, heads, D], cached and new."""
        c, k, P = self.chunks[i], self.cached[i], self.page_size
        at = int(self.offsets[i])
        rows = [self.pool[int(self.table[i, r // P]), :, layer, r % P] for r in range(k)]
        old = torch.stack(rows) if rows else torch.zeros(0, 2, self.heads, D)
        return torch.cat([old[:, 0], k_new[at:at + c]]), torch.cat([old[:, 1], v_new[at:at + c]])

    def want(self, layer, q, k_new, v_new, scale=SCALE):
        """The formula in float64, [tokens, heads, D]; rows no chunk holds are zero."""
        out = torch.zeros(self.tokens, self.heads, D, dtype=torch.float64)
        for i, (c, k) in enumerate(zip(self.chunks, self.cached)):
            keys, values = (x.double() for x in self.history(i, layer, k_new, v_new))
            at = int(self.offsets[i])
            for j in range(c):
                s = torch.einsum("hd,rhd->hr", q[at + j].double(), keys[:k + j + 1]) * scale
                out[at + j] = torch.einsum("hr,rhd->hd", torch.softmax(s, dim=1), values[:k + j + 1])
        return out

    def stored(self, layer, k_new, v_new):
        """The pool with the chunks' rows in it."""
        pool = self.pool.clone()
        for i, (c, k) in enumerate(zip(self.chunks, self.cached)):
            for j in range(c):
                page, slot = int(self.table[i, (k + j) // self.page_size]), (k + j) % self.page_size
                pool[page, 0, layer, slot] = k_new[int(self.offsets[i]) + j]
                pool[page, 1, layer, slot] = v_new[int(self.offsets[i]) + j]
        return pool


def _far(got, want) -> float:
    """The largest error of a token over that token's largest output."""
    if got.numel() == 0:
        return 0.0
    err = (got.double() - want).abs().flatten(1).amax(dim=1)
    return float((err / want.abs().flatten(1).amax(dim=1)).max())


def _tables(rows):
    cos, sin = _uocr().rope_tables(head_dim=D, seq_len=rows, theta=10000.0)
    return torch.from_numpy(cos), torch.from_numpy(sin)


def _same_bits(a, b) -> bool:
    return torch.equal(a.contiguous().view(torch.int32), b.contiguous().view(torch.int32))


SHAPES = [
    ([1], [0]), ([1], [1]), ([2], [127]), ([1], [128]), ([5], [123]), ([31], [1]), ([32], [0]), ([33], [95]),
    ([64], [64]), ([65], [0]), ([127], [300]), ([129], [129]), ([291], [0]), ([300], [517]), ([7], [2900]),
    ([1, 1, 1], [0, 5, 640]), ([4, 0, 9, 1], [300, 0, 0, 128]), ([0, 3], [0, 0]), ([513, 1, 70], [0, 999, 57]),
    ([3, 2, 1, 0] * 20, [0, 130, 64, 7] * 20),
]


@pytest.mark.parametrize(("chunks", "cached"), SHAPES, ids=lambda v: "-".join(map(str, v[:4])))
@pytest.mark.parametrize("form", ["plain", "qkv"])
def test_matches_the_formula(chunks, cached, form) -> None:
    u = _uocr()
    s = Setup(len(chunks) + sum(chunks) + sum(cached), chunks, cached)
    q, k, v = s.qkv.unbind(1)
    pool, kv = s.pool.to(DEV), None
    kv = s.kv(pool)
    if form == "qkv":
        cos, sin = _tables(s.attend_max)
        pos = s.positions()
        got = u.paged_chunk_attention_qkv(s.qkv.view(s.tokens, -1).to(DEV), pos.to(DEV), cos.to(DEV), sin.to(DEV),
                                          heads=s.heads, kv=kv, layer_idx=1, scale=SCALE)
        q, k, _ = u.rope(q.to(DEV), k.to(DEV), pos.to(DEV), cos.to(DEV), sin.to(DEV))
        q, k = q.cpu(), k.cpu()
    else:
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=1, scale=SCALE)
    assert _same_bits(pool.cpu(), s.stored(1, k, v)), "the pool's rows"
    assert _far(got.cpu(), s.want(1, q, k, v)) <= BAR


@pytest.mark.parametrize(("heads", "page_size", "layers", "layer"), [(1, 128, 1, 0), (3, 256, 3, 2), (10, 384, 1, 0)])
def test_head_counts_page_sizes_and_layers(heads, page_size, layers, layer) -> None:
    u = _uocr()
    s = Setup(heads, [70, 2], [200, 390], heads=heads, page_size=page_size, layers=layers)
    q, k, v = s.qkv.unbind(1)
    pool = s.pool.to(DEV)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(pool), layer_idx=layer, scale=0.2)
    assert _far(got.cpu(), s.want(layer, q, k, v, 0.2)) <= BAR
    assert _same_bits(pool.cpu(), s.stored(layer, k, v))


@pytest.mark.parametrize("chunk", [3, 40, 150])
def test_strides_and_rows_outside_the_chunks(chunk) -> None:
    """Views of one wide projection, of unlike strides and alignments; token rows before the first chunk and behind the
    last (NaN inputs) leave out and the pool alone."""
    u = _uocr()
    s = Setup(chunk, [chunk, 2], [130, 0], lead=3, tail=5)
    s.qkv[:3] = s.qkv[3 + chunk + 2:] = math.nan
    q, k, v = s.qkv.unbind(1)
    want = s.want(0, q, k, v)[s.covered()]
    wide = torch.zeros(s.tokens, 3 * s.heads * D + 4, device=DEV)
    wide[:, 4:] = s.qkv.view(s.tokens, -1).to(DEV)
    views = wide[:, 4:].view(s.tokens, 3, s.heads, D).unbind(1)
    shifted = torch.zeros(s.tokens * s.heads * D + 1, device=DEV)[1:].view(s.tokens, s.heads, D)
    shifted.copy_(views[1])
    flipped = views[2].transpose(1, 2).contiguous().transpose(1, 2)
    for inputs in (views, (views[0], shifted, flipped)):
        out, pool = torch.full((s.tokens, s.heads, D), 7.0, device=DEV), s.pool.to(DEV)
        got = u.paged_chunk_attention(*inputs, kv=s.kv(pool), layer_idx=0, scale=SCALE, out=out)
        assert got is out
        assert _far(out[s.covered()].cpu(), want) <= BAR
        assert (out[:3] == 7.0).all() and (out[s.covered().stop:] == 7.0).all()
        assert _same_bits(pool.cpu(), s.stored(0, k, v))
    # the fused form's rows may be strided too
    cos, sin = torch.ones(1, D, device=DEV), torch.zeros(1, D, device=DEV)
    got = u.paged_chunk_attention_qkv(wide[:, 4:], torch.zeros(s.tokens, dtype=torch.int32, device=DEV), cos, sin,
                                      heads=s.heads, kv=s.kv(), layer_idx=0, scale=SCALE)
    assert _far(got[s.covered()].cpu(), want) <= BAR


@pytest.mark.parametrize(("chunk", "cached"), [(1, 200), (5, 123), (33, 20), (200, 300)])
def test_what_a_token_does_not_attend_may_hold_anything(chunk, cached) -> None:
    """NaN and infinities in the pool's other rows (the rest of the request's last page, its later pages, other pages,
    the null page, the other layer) change nothing; a new row's reach only itself and later tokens."""
    u = _uocr()
    s = Setup(chunk * 7 + cached, [chunk], [cached])
    q, k, v = s.qkv.unbind(1)
    want = s.want(1, q, k, v)
    rows = torch.zeros(s.pool.shape[0], s.page_size, dtype=torch.bool)
    for r in range(cached):
        rows[int(s.table[0, r // s.page_size]), r % s.page_size] = True
    junk = torch.tensor([math.nan, math.inf, -math.inf, 3.4e38])
    bad = junk[torch.arange(s.pool[:, :, 1].numel()) % 4].view_as(s.pool[:, :, 1])
    keep = rows[:, None, :, None, None]
    s.pool[:, :, 1] = torch.where(keep, s.pool[:, :, 1], bad)
    s.pool[:, :, 0] = math.nan
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=1, scale=SCALE).cpu()
    assert _far(got, want) <= BAR
    # the last new token's own row: earlier tokens do not see it
    for which, value in ((k, math.nan), (v, math.inf), (v, math.nan), (k, -math.inf)):
        saved = which[-1].clone()
        which[-1, :, 5] = value
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=1, scale=SCALE).cpu()
        if chunk > 1:
            assert _far(got[:-1], want[:-1]) <= BAR, (value, which is k)
        if which is v:
            assert not torch.isfinite(got[-1, :, 5]).any()
            rest = [d for d in range(D) if d != 5]
            assert _far(got[-1:, :, rest], want[-1:, :, rest]) <= BAR
        elif math.isnan(value):
            assert torch.isnan(got[-1]).all()
        which[-1] = saved


def test_a_cached_row_of_infinities_is_seen_as_the_formula_has_it() -> None:
    """An attended key whose score is -inf has the weight 0; one of +inf or NaN makes the token NaN; a value of inf is
    the output's.  Tokens of another request beside it are untouched."""
    u = _uocr()
    s = Setup(5, [40, 3], [60, 30])
    q, k, v = s.qkv.unbind(1)
    q[:, 0, 0] = q[:, 0, 0].abs() + 0.1
    page, slot = int(s.table[0, 0]), 17
    s.pool[page, 0, 1, slot, 0, 0] = -math.inf  # head 0: scores of -inf
    s.pool[page, 1, 1, slot, 1, 9] = math.inf   # head 1: a value of inf
    want = s.want(1, q, k, v)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=1, scale=SCALE).cpu()
    fine = torch.isfinite(want)
    assert not fine[:40, 1, 9].any() and int((~fine).sum()) == 40
    assert (got[:40, 1, 9] == math.inf).all()
    assert _far(torch.where(fine, got.double(), 0.0), torch.where(fine, want, 0.0)) <= BAR
    s.pool[page, 0, 1, slot, 0, 0] = math.inf
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=1, scale=SCALE).cpu()
    assert torch.isnan(got[:40, 0]).all() and _far(got[40:], want[40:]) <= BAR


@pytest.mark.parametrize("chunk", [2, 64, 140])
@pytest.mark.parametrize(("ks", "vs"), [(1e-4, 1e-5), (1e3, 1e4), (1e-12, 1e-30), (1e12, 1e25), (1e22, 1e36)])
def test_magnitudes(chunk, ks, vs) -> None:
    """Keys and values of any size in fp32's range: the queries are scaled the other way, so that the scores are of
    unit size; the error stays relative."""
    u = _uocr()
    s = Setup(chunk, [chunk], [150])
    s.pool[:, 0] *= ks
    s.pool[:, 1] *= vs
    s.qkv[:, 0] /= ks
    s.qkv[:, 1] *= ks
    s.qkv[:, 2] *= vs
    q, k, v = s.qkv.unbind(1)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=0, scale=SCALE)
    assert _far(got.cpu(), s.want(0, q, k, v)) <= BAR


@pytest.mark.parametrize("chunk", [2, 64, 140])
def test_rows_of_unlike_sizes(chunk) -> None:
    """Small and large keys and values side by side, zero rows, and denormals: an output is off by no more than 1e-5 of
    the largest weighted value that goes into it."""
    u = _uocr()
    s = Setup(chunk + 1, [chunk], [200])
    g = torch.Generator().manual_seed(chunk)
    size = 10.0 ** torch.randint(-6, 1, s.pool.shape[:4], generator=g)
    s.pool *= size[..., None, None]
    s.pool[int(s.table[0, 0]), :, 0, 40:50] = 0.0
    s.pool[int(s.table[0, 0]), :, 0, 50] = 1e-41
    q, k, v = s.qkv.unbind(1)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=0, scale=SCALE)
    assert _far(got.cpu(), s.want(0, q, k, v)) <= BAR


def test_scores_far_apart() -> None:
    """Scores of hundreds (one key takes all the weight) and a negative scale.  A score of size S is off by about
    S 2^-22, S up to 600 here: 1.4e-4 of a weight where two keys are near each other."""
    u = _uocr()
    for scale in (SCALE, -SCALE):
        s = Setup(77, [50, 1], [100, 300])
        s.qkv[:, 0] *= 20
        q, k, v = s.qkv.unbind(1)
        got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=0, scale=scale)
        assert _far(got.cpu(), s.want(0, q, k, v, scale)) <= 1.5e-4


def test_a_single_token_is_the_decode_step() -> None:
    u = _uocr()
    s = Setup(3, [1, 1, 1], [409, 0, 128], heads=10)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    a, b = s.pool.to(DEV), s.pool.to(DEV)
    kv = s.kv(a)
    got = u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE)
    step = u.PagedKv(kv_blocks=b, lookup_table=kv.lookup_table, attend_lengths=kv.cache_lengths,
                     attend_max=kv.attend_max, write_index=kv.cache_lengths)
    want = u.paged_decode_attention(q, k, v, kv=step, layer_idx=1, scale=SCALE)
    assert _far(got.cpu(), want.cpu().double()) <= 2 * BAR
    assert _same_bits(a.cpu(), b.cpu())


@pytest.mark.parametrize("cuts", [(100,), (1, 33, 130), (256, 290)])
def test_a_prompt_in_pieces_is_the_prompt(cuts) -> None:
    u = _uocr()
    s = Setup(9, [300], [0], heads=2)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    whole_pool, pool = s.pool.to(DEV), s.pool.to(DEV)
    whole = u.paged_chunk_attention(q, k, v, kv=s.kv(whole_pool), layer_idx=0, scale=SCALE).cpu()
    parts = []
    for a, b in zip((0, *cuts), (*cuts, 300)):
        kv = u.PagedChunk(kv_blocks=pool, lookup_table=s.table.to(DEV),
                          cache_lengths=torch.tensor([a], dtype=torch.int32, device=DEV),
                          chunk_offsets=torch.tensor([0, b - a], dtype=torch.int32, device=DEV), attend_max=b)
        parts.append(u.paged_chunk_attention(q[a:b], k[a:b], v[a:b], kv=kv, layer_idx=0, scale=SCALE).cpu())
    assert _same_bits(pool.cpu(), whole_pool.cpu())
    assert _far(torch.cat(parts), whole.double()) <= 2 * BAR


@pytest.mark.parametrize("chunk", [2, 200])
def test_device_metadata_is_clamped(chunk) -> None:
    """Rows past what the lookup row addresses are neither stored nor attended, nor are rows past attend_max attended;
    page ids past the pool mean the null page; offsets past the tokens end there."""
    u = _uocr()
    s = Setup(21, [chunk], [256 - 1], heads=1, layers=1, spare=0)
    s.table = s.table[:, :2].contiguous()  # 256 rows: the chunk's first token is the last that fits
    s.attend_max = 256
    q, k, v = s.qkv.unbind(1)
    pool = s.pool.to(DEV)
    kv = s.kv(pool)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=0, scale=SCALE).cpu()
    keys, values = s.history(0, 0, k[:1], v[:1])
    w = torch.softmax(torch.einsum("thd,rhd->thr", q.double(), keys.double()) * SCALE, dim=2)
    assert _far(got, torch.einsum("thr,rhd->thd", w, values.double())) <= BAR
    stored = s.pool.clone()
    stored[int(s.table[0, 1]), 0, 0, 127], stored[int(s.table[0, 1]), 1, 0, 127] = k[0], v[0]
    assert _same_bits(pool.cpu(), stored)
    # a smaller attend_max, page ids past the pool, offsets past the tokens
    null = s.pool.shape[0] - 1
    s2 = Setup(22, [chunk], [100], heads=1, layers=1)
    q, k, v = s2.qkv.unbind(1)
    null = s2.pool.shape[0] - 1
    s2.attend_max = 90
    kv = s2.kv()
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=0, scale=SCALE).cpu()
    keys, values = (x[:90].double() for x in s2.history(0, 0, k, v))
    w = torch.softmax(torch.einsum("thd,rhd->thr", q.double(), keys) * SCALE, dim=2)
    assert _far(got, torch.einsum("thr,rhd->thd", w, values)) <= BAR
    s2.attend_max = 100 + chunk
    s2.table[0, 0] = 2 ** 31 - 1
    kv = s2.kv()
    kv.chunk_offsets[1] = 10 ** 6
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=0, scale=SCALE).cpu()
    s2.table[0, 0] = null
    assert _far(got, s2.want(0, q, k, v)) <= BAR


def test_offsets_that_hold_no_chunks_write_nothing() -> None:
    u = _uocr()
    s = Setup(23, [40, 40], [5, 5])
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    for offsets in ([0, 0, 0], [80, 80, 80], [-5, -3, 0], [200, 300, 400]):
        pool = s.pool.to(DEV)
        kv = s.kv(pool)
        kv.chunk_offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
        out = torch.full((80, s.heads, D), 3.0, device=DEV)
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE, out=out)
        assert (out == 3.0).all(), offsets
        assert _same_bits(pool.cpu(), s.pool), offsets


def test_no_tokens_or_no_requests() -> None:
    u = _uocr()
    s = Setup(1, [0], [7])
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    assert u.paged_chunk_attention(q, k, v, kv=s.kv(), layer_idx=0, scale=1.0).shape == (0, 2, D)
    s = Setup(1, [4], [7])
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    kv = s.kv()
    none = u.PagedChunk(kv.kv_blocks, kv.lookup_table[:0], kv.cache_lengths[:0], kv.chunk_offsets[:1], 1)
    out = torch.full_like(q, 2.0)
    assert (u.paged_chunk_attention(q, k, v, kv=none, layer_idx=0, scale=1.0, out=out) == 2.0).all()


@pytest.mark.parametrize("chunk", [3, 150])
def test_a_pool_past_32_bit_offsets(chunk) -> None:
    """Pages whose elements lie past 2^31 (and bytes past 2^33) of the pool."""
    u = _uocr()
    heads, page = 10, 2 * 128 * 10 * D
    pages = 2 ** 31 // page + 6
    s = Setup(chunk, [chunk], [200], heads=heads, layers=1)
    need = int((s.table[0] < s.pool.shape[0] - 1).sum())
    pool = torch.full((pages, 2, 1, 128, heads, D), math.nan, device=DEV)
    moved = s.table.clone()
    for c in range(need):
        pool[pages - 2 - c] = s.pool[int(s.table[0, c])].to(DEV)
        moved[0, c] = pages - 2 - c
    moved[0, need:] = pages - 1
    kv = u.PagedChunk(pool, moved.to(DEV), torch.tensor([200], dtype=torch.int32, device=DEV), s.offsets.to(DEV),
                      200 + chunk)
    q, k, v = s.qkv.unbind(1)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=0, scale=SCALE)
    assert _far(got.cpu(), s.want(0, q, k, v)) <= BAR
    stored = s.stored(0, k, v)
    for c in range(need):
        assert _same_bits(pool[pages - 2 - c].cpu(), stored[int(s.table[0, c])])


@pytest.mark.parametrize(("chunks", "cached"), [([4], [300]), ([5, 7], [640, 100]), ([200, 30], [0, 900])])
def test_repeats_streams_and_graphs_give_the_same_bits(chunks, cached) -> None:
    """A second call, one on a side stream, and replays of two captured graphs (replayed between each other's, with
    eager calls between) give the first call's bits."""
    u = _uocr()
    s = Setup(31, chunks, cached, heads=10)
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    kv = s.kv()
    run = lambda out=None: u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=1, scale=SCALE, out=out)  # noqa: E731
    want = run().clone()
    assert _same_bits(run(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert _same_bits(got, want)
    graphs = []
    for _ in range(2):
        out = torch.zeros_like(want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            run(out)
        graphs.append((g, out))
    for i in range(6):
        g, out = graphs[i % 2]
        out.zero_()
        g.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
            assert _same_bits(run(), want)
        assert _same_bits(out, want), i
    # both in flight at once, each with the workspace of its own capture
    other = torch.cuda.Stream()
    for _, out in graphs:
        out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0][0].replay()
    with torch.cuda.stream(other):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(_same_bits(out, want) for _, out in graphs)


@pytest.mark.parametrize("chunks", [(3, 2), (40, 90)])
def test_a_graph_replayed_for_other_lengths(chunks) -> None:
    """A serving loop's graph: captured once for the longest requests, replayed as the lengths, the offsets and the
    pages change in place."""
    u = _uocr()
    s = Setup(37, list(chunks), [600, 300], heads=3)
    s.attend_max = 700
    q, k, v = s.qkv.unbind(1)
    on = [x.to(DEV) for x in (q, k, v)]
    pool = s.pool.to(DEV)
    kv = s.kv(pool)
    run = lambda out: u.paged_chunk_attention(*on, kv=kv, layer_idx=1, scale=SCALE, out=out)  # noqa: E731
    out = torch.zeros_like(on[0])
    run(out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        run(out)
    total = sum(chunks)
    for lengths, cached in ((chunks, (600, 300)), ((total, 0), (5, 9)), ((1, total - 1), (127, 128)),
                            ((0, total), (0, 0)), (chunks, (0, 31))):
        s.chunks, s.cached = list(lengths), list(cached)
        s.offsets = torch.tensor([0, lengths[0], total], dtype=torch.int32)
        kv.chunk_offsets.copy_(s.offsets)
        kv.cache_lengths.copy_(torch.tensor(cached, dtype=torch.int32))
        null = s.pool.shape[0] - 1
        s.table = torch.where(s.table < null, (s.table + 1) % null, s.table)
        kv.lookup_table.copy_(s.table)
        pool.copy_(s.pool)
        out.zero_()
        g.replay()
        assert _far(out.cpu(), s.want(1, q, k, v)) <= BAR, (lengths, cached)
        assert _same_bits(pool.cpu(), s.stored(1, k, v)), (lengths, cached)
        assert _same_bits(run(torch.zeros_like(out)), out), (lengths, cached)


@pytest.mark.parametrize("chunk", [5, 70])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-30])
def test_a_scale_of_nothing_is_the_mean(chunk, scale) -> None:
    u = _uocr()
    s = Setup(39, [chunk], [90])
    q, k, v = s.qkv.unbind(1)
    got = u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=0, scale=scale)
    assert _far(got.cpu(), s.want(0, q, k, v, scale)) <= BAR


def test_the_callers_workspace_and_the_wrappers_refusals() -> None:
    from uocr_moe import UocrError, _lib

    u = _uocr()
    s = Setup(41, [6, 2], [500, 90])
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    kv = s.kv()
    want = u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE)
    need = _lib.load().uocr_paged_chunk_workspace_bytes(8, 2, s.heads, s.attend_max)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    got = u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE, workspace=ws[:need])
    assert _same_bits(got, want) and (ws[need:] == 0xFF).all()
    if need:
        with pytest.raises(UocrError, match="is smaller than"):
            u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE, workspace=ws[:need - 16])
    with pytest.raises(ValueError, match="disagree on shape"):
        u.paged_chunk_attention(q, k[:-1], v, kv=kv, layer_idx=0, scale=SCALE)
    with pytest.raises(ValueError, match="does not hold"):
        u.paged_chunk_attention(q[:, :1], k[:, :1], v[:, :1], kv=kv, layer_idx=0, scale=SCALE)
    with pytest.raises(ValueError, match="metadata is not for"):
        short = u.PagedChunk(kv.kv_blocks, kv.lookup_table, kv.cache_lengths, kv.chunk_offsets[:-1], kv.attend_max)
        u.paged_chunk_attention(q, k, v, kv=short, layer_idx=0, scale=SCALE)
    with pytest.raises(UocrError, match="layer 2 is not in the pool"):
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=2, scale=SCALE)
    with pytest.raises(UocrError, match="out must not overlap"):
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE, out=k)
    with pytest.raises(ValueError, match="out must be"):
        u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE, out=want[:-1])
    half = u.PagedChunk(kv.kv_blocks.half(), kv.lookup_table, kv.cache_lengths, kv.chunk_offsets, kv.attend_max)
    with pytest.raises(ValueError, match="kv_blocks must be a contiguous f32"):
        u.paged_chunk_attention(q, k, v, kv=half, layer_idx=0, scale=SCALE)


def test_uint32_metadata_and_positions_outside_the_tables() -> None:
    u = _uocr()
    s = Setup(51, [9], [130])
    q, k, v = (x.to(DEV) for x in s.qkv.unbind(1))
    kv = s.kv()
    want = u.paged_chunk_attention(q, k, v, kv=kv, layer_idx=0, scale=SCALE)
    as_u32 = u.PagedChunk(kv.kv_blocks, kv.lookup_table.view(torch.uint32), kv.cache_lengths.view(torch.uint32),
                          kv.chunk_offsets, kv.attend_max)
    assert _same_bits(u.paged_chunk_attention(q, k, v, kv=as_u32, layer_idx=0, scale=SCALE), want)
    cos, sin = (x.to(DEV) for x in _tables(20))
    qkv = s.qkv.view(9, -1).to(DEV)
    pos = torch.tensor([-7, 0, 19, 20, 2 ** 31 - 1, 3, 4, 5, -2 ** 31], dtype=torch.int32, device=DEV)
    args = {"heads": s.heads, "layer_idx": 0, "scale": SCALE}
    a = u.paged_chunk_attention_qkv(qkv, pos, cos, sin, kv=s.kv(), **args)
    b = u.paged_chunk_attention_qkv(qkv, pos.clamp(0, 19), cos, sin, kv=s.kv(), **args)
    assert _same_bits(a, b)


def test_numpy_rows_agree_with_the_decode_oracle(oracle) -> None:
    """Token by token against the decode op's own oracle (its float64 chain)."""
    u = _uocr()
    s = Setup(61, [5], [125], heads=10)
    q, k, v = s.qkv.unbind(1)
    got = n(u.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=1, scale=SCALE))
    pool = s.pool.numpy()
    lut = s.table.numpy().astype(np.uint32)
    for j in range(5):
        row = np.asarray([125 + j], np.uint32)
        want, pool = oracle.paged_decode_attention(q[j:j + 1].numpy(), k[j:j + 1].numpy(), v[j:j + 1].numpy(), pool, lut,
                                                   row, row, 1, SCALE)
        assert np.max(np.abs(got[j] - want[0])) <= BAR * np.max(np.abs(want[0]))
    assert t(pool).shape == s.pool.shape
