"""GPU tests of the chunk attention where keys, values or weights of unlike sizes meet, against the formula in 64 bits.

The bar is that of ``test_gpu_chunk`` (1e-5 of a token's largest output).  Plain fp32 arithmetic meets it on all of these
inputs: a row's weight is a normal fp32 number or contributes less than 2^-24 of the output, scores stay below 100 where
they count, and what is large has no weight, or a factor of zero.  So what a row weighs next to nothing for must not cost
the others their bits, in either kernel, with one split of the rows and with several.
"""

from __future__ import annotations

import math

import pytest
import torch

from _gpu import DEV
from test_gpu_chunk import BAR, SCALE, Setup, _far, _same_bits, _uocr

pytestmark = pytest.mark.gpu

#: Chunk, cached rows, token rows behind the chunk: tiles of 32 queries in one split and in several, tiles of 256 (which
#: many token rows call for) in one and in several.
SHAPES = {"few": (20, 150, 0), "few-splits": (20, 900, 0), "tiles": (70, 160, 2300), "tiles-splits": (300, 800, 600)}


@pytest.fixture(params=list(SHAPES))
def scene(request):
    chunk, cached, tail = SHAPES[request.param]
    s = Setup(chunk + cached, [chunk], [cached], tail=tail)
    splits = _uocr()._lib.load().uocr_paged_chunk_workspace_bytes(s.tokens, 1, s.heads, s.attend_max) > 0
    assert splits == ("splits" in request.param)
    s.qkv[:, 0, :, 0] = 4.0  # a direction that every query has, so that a key's score is chosen by its first element
    return s


def _slot(s, row):
    """Where cached row `row` is: k or v of it is s.pool[_slot(s, row)][which]."""
    return s.pool[int(s.table[0, row // s.page_size]), :, 1, row % s.page_size]


def _check(s, upto=None) -> None:
    q, k, v = s.qkv.unbind(1)
    pool = s.pool.to(DEV)
    got = _uocr().paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(pool), layer_idx=1, scale=SCALE).cpu()
    used = slice(0, s.chunks[0] if upto is None else upto)
    assert _far(got[used], s.want(1, q, k, v)[used]) <= BAR
    assert _same_bits(pool.cpu(), s.stored(1, k, v))


@pytest.mark.parametrize("size", [1e3, 1e6, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("rows", [(0,), (77,), (5, 40, 41, 100, 149)])
def test_a_large_value_without_weight(scene, size, rows) -> None:
    for r in rows:
        _slot(scene, r)[1] *= size
        _slot(scene, r)[0, :, 0] = -500.0  # a score of -177: a weight of 1e-77
    _check(scene)


@pytest.mark.parametrize("size", [1e3, 1e6, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("rows", [(0,), (77,), (5, 40, 41, 100, 149)])
def test_a_large_key_without_weight(scene, size, rows) -> None:
    for r in rows:
        _slot(scene, r)[0] *= 1e-3 * size
        _slot(scene, r)[0, :, 0] = -size
    _check(scene)


@pytest.mark.parametrize("size", [1e6, 1e12, 1e30])
def test_large_elements_that_meet_zeros(scene, size) -> None:
    """A large element of a key where the queries have a zero, and of a query where the keys have one."""
    scene.qkv[:, 0, :, 9] = 0.0
    _slot(scene, 60)[0, :, 9] = size
    scene.qkv[3, 1, :, 9] = -size
    _check(scene)
    scene.qkv[:, 1, :, 17] = 0.0
    scene.pool[:, 0, 1, :, :, 17] = 0.0
    scene.qkv[::3, 0, :, 17] = size
    _check(scene)


@pytest.mark.parametrize("size", [1e6, 1e12, 1e30])
@pytest.mark.parametrize("which", [1, 2])
def test_large_rows_that_a_token_does_not_attend(scene, size, which) -> None:
    """Finite ones: the second half of the chunk is large; the first half does not see it."""
    half = scene.chunks[0] // 2
    scene.qkv[half:scene.chunks[0], which] *= size
    _check(scene, half)


@pytest.mark.parametrize("above", [12.0, 18.0, 24.0, 40.0, 70.0])
@pytest.mark.parametrize("value", [0.0, 1e-4])
@pytest.mark.parametrize("row", [0, 77])
def test_one_row_has_nearly_all_the_weight_and_a_small_value(scene, above, value, row) -> None:
    """The output is what the others' small weights leave: e^-above each, about."""
    _slot(scene, row)[0] = 0.0
    _slot(scene, row)[0, :, 0] = above / (4.0 * SCALE)
    _slot(scene, row)[1] *= value
    scene.qkv[:, 2] += 0.5  # the others' values do not cancel
    scene.pool[:, 1] += 0.5 * (scene.pool[:, 1] != 0)
    _slot(scene, row)[1] *= 1.0 if value else 0.0
    _check(scene)


@pytest.mark.parametrize("nan", [False, True])
@pytest.mark.parametrize("row", [0, 77])
def test_values_as_far_apart_as_the_type_allows(scene, row, nan) -> None:
    """Values near 1e-30 beside one of 1e36 without weight; with a NaN in the last new row, which the others do not see."""
    scene.pool[:, 1] *= 1e-30
    scene.qkv[:, 2] *= 1e-30
    _slot(scene, row)[1] *= 1e33
    _slot(scene, row)[1] *= 1e33
    _slot(scene, row)[0, :, 0] = -1500.0
    last = scene.chunks[0] - 1
    if nan:
        scene.qkv[last, 2] = math.nan
    q, k, v = scene.qkv.unbind(1)
    got = _uocr().paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=scene.kv(), layer_idx=1, scale=SCALE).cpu()
    assert _far(got[:last], scene.want(1, q, k, v)[:last]) <= BAR
    assert torch.isnan(got[last]).all() == nan


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_values_far_apart_in_a_block_beside_one_that_is_not_finite(scene, odd) -> None:
    """The first new row is 1e36 and has no weight, the others 1e-30; the tenth, in the same block, is not finite."""
    scene.pool[:, 1] *= 1e-30
    scene.qkv[:, 2] *= 1e-30
    scene.qkv[0, 2] *= 1e33
    scene.qkv[0, 2] *= 1e33
    scene.qkv[0, 1, :, 0] = -1500.0
    q, k, v = scene.qkv.unbind(1)
    want = scene.want(1, q, k, v)
    scene.qkv[9, 2, :, 3] = odd
    got = _uocr().paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=scene.kv(), layer_idx=1, scale=SCALE).cpu()
    assert _far(got[1:9], want[1:9]) <= BAR
    assert not torch.isfinite(got[9:scene.chunks[0], :, 3]).any()
    rest = [d for d in range(128) if d != 3]
    assert _far(got[9:scene.chunks[0], :, rest], want[9:scene.chunks[0], :, rest]) <= BAR


@pytest.mark.parametrize("row", [40, 149])
def test_a_small_value_takes_over_from_large_ones(scene, row) -> None:
    """Rows of 1e30 that count until a row of size 1, or nearly as large a weight later, has a score 700 above theirs."""
    scene.pool[:, 1] *= 1e30
    scene.qkv[:, 2] *= 1e30
    _slot(scene, row)[1] *= 1e-30
    _slot(scene, row)[0] = 0.0
    _slot(scene, row)[0, :, 0] = 700.0 / (4.0 * SCALE)
    _check(scene)


def test_tiny_and_huge_queries_side_by_side(scene) -> None:
    """Each query's own size costs the others nothing."""
    n = scene.chunks[0]
    size = 10.0 ** torch.randint(-30, 2, (n,), generator=torch.Generator().manual_seed(7)).float()
    scene.qkv[:n, 0] *= size[:, None, None]
    _check(scene)


def test_values_of_zero() -> None:
    """Nothing but zeros, and zeros with one row that counts."""
    for chunk, cached, tail in SHAPES.values():
        s = Setup(chunk, [chunk], [cached], tail=tail)
        s.pool[:, 1] = 0.0
        s.qkv[:, 2] = 0.0
        q, k, v = s.qkv.unbind(1)
        run = lambda: _uocr().paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv=s.kv(), layer_idx=1,  # noqa: E731
                                                    scale=SCALE)[:chunk].cpu()
        assert (run() == 0).all()
        _slot(s, 50)[1] = 1e-3 * torch.randn(s.heads, 128, generator=torch.Generator().manual_seed(1))
        assert _far(run(), s.want(1, q, k, v)[:chunk]) <= BAR
