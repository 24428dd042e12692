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


def test_tiny_and_huge_queries_side_by_side(scene) -> None:
    """Each query's own size costs the others nothing."""
    n = scene.chunks[0]
    size = 10.0 ** torch.randint(-30, 2, (n,), generator=torch.Generator().manual_seed(7)).float()
    scene.qkv[:n, 0] *= size[:, None, None]
    _check(scene)
