"""The chunk attention's tests once more, with token rows behind the last chunk (of NaN, which nothing may read): so
many that the calls' size alone calls for the kernel of large chunks, which the small chunks would not reach."""

from __future__ import annotations

import math

import pytest
import torch

import test_gpu_chunk
from _gpu import DEV
from test_gpu_chunk import *  # noqa: F401,F403
from test_gpu_chunk import _far, _same_bits

pytestmark = pytest.mark.gpu

del test_offsets_that_hold_no_chunks_write_nothing  # noqa: F821  (its offsets would hold the rows behind)
del test_the_callers_workspace_and_the_wrappers_refusals  # noqa: F821  (its workspace is for the rows as they are)


def _padded(x, rows, fill=math.nan):
    return torch.cat([x, torch.full((rows, *x.shape[1:]), fill, dtype=x.dtype, device=x.device)])


@pytest.fixture(autouse=True)
def rows_behind(monkeypatch):
    import uocr_moe as u

    plain, qkv = u.paged_chunk_attention, u.paged_chunk_attention_qkv

    def behind(kv):
        return max(128 * max(8, len(kv.cache_lengths)), 2 ** 19 // max(8, kv.attend_max) + 1)

    def call(run, q, heads, head_dim, kv, out):
        wide = torch.empty(q.shape[0], heads, head_dim, device=q.device) if out is None else out.clone()
        got = run(_padded(wide, behind(kv), 5.0))
        if not torch.cuda.is_current_stream_capturing():
            assert (got[q.shape[0]:] == 5.0).all()
        return got[:q.shape[0]] if out is None else out.copy_(got[:q.shape[0]])

    def padded_plain(q, k, v, *, kv, out=None, **rest):
        past = not torch.cuda.is_current_stream_capturing() and (kv.chunk_offsets > len(q)).any()
        if len(q) == 0 or past:  # a last chunk that ends with the tokens would hold the rows behind
            return plain(q, k, v, kv=kv, out=out, **rest)
        rows = [_padded(x, behind(kv)) for x in (q, k, v)]
        return call(lambda o: plain(*rows, kv=kv, out=o, **rest), q, q.shape[1], q.shape[2], kv, out)

    def padded_qkv(x, positions, cos, sin, *, heads, kv, out=None, **rest):
        rows, where = _padded(x, behind(kv)), _padded(positions, behind(kv), 0)
        return call(lambda o: qkv(rows, where, cos, sin, heads=heads, kv=kv, out=o, **rest), x, heads,
                    x.shape[1] // (3 * heads), kv, out)

    monkeypatch.setattr(u, "paged_chunk_attention", padded_plain)
    monkeypatch.setattr(u, "paged_chunk_attention_qkv", padded_qkv)
    assert test_gpu_chunk._uocr().paged_chunk_attention is padded_plain


def test_a_long_chunk_and_offsets_past_the_tokens() -> None:
    import uocr_moe as u

    s = test_gpu_chunk.Setup(77, [1100], [40], heads=1)
    q, k, v = s.qkv.unbind(1)
    plain = u.paged_chunk_attention
    for end in (1100, 10 ** 6):
        kv = s.kv(s.pool.to(DEV))
        kv.chunk_offsets[1] = end
        got = plain(q.to(DEV), k.to(DEV), v.to(DEV), kv=kv, layer_idx=1, scale=SCALE).cpu()
        assert _far(got, s.want(1, q, k, v)) <= BAR
        assert _same_bits(kv.kv_blocks.cpu(), s.stored(1, k, v))
