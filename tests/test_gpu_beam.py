"""GPU tests of ``beam_select`` against the same step in float64 on the host.

What is chosen has to be equal: keys are in 64 bits but for the sum of exponentials, whose terms are rounded to
float32: an exponent x - max is off by 2^-24 of itself and its exponential by two units, so that a term of weight p is
off by p (|x - max| + 2) 2^-24 at most, and the sum's logarithm by less than 16 2^-24 = 1e-6 where no token 14 or more
below the largest carries the sum.  Candidates of different beams nearer than that could change places; the inputs here
have none (asserted), as candidates of one beam share its sum.  Scores are the keys rounded to float32, half a step
(2^-24 of the score) and that 1e-6 off.
"""

from __future__ import annotations

import math

import pytest
import torch

from _gpu import DEV

pytestmark = pytest.mark.gpu

EOS = 2
INF = float("inf")


def _uocr():
    import uocr_moe

    return uocr_moe


def _step(logits, scores, beams, ended=None, lengths=None, alpha=0.0, history=None):
    """The step on the host, in float64: the columns of Beams, and the smallest gap between the candidates that matter."""
    rows, vocab = logits.shape
    out: dict = {k: [] for k in ("tokens", "parents", "scores", "ended", "lengths", "history")}
    gap = INF
    for first in range(0, rows, beams):
        found = []
        for b in range(first, first + beams):
            over = bool(ended is not None and ended[b])
            length = int(lengths[b]) + (not over) if lengths is not None else 0
            score = float(scores[b])
            by = math.pow(length, alpha) if lengths is not None else 1.0
            if over:
                keys = torch.tensor([score], dtype=torch.float64)
                ids = [EOS]
            else:
                x = logits[b].double()
                keys = score + (x - torch.logsumexp(x, dim=0))
                ids = list(range(vocab))
            rank = keys / by if by else torch.full_like(keys, -INF)
            rank = torch.where(torch.isfinite(rank), rank, -INF)
            order = torch.sort(rank, descending=True, stable=True).indices[:2 * beams].tolist()
            found += [(-float(rank[i]), b, ids[i], float(keys[i]), length, over) for i in order]
        found.sort(key=lambda c: c[:3])
        for x, y in zip(found[:beams], found[1:beams + 1]):
            if x[1] != y[1] and math.isfinite(y[0]):
                gap = min(gap, y[0] - x[0])
        for rank, b, token, key, length, over in found[:beams]:
            out["tokens"].append(token)
            out["parents"].append(b)
            out["scores"].append(key if rank < INF else -INF)
            out["ended"].append(int(over or token == EOS))
            out["lengths"].append(length)
            if history is not None:
                h = history[b].tolist()
                out["history"].append(h if over else (h + [token])[1:])
    return out, gap


def _check(logits, scores, beams, ended=None, lengths=None, alpha=0.0, history=None, **kw):
    u = _uocr()
    want, gap = _step(logits, scores, beams, ended, lengths, alpha, history)
    assert gap > 4e-6 or gap == 0.0, "the inputs' candidates are apart, or equal"
    on = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    got = u.beam_select(on(logits), on(scores), beams=beams, eos=EOS, ended=on(ended), lengths=on(lengths), alpha=alpha,
                        history=on(history), **kw)
    assert got.tokens.tolist() == want["tokens"]
    assert got.parents.tolist() == want["parents"]
    assert got.ended.tolist() == want["ended"]
    for a, b in zip(got.scores.tolist(), want["scores"]):
        assert a == b or abs(a - b) <= 2 ** -24 * abs(b) + 1e-6, (a, b)
    assert (got.lengths is None) == (lengths is None) and (got.history is None) == (history is None)
    if lengths is not None:
        assert got.lengths.tolist() == want["lengths"]
    if history is not None:
        assert got.history.tolist() == want["history"]
    return got


def _inputs(seed, requests, beams, vocab, width=7):
    g = torch.Generator().manual_seed(seed)
    rows = requests * beams
    logits = 2.5 * torch.randn(rows, vocab, generator=g)
    logits[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 8.0
    scores = -10.0 * torch.rand(rows, generator=g)
    ended = (torch.rand(rows, generator=g) < 0.25).int()
    lengths = torch.randint(1, 60, (rows,), generator=g, dtype=torch.int32)
    history = torch.randint(0, vocab, (rows, width), generator=g, dtype=torch.int32)
    return logits, scores, ended, lengths, history


@pytest.mark.parametrize(("requests", "beams", "vocab"), [
    (1, 1, 1), (1, 1, 5), (3, 2, 3), (1, 4, 2047), (2, 4, 2048), (1, 3, 2049), (1, 8, 129280), (5, 5, 12345), (1, 32, 32),
    (2, 32, 4001), (40, 16, 10001), (70, 8, 1000), (300, 2, 600),
])
@pytest.mark.parametrize("penalty", [False, True])
def test_steps(requests, beams, vocab, penalty) -> None:
    logits, scores, ended, lengths, history = _inputs(requests + beams + vocab, requests, beams, vocab)
    if vocab <= EOS:
        logits, history = torch.randn(requests * beams, EOS + 1), None
    if penalty:
        _check(logits, scores, beams, ended, lengths, 0.8, history)
    else:
        _check(logits, scores, beams, history=history)


def test_each_option_alone() -> None:
    logits, scores, ended, lengths, history = _inputs(1, 4, 3, 777, width=1)
    _check(logits, scores, 3, ended)
    _check(logits, scores, 3, lengths=lengths, alpha=-0.5)
    _check(logits, scores, 3, lengths=lengths, alpha=0.0)
    _check(logits, scores, 3, history=history)
    _check(logits, scores, 3, ended, history=history[:, :0].contiguous())


def test_a_request_begins_with_one_beam() -> None:
    logits, scores, *_ = _inputs(2, 3, 4, 3000)
    logits = logits[::4].repeat_interleave(4, dim=0).contiguous()
    scores[:] = -INF
    scores[::4] = 0.0
    got = _check(logits, scores, 4)
    assert got.parents.tolist() == [r // 4 * 4 for r in range(12)]


def test_equal_candidates_go_to_the_lower_row_and_token() -> None:
    logits = torch.zeros(8, 5000)
    _check(logits, torch.zeros(8), 4)  # every candidate is equal
    logits[:, 4000:] = 1.0  # a thousand equal best ones of every beam
    _check(logits, torch.zeros(8), 4)
    logits[1, :3] = 1.0
    logits[6, 17] = logits[5, 16] = 1.0
    _check(logits, torch.zeros(8), 4)
    _check(torch.zeros(64, 9000), torch.zeros(64), 32)


def test_masked_tokens_come_last() -> None:
    """Tokens at -inf and at the guard's -3e38, whole rows of them, and beams that are not there."""
    logits, scores, *_ = _inputs(3, 2, 4, 4100)
    logits[:, 10:] = -INF
    _check(logits, scores, 4)
    logits[:, 1:] = -INF  # one finite candidate of each beam
    _check(logits, scores, 4)
    logits[1:] = -INF  # rows with nothing: their first tokens, last
    _check(logits, scores, 4)
    logits[:] = -INF
    _check(logits, scores, 4)
    logits, scores, *_ = _inputs(4, 2, 4, 4100)
    logits[:, 2:] = -3.0e38
    _check(logits, scores, 4)
    scores[2] = -INF
    scores[5:] = -INF
    _check(logits, scores, 4)


def test_values_that_are_not_finite() -> None:
    logits, scores, ended, lengths, history = _inputs(5, 3, 3, 2500)
    logits[1, 9] = float("nan")
    logits[4, 2499] = INF
    logits[6:, 0] = float("nan")  # a request without a finite row
    scores[3] = float("nan")
    _check(logits, scores, 3, history=history)
    lengths[:] = 0
    ended[:] = 1
    _check(logits, scores, 3, ended, lengths, 0.5)  # 0 ** 0.5: no finite rank


def test_ended_beams_alone() -> None:
    logits, scores, ended, lengths, history = _inputs(6, 2, 5, 300)
    ended[:] = 1
    got = _check(logits, scores, 5, ended, history=history)
    assert got.tokens.tolist() == [EOS] * 10 and got.ended.tolist() == [1] * 10


def test_logits_at_odd_places() -> None:
    """Rows that are not at 16-byte boundaries, of a size that is no multiple of four, and a view that is packed."""
    logits, scores, *_ = _inputs(7, 2, 3, 1001)
    _check(logits, scores, 3)
    u = _uocr()
    for wide in (torch.zeros(6, 1300, device=DEV), torch.zeros(6, 1300, device=DEV).half().float()):
        wide[:, 100:1101] = logits.to(DEV)
        a = u.beam_select(wide[:, 100:1101], scores.to(DEV), beams=3, eos=EOS)
        b = u.beam_select(logits.to(DEV), scores.to(DEV), beams=3, eos=EOS)
        assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))
    flat = torch.zeros(6 * 1000 + 1, device=DEV)[1:].view(6, 1000)  # a multiple of four, at an odd address
    flat.copy_(logits[:, :1000])
    a = u.beam_select(flat, scores.to(DEV), beams=3, eos=EOS)
    b = u.beam_select(flat.clone(), scores.to(DEV), beams=3, eos=EOS)
    assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))


def test_a_workspace_of_the_callers() -> None:
    u = _uocr()
    logits, scores, ended, lengths, history = _inputs(8, 4, 4, 5000)
    need = u._lib.load().uocr_beam_select_workspace_bytes(16, 5000, 4)
    ws = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device=DEV)
    _check(logits, scores, 4, ended, lengths, 1.0, history, workspace=ws)
    assert bool((ws[need:] == 0xAB).all())


def test_no_rows() -> None:
    u = _uocr()
    got = u.beam_select(torch.empty(0, 50, device=DEV), torch.empty(0, device=DEV), beams=4, eos=EOS)
    assert got.tokens.shape == (0,) and got.history is None


def test_captured_and_replayed() -> None:
    u = _uocr()
    logits, scores, ended, lengths, history = (x.to(DEV) for x in _inputs(9, 6, 4, 20000))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        got = u.beam_select(logits, scores, beams=4, eos=EOS, ended=ended, lengths=lengths, alpha=0.6, history=history)
    for seed in (10, 11, 12):
        for x, y in zip((logits, scores, ended, lengths, history), _inputs(seed, 6, 4, 20000)):
            x.copy_(y)
        eager = u.beam_select(logits, scores, beams=4, eos=EOS, ended=ended, lengths=lengths, alpha=0.6, history=history)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
