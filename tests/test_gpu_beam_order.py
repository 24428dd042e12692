"""GPU tests of the order that ``beam_select`` puts candidates in."""

from __future__ import annotations

import pytest
import torch

from _gpu import DEV

pytestmark = pytest.mark.gpu

EOS = 2
INF = float("inf")


def _select(logits, scores, beams, ended=None, lengths=None, alpha=0.0):
    import uocr_moe

    on = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    got = uocr_moe.beam_select(on(logits), on(scores), beams=beams, eos=EOS, ended=on(ended), lengths=on(lengths), alpha=alpha)
    return got.tokens.tolist(), got.parents.tolist()


@pytest.mark.parametrize(("beams", "low", "zeros"), [(2, -5.0, [4, 8]), (4, -1.0, [400, 404, 408, 412]),
                                                     (3, -2.0, [5, 2100, 4200])])
def test_zeros_of_either_sign_are_equal(beams, low, zeros) -> None:
    """Of equal candidates the lower token comes first; -0.0 equals 0.0."""
    logits = torch.full((beams, 5000), low)
    logits[:, zeros] = 0.0
    logits[:, 0] = -0.0
    scores = torch.full((beams,), -INF)
    scores[0] = 0.0
    tokens, parents = _select(logits, scores, beams)
    assert tokens == [0, *zeros][:beams] and parents == [0] * beams
    logits = -logits  # the other way about: 0.0 among -0.0, below the others
    logits[:, 10] = INF  # no finite sum but in the first row
    logits[0, 10] = -low
    logits[0, logits[0] == -low] = low
    tokens, parents = _select(logits, scores, beams)
    assert tokens == [0, *zeros][:beams] and parents == [0] * beams


def test_scores_of_either_zero_are_equal() -> None:
    ended = torch.ones(4, dtype=torch.int32)
    for scores in ([-0.0, 0.0, -0.0, 0.0], [0.0, -0.0, 0.0, 0.0]):
        assert _select(torch.randn(4, 50), torch.tensor(scores), 4, ended)[1] == [0, 1, 2, 3]
