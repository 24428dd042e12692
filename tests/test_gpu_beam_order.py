"""GPU tests of the order that ``beam_select`` puts candidates in: ties, candidates of different beams that are near one
another, and lengths whose penalties make equal ranks.

All is decided in 64 bits, the exponentials too: each is off by 1.1e-12 of itself, and so is their sum (its roundings add a few
2^-53 each), whose logarithm is then off by less than 2e-12.  A key near -1 adds its own roundings, 2^-53 each.  The nearest
candidates here are 1e-10 apart.
"""

from __future__ import annotations

import math

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


@pytest.mark.parametrize(("requests", "beams", "vocab"), [(1, 8, 129280), (3, 8, 2500), (64, 8, 9001)])
@pytest.mark.parametrize("gap", [1e-10, 1e-9, 1e-8, 1e-7, 1e-6])
def test_near_candidates_of_different_beams(requests, beams, vocab, gap) -> None:
    """Every beam has one likely token; the beams' scores put them `gap` apart, in an order of their own."""
    g = torch.Generator().manual_seed(vocab)
    rows = requests * beams
    logits = (2.5 * torch.randn(rows, vocab, generator=g)).clamp(max=7.0)  # log probabilities below -3
    top = torch.randint(0, vocab, (rows,), generator=g)
    at = torch.arange(rows)
    logits[at, top] = -INF
    rest = torch.cat([torch.logsumexp(x.double(), dim=1) for x in logits.split(64)])
    logits[at, top] = (rest - 1.0 - math.log1p(-math.exp(-1.0))).float()  # a log probability near -1
    best = logits[at, top].double()
    lse = rest + torch.log1p((best - rest).exp())
    order = torch.stack([torch.randperm(beams, generator=g) for _ in range(requests)])  # the place of each beam
    scores = (-1.0 - gap * order.flatten().double() - (best - lse)).float()
    keys = (scores.double() + (best - lse)).view(requests, beams)
    want = torch.sort(keys, dim=1, descending=True).indices
    assert torch.equal(want.argsort(dim=1), order)
    apart = keys.gather(1, want).diff(dim=1)
    assert bool((apart < -gap / 2).all()) and bool((keys > -1.5).all())
    tokens, parents = _select(logits, scores, beams)
    want = (want + beams * torch.arange(requests)[:, None]).flatten()
    assert parents == want.tolist() and tokens == top[want].tolist()


@pytest.mark.parametrize("top", [3e9, 2.0 ** 60, 3.4e38])
def test_large_logits(top) -> None:
    """Beside such a logit the next ones have no weight, however near they are for its size: the beams' scores decide."""
    logits = torch.full((4, 5000), top)
    logits *= 1.0 - torch.rand(4, 5000, generator=torch.Generator().manual_seed(5)) / 100 - 1e-5
    best = [7, 4000, 2100, 12]
    logits[range(4), best] = top
    scores = torch.tensor([-3.0, -1.0, -4.0, -2.0])
    tokens, parents = _select(logits, scores, 4)
    assert parents == [1, 3, 0, 2] and tokens == [4000, 12, 7, 2100]


def test_rows_without_a_finite_sum_come_last() -> None:
    """A NaN anywhere in a row, of either sign, and infinite logits."""
    logits = torch.randn(8, 5000, generator=torch.Generator().manual_seed(6))
    logits[0, 4999] = float("nan")
    logits[1, 2] = -float("nan")
    logits[2, 2047] = INF
    logits[3] = -INF
    logits[4] = float("nan")
    logits[5, 2048:] = -INF  # finite
    logits[6, 17] = 30.0
    logits[7, 18] = 40.0
    _, parents = _select(logits, torch.zeros(8), 8)
    assert parents[:2] == [6, 7] or parents[:2] == [7, 6]
    assert set(parents) == {5, 6, 7}


@pytest.mark.parametrize("alpha", [1.0, 2.0, 0.5, -1.0])
def test_equal_ranks_of_different_lengths(alpha) -> None:
    """Scores in proportion to length^alpha, whole numbers all: every rank is one number, so the rows keep their order."""
    g = torch.Generator().manual_seed(7)
    beams, requests = 8, 64
    rows = beams * requests
    if alpha == 0.5:
        root = torch.randint(1, 40, (rows,), generator=g)
        lengths, power = root * root, root.double()
    elif alpha == -1.0:
        of = torch.tensor([n for n in range(1, 841) if 840 % n == 0])
        lengths = of[torch.randint(0, len(of), (rows,), generator=g)]
        power = 840.0 / lengths.double()
    else:
        lengths = torch.randint(1, 300, (rows,), generator=g)
        power = lengths.double() ** alpha
    times = torch.randint(1, 50, (requests,), generator=g).repeat_interleave(beams)
    scores = (-times * power).float()
    assert torch.equal(scores.double(), -times * power)
    ended = torch.ones(rows, dtype=torch.int32)
    _, parents = _select(torch.zeros(rows, beams), scores, beams, ended, lengths.int(), alpha)
    assert parents == list(range(rows))


@pytest.mark.parametrize("score", [-1e20, torch.finfo(torch.float32).min, 1e18])
def test_a_beams_tokens_go_by_their_logits(score) -> None:
    """Beside such a score the keys of one beam are equal in 64 bits; its tokens' logits are not."""
    logits = torch.randn(4, 5000, generator=torch.Generator().manual_seed(3))
    logits[0, 4500] = 20.0
    logits[0, 30] = logits[0, 4400] = 19.0
    logits[0, 2500] = 18.0
    scores = torch.full((4,), -INF)
    scores[0] = score
    assert _select(logits, scores, 4) == ([4500, 30, 4400, 2500], [0] * 4)
    scores[1] = score  # of two beams the lower row comes first
    logits[1, 7] = 40.0
    assert _select(logits, scores, 4) == ([4500, 30, 4400, 2500], [0] * 4)
