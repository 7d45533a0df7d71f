"""What the header says of the beam search's operators at its ends: the selection's
error, its order.

u = 2^-24, the half step of an f32 at 1."""
import numpy as np
import pytest
import torch

from decode_util import TYPES
from search_util import beam_scores
from test_gpu_decode import U
from test_gpu_search import INF, run_beam

pytestmark = pytest.mark.gpu


def few_values(vocab, places, beams, kind):
    """beams: (score, values) each; the values at `places`, -inf elsewhere."""
    x = torch.full((1, len(beams), vocab), -INF)
    for b, (_, values) in enumerate(beams):
        x[0, b, places] = torch.tensor(values, dtype=torch.float32)
    return x.to(TYPES[kind]), np.array([[s for s, _ in beams]], np.float32)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [0, 50, 300, 1000, 3990, 4090, 4100, 60000, -50, -300, -1000, -4100])
@pytest.mark.parametrize("vocab,places", [(3, [0, 1, 2]), (70000, [7, 30001, 69999])])
def test_beam_large_logits(kind, top, vocab, places):
    """Three values whose largest is far from 0, side by side and in parts of the row
    of their own.  An exponential is off by 2 u, its argument by 1.3 u times the
    value's distance from the top (0.4 on average), three additions by 3 u, what c
    lacks is made up for with 3 u, and of the sums of other lanes, waves and parts (a
    fifth of the whole) an exponential each and 3 u times the distance: 12 u in
    all, and half a step of the f32 score."""
    x, s = few_values(vocab, places, [(-1.0, [top, top - 1.5, top - 3])], kind)
    ref = beam_scores(x[0].float().numpy(), s[0], None, 0)[0, places]
    parent, token, score = run_beam(x, s, 3)
    order = np.argsort(-ref, kind="stable")
    assert parent[0].tolist() == [0, 0, 0] and token[0].tolist() == [places[i] for i in order]
    assert (np.abs(score[0] - ref[order]) <= 12 * U + U * np.abs(ref[order])).all(), (score[0] - ref[order]) / U


@pytest.mark.parametrize("vocab,places", [(3, [0, 1, 2]), (70000, [7, 30001, 69999])])
def test_beam_order_of_unlike_beams(vocab, places):
    """Beams whose logits lie apart and whose scores differ by a few 1e-6, 50 u and more:
    the order is the scores', and no continuation counts more than its beam."""
    for high, low in ((900, 100), (300, 0), (3900, -1000), (4090, 4100), (50, -800)):
        for a, b in ((-1.00001, -1.0), (-1.000003, -1.0), (-1.0, -1.00001), (-1.0, -1.000003)):
            x, s = few_values(vocab, places, [(a, [high, high - 50, high - 100]), (b, [low, low - 50, low - 100])], "f32")
            parent, token, score = run_beam(x, s, 2)
            assert parent[0].tolist() == ([0, 1] if a > b else [1, 0]), (high, low, a, b, score)
            assert token[0].tolist() == [places[0]] * 2
            # (e^-50 of the whole: within the score's rounding)
            assert (np.abs(score[0] - np.sort(s[0])[::-1]) <= 12 * U).all(), (score, s)
