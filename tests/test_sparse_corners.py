"""Corner inputs of the operators over selected pages, without a GPU."""
import torch

from oracle import sparse as R

BF, I32 = torch.bfloat16, torch.int32
INF = float("inf")


def test_oracle_scores_of_infinite_bounds():
    """A page's score is the sum of max(q low, q high), also where one of them is infinite and the
    other is not: six pages, the second with a key of -inf in one element and the largest maxima."""
    bounds = torch.ones(6, 1, 2, 128, dtype=BF)
    bounds[:, :, 0] = -1.0
    bounds[1, :, 1] = 3.0
    bounds[1, 0, 0, 7] = -INF
    q = torch.ones(1, 1, 128, dtype=BF)
    table = torch.arange(6, dtype=I32).view(1, 6)
    assert R.scores(q[0], bounds, table, 0, 0, 1).tolist() == [128.0, 384.0] + [128.0] * 4
    pos = torch.tensor([95], dtype=I32)
    assert R.select(q, bounds, table, pos, 2, 0, 1).tolist() == [[[1, 5]]]
    # a zero times an infinity, or a NaN, is NaN and ranks last; an infinite score first
    q[0, 0, 7] = 0.0
    assert R.select(q, bounds, table, pos, 2, 0, 1).tolist() == [[[0, 5]]]
    q[0, 0, 7] = -1.0
    assert R.scores(q[0], bounds, table, 0, 0, 1)[1] == INF
    bounds[3, 0, 1, 9] = float("nan")
    assert R.scores(q[0], bounds, table, 0, 0, 1)[3].isnan()
