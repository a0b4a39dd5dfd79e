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


def test_select_scratch_grows_with_the_shape():
    """A workspace that is enough for the longest tables, the most rows and the largest batch is
    enough for less of each."""
    from snowllm_amd import ops
    need = ops.page_select_scratch_bytes
    assert need(1 << 60, 0, 32, 8, 128, 4096) == 0
    assert need(1, 1024, 32, 8, 128, 4096) <= need(1, 1024, 32, 8, 128, 8192)
    assert need(4, 512, 32, 8, 128, 2432) <= need(4, 512, 32, 8, 128, 3840)
    widths = [0, 1, 15, 16, 17, 100, 513, 1000, 2432, 3840, 4064, 4096, 8192, 13751, 20000, 40000, 1 << 17]
    rows = [1, 9, 15, 16, 17, 31, 32, 33, 64, 100, 500, 512, 1000, 1024, 2048, 10000]
    for hkv, d in ((1, 64), (8, 128), (2, 256)):
        table = torch.tensor([[[need(b, t, 4 * hkv, hkv, d, w) for w in widths] for t in rows]
                              for b in (1, 2, 3, 4, 16, 64, 256)])
        for dim in range(3):
            assert (table.diff(dim=dim) >= 0).all(), (hkv, d, dim)
        # and 256 MiB do, or sixteen rows' part
        sixteen = torch.tensor([[[need(b, 16, 4 * hkv, hkv, d, w) for w in widths] for _ in rows]
                                for b in (1, 2, 3, 4, 16, 64, 256)])
        assert (table <= sixteen.clamp(min=256 << 20)).all()
