"""Corner inputs of the operators over selected pages against their definition in 64 bits
(oracle/sparse.py), with the tolerances of tests/test_gpu_sparse.py."""
import pytest
import torch

from oracle import sparse as R
from tests.test_gpu_sparse import check_attend, pools, run_attend, run_select, say, tables

pytestmark = pytest.mark.gpu

INF = float("inf")
PAGE = 16


# ------------------------------------------------------------------------------------------
# select
# ------------------------------------------------------------------------------------------
def test_select_page_with_an_infinite_minimum(gpu):
    """Positive queries score a page by its maxima, whatever its minima: the second page, whose
    maxima are the largest, holds a key of -inf."""
    bounds = torch.ones(6, 1, 2, 128, dtype=torch.bfloat16)
    bounds[:, :, 0] = -1.0
    bounds[1, :, 1] = 3.0
    bounds[1, 0, 0, 7] = -INF
    table = torch.arange(6, dtype=torch.int32).view(1, 6)
    pos = torch.tensor([95], dtype=torch.int32)
    for sign, low, high in ((1.0, bounds[:, :, 0], bounds[:, :, 1]), (-1.0, -bounds[:, :, 1], -bounds[:, :, 0])):
        q = torch.full((1, 2, 128), sign).bfloat16()
        got = run_select(q, torch.stack([low, high], 2), table, pos, 2, 0, 1, 1)
        assert got.tolist() == [[[1, 5]]], sign


@pytest.mark.parametrize("Hq,Hkv,d", [(8, 2, 128), (6, 1, 64), (3, 3, 256)])
@pytest.mark.parametrize("T", [1, 15, 40])
def test_select_infinite_bounds(gpu, Hq, Hkv, d, T):
    """Infinite keys among ordinary ones, for queries of one sign, of both, with zeros and with
    infinities: scores that are finite, infinite and NaN."""
    say("select inf", Hq, Hkv, d, T)
    g = torch.Generator().manual_seed(d + T)
    width, budget = 90, 20
    table = tables(g, 1, width, width)
    x = torch.randn(width, Hkv, 2, d, generator=g)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    bounds[::4, :, 0, 3] = -INF
    bounds[1::4, :, 1, 5] = INF
    bounds[2::8, :, 0, 7], bounds[2::8, :, 1, 7] = -INF, INF
    bounds[6::8, :, :, 9] = INF
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    q[0::5] = q[0::5].abs()
    q[1::5] = -q[1::5].abs()
    q[3::5, :, 3:6] = 0.0
    q[4::5, ::2, 11] = -INF
    pos = torch.full((T,), width * PAGE - 1, dtype=torch.int32)
    got = run_select(q, bounds, table, pos, budget, 1, 2, Hkv)
    assert torch.equal(got, R.select(q, bounds, table, pos, budget, 1, 2))


@pytest.mark.parametrize("T", [150, 140, 129])
def test_select_two_requests_in_parts_of_row_tiles(gpu, T):
    """Rows of two requests that pass the scratch in parts of four row tiles, the last part of two,
    of less than one and of a single row; rows at the parts' ends."""
    from snowllm_amd import ops
    say("select in parts", T)
    g = torch.Generator().manual_seed(T)
    B, Hq, Hkv, d, width, blocks, budget = 2, 16, 8, 64, 20000, 700, 90
    need = ops.page_select_scratch_bytes(B, T, Hq, Hkv, d, width)
    # a part is a multiple of sixteen rows: 64 rows fit, 80 do not
    fits = [r for r in range(16, T, 16) if ops.page_select_scratch_bytes(B, r, Hq, Hkv, d, width) < need]
    assert fits == [16, 32, 48, 64]
    table = torch.randint(0, blocks, (B, width), generator=g, dtype=torch.int32)
    x = torch.randn(blocks, Hkv, 2, d, generator=g)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    q = torch.randn(B * T, Hq, d, generator=g).bfloat16()
    pos = torch.randint(width // 2 * PAGE, width * PAGE, (B * T,), generator=g, dtype=torch.int32)
    pos[T - 1], pos[70], pos[T + 65] = width * PAGE - 1, -1, 50 * PAGE
    got = run_select(q, bounds, table, pos, budget, 1, 2, Hkv)
    for b in range(B):
        for t in (0, 15, 16, 63, 64, 65, 70, 127, 128, T - 1):
            m = b * T + t
            one = R.select(q[m:m + 1], bounds, table[b:b + 1], pos[m:m + 1], budget, 1, 2)
            assert torch.equal(got[m:m + 1], one), (b, t)


# ------------------------------------------------------------------------------------------
# attend
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 130, 799])
def test_attend_at_the_last_position(gpu, T):
    """Rows at position 2^31 - 1, which see every listed page whole, page 0 among them as the first
    and as the second page of a pair: a wave takes every fourth entry of a list, the union of the
    lists of many rows begins with the first one's."""
    say("attend at 2^31 - 1", T)
    g = torch.Generator().manual_seed(T)
    Hq, Hkv, d, width, budget = (16, 4, 128, 24, 20) if T == 799 else (8, 2, 128, 24, 20)
    table = tables(g, 1, width, width + 2)
    kp, vp = pools(g, width + 2, Hkv, d)
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    pos = torch.full((T,), 2 ** 31 - 1, dtype=torch.int32)
    pages = torch.stack([torch.randperm(width - 1, generator=g)[:budget] + 1 for _ in range(T * Hkv)])
    pages = pages.view(T, Hkv, budget).int()
    pages[:, :, 1 if T == 799 else 4] = 0
    pages[3::7, :, 0] = 0
    pages[3::7, :, 1:5] = pages[3::7, :, 5:9]
    pages[3::7, :, 5:9] = -1
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)


@pytest.mark.parametrize("T,budget", [(1, 20), (1, 131), (130, 20), (799, 20)])
def test_attend_infinite_values(gpu, T, budget):
    """An infinite value that a row sees makes its element infinite, and NaN only together with one
    of the other sign: also under the largest weight, which is a power of two."""
    say("attend infinite v", T, budget)
    g = torch.Generator().manual_seed(T + budget)
    Hq, Hkv, d, width = (16, 4, 128, 140) if T == 799 else (8, 2, 128, 140)
    table = tables(g, 1, width, width)
    kp, vp = pools(g, width, Hkv, d)
    vp[:, :, :, 5], vp[:, :, :, 6] = INF, -INF         # [blocks, Hkv, 4, d, 4]
    vp[table[0, 0].long(), :, 0, 7, 0] = INF           # one key
    vp[table[0, 1].long(), :, 0, 8, 1], vp[table[0, 2].long(), :, 0, 8, 1] = INF, -INF
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    pos = torch.full((T,), width * PAGE - 1, dtype=torch.int32)
    pages = torch.stack([torch.randperm(width - 3, generator=g)[:budget].sort().values + 3
                         for _ in range(T * Hkv)]).view(T, Hkv, budget).int()
    pages[::2, :, 0], pages[1::4, :, 1], pages[::3, :, 2] = 0, 1, 2
    if T > 1:
        pos[4], pos[6] = 0, 2                          # one key, whose weight is 1, and three
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)
    assert (got[:, :, 5] == INF).all(-1)[pos > 15].all() and (got[:, :, 6] == -INF).all(-1)[pos > 15].all()
