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
    spread = 60 if T == 799 else width - 3             # few pages: rows over the union of their lists
    pages = torch.stack([torch.randperm(spread, generator=g)[:budget].sort().values + 3
                         for _ in range(T * Hkv)]).view(T, Hkv, budget).int()
    pages[::2, :, 0], pages[1::4, :, 1], pages[::3, :, 2] = 0, 1, 2
    if T > 1:
        pos[4], pos[6] = 0, 2                          # one key, whose weight is 1, and three
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)
    assert (got[:, :, 5] == INF).all(-1)[pos > 15].all() and (got[:, :, 6] == -INF).all(-1)[pos > 15].all()


# rows of a wave that go over the union of their lists, and the most pages of a union, as the host
# chooses them: without these the tests below would test the form row by row
def union_form(G, d, budget):
    rows = 4 * min(16 // G, 4)
    return rows, rows * budget // (3 if d == 256 else 4)


def unions(pos, pages, G, d):
    """(pages, pages that several rows share) of the unions of every group of rows and kv head."""
    T, Hkv, budget = pages.shape
    R_, _ = union_form(G, d, budget)
    found = []
    for h in range(Hkv):
        for t0 in range(0, T, R_):
            here = range(t0, min(T, t0 + R_))
            low = min([int(pos[t]) for t in here if pos[t] >= 0], default=-1)
            count = {}
            for t in here:
                for p in pages[t, h].tolist():
                    if p >= 0 and pos[t] >= 0 and p <= int(pos[t]) // PAGE:
                        k = p if p * PAGE + PAGE - 1 <= low else (p, t)
                        count[k] = count.get(k, 0) + 1
            found.append((len(count), sum(n > 1 for n in count.values())))
    return found


UNION = [
    # Hq, Hkv, d, batch, T, width, budget: 2, 2, 4, 4, 4, 4, 3, 3 rows of a matrix instruction
    (16, 2, 256, 1, 781, 200, 64),
    (32, 4, 128, 1, 397, 160, 70),
    (8, 8, 128, 2, 199, 300, 100),
    (4, 4, 256, 1, 800, 180, 64),
    (15, 5, 256, 1, 623, 150, 64),
    (15, 5, 128, 1, 623, 150, 65),
    (20, 4, 128, 1, 590, 400, 130),
    (10, 2, 256, 1, 1204, 170, 64),
]


@pytest.mark.parametrize("Hq,Hkv,d,B,T,width,budget", UNION)
def test_attend_over_unions(gpu, Hq, Hkv, d, B, T, width, budget):
    """A chunk of a prompt: consecutive positions behind a long context, lists that the rows of a
    group have mostly in common, the first page and the row's last two in each; a few rows with a
    short list or none, and padding rows. Rows of some groups against the definition, all rows
    against the form that takes them one by one."""
    say("attend over unions", Hq, Hkv, d, B, T, width, budget)
    g = torch.Generator().manual_seed(budget * 7 + d)
    G, M = Hq // Hkv, B * T
    rows, most = union_form(G, d, budget)
    groups = B * Hkv * ((T + rows - 1) // rows)
    assert 4 * B * Hkv * T >= 3 * rows * ((groups + 255) // 256 * 256)      # rows fill the workgroups
    table = tables(g, B, width, B * width + 3)
    kp, vp = pools(g, B * width + 3, Hkv, d)
    q = torch.randn(M, Hq, d, generator=g).bfloat16()
    context = width * PAGE - T - 3
    pos = (context + torch.arange(T)).repeat(B).int()
    first = context // PAGE - 1                     # pages 1 .. first - 1 are whole to every row
    pages = torch.empty(B, T, Hkv, budget, dtype=torch.int32)
    for b in range(B):
        for t in range(T):
            if t % rows == 0:
                common = [torch.randperm(first - 1, generator=g)[:budget * 5 // 4] + 1 for _ in range(Hkv)]
            last = int(pos[t]) // PAGE
            for h in range(Hkv):
                pick = common[h][torch.randperm(len(common[h]), generator=g)[:budget - 3]].sort().values
                pages[b, t, h] = torch.cat([torch.tensor([0]), pick, torch.tensor([last - 1, last])])
    pages = pages.view(M, Hkv, budget)
    pages[5::41, :, budget // 3:] = -1
    pages[17::97] = -1
    pos[rows + 1::89] = -1
    for b in range(B):
        found = unions(pos[b * T:(b + 1) * T], pages[b * T:(b + 1) * T], G, d)
        assert all(n <= most and shared >= budget // 2 for n, shared in found), (most, found)
    scale = d ** -0.5
    got = run_attend(q, kp, vp, table, pos, pages, scale)
    assert (got[pos < 0] == 0).all() and (got[17::97] == 0).all()
    for b in range(B):
        some = torch.cat([torch.arange(rows), torch.arange(T // 2 // rows * rows, T // 2 // rows * rows + rows),
                          torch.arange((T - 1) // rows * rows, T)]) + b * T
        check_attend(got[some], q[some], kp, vp, table[b:b + 1], pos[some], pages[some], scale)
        # one by one. Each form is within one rounding (2^-8) and twice the weights' error times the sum
        # of weights times |v| (at most 1.3 here) of the definition; weights are off by at most (d + 4) u
        # of a score's terms (at most 14) + 2^-16 + (keys + 64) u = 3.7e-4: 2 . 2 . 3.7e-4 . 1.3 < 2^-9
        for t0 in range(b * T, b * T + T, 32):
            part = slice(t0, min(t0 + 32, b * T + T))
            alone = run_attend(q[part], kp, vp, table[b:b + 1], pos[part], pages[part], scale)
            err = (alone.double() - got[part].double()).abs()
            assert (err <= 2.0 ** -7 * alone.double().abs() + 2.0 ** -9).all(), (t0, err.max())


@pytest.mark.parametrize("Hq,Hkv,d,T,budget", [(40, 1, 128, 2, 9), (33, 1, 256, 1, 33), (80, 2, 64, 3, 20)])
def test_attend_three_head_tiles(gpu, Hq, Hkv, d, T, budget):
    say("attend", Hq, Hkv, d, T, budget)
    g = torch.Generator().manual_seed(Hq)
    width = 40
    table = tables(g, 1, width, width)
    kp, vp = pools(g, width, Hkv, d)
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    pos = torch.randint(20 * PAGE, width * PAGE, (T,), generator=g, dtype=torch.int32)
    pages = torch.stack([torch.randperm(width, generator=g)[:budget] for _ in range(T * Hkv)])
    pages = pages.view(T, Hkv, budget).int()
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)


@pytest.mark.parametrize("T,budget", [(1, 20), (1, 131), (130, 20), (799, 20)])
def test_attend_keys_of_minus_infinity(gpu, T, budget):
    """Keys that score -inf have no weight beside others; alone they leave nothing, and the row is
    zeros as one without keys is."""
    say("attend -inf keys", T, budget)
    g = torch.Generator().manual_seed(T + budget)
    Hq, Hkv, d, width = (16, 4, 128, 140) if T == 799 else (8, 2, 128, 140)
    table = tables(g, 1, width, width)
    kp, vp = pools(g, width, Hkv, d)
    kp[table[0, :70].long(), :, 2, ::3, 5] = -INF
    kp[table[0, 133].long(), :, 2, :, 5] = -INF
    q = torch.randn(T, Hq, d, generator=g).abs().bfloat16()
    pos = torch.full((T,), width * PAGE - 1, dtype=torch.int32)
    spread = 60 if T == 799 else 133                   # few pages: rows over the union of their lists
    pages = torch.stack([torch.randperm(spread, generator=g)[:budget].sort().values + 133 - spread
                         for _ in range(T * Hkv)]).view(T, Hkv, budget).int()
    alone = torch.zeros(T, dtype=torch.bool)
    alone[5::9] = True
    pages[alone], pages[alone, :, 0] = -1, 133
    if T == 1:
        got = run_attend(q, kp, vp, table, pos, torch.full_like(pages, 133), d ** -0.5)
        assert (got == 0).all()
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    assert (got[alone] == 0).all()
    pages[alone] = -1                    # zeros by the definition too
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)
