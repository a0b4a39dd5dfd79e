"""Attention over selected pages against its definition in 64 bits (oracle/sparse.py): the cache
write with page bounds, bounds of pages another writer filled, the choice of pages, the attention
over them, and the four in a row.

Tolerances count roundings, with u = 2^-24 (fp32) and one rounding to bf16 of at most 2^-8 of the
value. Rotated values: two products and their sum (4 u of the terms), and with the norm the sum of
d squares in any order, its root and two more products ((d + 8) u). Attention: a score of d products
is off by at most (d + 4) u of its terms' sum, and as an exponent moves a weight by that; the weight
itself is held to 2^-16 and exp2 and the sums add (keys + 64) u; each of these enters the weights
and their sum."""
import pytest
import torch

from oracle import sparse as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = 2.0 ** -8
PAGE = 16


def say(*a):
    print(*a, flush=True)


def pools(g, blocks, hkv, d):
    return (torch.randn(blocks, hkv, d // 16, PAGE, 16, generator=g).bfloat16(),
            torch.randn(blocks, hkv, 4, d, 4, generator=g).bfloat16())


def tables(g, batch, width, blocks):
    return torch.randperm(blocks, generator=g)[:batch * width].int().view(batch, width)


def bits(t):
    return t.contiguous().view(torch.int16)


# ------------------------------------------------------------------------------------------
# append and bounds
# ------------------------------------------------------------------------------------------
APPEND = [
    # Hq, Hkv, d, half, norm, T, starts, counts
    (32, 8, 128, 64, False, 1, [8191], [1]),
    (16, 2, 256, 32, True, 9, [5, 16, 31], [9, 1, 9]),
    (4, 4, 64, 32, False, 33, [0, 15, 1], [33, 17, 0]),
    (5, 1, 128, 8, True, 40, [7, 0], [40, 16]),
    (6, 3, 64, 0, True, 16, [16, 3], [16, 13]),
    (4, 2, 256, 128, False, 21, [100, 47, 2], [21, 99, -4]),
    (3, 3, 128, 24, True, 2, [14, -1, 15], [2, 2, 2]),
]


@pytest.mark.parametrize("Hq,Hkv,d,half,norm,T,starts,counts", APPEND)
def test_append(gpu, Hq, Hkv, d, half, norm, T, starts, counts):
    from snowllm_amd import ops
    say("append", Hq, Hkv, d, half, norm, T, starts, counts)
    g = torch.Generator().manual_seed(T * 1000 + d)
    B = len(starts)
    M = B * T
    width = max(max(s, 0) + T for s in starts) // PAGE + 1
    blocks = B * width + 3
    table = tables(g, B, width, blocks)
    kp, vp = pools(g, blocks, Hkv, d)
    bounds = torch.randn(blocks, Hkv, 2, d, generator=g).bfloat16()
    n = (Hq + 2 * Hkv) * d
    proj = torch.randn(M, n + 24, generator=g).bfloat16()          # rows at a pitch of their own
    cut = [proj[:, 8:8 + Hq * d], proj[:, 8 + Hq * d:8 + (Hq + Hkv) * d],
           proj[:, 8 + (Hq + Hkv) * d:8 + n]]
    q, k, v = (x.unflatten(1, (h, d)) for x, h in zip(cut, (Hq, Hkv, Hkv)))
    angle = torch.rand(M, half, generator=g) * 6.28
    cos, sin = angle.cos(), angle.sin()
    qg = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16() if norm else None
    kg = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16() if norm else None
    q_out = torch.full((M, Hq, d), 7.0).bfloat16()
    st, ct = torch.tensor(starts, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)

    pc = proj.cuda()
    cu = [pc[:, 8:8 + Hq * d], pc[:, 8 + Hq * d:8 + (Hq + Hkv) * d], pc[:, 8 + (Hq + Hkv) * d:8 + n]]
    qc, kc, vc = (x.unflatten(1, (h, d)) for x, h in zip(cu, (Hq, Hkv, Hkv)))
    gk, gv, gb, gq = kp.cuda(), vp.cuda(), bounds.cuda(), q_out.cuda()
    dev = [x.cuda() if x is not None else None for x in (cos, sin, table, st, ct, qg, kg)]
    ops.kv_append(kc, vc, dev[0], dev[1], gk, gv, dev[2], dev[3], dev[4], bounds=gb, q=qc, q_out=gq,
                  q_gamma=dev[5], k_gamma=dev[6], eps=1e-6)
    torch.cuda.synchronize()

    wk, wv = R.norm_rotate(k, kg, cos, sin, 1e-6), R.norm_rotate(q, qg, cos, sin, 1e-6)
    want_k, want_v, tol_k = kp.double(), vp.clone(), torch.zeros(kp.shape, dtype=torch.float64)
    for m, blk, off in R.slots(table, st, ct, T, blocks):
        want_k[blk, :, :, off] = wk[0][m].view(Hkv, d // 16, 16)
        tol_k[blk, :, :, off] = (BF * wk[0][m].abs() + (d + 12) * U * wk[1][m]).view(Hkv, d // 16, 16)
        want_v[blk, :, off // 4, :, off % 4] = v[m]
    got = gk.cpu()
    assert ((got.double() - want_k).abs() <= tol_k).all()
    assert torch.equal(bits(gv.cpu()), bits(want_v))
    live = torch.zeros(M, dtype=torch.bool)
    for b in range(B):
        if starts[b] >= 0:
            live[b * T:b * T + min(max(counts[b], 0), T)] = True
    tol = BF * wv[0].abs() + (d + 12) * U * wv[1]
    assert ((gq.cpu().double() - wv[0]).abs() <= tol)[live].all()
    assert (gq.cpu()[~live] == 7.0).all()
    # the bounds are those of the keys as cached, exactly
    assert torch.equal(gb.cpu().float(), R.page_limits(got, bounds, table, st, ct, T).float())


def test_append_refused_slots_and_dead_keys(gpu):
    """Pages without a block are skipped; what lies behind the last row stays and stays out of the
    bounds; NaN and infinite keys are in them."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(3)
    Hkv, d, T, blocks = 2, 64, 20, 6
    table = torch.tensor([[3, -1, 2], [0, 6, 5]], dtype=torch.int32)
    st, ct = torch.tensor([12, 10], dtype=torch.int32), torch.tensor([20, 20], dtype=torch.int32)
    kp, vp = pools(g, blocks, Hkv, d)
    kp[:] = float("nan")
    kp[3, :, :, :12] = 0.5
    kp[0, :, :, :10] = -0.5
    k = torch.randn(2 * T, Hkv, d, generator=g).bfloat16()
    k[1, 0, 3], k[2, 1, 5], k[21, 0, 7], k[22, 1, 9] = float("nan"), float("inf"), float("-inf"), -float("nan")
    v = torch.randn(2 * T, Hkv, d, generator=g).bfloat16()
    bounds = torch.zeros(blocks, Hkv, 2, d).bfloat16()
    none = torch.zeros(2 * T, 0)
    gk, gv, gb = kp.cuda(), vp.cuda(), bounds.cuda()
    ops.kv_append(k.cuda(), v.cuda(), none.cuda(), none.cuda(), gk, gv, table.cuda(), st.cuda(),
                  ct.cuda(), bounds=gb)
    torch.cuda.synchronize()
    written = R.slots(table, st, ct, T, blocks)
    assert len(written) == 4 + 6                 # pages 1 of both requests have no block
    for m, blk, off in written:
        kp[blk, :, :, off] = k[m].view(Hkv, d // 16, 16)
        vp[blk, :, off // 4, :, off % 4] = v[m]
    assert torch.equal(gk.cpu().isnan(), kp.isnan())
    assert torch.equal(gk.cpu().nan_to_num(9.0), kp.nan_to_num(9.0))
    assert torch.equal(bits(gv.cpu()), bits(vp))
    want = R.page_limits(kp, bounds, table, st, ct, T).float()
    assert torch.equal(gb.cpu().float().nan_to_num(9.0), want.nan_to_num(9.0))
    assert want[3, 0, 0, 3].isnan() and want[3, 1, 1, 5] == float("inf") and want[0, 0, 0, 7] == float("-inf")


@pytest.mark.parametrize("Hkv,d,starts,counts,tokens", [
    (8, 128, [8190, 100, 0], [9, 1, 5], 9), (2, 256, [0], [1000], 1000), (3, 64, [7, 5], [90, 0], 64),
    (1, 64, [15, 16, -3], [1, 1, 1], 1)])
def test_bounds(gpu, Hkv, d, starts, counts, tokens):
    from snowllm_amd import ops
    say("bounds", Hkv, d, starts, counts, tokens)
    g = torch.Generator().manual_seed(d)
    B = len(starts)
    width = max(max(s, 0) + tokens for s in starts) // PAGE + 1
    blocks = B * width + 2
    table = tables(g, B, width, blocks)
    kp, _ = pools(g, blocks, Hkv, d)
    kp[::3, 0, 0, 5, 3] = float("nan")
    kp[1::3, 0, 0, 2, 4] = -float("inf")
    bounds = torch.randn(blocks, Hkv, 2, d, generator=g).bfloat16()
    st, ct = torch.tensor(starts, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)
    gb = bounds.cuda()
    ops.page_bounds(kp.cuda(), gb, table.cuda(), st.cuda(), ct.cuda(), tokens)
    want = R.page_limits(kp, bounds, table, st, ct, tokens).float()
    assert torch.equal(gb.cpu().float().nan_to_num(9.0), want.nan_to_num(9.0))


# ------------------------------------------------------------------------------------------
# select
# ------------------------------------------------------------------------------------------
def run_select(q, bounds, table, positions, budget, sink, recent, hkv):
    from snowllm_amd import ops
    M, Hq, d = q.shape
    B = table.shape[0]
    scratch = ops.empty_bytes(ops.page_select_scratch_bytes(B, M // B, Hq, hkv, d, table.shape[1]))
    pages = torch.full((M, hkv, budget), 77, dtype=torch.int32, device="cuda")
    ops.page_select(q.cuda(), bounds.cuda(), table.cuda(), positions.cuda(), pages, scratch,
                    sink=sink, recent=recent)
    torch.cuda.synchronize()
    return pages.cpu()


SELECT = [
    # Hq, Hkv, d, batch, T, width, budget, sink, recent
    (16, 2, 256, 1, 1, 513, 64, 1, 2),
    (32, 8, 128, 3, 1, 100, 17, 1, 2),
    (32, 8, 128, 2, 5, 70, 64, 0, 1),
    (6, 3, 64, 2, 19, 200, 9, 2, 3),
    (20, 1, 64, 1, 33, 130, 5, 1, 4),
    (4, 4, 128, 1, 2, 65, 65, 1, 2),
    (4, 4, 128, 1, 2, 65, 200, 1, 2),
    (2, 1, 256, 1, 17, 1030, 300, 3, 2),
    (8, 2, 64, 4, 3, 64, 1, 0, 1),
    (1, 1, 64, 1, 1, 1, 1, 0, 1),
    (4, 2, 128, 1, 3, 5000, 128, 1, 2),
    (2, 2, 64, 1, 2, 4096, 4000, 1, 2),
    (2, 1, 64, 1, 2, 17000, 257, 0, 5),
]


@pytest.mark.parametrize("Hq,Hkv,d,B,T,width,budget,sink,recent", SELECT)
def test_select(gpu, Hq, Hkv, d, B, T, width, budget, sink, recent):
    say("select", Hq, Hkv, d, B, T, width, budget, sink, recent)
    g = torch.Generator().manual_seed(width * 7 + budget)
    blocks = B * width + 2
    table = tables(g, B, width, blocks)
    x = torch.randn(blocks, Hkv, 2, d, generator=g)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    q = torch.randn(B * T, Hq, d, generator=g).bfloat16()
    # rows over the whole range, the last one at the table's end, padding rows between
    pos = torch.randint(0, width * PAGE, (B * T,), generator=g, dtype=torch.int32)
    pos[-1] = width * PAGE - 1
    if B * T > 2:
        pos[1] = -1
        pos[0] = min(budget + 1, width) * PAGE - 1     # one page more than the budget holds
    got = run_select(q, bounds, table, pos, budget, sink, recent, Hkv)
    assert torch.equal(got, R.select(q, bounds, table, pos, budget, sink, recent))


@pytest.mark.parametrize("width,budget", [(4096, 40), (8400, 40), (17000, 300)])
def test_select_every_length(gpu, width, budget):
    """Rows that end in every group of 64 pages, at its start, in it and at its end."""
    g = torch.Generator().manual_seed(width)
    table = tables(g, 1, width, width)
    x = torch.randn(width, 1, 2, 64, generator=g)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    groups = torch.arange((width + 63) // 64)
    last = torch.stack([groups * 64, groups * 64 + torch.randint(1, 63, groups.shape, generator=g),
                        groups * 64 + 63], 1).view(-1).clamp(max=width - 1)
    pos = (last * PAGE + 5).int()
    q = torch.randn(len(pos), 2, 64, generator=g).bfloat16()
    got = run_select(q, bounds, table, pos, budget, 1, 2, 1)
    assert torch.equal(got, R.select(q, bounds, table, pos, budget, 1, 2))


@pytest.mark.parametrize("width,budget", [(300, 40), (1500, 40), (1500, 1400)])
@pytest.mark.parametrize("kind", ["equal", "near", "same", "zero", "nan", "inf", "holes", "few", "past",
                                  "tiny", "huge", "far"])
def test_select_borders(gpu, kind, width, budget):
    """Equal and nearly equal scores, NaN and infinite bounds, pages that are none, positions past
    the table, values at the ends of the type's range, one page far above the others."""
    g = torch.Generator().manual_seed(11)
    Hq, Hkv, d, T = 8, 2, 128, 18
    blocks = width + 5
    table = tables(g, 1, width, blocks)
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    x = torch.randn(blocks, Hkv, 2, d, generator=g)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    pos = torch.randint(width // 2 * PAGE, width * PAGE, (T,), generator=g, dtype=torch.int32)
    if kind == "equal":                 # a few distinct pages, each many times
        bounds = bounds[torch.randint(0, 7, (blocks,), generator=g)].contiguous()
    if kind == "near":                  # all pages alike but for one element's last bit
        bounds[:] = bounds[:1]
        at = torch.randint(0, d, (blocks,), generator=g)
        lines = bits(bounds).view(blocks, Hkv, 2, d)
        lines[torch.arange(blocks), :, 1, at] += 1
        bounds = lines.view(torch.bfloat16)
    if kind == "same":                  # one page, many times
        bounds[:] = bounds[:1]
    if kind == "zero":
        bounds[:] = 0.0
    if kind == "tiny":                  # subnormal operands and products
        bounds = (bounds.float() * 2.0 ** -125).bfloat16()
        q[::2] = (q[::2].float() * 2.0 ** -100).bfloat16()
    if kind == "huge":                  # scores past the 32-bit range
        bounds = (bounds.float() * 2.0 ** 120).bfloat16()
    if kind == "far":
        bounds[5::400] *= 2.0 ** 30
    if kind == "nan":
        bounds[::2, :, 0, 3] = float("nan")
        q[3, 2, 5] = float("nan")       # every score of that row and kv head
    if kind == "inf":
        bounds[::5, :, 1, 3] = float("inf")
        bounds[1::5, :, 0, 4] = float("-inf")
        q[::2, :, 3] = 0.0              # 0 . inf: NaN
    if kind == "holes":
        table[0, 5:60:3] = -1
        table[0, 6:60:3] = blocks
    if kind == "few":                   # fewer pages than the budget
        table[0, 7:] = -1
    if kind == "past":
        pos[::2] = 2 ** 31 - 1
    got = run_select(q, bounds, table, pos, budget, 1, 2, Hkv)
    assert torch.equal(got, R.select(q, bounds, table, pos, budget, 1, 2))


def test_select_rows_in_parts_of_a_wide_table(gpu):
    """The widest table: the rows' scores pass the scratch a part at a time."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(5)
    Hkv, d, T, width, blocks = 8, 64, 34, 1 << 17, 500
    assert ops.page_select_scratch_bytes(1, T, Hkv, Hkv, d, width) < T * Hkv * width * 8
    table = torch.randint(0, blocks, (1, width), generator=g, dtype=torch.int32)
    x = torch.randn(blocks, Hkv, 2, d, generator=g)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    q = torch.randn(T, Hkv, d, generator=g).bfloat16()
    pos = torch.full((T,), width * PAGE - 1, dtype=torch.int32)
    pos[2] = 70000 * PAGE
    got = run_select(q, bounds, table, pos, 600, 1, 2, Hkv)
    for m in (0, 2, 31, 33):            # the rows at the parts' ends
        one = R.select(q[m:m + 1], bounds, table, pos[m:m + 1], 600, 1, 2)
        assert torch.equal(got[m:m + 1], one)


def test_select_no_scratch_when_refused(gpu):
    from snowllm_amd import ops
    from snowllm_amd.errors import SnowLLMError
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    bounds = torch.zeros(9, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, 9, dtype=torch.int32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    pages = torch.zeros(1, 1, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(SnowLLMError, match="scratch"):
        ops.page_select(q, bounds, table, pos, pages, None)
    with pytest.raises(SnowLLMError, match="budget"):
        ops.page_select(q, bounds, table, pos, pages, None, sink=3, recent=2)
    with pytest.raises(SnowLLMError, match="budget"):
        ops.page_select(q, bounds, table, pos, pages, None, sink=1, recent=0)


# ------------------------------------------------------------------------------------------
# attend
# ------------------------------------------------------------------------------------------
def run_attend(q, kp, vp, table, positions, pages, scale):
    from snowllm_amd import ops
    M, Hq, d = q.shape
    B, hkv = table.shape[0], kp.shape[1]
    need = ops.sparse_attention_scratch_bytes(B, M // B, Hq, hkv, d, pages.shape[2])
    scratch = ops.empty_bytes(need) if need else None
    out = torch.full((M, Hq, d), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.sparse_attention(q.cuda(), kp.cuda(), vp.cuda(), out, table.cuda(), positions.cuda(),
                         pages.cuda(), scale, scratch)
    torch.cuda.synchronize()
    return out.cpu()


def check_attend(got, q, kp, vp, table, positions, pages, scale):
    want, size, reach = R.attend(q, kp, vp, table, positions, pages, scale)
    keys = pages.shape[2] * PAGE
    weight = (q.shape[2] + 4) * U * reach + 2.0 ** -16 + (keys + 64) * U
    tol = BF * want.abs() + 2 * weight * size + 1e-30
    err = (got.double() - want).abs()
    ok = (err <= tol) | (want.isnan() & got.isnan()) | (got.double() == want)
    assert ok.all(), float((err / tol).nan_to_num(1e9).max())


ATTEND = [
    # Hq, Hkv, d, batch, T, width, budget
    (16, 2, 256, 1, 1, 40, 16),
    (32, 8, 128, 2, 1, 30, 64),
    (4, 1, 64, 3, 7, 9, 5),
    (32, 1, 64, 1, 2, 12, 12),
    (20, 1, 256, 1, 3, 20, 9),
    (5, 5, 128, 2, 3, 10, 1),
    (40, 2, 128, 1, 1, 70, 33),
    (12, 1, 256, 2, 1, 6, 2),
    (16, 2, 64, 2, 150, 8, 7),
    (3, 3, 256, 1, 1, 140, 131),
    (8, 8, 64, 2, 40, 20, 17),
    # many rows one by one
    (16, 2, 256, 1, 517, 30, 12),
    (8, 2, 128, 2, 600, 25, 20),
    (16, 1, 64, 1, 520, 20, 20),
    (3, 3, 64, 1, 700, 6, 1),
    # rows over the union of their lists: 2, 4, 4, 3, 4 rows a tile, a last group that is not full
    (32, 4, 256, 1, 397, 30, 12),
    (8, 2, 128, 2, 789, 25, 20),
    (15, 5, 256, 2, 310, 12, 9),
    (20, 4, 128, 1, 590, 40, 130),
    (4, 4, 128, 1, 799, 6, 1),
    # the same with lists that have little in common
    (32, 4, 256, 1, 397, 90, 12),
    (16, 4, 128, 1, 801, 200, 20),
    (24, 8, 256, 1, 390, 40, 9),
]


@pytest.mark.parametrize("Hq,Hkv,d,B,T,width,budget", ATTEND)
def test_attend(gpu, Hq, Hkv, d, B, T, width, budget):
    say("attend", Hq, Hkv, d, B, T, width, budget)
    g = torch.Generator().manual_seed(budget * 31 + d)
    M, blocks = B * T, B * width + 2
    table = tables(g, B, width, blocks)
    kp, vp = pools(g, blocks, Hkv, d)
    q = torch.randn(M, Hq, d, generator=g).bfloat16()
    pos = torch.randint(0, width * PAGE, (M,), generator=g, dtype=torch.int32)
    pos[-1] = width * PAGE - 1
    # lists in any order, -1 among them, pages past the row's position
    pages = torch.randint(-1, width, (M, Hkv, budget), generator=g, dtype=torch.int32)
    if T > 300:        # ascending, as they are chosen; a few rows in any order
        keep = pages[::97].clone()
        pages = torch.stack([torch.randperm(width, generator=g)[:min(budget, width)].sort().values
                             for _ in range(M * Hkv)]).int()
        pages = torch.nn.functional.pad(pages, (0, max(0, budget - width)), value=-1).view(M, Hkv, budget)
        pages[::97] = keep
    if M > 2:
        pos[0], pos[1] = 0, -1
        pages[2] = -1
        pages[0, :, 0] = 0
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)
    if M > 2:
        assert (got[1:3] == 0).all()


@pytest.mark.parametrize("kind", ["dead", "holes", "twice", "past", "large", "tiny", "other", "ends"])
@pytest.mark.parametrize("T", [1, 130, 799])
def test_attend_borders(gpu, kind, T):
    """NaN and infinities behind the last position, table entries that are no page, listed pages
    outside the table or listed twice, scores that differ by hundreds."""
    g = torch.Generator().manual_seed(8)
    Hq, Hkv, d, width, budget = (16, 4, 128, 24, 20) if T == 799 else (8, 2, 128, 24, 20)
    blocks = width + 4
    table = tables(g, 1, width, blocks)
    kp, vp = pools(g, blocks, Hkv, d)
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    last = 20 * PAGE + 4
    pos = torch.full((T,), last, dtype=torch.int32)
    pages = torch.stack([torch.randperm(21, generator=g)[:budget] for _ in range(T * Hkv)])
    pages = pages.view(T, Hkv, budget).int()
    pages[:, :, 3] = 20                  # the page that the row ends in
    if T == 799:                         # ascending: rows over the union of their lists
        pages = torch.stack([torch.randperm(20, generator=g)[:budget - 2].sort().values
                             for _ in range(T * Hkv)]).view(T, Hkv, -1).int()
        pages = torch.cat([pages, torch.full((T, Hkv, 1), 20), torch.full((T, Hkv, 1), -1)], 2).int()
    if kind == "dead":
        blk = int(table[0, 20])
        kp[blk, :, :, 5:] = float("nan")
        vp[blk, :, 1, :, 1:] = float("inf")
        vp[blk, :, 2:] = float("nan")
    if kind == "holes":
        table[0, 3], table[0, 7], table[0, 11] = -1, blocks, 2 ** 31 - 1
    if kind == "twice":
        pages[:, :, 1::2] = pages[:, :, :1]
    if kind == "past":
        pages[:, :, ::3] = 2 ** 31 - 1
        pages[:, :, 1::3] = -2 ** 31
    if kind == "large":
        q *= 64
    if kind == "other":                  # pages that only some rows list hold no numbers
        bad = table[0, 7].long()
        vp[bad, 0, 2, 5, 1], vp[bad, 1, 0, 3, 2], kp[bad, 1, 2, 4, 5] = float("nan"), float("inf"), float("nan")
        pages[::2] = torch.where(pages[::2] == 7, -1, pages[::2]).sort(dim=2, descending=False).values
        pages[::2] = torch.where(pages[::2] == -1, 2 ** 30, pages[::2]).sort(dim=2).values
    if kind == "ends":                   # rows of a group end in the same page, or pages apart
        pos = (last - torch.arange(T) % 37).int()
        vp[int(table[0, 20]), :, 1:, :, 1:] = float("nan")
        pos[5::11] = -1
    if kind == "tiny":
        q *= 2.0 ** -100
    got = run_attend(q, kp, vp, table, pos, pages, d ** -0.5)
    check_attend(got, q, kp, vp, table, pos, pages, d ** -0.5)


def test_offsets_past_32_bits(gpu):
    """Pools of more than 2^31 elements: the last blocks are written, bounded, chosen and read."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(2)
    Hq, Hkv, d, blocks, width = 16, 8, 128, 140000, 12
    assert blocks * Hkv * PAGE * d > 2 ** 31
    kp = torch.empty(blocks, Hkv, d // 16, PAGE, 16, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty(blocks, Hkv, 4, d, 4, dtype=torch.bfloat16, device="cuda")
    bounds = torch.empty(blocks, Hkv, 2, d, dtype=torch.bfloat16, device="cuda")
    table = (blocks - 1 - torch.arange(width)).int().view(1, width)
    T = width * PAGE
    k, v = (torch.randn(T, Hkv, d, generator=g).bfloat16() for _ in range(2))
    none = torch.zeros(T, 0, device="cuda")
    st, ct = torch.zeros(1, dtype=torch.int32), torch.tensor([T], dtype=torch.int32)
    ops.kv_append(k.cuda(), v.cuda(), none, none, kp, vp, table.cuda(), st.cuda(), ct.cuda(),
                  bounds=bounds)
    small = table.long()[0].flip(0)
    lk, lv, lb = (x[blocks - width:].cpu() for x in (kp, vp, bounds))
    ltable = (width - 1 - torch.arange(width)).int().view(1, width)
    assert torch.equal(R.key(lk, width - 1, 3), k[3]) and torch.equal(R.value(lv, 0, 15), v[T - 1])
    assert torch.equal(lb.float(), R.page_limits(lk, lb, ltable, st, ct, T).float())
    bounds[blocks - width:] = 0
    ops.page_bounds(kp, bounds, table.cuda(), st.cuda(), ct.cuda(), T)
    assert torch.equal(bounds[blocks - width:].cpu(), lb) and len(small) == width
    q = torch.randn(1, Hq, d, generator=g).bfloat16()
    pos = torch.tensor([T - 1], dtype=torch.int32)
    scratch = ops.empty_bytes(ops.page_select_scratch_bytes(1, 1, Hq, Hkv, d, width))
    pages = torch.empty(1, Hkv, 6, dtype=torch.int32, device="cuda")
    ops.page_select(q.cuda(), bounds, table.cuda(), pos.cuda(), pages, scratch)
    assert torch.equal(pages.cpu(), R.select(q, lb, ltable, pos, 6, 1, 2))
    out = torch.empty(1, Hq, d, dtype=torch.bfloat16, device="cuda")
    need = ops.sparse_attention_scratch_bytes(1, 1, Hq, Hkv, d, 6)
    ops.sparse_attention(q.cuda(), kp, vp, out, table.cuda(), pos.cuda(), pages, d ** -0.5,
                         ops.empty_bytes(need) if need else None)
    check_attend(out.cpu(), q, lk, lv, ltable, pos, pages.cpu(), d ** -0.5)


# ------------------------------------------------------------------------------------------
# the four together
# ------------------------------------------------------------------------------------------
class Cache:
    """A layer's cache and buffers, as a decoding program keeps them."""

    def __init__(self, Hq, Hkv, d, half, batch, T, width, budget, seed):
        from snowllm_amd import ops
        self.ops, self.g = ops, torch.Generator(device="cuda").manual_seed(seed)
        self.Hq, self.Hkv, self.d, self.B, self.T, self.M = Hq, Hkv, d, batch, T, batch * T
        blocks = batch * width + 3
        def rand(*s):
            return torch.randn(*s, device="cuda", generator=self.g).bfloat16()
        self.kp, self.vp = rand(blocks, Hkv, d // 16, PAGE, 16), rand(blocks, Hkv, 4, d, 4)
        self.bounds = torch.zeros(blocks, Hkv, 2, d, dtype=torch.bfloat16, device="cuda")
        self.table = torch.randperm(blocks, device="cuda", generator=self.g)[:batch * width].int().view(batch, width)
        self.proj = rand(self.M, (Hq + 2 * Hkv) * d)
        self.cos, self.sin = (torch.rand(self.M, half, device="cuda", generator=self.g) for _ in range(2))
        i32 = dict(dtype=torch.int32, device="cuda")
        self.starts, self.counts = torch.zeros(batch, **i32), torch.full((batch,), T, **i32)
        self.positions = torch.zeros(self.M, **i32)
        self.pages = torch.empty(self.M, Hkv, budget, **i32)
        self.q = torch.zeros(self.M, Hq, d, dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.s1 = ops.empty_bytes(ops.page_select_scratch_bytes(batch, T, Hq, Hkv, d, width))
        self.s2 = ops.empty_bytes(ops.sparse_attention_scratch_bytes(batch, T, Hq, Hkv, d, budget) + 16)

    def at(self, contexts):
        """Stage a block at each request's context; its older pages get their bounds."""
        c = torch.tensor(contexts, dtype=torch.int32, device="cuda")
        self.ops.page_bounds(self.kp, self.bounds, self.table, torch.zeros_like(c), c, max(contexts))
        self.starts.copy_(c)
        self.positions.copy_((c[:, None] + torch.arange(self.T, dtype=torch.int32, device="cuda")).view(-1))

    def step(self):
        Hq, Hkv, d = self.Hq, self.Hkv, self.d
        q = self.proj[:, :Hq * d].unflatten(1, (Hq, d))
        k = self.proj[:, Hq * d:(Hq + Hkv) * d].unflatten(1, (Hkv, d))
        v = self.proj[:, (Hq + Hkv) * d:].unflatten(1, (Hkv, d))
        self.ops.kv_append(k, v, self.cos, self.sin, self.kp, self.vp, self.table, self.starts,
                           self.counts, bounds=self.bounds, q=q, q_out=self.q)
        self.ops.page_select(self.q, self.bounds, self.table, self.positions, self.pages, self.s1)
        self.ops.sparse_attention(self.q, self.kp, self.vp, self.out, self.table, self.positions,
                                  self.pages, d ** -0.5, self.s2)
        return self.out

    def check(self):
        torch.cuda.synchronize()
        q, table, pos = self.q.cpu(), self.table.cpu(), self.positions.cpu()
        kp, vp, bounds = self.kp.cpu(), self.vp.cpu(), self.bounds.cpu()
        # the bounds of every page that a row sees
        live = torch.zeros(self.B, dtype=torch.int32)
        ends = (self.starts + self.counts).cpu()
        assert torch.equal(bounds.float(), R.page_limits(kp, bounds, table, live, ends, int(ends.max())).float())
        pages = R.select(q, bounds, table, pos, self.pages.shape[2], 1, 2)
        assert torch.equal(self.pages.cpu(), pages)
        check_attend(self.out.cpu(), q, kp, vp, table, pos, pages, self.d ** -0.5)


@pytest.mark.parametrize("Hq,Hkv,d,B,T,width,budget", [
    (16, 2, 256, 1, 9, 60, 16), (32, 8, 128, 3, 1, 40, 12), (8, 2, 64, 2, 20, 30, 8)])
def test_step(gpu, Hq, Hkv, d, B, T, width, budget):
    """Append, choose, attend, at contexts that grow (with rejected rows behind them)."""
    c = Cache(Hq, Hkv, d, 32, B, T, width, budget, seed=d + T)
    for contexts in ([300 - 7 * b for b in range(B)], [303 + 5 * b for b in range(B)]):
        say("step", Hq, Hkv, d, B, T, contexts)
        c.at(contexts)
        c.step()
        c.check()


def test_step_with_every_page_is_the_paged_attention(gpu):
    """A budget that holds all pages: the paged attention of the same rows, whose causal block the
    positions give."""
    from snowllm_amd import ops
    c = Cache(16, 2, 256, 32, 2, 9, 20, 20, seed=4)
    c.at([200, 281])
    got = c.step().clone()
    lens = c.starts + c.T
    want = torch.empty_like(got)
    scratch = ops.empty_bytes(ops.paged_attention_explicit_scratch_bytes(2, 9, 16, 2, 256))
    ops.paged_attention_explicit(c.q, c.kp, c.vp, want, c.table, lens, 256 ** -0.5, scratch)
    c.check()
    # both hold the definition to about one bf16 rounding: two roundings apart at most, and the
    # paged attention's own arithmetic (2e-3 of the norm)
    assert ((got.double() - want.double()).norm() / want.double().norm()).item() < 2 * BF + 2e-3


def test_step_in_a_graph_and_on_another_stream(gpu):
    """Captured once, replayed at other contexts between eager steps; each replay against the
    oracle and bit for bit against the eager step."""
    c = Cache(32, 8, 128, 64, 2, 4, 50, 10, seed=6)
    c.at([333, 290])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.step()
    torch.cuda.current_stream().wait_stream(side)
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step()
    for contexts in ([340, 17], [600, 401], [0, 100], [600, 401]):
        say("replay", contexts)
        c.at(contexts)
        eager = c.step().clone()
        torch.cuda.synchronize()
        c.out.fill_(5.0)
        graph.replay()
        c.check()
        assert torch.equal(bits(c.out.cpu()), bits(eager.cpu()))


def test_many_rows_in_two_graphs(gpu):
    """A prompt chunk's step, captured for two caches, replayed in turn and on two streams at once,
    between eager steps."""
    caches = [Cache(32, 4, 256, 32, 1, 397, 60, 8, seed=s) for s in (11, 12)]
    graphs = []
    for c in caches:
        c.at([500])
        c.step()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c.step()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n, contexts in enumerate(([500], [530], [101])):
        say("replay", contexts)
        for c in caches:
            c.at(contexts)
        eager = [c.step().clone() for c in caches]
        for c in caches:
            c.out.fill_(5.0)
            c.pages.fill_(3)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream if n == 2 else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        for c, e in zip(caches, eager):
            assert torch.equal(bits(c.out.cpu()), bits(e.cpu()))
    caches[0].check()


def test_in_place_and_unaligned_views(gpu):
    """q rotated in place, and positions, tables, lists, starts and angles that begin anywhere in
    their buffers."""
    from snowllm_amd import ops
    def inside(t):
        t = t.cuda()
        return torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)
    g = torch.Generator().manual_seed(77)
    Hq, Hkv, d, half, B, T, width, budget = 8, 2, 128, 32, 2, 21, 20, 7
    blocks, M = B * width + 1, B * T
    table = tables(g, B, width, blocks)
    kp, vp = pools(g, blocks, Hkv, d)
    bounds = torch.zeros(blocks, Hkv, 2, d, dtype=torch.bfloat16)
    c = [t.cuda() for t in (kp, vp, bounds)]
    proj = torch.randn(M, Hq + 2 * Hkv, d, generator=g).bfloat16()
    q, k, v = proj[:, :Hq].contiguous(), proj[:, Hq:Hq + Hkv], proj[:, Hq + Hkv:]
    cos, sin = torch.rand(M, half, generator=g), torch.rand(M, half, generator=g)
    st, ct = torch.tensor([200, 31], dtype=torch.int32), torch.tensor([21, 20], dtype=torch.int32)
    pos = (st[:, None] + torch.arange(T, dtype=torch.int32)).view(-1)
    out, qd = torch.zeros_like(q).cuda(), q.cuda()
    ops.page_bounds(c[0], c[2], inside(table), inside(torch.zeros_like(st)), inside(st), 200)
    ops.kv_append(k.cuda(), v.cuda(), inside(cos), inside(sin), c[0], c[1], inside(table), inside(st),
                  inside(ct), bounds=c[2], q=qd, q_out=qd)
    other = torch.full_like(q, 4.0).cuda()
    ops.kv_append(k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), c[0], c[1], table.cuda(), st.cuda(),
                  ct.cuda(), bounds=c[2], q=q.cuda(), q_out=other)
    assert torch.equal(bits(qd[:-1].cpu()), bits(other[:-1].cpu()))
    assert torch.equal(bits(qd[-1].cpu()), bits(q[-1])) and (other[-1] == 4).all()
    scratch = ops.empty_bytes(ops.page_select_scratch_bytes(B, T, Hq, Hkv, d, width))
    pages = inside(torch.zeros(M, Hkv, budget, dtype=torch.int32))
    assert pages.data_ptr() % 16 and pages.is_contiguous()
    ops.page_select(qd, c[2], inside(table), inside(pos), pages, scratch)
    assert torch.equal(pages.cpu(), R.select(qd.cpu(), c[2].cpu(), table, pos, budget, 1, 2))
    need = ops.sparse_attention_scratch_bytes(B, T, Hq, Hkv, d, budget)
    ops.sparse_attention(qd, c[0], c[1], out, inside(table), inside(pos), pages, d ** -0.5,
                         ops.empty_bytes(need) if need else None)
    check_attend(out.cpu(), qd.cpu(), c[0].cpu(), c[1].cpu(), table, pos, pages.cpu(), d ** -0.5)


def test_two_streams_at_once(gpu):
    """Two caches stepped on two streams without an order between them."""
    a, b = Cache(16, 2, 256, 32, 1, 3, 40, 9, seed=1), Cache(16, 2, 256, 32, 1, 3, 40, 9, seed=2)
    a.at([500])
    b.at([611])
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s):
            a.step()
        with torch.cuda.stream(t):
            b.step()
    a.check()
    b.check()


def test_empty_calls(gpu):
    from snowllm_amd import ops
    z = dict(device="cuda")
    kp, vp = (x.cuda() for x in pools(torch.Generator().manual_seed(0), 3, 1, 64))
    table = torch.zeros(2, 3, dtype=torch.int32, **z)
    none = torch.zeros(0, 1, 64, dtype=torch.bfloat16, **z)
    i0, i2 = torch.zeros(0, dtype=torch.int32, **z), torch.zeros(2, dtype=torch.int32, **z)
    cs = torch.zeros(0, 32, **z)
    before = bits(kp.cpu())
    ops.kv_append(none, none, cs, cs, kp, vp, table, i2, i2, q=none, q_out=none.clone())
    bounds = torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16, **z)
    ops.page_bounds(kp, bounds, table, i2, i2, 0)
    ops.page_bounds(kp, bounds, table, i2, i2, 50)          # counts of zero
    ops.page_select(none, bounds, table, i0, torch.zeros(0, 1, 4, dtype=torch.int32, **z), None)
    ops.sparse_attention(none, kp, vp, none.clone(), table, i0, torch.zeros(0, 1, 4, dtype=torch.int32, **z), 1.0)
    # rows, but an empty list, and a table without pages
    q = torch.ones(2, 1, 64, dtype=torch.bfloat16, **z)
    out = torch.ones_like(q)
    ops.sparse_attention(q, kp, vp, out, table, i2, torch.zeros(2, 1, 0, dtype=torch.int32, **z), 1.0)
    assert (out == 0).all()
    pages = torch.zeros(2, 1, 4, dtype=torch.int32, **z)
    wide = torch.zeros(2, 0, dtype=torch.int32, **z)
    ops.page_select(q, bounds, wide, i2, pages, None)
    assert (pages == -1).all() and (bounds == 0).all() and torch.equal(bits(kp.cpu()), before)
