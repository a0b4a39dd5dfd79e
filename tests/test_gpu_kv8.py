"""The cache in 8 bits against its definitions in 64 bits (oracle/kv8.py): angles of several axes,
quantised write, read back, attention, and the four in a row.

Tolerances count roundings, with u = 2^-24 (fp32) and one rounding to bf16 of at most 2^-8 of the
value. A quantised row: y (rotated: 4 u of its terms, with the norm (d + 8) u) is off by e, its scale
by e + 2 u of it, so a code's place before its rounding by e / scale + 4 u 127: a code is one of those
within half a step and that of the place in 64 bits. The attention's errors are counted in the oracle.
Angles: the reduced turn is rounded once to 32 bits (half a turn: 2 pi 2^-25) and the functions of it
are taken to be within 4 u."""
import pytest
import torch

from oracle import kv8 as R
from oracle import sparse as RS

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = 2.0 ** -8
PAGE = 16
NAN = float("nan")


def say(*a):
    print(*a, flush=True)


def random_cache(g, blocks, hkv, d):
    def codes(*shape):
        return (torch.randn(*shape, generator=g) * 42).round().clamp(-127, 127).to(torch.int8)

    return (codes(blocks, hkv, 4, d // 16, 4, 16), codes(blocks, hkv, d, PAGE),
            0.024 * torch.randn(blocks, hkv, PAGE, generator=g).mul(0.4).exp(),
            0.020 * torch.randn(blocks, hkv, PAGE, generator=g).mul(0.8).exp())


def tables(g, batch, width, blocks):
    return torch.randperm(blocks, generator=g)[:batch * width].int().view(batch, width)


def on_gpu(*xs):
    return [None if x is None else tuple(y.cuda() for y in x) if isinstance(x, tuple) else x.cuda() for x in xs]


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def tree_masks(g, T):
    masks = []
    for t in range(T):
        p = int(torch.randint(max(0, t - 4), t, (1,), generator=g)) if t else -1
        masks.append(1 << t | (masks[p] if t else 0))
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


# ------------------------------------------------------------------------------------------
# angles
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,half,sections,interleaved", [
    (1, 32, (12, 10, 10), True), (9, 32, (12, 10, 10), False), (333, 64, (24, 20, 20), True),
    (7, 5, (5,), False), (7, 5, (5,), True), (100, 9, (3, 2, 2, 2), True), (100, 9, (0, 4, 0, 5), False)])
def test_axes(gpu, M, half, sections, interleaved):
    from snowllm_amd import ops
    say("axes", M, half, sections, interleaved)
    g = torch.Generator().manual_seed(M)
    pos = torch.randint(0, 1 << 20, (len(sections), M), generator=g)
    pos[0, 0], pos[-1, -1] = (1 << 31) - 1, -220000
    freq = (1e7 ** (-torch.arange(half, dtype=torch.float64) / half)).float()
    cos, sin = torch.full((M, half), 9.0).cuda(), torch.full((M, half), 9.0).cuda()
    ops.rope_axes(pos.cuda(), freq.cuda(), cos, sin, sections, interleaved=interleaved)
    want = R.angles(pos, freq, sections, interleaved)
    # the product's 64 bits: 2^-52 of up to 2^31 radians
    tol = 3.1416 * U + 4 * U + 2.0 ** -20 * (want.abs() > 2.0 ** 28)
    assert ((cos.cpu() - want.cos()).abs() <= tol).all()
    assert ((sin.cpu() - want.sin()).abs() <= tol).all()


def test_axes_of_equal_positions_is_the_plain_table(gpu):
    """Text: all axes alike. Near positions: where the 32-bit angles of rope_cos_sin are good."""
    from snowllm_amd import layers, ops
    pos = torch.arange(40).cuda()
    freq = (1e6 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    a, b, c, s = (torch.empty(40, 32, device="cuda") for _ in range(4))
    layers.rope_cos_sin(pos, freq, a, b)
    ops.rope_axes(pos.repeat(3, 1), freq, c, s, (12, 10, 10), interleaved=True)
    assert (a - c).abs().max() <= 40 * U + 8 * U and (b - s).abs().max() <= 40 * U + 8 * U


def test_axes_without_rows(gpu):
    from snowllm_amd import ops
    none = torch.zeros(0, 32).cuda()
    ops.rope_axes(torch.zeros(3, 0, dtype=torch.int64).cuda(), torch.ones(32).cuda(), none, none, (32, 0, 0))


# ------------------------------------------------------------------------------------------
# append and read
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


def check_code(code, scale, y, off, what):
    """Codes and scales of a row y known to `off`."""
    place, want = R.quantise(y)
    off = off + torch.zeros_like(y)
    assert ((scale.double() - want).abs() <= off.amax(-1) / 127 + 2 * U * want).all(), what
    slack = off / want[..., None] + off.amax(-1, keepdim=True) / want[..., None] + 4 * U * 127
    assert ((code.double() - place).abs() <= 0.5 + slack).all(), what
    assert code.abs().max() <= 127


@pytest.mark.parametrize("Hq,Hkv,d,half,norm,T,starts,counts", APPEND)
def test_append_and_read(gpu, Hq, Hkv, d, half, norm, T, starts, counts):
    from snowllm_amd import ops
    say("append", Hq, Hkv, d, half, norm, T, starts, counts)
    g = torch.Generator().manual_seed(T * 1000 + d)
    B = len(starts)
    M = B * T
    width = max(max(s, 0) + T for s in starts) // PAGE + 1
    blocks = B * width + 3
    table = tables(g, B, width, blocks)
    cache = random_cache(g, blocks, Hkv, d)
    n = (Hq + 2 * Hkv) * d
    proj = torch.randn(M, n + 24, generator=g).bfloat16()          # rows at a pitch of their own
    angle = torch.rand(M, half, generator=g) * 6.28
    cos, sin = angle.cos(), angle.sin()
    qg = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16() if norm else None
    kg = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16() if norm else None
    st, ct = ints(starts), ints(counts)

    def cut(p):
        at = (8, 8 + Hq * d, 8 + (Hq + Hkv) * d, 8 + n)
        return [p[:, at[i]:at[i + 1]].unflatten(1, (h, d)) for i, h in enumerate((Hq, Hkv, Hkv))]

    q, k, v = cut(proj)
    qc, kc, vc = cut(proj.cuda())
    gc, gcos, gsin, gt, gs, gn, gqg, gkg = on_gpu(cache, cos, sin, table, st, ct, qg, kg)
    gq = torch.full((M, Hq, d), 7.0).bfloat16().cuda()
    ops.kv8_append(kc, vc, gcos, gsin, gc, gt, gs, gn, q=qc, q_out=gq, q_gamma=gqg, k_gamma=gkg, eps=1e-6)
    torch.cuda.synchronize()

    wk, wv = RS.norm_rotate(k, kg, cos, sin, 1e-6), RS.norm_rotate(q, qg, cos, sin, 1e-6)
    got = [x.cpu() for x in gc]
    written = RS.slots(table, st, ct, T, blocks)
    touched = torch.zeros(blocks, PAGE, dtype=torch.bool)
    for m, blk, off in written:
        touched[blk, off] = True
        ck, cv, ks, vs = R.code_of(got, blk, off)
        check_code(ck, ks, wk[0][m], (d + 12) * U * wk[1][m], "K")
        check_code(cv, vs, v[m].double(), torch.zeros(1), "V")
    # everything else is as it was
    for blk in range(blocks):
        for off in range(PAGE):
            if not touched[blk, off]:
                for a, b in zip(R.code_of(got, blk, off), R.code_of(cache, blk, off)):
                    assert torch.equal(a, b)
    live = torch.zeros(M, dtype=torch.bool)
    for b in range(B):
        if starts[b] >= 0:
            live[b * T:b * T + min(max(counts[b], 0), T)] = True
    tol = BF * wv[0].abs() + (d + 12) * U * wv[1]
    assert ((gq.cpu().double() - wv[0]).abs() <= tol)[live].all()
    assert (gq.cpu()[~live] == 7.0).all()

    # read back: the values the codes stand for, rounded once
    ko, vo = (torch.full((M, Hkv, d), 5.0).bfloat16().cuda() for _ in range(2))
    ops.kv8_read(gc, gt, gs, gn, ko, vo)
    ko, vo = ko.cpu(), vo.cpu()
    for m, blk, off in written:
        ck, cv, ks, vs = R.code_of(got, blk, off)
        assert torch.equal(ko[m], (ck.float() * ks[:, None]).bfloat16())
        assert torch.equal(vo[m], (cv.float() * vs[:, None]).bfloat16())
    rest = torch.ones(M, dtype=torch.bool)
    rest[[m for m, _, _ in written]] = False
    assert (ko[rest] == 5.0).all() and (vo[rest] == 5.0).all()


def test_append_extremes(gpu):
    """Zeros, the smallest and the largest numbers, infinities and NaN; pages without a block."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(3)
    Hkv, d, T, blocks = 2, 64, 20, 6
    table = ints([[3, -1, 2], [0, 6, 5]])
    st, ct = ints([12, 10]), ints([20, 20])
    cache = random_cache(g, blocks, Hkv, d)
    k = torch.randn(2 * T, Hkv, d, generator=g).bfloat16()
    v = torch.randn(2 * T, Hkv, d, generator=g).bfloat16()
    k[0], v[0] = 0.0, -0.0
    k[1] *= 2.0 ** -130
    k[2] *= 2.0 ** -90
    v[1], v[2] = 3.3e38, k[1]
    k[3, 0, 3], k[20, 1, 5], v[21, 0, 7], v[22, 1, 9] = NAN, float("inf"), float("-inf"), -NAN
    none = torch.zeros(2 * T, 0)
    gk, gv, gn, gc, gt, gs, gct = on_gpu(k, v, none, cache, table, st, ct)
    ops.kv8_append(gk, gv, gn, gn, gc, gt, gs, gct)
    ko, vo = torch.zeros_like(gk), torch.zeros_like(gv)
    ops.kv8_read(gc, gt, gs, gct, ko, vo)
    got, ko, vo = [x.cpu() for x in gc], ko.cpu(), vo.cpu()
    written = RS.slots(table, st, ct, T, blocks)
    assert len(written) == 4 + 6                 # pages 1 of both requests have no block
    for m, blk, off in written:
        ck, cv, ks, vs = R.code_of(got, blk, off)
        for code, scale, x, out in ((ck, ks, k[m], ko[m]), (cv, vs, v[m], vo[m])):
            fine = x.isfinite().all(-1)
            assert torch.equal(scale.isnan(), ~fine) and (code[~fine] == 0).all() and out[~fine].isnan().all()
            if fine.any():
                check_code(code[fine], scale[fine], x[fine].double(), torch.zeros(1), "extremes")
                assert torch.equal(out[fine], (code[fine].float() * scale[fine, None]).bfloat16())
    assert (ko[0] == 0).all() and (vo[0] == 0).all() and (ko[1] == 0).all() and (ko[2] != 0).any()
    assert vo[1].isfinite().all()


def test_append_q_in_place_and_without_rows(gpu):
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(5)
    d, T = 128, 6
    cache = random_cache(g, 3, 1, d)
    q, k = torch.randn(T, 2, d, generator=g).bfloat16(), torch.randn(T, 1, d, generator=g).bfloat16()
    angle = torch.rand(T, 64, generator=g)
    gq, gk, gc, cos, sin, gt, gs, gn = on_gpu(q, k, cache, angle.cos(), angle.sin(), ints([[2]]), ints([3]), ints([5]))
    other = torch.zeros_like(gq)
    ops.kv8_append(gk, gk, cos, sin, gc, gt, gs, gn, q=gq, q_out=other)
    ops.kv8_append(gk, gk, cos, sin, gc, gt, gs, gn, q=gq, q_out=gq)
    assert torch.equal(gq[:5], other[:5]) and torch.equal(gq[5].cpu(), q[5])
    none = torch.zeros(0, 1, d).bfloat16().cuda()
    zero = torch.zeros(0, 0).cuda()
    before = [x.clone() for x in gc]
    ops.kv8_append(none, none, zero, zero, gc, gt, gs, gn)
    ops.kv8_read(gc, gt, gs, gn, none, none)
    ops.kv8_attention(none, gc, none, gt, gs, gn, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(before, gc))


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
def form_tables(table, form, Hq, Hkv, d, T):
    """The same requests for one of the attention's two forms: tables of many pages that are not there
    take the one whose tiles of 16 rows of a head share their keys (from 2^21 / d tiles times chunks of
    four pages times heads on)."""
    if form == "tiles":
        return table
    B, width = table.shape
    tiles = -(-T * (Hq // Hkv) // 16)
    most = 4 * -(-(1 << 21) // (d * tiles * B * Hkv))
    return torch.nn.functional.pad(table, (0, max(0, most - width)), value=-1)


FORMS = ["tiles", "ring"]


def run_attention(q, cache, table, starts, counts, scale, tree=None, fill=3.0, out=None):
    from snowllm_amd import ops
    M, Hq, d = q.shape
    B, width = table.shape
    need = ops.kv8_attention_scratch_bytes(B, M // B, Hq, cache[1].shape[1], d, width)
    scratch = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")   # NaN
    out = torch.full((M, Hq, d), fill).bfloat16().cuda() if out is None else out
    ops.kv8_attention(q, cache, out, table, starts, counts, scale, scratch, tree=tree)
    return out


def check_attention(got, want, error, live, fill=3.0):
    got = got.cpu().double()
    assert (got[~live] == fill).all()
    tol = BF * (want.abs() + error) + error
    over = ((got - want).abs() - tol)[live]
    assert got[live].isfinite().all() and (over <= 0).all(), float(over.max())


ATTEND = [
    # Hq, Hkv, d, T, starts, counts, tree
    (16, 2, 256, 1, [0], [1], False),
    (16, 2, 256, 1, [130, 15, 16, 64, 63], [1] * 5, False),
    (8, 2, 64, 1, [1000], [1], False),
    (4, 4, 128, 3, [61, 62, 0], [3, 2, 1], False),
    (32, 8, 128, 9, [100, 7], [9, 9], False),
    (16, 2, 256, 9, [259], [9], False),
    (16, 2, 256, 11, [300, 5], [11, 7], True),
    (6, 2, 64, 17, [40], [17], False),
    (5, 1, 128, 13, [33, 0, 200], [13, 0, 5], False),
    (20, 1, 64, 5, [90], [5], True),
    (2, 2, 128, 64, [70], [64], True),
    (8, 1, 256, 40, [0, 129], [40, 33], False),
    (3, 3, 64, 130, [0, 50], [130, 129], False),
    (16, 1, 128, 2, [-1, 17], [2, 9], False),
    (34, 2, 64, 2, [77], [2], False),
    # requests of very different lengths share the workgroups
    (16, 2, 256, 9, [1700, 3, 800, 0, -1], [9, 9, 4, 1, 9], False),
    (8, 2, 64, 1, [3000, 100, 0, 1999], [1, 1, 1, 0], False),
    (8, 1, 128, 7, [900, 5, 640], [7, 7, 5], True),
    (4, 1, 128, 1, [40 * i for i in range(40)], [1] * 40, False),
    (8, 2, 64, 9, [(53 * i) % 300 for i in range(66)], [9 - i % 10 for i in range(66)], False),
    # tiles of many short prompts
    (32, 16, 128, 64, [11 * i for i in range(16)], [64 - i for i in range(16)], False),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,T,starts,counts,tree", ATTEND)
def test_attention(gpu, Hq, Hkv, d, T, starts, counts, tree, form):
    say("attention", Hq, Hkv, d, T, starts, counts, tree, form)
    g = torch.Generator().manual_seed(Hq * 1000 + T)
    B = len(starts)
    width = max(max(s, 0) + T for s in starts) // PAGE + 1
    blocks = B * width + 3
    table = form_tables(tables(g, B, width, blocks), form, Hq, Hkv, d, T)
    cache = random_cache(g, blocks, Hkv, d)
    q = (torch.randn(B * T, Hq, d, generator=g) * 2).bfloat16()
    masks = torch.cat([tree_masks(g, T) for _ in range(B)]) if tree else None
    st, ct = ints(starts), ints(counts)
    scale = d ** -0.5
    got = run_attention(*on_gpu(q, cache, table, st, ct), scale, on_gpu(masks)[0])
    check_attention(got, *R.attention(q, cache, table, st, ct, scale, T, masks))


@pytest.mark.parametrize("form", FORMS)
def test_attention_over_holes(gpu, form):
    """Pages without a block and positions past the table; a row that sees nothing; masks of nothing;
    NaN in the places that no row sees."""
    g = torch.Generator().manual_seed(11)
    Hq, Hkv, d, T = 16, 2, 128, 4
    table = ints([[3, -1, 2, 9, 1], [-1, -1, -1, -1, -1], [0, 4, 5, 6, 7]])
    table = form_tables(table, form, Hq, Hkv, d, T)
    st, ct = ints([78, 20, 0]), ints([4, 4, 4])
    cache = random_cache(g, 9, Hkv, d)
    for x in cache[2:]:
        x[1, :, 14:] = NAN              # request 0 ends at position 81, its table at 80
        x[0, :, 4:] = NAN
        x[8] = NAN
    q = torch.randn(3 * T, Hq, d, generator=g).bfloat16()
    cache2 = tuple(x.clone() for x in cache)
    got = run_attention(*on_gpu(q, cache2, table, st, ct), -0.3)
    # every row of request 0 sees the NaN place 78
    got2 = got.cpu().double()
    assert got2[0:4].isnan().all() and (got2[4:8] == 0).all()
    for x in cache2[2:]:
        x[1, :, 14:] = 0.02
    want = R.attention(q, cache2, table, st, ct, -0.3, T)
    got = run_attention(*on_gpu(q, cache2, table, st, ct), -0.3)
    check_attention(got, *want)
    # masks: row 0 sees no row of its block, not even itself
    masks = torch.tensor([0, 2, 6, 9] * 3)
    want = R.attention(q, cache2, table, st, ct, 0.1, T, masks)
    got = run_attention(*on_gpu(q, cache2, table, st, ct), 0.1, masks.cuda())
    check_attention(got, *want)
    assert (got.cpu()[8] == 0).all()


@pytest.mark.parametrize("B", [1, 3, 70])
@pytest.mark.parametrize("T,W", [(1, 100), (9, 100), (9, 9000)])
def test_attention_without_blocks_or_pages(gpu, B, T, W):
    """A cache of no blocks, tables of no pages or of none that is there: zeros for every row of a request."""
    Hq, Hkv, d = 16, 2, 128
    g = torch.Generator().manual_seed(20)
    q = torch.randn(B * T, Hq, d, generator=g).bfloat16().cuda()
    counts = torch.tensor([T - b % 2 for b in range(B)], dtype=torch.int32)
    live = torch.arange(T)[None] < counts[:, None]
    empty = (torch.empty(0, Hkv, 4, 8, 4, 16, dtype=torch.int8), torch.empty(0, Hkv, d, 16, dtype=torch.int8),
             torch.empty(0, Hkv, 16), torch.empty(0, Hkv, 16))
    some = random_cache(g, 2, Hkv, d)
    for cache, table in ((empty, torch.zeros(B, W, dtype=torch.int32)), (some, torch.zeros(B, 0, dtype=torch.int32)),
                         (some, torch.full((B, W), -1, dtype=torch.int32)),
                         (some, torch.full((B, W), 2, dtype=torch.int32))):
        starts = torch.tensor([(37 * b) % 1500 for b in range(B)], dtype=torch.int32)
        got = run_attention(*on_gpu(q, cache, table, starts, counts), 0.1).cpu()
        assert (got[live.view(-1)] == 0).all() and (got[~live.view(-1)] == 3).all()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("T,form", [(1, "tiles"), (9, "tiles"), (9, "ring")])
def test_attention_nan_reaches_the_rows_that_see_it(gpu, which, T, form):
    g = torch.Generator().manual_seed(12)
    Hq, Hkv, d = 8, 2, 64
    cache = random_cache(g, 30, Hkv, d)
    table = form_tables(ints([list(range(29, -1, -1))]), form, Hq, Hkv, d, T)
    cache[2 if which == "k" else 3][29 - 2, 1, 5] = NAN          # position 37 of kv head 1
    for start in (0, 37 - T // 2, 400):
        q = torch.randn(T, Hq, d, generator=g).bfloat16()
        got = run_attention(*on_gpu(q, cache, table, ints([start]), ints([T])), 0.1).cpu()
        sees = start + torch.arange(T) >= 37
        assert got[:, :4].isfinite().all()
        assert got[sees, 4:].isnan().all() and got[~sees, 4:].isfinite().all()


def test_attention_of_queries_that_are_not_finite_or_zero(gpu):
    g = torch.Generator().manual_seed(13)
    cache = random_cache(g, 4, 1, 64)
    table, st, ct = ints([[1, 2, 3]]), ints([40]), ints([4])
    q = torch.randn(4, 2, 64, generator=g).bfloat16()
    q[0, 0, 5], q[1, 1, 60], q[2], q[3, 1] = NAN, float("inf"), 0.0, 2.0 ** -120
    got = run_attention(*on_gpu(q, cache, table, st, ct), 1.0).cpu()
    assert got[0, 0].isnan().all() and got[1, 1].isnan().all()
    ok = [(0, 1), (1, 0), (2, 0), (2, 1), (3, 0), (3, 1)]
    q[0, 0], q[1, 1] = 0.0, 0.0
    want, error, _ = R.attention(q, cache, table, st, ct, 1.0, 4)
    for m, h in ok:
        assert ((got[m, h].double() - want[m, h]).abs() <= BF * want[m, h].abs() + (1 + BF) * error[m, h]).all()
    # no scale at all: the mean of the visible values
    got = run_attention(*on_gpu(q, cache, table, st, ct), 0.0).cpu()
    want, error, live = R.attention(q, cache, table, st, ct, 0.0, 4)
    check_attention(got, want, error, live)


def test_attention_of_a_sink_and_small_weights(gpu):
    """One key far above the others whose values are as large: the small weights keep their precision
    (their sum counts as much as the sink's)."""
    g = torch.Generator().manual_seed(14)
    d, n = 128, 6000
    W = (n + PAGE) // PAGE
    cache = list(random_cache(g, W, 1, d))
    cache[2][:] = 1e-3
    cache[3][:] = 0.02
    table = torch.arange(W).int().view(1, W)
    q = torch.ones(1, 4, d).bfloat16()
    cache[0][0, 0, 0, :, 0, :] = 127          # position 0: score 8.7 nats above the mean
    cache[2][0, 0, 0] = 8.7 / 127 / d
    cache = tuple(cache)
    got = run_attention(*on_gpu(q, cache, table, ints([n]), ints([1])), 1.0)
    want, error, live = R.attention(q, cache, table, ints([n]), ints([1]), 1.0, 1)
    check_attention(got, want, error, live)
    # 192 keys at most share the sink's factor: 192 * 33 * 0.47 * 0.02 / 65024 = 9e-4, and 2e-4 from the
    # scores; with one factor for all 6000 it were 3e-2
    assert (error[0] < 2e-3).all()


@pytest.mark.parametrize("Hq,Hkv,d,T,start", [(16, 2, 256, 11, 20011), (16, 2, 256, 11, 50011), (8, 2, 64, 1, 33333), (32, 8, 128, 9, 9001),
                                                   (32, 8, 128, 9, 45001), (16, 2, 64, 33, 62001)])
def test_attention_long(gpu, Hq, Hkv, d, T, start):
    """Many splits, joined."""
    say("long", Hq, Hkv, d, T, start)
    g = torch.Generator().manual_seed(start)
    W = (start + T) // PAGE + 1
    cache = random_cache(g, W, Hkv, d)
    table = tables(g, 1, W, W)
    q = (torch.randn(T, Hq, d, generator=g) * 2).bfloat16()
    masks = tree_masks(g, T) if T == 11 else None
    got = run_attention(*on_gpu(q, cache, table, ints([start]), ints([T])), d ** -0.5, on_gpu(masks)[0])
    # the rows 0 and T - 1 of every head, in full
    rows = [0, T - 1]
    for t in rows:
        if masks is None:
            want, error, _ = R.attention(q[t:t + 1], cache, table, ints([start + t]), ints([1]), d ** -0.5, 1)
        else:
            want, error = whole_tree_row(q, cache, table, start, T, t, masks, d ** -0.5)
        tol = BF * want.abs() + (1 + BF) * error
        assert ((got[t].cpu().double() - want[0]).abs() <= tol[0]).all()


def whole_tree_row(q, cache, table, start, T, t, masks, scale):
    """The oracle for row t of a tree alone."""
    n = start + T
    k, v, ks, vs, there = R.rows_of(cache, table, 0, n)
    vis = R.seen(start, T, t, n, masks[t]) & there
    sub = q[t:t + 1]
    out, error = torch.zeros(1, *q.shape[1:], dtype=torch.float64), torch.zeros(1, *q.shape[1:], dtype=torch.float64)
    hkv = v.shape[1]
    G = q.shape[1] // hkv
    for h in range(hkv):
        key = k[vis, h].double() * ks[vis, h].double()[:, None]
        val = v[vis, h].double() * vs[vis, h].double()[:, None]
        for e in range(G):
            x = sub[0, h * G + e].double()
            s = key @ x * scale
            w = s.softmax(0)
            off = abs(scale) * x.abs().max() / 65024 * key.abs().sum(1).max() + 8 * U * (s.abs().max() + 1)
            big = w @ val.abs()
            wv = w * vs[vis, h].double()
            group = torch.arange(n)[vis] // R.GROUP
            most = R.largest_near(wv, group, n // R.GROUP + 1)
            out[0, h * G + e] = w @ val
            error[0, h * G + e] = (2 * off * big + (most[group] / 65024) @ v[vis, h].double().abs()
                                   + (n / R.GROUP + 64) * U * big)
    return out, error


def test_far_blocks(gpu):
    """Offsets past 2^32 bytes in the pools."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(15)
    Hkv, d, blocks = 8, 256, 140000                    # 32 KiB a block: 4.6 GB a pool
    near = random_cache(g, 3, Hkv, d)
    at = ints([[139999, 70001, 131073]])
    far = (torch.empty(blocks, Hkv, 4, 16, 4, 16, dtype=torch.int8, device="cuda"),
           torch.empty(blocks, Hkv, d, 16, dtype=torch.int8, device="cuda"),
           torch.full((blocks, Hkv, 16), NAN, device="cuda"), torch.full((blocks, Hkv, 16), NAN, device="cuda"))
    for f, x in zip(far, near):
        f[at[0].long().cuda()] = x.cuda()
    q = torch.randn(2, 16, d, generator=g).bfloat16()
    k = torch.randn(2, Hkv, d, generator=g).bfloat16()
    here = ints([[0, 1, 2]])
    none = torch.zeros(2, 0).cuda()
    args = on_gpu(ints([38]), ints([2]))
    small = on_gpu(near)[0]
    ops.kv8_append(k.cuda(), k.cuda(), none, none, far, at.cuda(), *args)
    ops.kv8_append(k.cuda(), k.cuda(), none, none, small, here.cuda(), *args)
    a = run_attention(q.cuda(), far, at.cuda(), *args, 0.06)
    b = run_attention(q.cuda(), small, here.cuda(), *args, 0.06)
    assert torch.equal(a, b) and a.isfinite().all()
    outs = [torch.zeros(80, Hkv, d).bfloat16().cuda() for _ in range(4)]
    whole = on_gpu(ints([0]), ints([40]))
    ops.kv8_read(far, at.cuda(), *whole, *outs[:2])
    ops.kv8_read(small, here.cuda(), *whole, *outs[2:])
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_attention_takes_queries_at_a_pitch_and_repeats(gpu):
    """Views of a projection; the same bits every time, also from another stream."""
    g = torch.Generator().manual_seed(16)
    Hq, Hkv, d, T, n = 8, 2, 128, 3, 3000
    W = (n + T) // PAGE + 1
    cache, table = on_gpu(random_cache(g, W, Hkv, d), tables(g, 1, W, W))
    proj = torch.randn(T, Hq * d + 40, generator=g).bfloat16().cuda()
    q = proj[:, 16:16 + Hq * d].unflatten(1, (Hq, d))
    st, ct = on_gpu(ints([n]), ints([T]))
    a = run_attention(q.contiguous(), cache, table, st, ct, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = run_attention(q, cache, table, st, ct, 0.1)
    side.synchronize()
    assert torch.equal(a, b)


def test_graph(gpu):
    """Write, attention and read back captured once and replayed on other data: the bits of the calls."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(17)
    B, Hq, Hkv, d, T, n = 2, 16, 2, 256, 5, 700
    W = (n + 4 * T) // PAGE + 1
    first = random_cache(g, B * W, Hkv, d)
    cache, table = on_gpu(first, tables(g, B, W, B * W))
    pos = torch.zeros(3, B * T, dtype=torch.int64, device="cuda")
    freq = (1e7 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    cos, sin = torch.empty(B * T, 32, device="cuda"), torch.empty(B * T, 32, device="cuda")
    proj = torch.zeros(B * T, (Hq + 2 * Hkv) * d, dtype=torch.bfloat16, device="cuda")
    q, k, v = (x.unflatten(1, (-1, d)) for x in proj.split([Hq * d, Hkv * d, Hkv * d], 1))
    gamma = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    starts, counts = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    qo, out = (torch.zeros(B * T, Hq, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ko, vo = (torch.zeros(B * T, Hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scratch = ops.empty_bytes(max(16, ops.kv8_attention_scratch_bytes(B, T, Hq, Hkv, d, W)))

    def step():
        ops.rope_axes(pos, freq, cos, sin, (12, 10, 10), interleaved=True)
        ops.kv8_append(k, v, cos, sin, cache, table, starts, counts, q=q, q_out=qo, q_gamma=gamma, k_gamma=gamma)
        ops.kv8_attention(qo, cache, out, table, starts, counts, d ** -0.5, scratch)
        ops.kv8_read(cache, table, starts, counts, ko, vo)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        proj.copy_(torch.randn(proj.shape, generator=g).bfloat16())
        starts.copy_(ints([n + i * T, 3 + 61 * i]))
        counts.copy_(ints([T, T - i]))
        pos.copy_(torch.randint(0, 10000, (3, B * T), generator=g))
        kept = [x.clone() for x in cache]
        for x in (qo, out, ko, vo):
            x.fill_(2.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*cache, qo, out, ko, vo, cos, sin)]
        for x, y in zip(cache, kept):
            x.copy_(y)
        for x in (qo, out, ko, vo):
            x.fill_(2.0)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, (*cache, qo, out, ko, vo, cos, sin)))


def test_two_graphs_share_a_scratch_and_two_streams_do_not(gpu):
    """Graphs of single tokens and of blocks over one scratch, replayed in turn; then both at once, each
    with its own: the bits of the calls."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(21)
    Hq, Hkv, d, n = 16, 2, 128, 5000
    W = n // PAGE + 2
    cache, table = on_gpu(random_cache(g, W, Hkv, d), tables(g, 1, W, W))
    sizes = (1, 9)
    qs = [torch.randn(T, Hq, d, generator=g).bfloat16().cuda() for T in sizes]
    outs = [torch.empty_like(q) for q in qs]
    spans = [on_gpu(ints([n - 77 * T]), ints([T])) for T in sizes]
    needs = [ops.kv8_attention_scratch_bytes(1, T, Hq, Hkv, d, W) for T in sizes]
    assert min(needs) > 0
    shared = ops.empty_bytes(max(needs))
    own = [ops.empty_bytes(x) for x in needs]
    want = [run_attention(q, cache, table, *span, 0.1) for q, span in zip(qs, spans)]
    graphs = []
    for q, out, span in zip(qs, outs, spans):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.kv8_attention(q, cache, out, table, *span, 0.1, shared)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            outs[i].fill_(5.0)
            graphs[i].replay()
            assert torch.equal(outs[i], want[i])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for out in outs:
        out.fill_(5.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                ops.kv8_attention(qs[i], cache, outs[i], table, *spans[i], 0.1, own[i])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_attention_of_many_heads(gpu):
    """More workgroups of heads and rows than 65535: the first and the last heads as by themselves."""
    heads, d, T = 4096, 64, 2049
    W = T // PAGE + 1
    g = torch.Generator(device="cuda").manual_seed(22)
    codes = dict(dtype=torch.int8, device="cuda", generator=g)
    cache = (torch.randint(-127, 128, (W, heads, 4, 4, 4, 16), **codes),
             torch.randint(-127, 128, (W, heads, d, 16), **codes),
             torch.rand(W, heads, 16, device="cuda", generator=g) * 0.02,
             torch.rand(W, heads, 16, device="cuda", generator=g) * 0.02)
    q = torch.empty(T, heads, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    table = torch.randperm(W, device="cuda", generator=g).int()[None]
    span = on_gpu(ints([0]), ints([T]))
    got = run_attention(q, cache, table, *span, 0.1)
    for at in (slice(0, 64), slice(heads - 64, heads)):
        want = run_attention(q[:, at].contiguous(), tuple(x[:, at].contiguous() for x in cache), table, *span, 0.1)
        assert torch.equal(got[:, at], want) and want.isfinite().all()


def test_a_prompt_and_its_continuation(gpu):
    """Angles, writes in chunks, attention of each chunk, then single tokens: every row against the
    attention of the definition over the cache as it then is."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(18)
    Hq, Hkv, d, half = 8, 2, 64, 32
    W = 12
    cache = ops.kv8_cache(W + 2, Hkv, d)
    table = tables(g, 1, W, W + 2)
    gt = table.cuda()
    freq = (1e4 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
    start = 0
    for T in (77, 50, 1, 1, 9, 1):
        x = torch.randn(T, (Hq + 2 * Hkv) * d, generator=g).bfloat16().cuda()
        q, k, v = (y.unflatten(1, (-1, d)) for y in x.split([Hq * d, Hkv * d, Hkv * d], 1))
        pos = (torch.arange(T) + start).repeat(3, 1)
        pos[1] += 3
        cos, sin = torch.empty(T, half, device="cuda"), torch.empty(T, half, device="cuda")
        ops.rope_axes(pos.cuda(), freq, cos, sin, (12, 10, 10))
        st, ct = on_gpu(ints([start]), ints([T]))
        qo = torch.empty(T, Hq, d, dtype=torch.bfloat16, device="cuda")
        ops.kv8_append(k, v, cos, sin, cache, gt, st, ct, q=q, q_out=qo)
        got = run_attention(qo, cache, gt, st, ct, d ** -0.5)
        host = tuple(y.cpu() for y in cache)
        check_attention(got, *R.attention(qo.cpu(), host, table, ints([start]), ints([T]), d ** -0.5, T))
        start += T


def test_refusals_on_the_gpu(gpu):
    from snowllm_amd import ops
    from snowllm_amd.errors import SnowLLMError as Err
    cache = ops.kv8_cache(4, 2, 64)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16).cuda()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16).cuda()
    out = torch.zeros_like(q)
    cs = torch.zeros(2, 32).cuda()
    table, n = ints([[0, 1, 2]]).cuda(), ints([0]).cuda()
    wide = torch.zeros(1, 5000, dtype=torch.int32, device="cuda")
    bad = [
        (lambda: ops.kv8_append(k.float(), k, cs, cs, cache, table, n, n), "bfloat16"),
        (lambda: ops.kv8_append(k, k, cs[:, :30], cs, cache, table, n, n), "half a multiple"),
        (lambda: ops.kv8_append(k, k, cs, cs[:1], cache, table, n, n), "sin: expected shape"),
        (lambda: ops.kv8_append(k, k, cs, cs, cache, table, n, n, q=q), "together"),
        (lambda: ops.kv8_append(k, k[:, :1], cs, cs, cache, table, n, n), "v: expected shape"),
        (lambda: ops.kv8_append(k, k, cs, cs, cache, table.long(), n, n), "int32"),
        (lambda: ops.kv8_append(k, k, cs, cs, (cache[0], cache[1], cache[2].half(), cache[3]), table, n, n), "float32"),
        (lambda: ops.kv8_append(k, k, cs, cs, (cache[0], cache[0], *cache[2:]), table, n, n), "V pool"),
        (lambda: ops.kv8_read(cache, table, n, n, k, k), "must not be"),
        (lambda: ops.kv8_read(cache, table, n, n, k, k[:1]), "v: expected shape"),
        (lambda: ops.kv8_read(cache, table, n, n, k.transpose(0, 1), k), "contiguous"),
        (lambda: ops.kv8_attention(q, cache, q, table, n, n, 1.0), "must not be q"),
        (lambda: ops.kv8_attention(q[:, :3], cache, out, table, n, n, 1.0), "heads"),
        (lambda: ops.kv8_attention(q, cache, out, table, n, n[:0], 1.0), "counts"),
        (lambda: ops.kv8_attention(q, cache, out, wide, n, n, 1.0), "scratch bytes"),
        (lambda: ops.kv8_attention(q, cache, out, wide, n, n, 1.0, torch.zeros(16, dtype=torch.uint8).cuda()), "scratch bytes"),
        (lambda: ops.kv8_attention(q, cache, out, table, n, n, 1.0, tree=table), "tree masks"),
        (lambda: ops.kv8_attention(q, cache, out, table, n, n, float("nan")), "kv8_attention"),
        (lambda: ops.kv8_attention(q.repeat(33, 1, 1), cache, out.repeat(33, 1, 1), table, n, n, 1.0,
                                   tree=torch.zeros(66, dtype=torch.int64).cuda()), "64 rows"),
    ]
    for call, what in bad:
        with pytest.raises(Err, match=what):
            call()
