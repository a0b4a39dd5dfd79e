"""The cache in 8 bits where it can go wrong: the ends of the attention's range of values, rows that are not
there or see nothing, writes of many queries, several position axes in the step. Tolerances are those of
test_gpu_kv8.py and of the oracle (oracle/kv8.py)."""
import pytest
import torch

from oracle import kv8 as R
from tests.test_gpu_kv8 import (FORMS, check_attention, check_code, form_tables, ints, on_gpu, random_cache,
                                run_attention, say, tables, tree_masks)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,T,start", [(8, 2, 64, 9, 700), (16, 2, 128, 5, 300), (16, 2, 256, 9, 1500)])
def test_values_near_the_least_scale(gpu, Hq, Hkv, d, T, start, form):
    """Rows of V whose largest magnitudes are from 2^-100 to 2^-98 or, every other page, zeros (whose scale
    is the least one): weights times scales of 2^-107 and less."""
    say("least", Hq, Hkv, d, T, start, form)
    g = torch.Generator().manual_seed(d + T)
    W = (start + T) // 16 + 1
    cache = list(random_cache(g, W, Hkv, d))
    cache[3] = 2.0 ** -100 / 127 * 4 ** torch.rand(W, Hkv, 16, generator=g)
    cache[1][::2], cache[3][::2] = 0, 2.0 ** -100 / 127
    cache = tuple(cache)
    table = form_tables(tables(g, 1, W, W), form, Hq, Hkv, d, T)
    q = (torch.randn(T, Hq, d, generator=g) * 2).bfloat16()
    st, ct = ints([start]), ints([T])
    got = run_attention(*on_gpu(q, cache, table, st, ct), d ** -0.5)
    want, error, live = R.attention(q, cache, table, st, ct, d ** -0.5, T)
    assert (error < 0.1 * want.abs().amax()).all()
    check_attention(got, want, error, live)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,T,start", [(8, 2, 64, 9, 700), (16, 2, 128, 5, 300), (16, 2, 256, 9, 1500)])
def test_values_near_the_largest_number(gpu, Hq, Hkv, d, T, start, form):
    """A key whose score is 2^6 above those before it and whose value is the largest that bf16 holds, so that
    the weights, relative to the row's first keys, times its value are past fp32.
    Relative to the largest score the weights times the values are within it."""
    say("largest", Hq, Hkv, d, T, start, form)
    g = torch.Generator().manual_seed(d + T)
    W = (start + T) // 16 + 1
    cache = list(random_cache(g, W, Hkv, d))
    q = 1 + 0.1 * torch.randn(T, Hq, d, generator=g)
    q = q.bfloat16()
    # scores 0.02 nats about 0, but for position 270: about 4.5
    cache[0] = torch.randint(-127, 128, cache[0].shape, generator=g).to(torch.int8)
    cache[2][:] = 0.02 / 127 / d ** 0.5
    page, at = 270 // 16, 270 % 16
    cache[0][page, :, at // 4, :, at % 4], cache[2][page, :, at] = 127, 4.5 / 127 / d
    cache[3][page, :, at] = 2.0 ** 128 * (1 - 2.0 ** -8) / 127
    cache = tuple(cache)
    table = form_tables(torch.arange(W).int().view(1, W), form, Hq, Hkv, d, T)
    st, ct = ints([start]), ints([T])
    got = run_attention(*on_gpu(q, cache, table, st, ct), 1.0)
    want, error, live = R.attention(q, cache, table, st, ct, 1.0, T)
    assert want.isfinite().all() and (error < 0.1 * want.abs().amax()).all()
    check_attention(got, want, error, live)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,T,start", [(8, 2, 64, 9, 700), (16, 2, 128, 5, 300), (16, 2, 256, 9, 1500)])
def test_keys_and_queries_far_from_one(gpu, Hq, Hkv, d, T, start, form):
    """The largest keys that scores are held for (2^104) against queries of 2^-98, and the other way round:
    keys of 2^-98 against the largest queries."""
    say("far", Hq, Hkv, d, T, start, form)
    g = torch.Generator().manual_seed(d + T)
    W = (start + T) // 16 + 1
    first = random_cache(g, W, Hkv, d)
    table = form_tables(tables(g, 1, W, W), form, Hq, Hkv, d, T)
    x = torch.randn(T, Hq, d, generator=g).clamp(-3, 3)
    st, ct = ints([start]), ints([T])
    # codes of 42, scores of about 42 / 127 * sqrt(d) * 2^6 scale
    for key, query, scale in ((2.0 ** 104, 2.0 ** -98, 2.0 ** -6), (2.0 ** -98, 2.0 ** 126, 2.0 ** -28)):
        cache = (*first[:2], torch.full_like(first[2], key / 127), first[3])
        q = (x * query).bfloat16()
        got = run_attention(*on_gpu(q, cache, table, st, ct), scale)
        want, error, live = R.attention(q, cache, table, st, ct, scale, T)
        assert (error < 0.1 * want.abs().amax()).all()
        check_attention(got, want, error, live)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,T,starts,counts,tree", [
    (8, 1, 64, 9, [3000], [5], False), (16, 2, 256, 9, [2000], [3], True), (32, 8, 128, 4, [700, 90], [1, 3], False),
    (8, 2, 128, 70, [400], [33], False), (64, 8, 64, 9, [6000], [5], False)])
def test_padding_rows_do_not_reach_the_others(gpu, Hq, Hkv, d, T, starts, counts, tree, form):
    """The bits of a request's rows are the same whatever the rows past its count hold."""
    say("padding", Hq, Hkv, d, T, starts, counts, tree, form)
    g = torch.Generator().manual_seed(d + T)
    B = len(starts)
    W = (max(starts) + T) // 16 + 1
    cache = random_cache(g, B * W, Hkv, d)
    table = form_tables(tables(g, B, W, B * W), form, Hq, Hkv, d, T)
    q = torch.randn(B * T, Hq, d, generator=g).bfloat16()
    noise = torch.randn(B * T, Hq, d, generator=g)
    masks = torch.cat([tree_masks(g, T) for _ in range(B)]) if tree else None
    live = (torch.arange(T)[None] < torch.tensor(counts)[:, None]).view(-1)
    gc, gt, gs, gn, gm = on_gpu(cache, table, ints(starts), ints(counts), masks)
    seen = []
    for padding in (torch.zeros_like(noise), noise * 40, noise * 1e30, torch.full_like(noise, float("nan")),
                    torch.full_like(noise, float("inf"))):
        x = torch.where(live[:, None, None], q, padding.bfloat16())
        seen.append(run_attention(x.cuda(), gc, gt, gs, gn, d ** -0.5, gm).cpu())
    check_attention(seen[0], *R.attention(q, cache, table, ints(starts), ints(counts), d ** -0.5, T, masks))
    for other in seen[1:]:
        assert torch.equal(other, seen[0])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,start", [(16, 2, 256, 0), (8, 2, 64, 0), (16, 2, 128, 3000), (8, 1, 128, 300)])
def test_queries_that_are_not_finite_and_see_nothing(gpu, Hq, Hkv, d, start, form):
    """Zeros for a row that sees no key, NaN for one that does: by ancestor masks, over pages without a block."""
    say("nothing", Hq, Hkv, d, start, form)
    g = torch.Generator().manual_seed(d + start)
    T = 8
    W = (start + T) // 16 + 1
    cache = random_cache(g, W, Hkv, d)
    table = tables(g, 1, W, W)
    if start:
        table[0, :start // 16] = -1     # the context has no block but for its last page
        start = start // 16 * 16
    table = form_tables(table, form, Hq, Hkv, d, T)
    q = torch.randn(T, Hq, d, generator=g).bfloat16()
    q[0, :, 3], q[1, 0, 5], q[2, :, 7], q[3, 1, 9] = float("nan"), float("inf"), float("-inf"), float("nan")
    masks = torch.tensor([0, 0, 4, 1, 16, 0, 64, 255])
    args = on_gpu(q, cache, table, ints([start]), ints([T]))
    got = run_attention(*args, d ** -0.5, masks.cuda()).cpu()
    fine = q.isfinite().all(-1)
    nothing = masks == 0
    assert (got[nothing] == 0).all()
    assert got[~nothing][~fine[~nothing]].isnan().all()
    want, error, live = R.attention(torch.where(fine[..., None], q, 0), cache, table, ints([start]), ints([T]),
                                    d ** -0.5, T, masks)
    rest = fine & ~nothing[:, None]
    assert rest.any() and ((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + error) + error)[rest].all()
    # nothing at all
    args[2] = torch.full_like(args[2], -1)
    assert (run_attention(*args, d ** -0.5).cpu() == 0).all()


@pytest.mark.parametrize("writer", ["kv_append", "kv8_append"])
def test_many_queries_as_in_parts(gpu, writer):
    """A cache write whose queries go past the caches (40 MiB of them) and the same rows in two calls whose do
    not: the same bits."""
    from snowllm_amd import ops
    say("many queries", writer)
    Hq, Hkv, d, half, T = 32, 2, 128, 64, 5121
    W = T // 16 + 1
    g = torch.Generator(device="cuda").manual_seed(9)
    bf = dict(dtype=torch.bfloat16, device="cuda")
    q = torch.empty(T, Hq, d, **bf).normal_(generator=g)
    k, v = torch.empty(2, T, Hkv, d, **bf).normal_(generator=g)
    gamma = torch.empty(d, **bf).normal_(generator=g)
    cos, sin = torch.rand(2, T, half, device="cuda", generator=g)
    table = torch.randperm(W, device="cuda", generator=g).int()[None]
    got = []
    for cuts in ((0, T), (0, 2000, T)):
        if writer == "kv8_append":
            cache = list(ops.kv8_cache(W, Hkv, d))
        else:
            cache = [torch.zeros(W, Hkv, d // 16, 16, 16, **bf), torch.zeros(W, Hkv, 4, d, 4, **bf)]
        out = torch.zeros_like(q)
        for a, b in zip(cuts, cuts[1:]):
            rows = slice(a, b)
            span = on_gpu(ints([a]), ints([b - a - (b == T)]))      # the last row is none of the request's
            args = (k[rows], v[rows], cos[rows], sin[rows], *((cache,) if writer == "kv8_append" else cache), table, *span)
            getattr(ops, writer)(*args, q=q[rows], q_out=out[rows], q_gamma=gamma, k_gamma=gamma)
        got.append(cache + [out])
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert (got[0][-1][-1] == 0).all() and (got[0][-1][:-1] != 0).any()


def test_rows_about_the_least_scale_read_back(gpu):
    """Rows whose largest magnitude is below 2^-100 keep what half of the least scale resolves."""
    from snowllm_amd import ops
    g = torch.Generator().manual_seed(8)
    T, Hkv, d = 16, 2, 64
    x = torch.randn(T, Hkv, d, generator=g)
    x = x / x.abs().amax(-1, keepdim=True)
    size = 2.0 ** -torch.tensor([100, 100.2, 101, 102, 103, 104, 105, 106, 107, 108, 108.5, 110, 120, 126, 130, 133])
    x = (x * size[:, None, None]).bfloat16()
    cache = ops.kv8_cache(1, Hkv, d)
    none = torch.zeros(T, 0).cuda()
    args = on_gpu(ints([[0]]), ints([0]), ints([T]))
    ops.kv8_append(x.cuda(), x.cuda(), none, none, cache, *args)
    k, v = torch.ones(2, T, Hkv, d, dtype=torch.bfloat16, device="cuda")
    ops.kv8_read(cache, *args, k, v)
    host = tuple(y.cpu() for y in cache)
    for t in range(T):
        ck, cv, ks, vs = R.code_of(host, 0, t)
        check_code(ck, ks, x[t].double(), torch.zeros(1), "K")
        check_code(cv, vs, x[t].double(), torch.zeros(1), "V")
    # half of the least scale is 2^-107.99: rows of 2^-107 are there, those of 2^-108.5 are not
    there = (size >= 2.0 ** -107)
    for y in (k.cpu(), v.cpu()):
        assert (y[there].abs().amax(-1) > 0).all() and (y[size < 2.0 ** -108.2] == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_queries_below_the_least_unit(gpu, form):
    """Queries of 2^-104 to 2^-102 against keys of 2^104: their scores count."""
    g = torch.Generator().manual_seed(10)
    Hq, Hkv, d, T, start = 16, 2, 128, 5, 300
    W = (start + T) // 16 + 1
    first = random_cache(g, W, Hkv, d)
    cache = (*first[:2], torch.full_like(first[2], 2.0 ** 104 / 127), first[3])
    table = form_tables(tables(g, 1, W, W), form, Hq, Hkv, d, T)
    q = (torch.randn(T, Hq, d, generator=g).clamp(-4, 4) * 2.0 ** -104).bfloat16()
    got = run_attention(*on_gpu(q, cache, table, ints([start]), ints([T])), 0.5)
    want, error, live = R.attention(q, cache, table, ints([start]), ints([T]), 0.5, T)
    mean, _, _ = R.attention(q * 0, cache, table, ints([start]), ints([T]), 0.5, T)
    assert (error < 0.1 * want.abs().amax()).all() and ((want - mean).abs() > error).any(-1).all()
    check_attention(got, want, error, live)


@pytest.mark.parametrize("kind,change", [("dense", {}), ("moe", {}), ("dense", dict(sparse_pages=8)), ("moe", dict(kv8=True))])
def test_step_with_several_axes_over_every_cache(gpu, monkeypatch, kind, change):
    """rope_sections beside each kind of cache: the step's angles are those of the axes, and with the same
    angles the step is the one of a single axis, bit for bit."""
    from dataclasses import replace

    from snowllm_amd import layers, ops
    from snowllm_amd.verify import VerifyModel
    from tests.test_gpu_batch import tiny
    say("step", kind, change)
    cfg = replace(tiny(kind), **change)
    half = cfg.rot_half
    several = replace(cfg, rope_sections=(half - 16, 8, 8), rope_interleaved=False)
    one, m = VerifyModel(cfg, seed=3), VerifyModel(several, seed=3)
    ids = torch.arange(cfg.block).view(1, -1) * 7 % cfg.vocab
    for x in (one, m):
        x.set_batch(ids, [200])
    want = one.forward().clone()
    m.forward()
    angles = R.angles(m.positions.cpu(), m.inv_freq.cpu(), several.rope_sections, False)
    assert ((m.cos.cpu() - angles.cos()).abs() <= 8 * 2.0 ** -24).all()
    assert ((m.sin.cpu() - angles.sin()).abs() <= 8 * 2.0 ** -24).all()
    again = VerifyModel(several, seed=3)
    again.set_batch(ids, [200])
    monkeypatch.setattr(ops, "rope_axes", lambda p, f, c, s, *_, **__: layers.rope_cos_sin(p[0].contiguous(), f, c, s))
    assert torch.equal(again.forward(), want)
