"""Refusals of the operators over the cache in 8 bits, without a GPU, and their oracle against plain
loops: the wrappers' checks come before any launch, and the C entry points return
hipErrorInvalidValue for what they do not take."""
import ctypes

import pytest
import torch

from oracle import kv8 as R

BF, I32 = torch.bfloat16, torch.int32
EINVAL = 1


def entry():
    from snowllm_amd import kv8, ops
    from snowllm_amd._capi import lib
    from snowllm_amd.errors import SnowLLMError
    return ops, kv8, lib, SnowLLMError


def test_wrappers_refuse_host_tensors():
    ops, _, _, Err = entry()
    cache = ops.kv8_cache(4, 2, 64, device="cpu")
    k, cs = torch.zeros(2, 2, 64, dtype=BF), torch.zeros(2, 32)
    table, n = torch.zeros(1, 4, dtype=I32), torch.zeros(1, dtype=I32)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.kv8_append(k, k, cs, cs, cache, table, n, n)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.kv8_read(cache, table, n, n, k, k)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.kv8_attention(k, cache, k, table, n, n, 1.0)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.rope_axes(torch.zeros(3, 2, dtype=torch.int64), torch.ones(32), cs, cs, (12, 10, 10))


def test_caches():
    ops, kv8, _, Err = entry()
    cache = ops.kv8_cache(5, 3, 128, device="cpu")
    assert sum(x.nbytes for x in cache) == ops.kv8_bytes(5, 3, 128)
    with pytest.raises(Err, match="head size"):
        ops.kv8_cache(4, 2, 96, device="cpu")
    with pytest.raises(Err, match="expected a cache"):
        kv8._cache(cache[:3])
    for shape in ((4, 2, 4, 6, 4, 16), (4, 2, 4, 4, 16), (4, 2, 4, 4, 16, 4)):
        with pytest.raises(Err, match="K pool: expected"):
            kv8._cache((torch.zeros(shape, dtype=torch.int8), *cache[1:]))


@pytest.mark.parametrize("sections,interleaved,what", [
    ((12, 10), False, "do not share"), ((12, 10, 11), False, "do not share"),
    ((42, -5, -5), False, "do not share"), ((0, 0, 32), True, "cannot take turns"),
    ((8, 12, 12), True, "cannot take turns")])
def test_sections(sections, interleaved, what):
    ops, _, lib, Err = entry()
    pos, f, cs = torch.zeros(3, 2, dtype=torch.int64), torch.ones(32), torch.zeros(2, 32)
    with pytest.raises(Err, match=what):
        ops.rope_axes(pos, f, cs, cs, sections, interleaved=interleaved)
    s = (ctypes.c_int64 * 3)(*(tuple(sections) + (0,))[:3])
    if sum(s) != 32 or min(s) < 0 or interleaved:
        assert lib.snowverify_rope_axes(16, 16, 16, 16, 2, 32, 3, s, interleaved, None) == EINVAL
    with pytest.raises(Err, match="one to four axes"):
        ops.rope_axes(torch.zeros(5, 2, dtype=torch.int64), f, cs, cs, (32, 0, 0, 0, 0))


def attention_args(**change):
    a = dict(q=16, q_stride=512, k=16, v=16, ks=16, vs=16, out=32, table=16, starts=16, counts=16, tree=None,
             batch=1, tokens=2, heads=8, hkv=2, d=64, width=4, blocks=4, scale=1.0, scratch=None, n=0)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [
    dict(d=96), dict(heads=7), dict(hkv=0), dict(batch=-1), dict(tokens=-1), dict(width=-1),
    dict(width=(1 << 26) + 1), dict(blocks=-1), dict(q_stride=513), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(tree=16, tokens=65), dict(q=None), dict(out=None), dict(out=16),
    dict(k=None), dict(vs=None), dict(table=None), dict(starts=None), dict(counts=None),
    dict(batch=1 << 20, tokens=1 << 10), dict(width=4000)])   # the last: no scratch
def test_attention_refuses(change):
    _, _, lib, _ = entry()
    assert lib.snowverify_kv8_attention(*attention_args(**change), None) == EINVAL


def test_attention_takes_no_rows_and_no_grid():
    _, _, lib, _ = entry()
    assert lib.snowverify_kv8_attention(*attention_args(tokens=0), None) == 0
    assert lib.snowverify_kv8_attention(*attention_args(batch=0), None) == 0
    need = lib.snowverify_kv8_attention_scratch_bytes(1, 2, 8, 2, 64, 4000)
    assert need > 0 and need % 16 == 0
    assert lib.snowverify_kv8_attention_scratch_bytes(1, 2, 8, 2, 64, 0) == 0
    assert lib.snowverify_kv8_attention_scratch_bytes(1, 2, 8, 3, 64, 9) == 0
    # more heads' rows than a launch holds, more requests
    assert lib.snowverify_kv8_attention(*attention_args(tokens=1 << 24, heads=4096, hkv=64), None) == 801
    assert lib.snowverify_kv8_attention(*attention_args(batch=70000, scratch=16, n=1 << 60), None) == 801


def append_args(**change):
    a = dict(k=16, ks=128, v=16, vs=128, q=None, qs=0, cos=16, sin=16, cst=32, half=32, qg=None, kg=None,
             eps=1e-6, kp=16, vp=16, ksc=16, vsc=16, qo=None, table=16, starts=16, counts=16, batch=1,
             tokens=1, heads=2, hkv=2, d=64, width=4, blocks=4)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [
    dict(half=4), dict(half=40), dict(half=-8), dict(d=96), dict(ks=12), dict(vs=12), dict(q=16, qs=8),
    dict(k=None), dict(v=None), dict(kp=None), dict(vsc=None), dict(table=None), dict(starts=None),
    dict(counts=None), dict(cos=None), dict(heads=3), dict(width=-1), dict(blocks=-1)])
def test_append_refuses(change):
    _, _, lib, _ = entry()
    assert lib.snowverify_kv8_append(*append_args(**change), None) == EINVAL


@pytest.mark.parametrize("i,value", [(0, None), (3, None), (4, None), (5, None), (6, None), (7, None), (8, None),
                                     (9, -1), (10, -1), (11, 0), (12, 80), (13, -1), (14, -1)])
def test_read_refuses(i, value):
    _, _, lib, _ = entry()
    a = [16] * 9 + [1, 1, 2, 64, 4, 4]
    a[i] = value
    assert lib.snowverify_kv8_read(*a, None) == EINVAL


def test_oracle_against_loops():
    """The oracle's rows, masks and attention against the layout written out."""
    g = torch.Generator().manual_seed(1)
    hkv, d, blocks = 2, 64, 5
    cache = (torch.randint(-127, 128, (blocks, hkv, 4, d // 16, 4, 16), generator=g).to(torch.int8),
             torch.randint(-127, 128, (blocks, hkv, d, 16), generator=g).to(torch.int8),
             torch.rand(blocks, hkv, 16, generator=g), torch.rand(blocks, hkv, 16, generator=g))
    table = torch.tensor([[3, -1, 1]], dtype=I32)
    k, v, ks, vs, there = R.rows_of(cache, table, 0, 40)
    assert there.tolist() == [True] * 16 + [False] * 16 + [True] * 8
    for p, blk in ((0, 3), (5, 3), (33, 1), (39, 1)):
        t = p % 16
        for h, e in ((0, 0), (1, 63), (1, 17)):
            assert k[p, h, e] == cache[0][blk, h, t // 4, e // 16, t % 4, e % 16]
            assert v[p, h, e] == cache[1][blk, h, e, t]
        assert ks[p, 1] == cache[2][blk, 1, t] and vs[p, 0] == cache[3][blk, 0, t]
        ck, cv, cks, _ = R.code_of(cache, blk, t)
        assert torch.equal(ck, k[p]) and torch.equal(cv, v[p]) and torch.equal(cks, ks[p])
    q = torch.randn(3, 4, d, generator=g).bfloat16()
    tree = torch.tensor([1, 3, 5])
    out, _, live = R.attention(q, cache, table, [34], [3], 0.01, 3, tree)
    assert live.all()
    # row 2 sees the context and the block's rows 0 and 2; positions 16 .. 31 have no block
    at = list(range(16)) + [32, 33, 34, 36]
    s = torch.tensor([float((q[2, 3].double() * k[p, 1].double()).sum() * ks[p, 1].double() * 0.01) for p in at],
                     dtype=torch.float64)
    w = (s - s.max()).exp()
    want = sum(w[i] * v[p, 1].double() * vs[p, 1].double() for i, p in enumerate(at)) / w.sum()
    assert torch.allclose(out[2, 3], want, rtol=1e-12, atol=1e-12)
    assert [R.axis_of(i, (4, 3, 1), True) for i in range(8)] == [0, 1, 2, 0, 1, 0, 0, 1]
    assert [R.axis_of(i, (4, 3, 1), False) for i in range(8)] == [0, 0, 0, 0, 1, 1, 1, 2]
