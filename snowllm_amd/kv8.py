"""The paged KV cache in 8 bits (extension): half the bytes of the bf16 cache, for twice the context in
the same memory and an attention that reads half as much.

    rope_axes      cos and sin of positions with several axes (time, height, width)
    kv8_append     the cache write of new rows (norm, rotation), quantised
    kv8_read       cached rows back in bf16
    kv8_attention  softmax attention of new rows over the cache: single tokens, verify blocks and trees,
                   prompts

A cache is (k_pool, v_pool, k_scale, v_scale), as kv8_cache makes it: int8 codes K [blocks, Hkv, 4,
d/16, 4, 16] (token t of a page is group t // 4, place t % 4) and V [blocks, Hkv, d, 16], and one
float32 scale per (token, kv head), [blocks, Hkv, 16]. The row x of a head is held as code * scale,
scale = max(max |x|, 2^-100) / 127; a row with an element that is not finite has a NaN scale (it reads
back as NaN, and rows that see it get NaN). Rows are padded [batch, tokens]: row t of request b is row
b * tokens + t, request b's page p is block table[b, p], its rows lie at positions starts[b],
starts[b] + 1, .. and there are counts[b] of them (more than `tokens` count as tokens; none where the
count or the start is negative). Nothing allocates or synchronises, and no scratch is shared between
calls.
"""
import ctypes
from functools import lru_cache
from typing import NamedTuple

import torch

from ._capi import SnowLLMError, check, lib
from .sparse import (BF16, F32, HEAD_SIZES, I32, PAGE, _groups, _need, _refuse, _requests, _rows,
                     _scratch, _stream)

I8, I64 = torch.int8, torch.int64
MAX_TREE = 64   # rows of a block with ancestor masks


class Kv8Cache(NamedTuple):
    k_pool: torch.Tensor
    v_pool: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv8_cache(blocks, num_kv_heads, head_size, device="cuda") -> Kv8Cache:
    """An empty cache of `blocks` pages."""
    if head_size not in HEAD_SIZES:
        raise SnowLLMError(f"head size {head_size} is none of {HEAD_SIZES}")
    pool = dict(dtype=I8, device=device)
    scale = dict(dtype=F32, device=device)
    return Kv8Cache(torch.zeros(blocks, num_kv_heads, 4, head_size // 16, 4, 16, **pool),
                    torch.zeros(blocks, num_kv_heads, head_size, PAGE, **pool),
                    torch.zeros(blocks, num_kv_heads, PAGE, **scale),
                    torch.zeros(blocks, num_kv_heads, PAGE, **scale))


def kv8_bytes(blocks, num_kv_heads, head_size) -> int:
    """Bytes of a cache."""
    return blocks * num_kv_heads * PAGE * (2 * head_size + 8)


def _cache(cache):
    """(four addresses, blocks, Hkv, d, device) of a cache."""
    if len(cache) != 4:
        raise SnowLLMError("expected a cache (k_pool, v_pool, k_scale, v_scale)")
    k, v, ks, vs = cache
    shape = k.shape
    if len(shape) != 6 or shape[2] != 4 or shape[3] * 16 not in HEAD_SIZES or shape[4] != 4 or shape[5] != 16:
        raise SnowLLMError(f"K pool: expected [blocks, Hkv, 4, d/16, 4, 16] with d in {HEAD_SIZES}, "
                           f"got {tuple(shape)}")
    dev = k.get_device()
    blocks, hkv, d = shape[0], shape[1], shape[3] * 16
    per_token = (blocks, hkv, PAGE)
    # (as _need, in one condition)
    if (dev < 0 or k.dtype is not I8 or v.dtype is not I8 or ks.dtype is not F32 or vs.dtype is not F32
            or v.shape != (blocks, hkv, d, PAGE) or ks.shape != per_token or vs.shape != per_token
            or v.get_device() != dev or ks.get_device() != dev or vs.get_device() != dev
            or not k.is_contiguous() or not v.is_contiguous() or not ks.is_contiguous()
            or not vs.is_contiguous()):
        if dev < 0:
            _refuse(k, "K pool", I8, shape, dev)
        _need(k, "K pool", I8, shape, dev)
        _need(v, "V pool", I8, (blocks, hkv, d, PAGE), dev)
        _need(ks, "K scales", F32, per_token, dev)
        _need(vs, "V scales", F32, per_token, dev)
    kp, vp, ksp, vsp = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if (kp | vp | ksp | vsp) & 15:
        raise SnowLLMError("cache: every part must be 16-byte aligned")
    return kp, vp, ksp, vsp, blocks, hkv, d, dev


def _spans(table, starts, counts, M, dev):
    """(addresses of the three, batch, tokens, pages per request) of M padded rows."""
    shape = table.shape
    # (as _requests and _need, in one condition)
    if (len(shape) == 2 and table.dtype is I32 and starts.dtype is I32 and counts.dtype is I32
            and starts.shape == shape[:1] and counts.shape == shape[:1] and table.get_device() == dev
            and starts.get_device() == dev and counts.get_device() == dev and table.is_contiguous()
            and starts.is_contiguous() and counts.is_contiguous()):
        batch, width = shape
        if batch and M % batch == 0:
            return table.data_ptr(), starts.data_ptr(), counts.data_ptr(), batch, M // batch, width
    tp, batch, tokens, width = _requests(table, M, dev)
    st = _need(starts, "starts", I32, (batch,), dev)
    ct = _need(counts, "counts", I32, (batch,), dev)
    return tp, st, ct, batch, tokens, width


@lru_cache(maxsize=64)
def _sections(sections, axes, half, interleaved):
    """The C array of an axes' sections, checked."""
    if len(sections) != axes or min(sections) < 0 or sum(sections) != half or half < 1:
        raise SnowLLMError(f"sections {sections} do not share {half} pairs between {axes} axes")
    if interleaved and any(n and a + axes * (n - 1) >= half for a, n in enumerate(sections) if a):
        raise SnowLLMError(f"sections {sections} of {half} pairs cannot take turns")
    return (ctypes.c_int64 * axes)(*sections)


def rope_axes(positions, inv_freq, cos, sin, sections, *, interleaved=False):
    """cos, sin [M, half] f32 of the angles positions[axis(i), m] * inv_freq[i], i < half.

    positions int64 [axes, M] (one to four axes); inv_freq f32 [half]; sections: the pairs of every
    axis, half in all. Pairs belong to the axes one section behind the other or, interleaved, in
    turn: pair i to axis i % axes while i // axes < sections[axis], to the first axis else. Angles
    are taken in 64 bits.
    """
    shape = positions.shape
    if len(shape) != 2 or not 1 <= shape[0] <= 4:
        raise SnowLLMError(f"positions: expected [axes, M] with one to four axes, got {tuple(shape)}")
    axes, M = shape
    half = inv_freq.shape[0] if inv_freq.dim() == 1 else 0
    shares = _sections(tuple(sections), axes, half, bool(interleaved))
    dev = positions.get_device()
    if dev < 0:
        _refuse(positions, "positions", I64, shape, dev)
    pp = _need(positions, "positions", I64, shape, dev)
    fp = _need(inv_freq, "inv_freq", F32, (half,), dev)
    cp = _need(cos, "cos", F32, (M, half), dev)
    sp = _need(sin, "sin", F32, (M, half), dev)
    check(lib.snowverify_rope_axes(pp, fp, cp, sp, M, half, axes, shares, interleaved, _stream(dev)), "rope_axes")


def kv8_append(k, v, cos, sin, cache, table, starts, counts, *, q=None, q_out=None, q_gamma=None,
               k_gamma=None, eps=1e-6):
    """Write counts[b] rows of request b into its pages at positions starts[b], starts[b] + 1, ..

    k, v [batch*tokens, Hkv, d] and q [batch*tokens, Hq, d] bf16, rows at any pitch (views of a
    projection); cos, sin [batch*tokens, half] f32, half % 8 == 0; starts, counts int32 [batch].
    K (and q, into q_out) is normalised per head where its gamma [d] is given and its first 2 half
    elements rotated in the pairs (i, i + half); K and V are quantised from fp32, q_out is rounded
    once to bf16 and may be q. Rows past a request's count are left as they were, in the pages and in
    q_out. No page may be written twice in a call: requests must not share those they write, and a
    request's are different ones.
    """
    kp, vp, ksp, vsp, blocks, hkv, d, dev = _cache(cache)
    M = k.shape[0]
    tp, st, ct, batch, tokens, width = _spans(table, starts, counts, M, dev)
    rows = (M, hkv, d)
    k_at, ks = _rows(k, "k", rows, dev)
    v_at, vs = _rows(v, "v", rows, dev)
    half = cos.shape[1] if cos.dim() == 2 else -1
    if half < 0 or half % 8 or 2 * half > d:
        raise SnowLLMError(f"cos: expected [rows, half] with half a multiple of 8 up to {d // 2}, "
                           f"got {tuple(cos.shape)}")
    cp = _need(cos, "cos", F32, (M, half), dev)
    sp = _need(sin, "sin", F32, (M, half), dev)
    qg = 0 if q_gamma is None else _need(q_gamma, "q gamma", BF16, (d,), dev)
    kg = 0 if k_gamma is None else _need(k_gamma, "k gamma", BF16, (d,), dev)
    heads, qp, qs, qo = hkv, 0, 0, 0
    if (q is None) != (q_out is None):
        raise SnowLLMError("q and q_out must be given together")
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        _groups(heads, hkv)
        qp, qs = _rows(q, "q", (M, heads, d), dev)
        qo = _need(q_out, "q_out", BF16, (M, heads, d), dev)
    check(lib.snowverify_kv8_append(k_at, ks, v_at, vs, qp, qs, cp, sp, half, half, qg, kg, eps, kp,
                                    vp, ksp, vsp, qo, tp, st, ct, batch, tokens, heads, hkv, d, width,
                                    blocks, _stream(dev)), "kv8_append")


def kv8_read(cache, table, starts, counts, k, v):
    """k, v [batch*tokens, Hkv, d] bf16: the cached rows at positions starts[b] .. starts[b] +
    counts[b] - 1 of request b, code * scale rounded once. Rows past a request's count, and those of
    pages without a block, are left as they were."""
    kp, vp, ksp, vsp, blocks, hkv, d, dev = _cache(cache)
    M = k.shape[0]
    tp, st, ct, batch, tokens, width = _spans(table, starts, counts, M, dev)
    ko = _need(k, "k", BF16, (M, hkv, d), dev)
    vo = _need(v, "v", BF16, (M, hkv, d), dev)
    if ko == vo and M:
        raise SnowLLMError("v must not be k")
    check(lib.snowverify_kv8_read(kp, vp, ksp, vsp, tp, st, ct, ko, vo, batch, tokens, hkv, d, width,
                                  blocks, _stream(dev)), "kv8_read")


@lru_cache(maxsize=256)
def kv8_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads, head_size, width) -> int:
    """width: pages per request (the table's second dimension). For this shape: few rows' keys are
    split, so fewer rows may need more than many."""
    return int(lib.snowverify_kv8_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                          head_size, width))


def kv8_attention(q, cache, out, table, starts, counts, scale, scratch=None, *, tree=None):
    """out[m, h] = softmax(scale q k^T) v over the cached keys that row m sees.

    q [batch*tokens, Hq, d] bf16, rows at any pitch; out [batch*tokens, Hq, d]; starts, counts int32
    [batch]. Row t of request b sees the positions up to starts[b] + t; with tree (int64 [batch*tokens]
    ancestor masks, at most 64 tokens) those before starts[b] and the block's rows j < counts[b] whose
    bit j is set. The rows' own K and V must be in the cache. Keys in pages without a block, or past
    the table, are passed over; a row that sees no key gets zeros; rows past a request's count are
    left as they were. out must not overlap q. scratch: kv8_attention_scratch_bytes (may be 0: None).

    Range: cached keys up to 2^104 in magnitude, scores and, summed over the keys, a row's values times
    their weights relative to its largest within fp32; beyond that a row may not be finite. Queries
    count from 2^-101 / 32512 on.

    Time: two to 64 requests share the workgroups by their lengths, where there are enough for a split of
    each; one request, or more than 64, are split by the table's width, so that a table much wider
    than its contexts costs time (9 rows of 32 heads of 128 behind 8K tokens 14 us, with a table
    for 131K 66).
    """
    kp, vp, ksp, vsp, blocks, hkv, d, dev = _cache(cache)
    if q.dim() != 3:
        raise SnowLLMError(f"q: expected [rows, Hq, d], got {tuple(q.shape)}")
    M, heads = q.shape[0], q.shape[1]
    tp, st, ct, batch, tokens, width = _spans(table, starts, counts, M, dev)
    _groups(heads, hkv)
    shape = (M, heads, d)
    qp, qs = _rows(q, "q", shape, dev)
    op = _need(out, "out", BF16, shape, dev)
    if op == qp and M:
        raise SnowLLMError("out must not be q")
    if tree is None:
        mp = 0
    else:
        if tokens > MAX_TREE:
            raise SnowLLMError(f"ancestor masks hold {MAX_TREE} rows, got {tokens}")
        mp = _need(tree, "tree masks", I64, (M,), dev)
    need = kv8_attention_scratch_bytes(batch, tokens, heads, hkv, d, width)
    scp, scn = _scratch(scratch, need, "8-bit attention", dev)
    check(lib.snowverify_kv8_attention(qp, qs, kp, vp, ksp, vsp, op, tp, st, ct, mp, batch, tokens, heads,
                                       hkv, d, width, blocks, float(scale), scp, scn, _stream(dev)),
          "kv8_attention")
