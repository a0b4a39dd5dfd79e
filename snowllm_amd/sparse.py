"""Attention over selected pages of the paged KV cache (extension): a row reads a bounded number
of pages of a long context, chosen by the bounds of their keys.

    kv_append         the cache write of new rows (norm, rotation), with the bounds of their pages
    page_bounds       the bounds of pages that another writer filled
    page_select       the pages each row reads
    sparse_attention  softmax attention over them

Pools as in attention.py: K [blocks, Hkv, d/16, 16, 16], V [blocks, Hkv, 4, d, 4]; bounds [blocks,
Hkv, 2, d] (element-wise minimum and maximum of a page's keys), all bf16. Rows are padded [batch,
tokens]: row t of request b is row b * tokens + t, request b's page p is block table[b, p]. Nothing
allocates or synchronises, and no scratch is shared between calls.
"""
from functools import lru_cache

import torch

from ._capi import SnowLLMError, check, lib

PAGE = 16
HEAD_SIZES = (64, 128, 256)
BF16, I32, F32 = torch.bfloat16, torch.int32, torch.float32


# The checks are most of what a small call costs on the host, so a tensor that passes is looked at
# once per property; what is wrong is found out afterwards.
def _need(t, name, dtype, shape, dev):
    """The address of a contiguous tensor of this dtype, shape and device (bf16: 16-byte aligned)."""
    if t.dtype != dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        _refuse(t, name, dtype, shape, dev)
    p = t.data_ptr()
    if p & 15 and dtype is BF16:
        raise SnowLLMError(f"{name}: must be 16-byte aligned")
    return p


def _refuse(t, name, dtype, shape, dev):
    if t.dtype != dtype:
        raise SnowLLMError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise SnowLLMError(f"{name}: expected a CUDA tensor, got {t.device}")
    if t.get_device() != dev:
        raise SnowLLMError(f"{name}: expected a tensor on cuda:{dev}, got {t.device}")
    if t.shape != shape:
        raise SnowLLMError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    raise SnowLLMError(f"{name}: must be contiguous")


def _rows(t, name, shape, dev):
    """(address, row stride) of [M, heads, d] bf16 rows at any pitch, each row's heads contiguous."""
    M, heads, d = shape
    if t.dtype != BF16 or t.get_device() != dev or t.shape != shape:
        _refuse(t, name, BF16, shape, dev)
    rs, hs, es = t.stride()
    if es != 1 or (hs != d and heads > 1) or (M > 1 and (rs % 8 or rs < heads * d)):
        raise SnowLLMError(f"{name}: a row's heads must be contiguous and rows a multiple of 8 "
                           f"elements apart, got stride {t.stride()}")
    p = t.data_ptr()
    if p & 15:
        raise SnowLLMError(f"{name}: must be 16-byte aligned")
    return p, rs if M > 1 else heads * d


def _stream(dev):
    """The current stream of the tensors' device, which has to be the current one."""
    if dev != torch._C._cuda_getDevice():
        raise SnowLLMError(f"tensors on cuda:{dev}, the current device is {torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(dev)


def _pool(t, name):
    """(address, blocks, Hkv, d, device) of a K pool."""
    shape = t.shape
    if len(shape) != 5 or shape[3] != PAGE or shape[4] != 16 or shape[2] * 16 not in HEAD_SIZES:
        raise SnowLLMError(f"{name}: expected [blocks, Hkv, d/16, 16, 16] with d in {HEAD_SIZES}, "
                           f"got {tuple(shape)}")
    dev = t.get_device()
    if dev < 0:
        _refuse(t, name, BF16, shape, dev)
    blocks, hkv, d16 = shape[:3]
    return _need(t, name, BF16, shape, dev), blocks, hkv, d16 * 16, dev


def _requests(table, M, dev):
    """(address, batch, tokens, pages per request) of the block table of M padded rows."""
    shape = table.shape
    if len(shape) != 2:
        raise SnowLLMError(f"block table: expected [batch, pages], got {tuple(shape)}")
    p = _need(table, "block table", I32, shape, dev)
    batch, width = shape
    if M == 0:
        return p, batch, 0, width
    if batch == 0 or M % batch:
        raise SnowLLMError("rows are not a whole number of requests")
    return p, batch, M // batch, width


def _scratch(scratch, need, what, dev):
    if not need:
        return 0, 0
    if scratch is None or scratch.nbytes < need or not scratch.is_contiguous():
        raise SnowLLMError(f"{what} needs {need} scratch bytes")
    if scratch.get_device() != dev:
        raise SnowLLMError(f"scratch: expected a tensor on cuda:{dev}, got {scratch.device}")
    p = scratch.data_ptr()
    if p & 15:
        raise SnowLLMError("scratch: must be 16-byte aligned")
    return p, scratch.nbytes


def _groups(heads, hkv):
    if heads <= 0 or hkv <= 0 or heads % hkv:
        raise SnowLLMError(f"{heads} heads over {hkv} kv heads")


def kv_append(k, v, cos, sin, k_pool, v_pool, table, starts, counts, *, bounds=None, q=None,
              q_out=None, q_gamma=None, k_gamma=None, eps=1e-6):
    """Write counts[b] rows of request b into its pages at positions starts[b], starts[b] + 1, ..

    k, v [batch*tokens, Hkv, d] and q [batch*tokens, Hq, d] bf16, rows at any pitch (views of a
    projection); cos, sin [batch*tokens, half] f32, half % 8 == 0; starts, counts int32 [batch].
    K (and q, into q_out) is normalised per head where its gamma [d] is given, its first 2 half
    elements rotated in the pairs (i, i + half), and rounded once. bounds: those of the pages
    written, over their keys up to the last one written. q_out may be q. Rows past a request's count
    are left as they were, in q_out too. Requests must not share the pages they write.
    """
    kp, blocks, hkv, d, dev = _pool(k_pool, "K pool")
    M = k.shape[0]
    tp, batch, tokens, width = _requests(table, M, dev)
    vp = _need(v_pool, "V pool", BF16, (blocks, hkv, PAGE // 4, d, 4), dev)
    rows = (M, hkv, d)
    k_at, ks = _rows(k, "k", rows, dev)
    v_at, vs = _rows(v, "v", rows, dev)
    half = cos.shape[1] if cos.dim() == 2 else -1
    if half < 0 or half % 8 or 2 * half > d:
        raise SnowLLMError(f"cos: expected [rows, half] with half a multiple of 8 up to {d // 2}, "
                           f"got {tuple(cos.shape)}")
    cp = _need(cos, "cos", F32, (M, half), dev)
    sp = _need(sin, "sin", F32, (M, half), dev)
    st = _need(starts, "starts", I32, (batch,), dev)
    ct = _need(counts, "counts", I32, (batch,), dev)
    bp = 0 if bounds is None else _need(bounds, "bounds", BF16, (blocks, hkv, 2, d), dev)
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
    check(lib.snowverify_kv_append(k_at, ks, v_at, vs, qp, qs, cp, sp, half, half, qg, kg, eps, kp,
                                   vp, bp, qo, tp, st, ct, batch, tokens, heads, hkv, d, width,
                                   blocks, _stream(dev)), "kv_append")


def page_bounds(k_pool, bounds, table, starts, counts, tokens):
    """The bounds of the pages that hold positions starts[b] .. starts[b] + counts[b] - 1, over
    their keys up to the last of these, from the K pool: for pages that another writer filled
    (attention.qk_norm_rope_cache, paged_attention_qk, a restored cache). tokens: the most that
    any counts[b] is."""
    kp, blocks, hkv, d, dev = _pool(k_pool, "K pool")
    tp, batch, _, width = _requests(table, 0, dev)
    bp = _need(bounds, "bounds", BF16, (blocks, hkv, 2, d), dev)
    st = _need(starts, "starts", I32, (batch,), dev)
    ct = _need(counts, "counts", I32, (batch,), dev)
    check(lib.snowverify_page_bounds(kp, bp, tp, st, ct, batch, tokens, hkv, d, width, blocks,
                                     _stream(dev)), "page_bounds")


@lru_cache(maxsize=256)
def page_select_scratch_bytes(batch, tokens, num_heads, num_kv_heads, head_size, width) -> int:
    """width: pages per request (the table's second dimension). Scratch for the largest of each size
    is enough for smaller ones."""
    return int(lib.snowverify_page_select_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                        head_size, width))


def page_select(q, bounds, table, positions, pages, scratch, *, sink=1, recent=2):
    """pages [batch*tokens, Hkv, budget] int32: the pages row m reads, ascending, -1 behind the last.

    q [batch*tokens, Hq, d]; positions int32 [batch*tokens], the last position a row sees (negative:
    a padding row, all -1). Every page where there are at most budget; else the first `sink`, the
    last `recent` (at least 1) and, of the others, those with the largest sum over the kv head's q
    heads and the elements of max(q low, q high), the most that a key within the bounds could
    score; taken in 64 bits, the lowest page first among equals, a sum with a NaN product (0 . inf)
    as -inf.
    """
    qs, bs, ps = q.shape, bounds.shape, pages.shape
    if len(qs) != 3 or len(ps) != 3 or len(bs) != 4:
        raise SnowLLMError("expected q [rows, Hq, d], pages [rows, Hkv, budget] and bounds [blocks, Hkv, 2, d]")
    M, heads, d = qs
    blocks, hkv = bs[0], bs[1]
    budget = ps[2]
    if d not in HEAD_SIZES:
        raise SnowLLMError(f"head size {d} is none of {HEAD_SIZES}")
    dev = q.get_device()
    if dev < 0:
        _refuse(q, "q", BF16, qs, dev)
    tp, batch, tokens, width = _requests(table, M, dev)
    qp = _need(q, "q", BF16, qs, dev)
    bp = _need(bounds, "bounds", BF16, (blocks, hkv, 2, d), dev)
    _groups(heads, hkv)
    at = _need(positions, "positions", I32, (M,), dev)
    out = _need(pages, "pages", I32, (M, hkv, budget), dev)
    if sink < 0 or recent < 1 or sink + recent > budget:
        raise SnowLLMError(f"a budget of {budget} pages holds {sink} first and {recent} last pages "
                           f"(at least one last)")
    need = page_select_scratch_bytes(batch, tokens, heads, hkv, d, width)
    scp, scn = _scratch(scratch, need, "page select", dev)
    check(lib.snowverify_page_select(qp, bp, tp, at, out, batch, tokens, heads, hkv, d, width, blocks,
                                     budget, sink, recent, scp, scn, _stream(dev)), "page_select")


@lru_cache(maxsize=256)
def sparse_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads, head_size, budget) -> int:
    """For this shape: few rows' lists are split, so fewer rows may need more than many."""
    return int(lib.snowverify_sparse_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                             head_size, budget))


def sparse_attention(q, k_pool, v_pool, out, table, positions, pages, scale, scratch=None):
    """out[m, h] = softmax(scale q k^T) v over the keys at positions <= positions[m] of the pages
    listed for row m and head h's kv head.

    q, out [batch*tokens, Hq, d]; positions int32 [batch*tokens]; pages int32 [batch*tokens, Hkv,
    budget] as page_select gives them, or any other: -1, pages past the row's position and pages
    outside the table are passed over, a page counts as often as it is listed, order is free. A
    row that sees no key, or only keys that score -inf, gets zeros. out must not overlap q. scratch:
    sparse_attention_scratch_bytes (may be 0: None).
    """
    kp, blocks, hkv, d, dev = _pool(k_pool, "K pool")
    qs, ps = q.shape, pages.shape
    if len(qs) != 3 or len(ps) != 3:
        raise SnowLLMError("expected q [rows, Hq, d] and pages [rows, Hkv, budget]")
    M, heads, budget = qs[0], qs[1], ps[2]
    tp, batch, tokens, width = _requests(table, M, dev)
    rows = (M, heads, d)
    qp = _need(q, "q", BF16, rows, dev)
    op = _need(out, "out", BF16, rows, dev)
    if op == qp and M:
        raise SnowLLMError("out must not be q")
    _groups(heads, hkv)
    vp = _need(v_pool, "V pool", BF16, (blocks, hkv, PAGE // 4, d, 4), dev)
    at = _need(positions, "positions", I32, (M,), dev)
    lp = _need(pages, "pages", I32, (M, hkv, budget), dev)
    need = sparse_attention_scratch_bytes(batch, tokens, heads, hkv, d, budget)
    scp, scn = _scratch(scratch, need, "sparse attention", dev)
    check(lib.snowverify_sparse_attention(qp, kp, vp, op, tp, at, lp, batch, tokens, heads, hkv, d,
                                          width, blocks, budget, float(scale), scp, scn, _stream(dev)),
          "sparse_attention")
