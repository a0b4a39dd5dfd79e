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
import torch

from ._capi import SnowLLMError, check, lib
from ._common import _p

PAGE = 16
HEAD_SIZES = (64, 128, 256)


def _need(t, name, dtype, shape=None):
    """A contiguous tensor of the dtype (and shape), or an error; 0 dims match anything."""
    if t.dtype != dtype:
        raise SnowLLMError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise SnowLLMError(f"{name}: expected a CUDA tensor, got {t.device}")
    if shape is not None and t.shape != shape:
        raise SnowLLMError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise SnowLLMError(f"{name}: must be contiguous")
    if t.data_ptr() % 16:
        raise SnowLLMError(f"{name}: must be 16-byte aligned")


def _rows(t, name, M, heads, d):
    """[M, heads, d] bf16 rows at any pitch: the row stride of the heads' contiguous elements."""
    if t.dtype != torch.bfloat16:
        raise SnowLLMError(f"{name}: expected {torch.bfloat16}, got {t.dtype}")
    if not t.is_cuda:
        raise SnowLLMError(f"{name}: expected a CUDA tensor, got {t.device}")
    if t.shape != (M, heads, d):
        raise SnowLLMError(f"{name}: expected shape {(M, heads, d)}, got {tuple(t.shape)}")
    rs, hs, es = t.stride()
    if es != 1 or (hs != d and heads > 1) or (M > 1 and (rs % 8 or rs < heads * d)):
        raise SnowLLMError(f"{name}: a row's heads must be contiguous and rows a multiple of 8 "
                           f"elements apart, got stride {t.stride()}")
    if t.data_ptr() % 16:
        raise SnowLLMError(f"{name}: must be 16-byte aligned")
    return rs if M > 1 else heads * d


def _one_device(first, *tensors):
    """All on one device, the current one: its stream is what the launch goes to."""
    dev = first.device
    for t in tensors:
        if t is not None and t.device != dev:
            raise SnowLLMError(f"tensors on {dev} and {t.device}")
    if dev.index != torch.cuda.current_device():
        raise SnowLLMError(f"tensors on {dev}, the current device is {torch.cuda.current_device()}")
    return torch.cuda.current_stream().cuda_stream


def _pool(t, name):
    """(blocks, Hkv, d) of a K pool."""
    if t.dim() != 5 or t.shape[3:] != (PAGE, 16) or t.shape[2] * 16 not in HEAD_SIZES:
        raise SnowLLMError(f"{name}: expected [blocks, Hkv, d/16, 16, 16] with d in {HEAD_SIZES}, "
                           f"got {tuple(t.shape)}")
    _need(t, name, torch.bfloat16)
    return t.shape[0], t.shape[1], t.shape[2] * 16


def _requests(table, M):
    """(batch, tokens, pages per request) of M padded rows."""
    if table.dim() != 2:
        raise SnowLLMError(f"block table: expected [batch, pages], got {tuple(table.shape)}")
    _need(table, "block table", torch.int32)
    batch = table.shape[0]
    if batch == 0 and M == 0:
        return 0, 0, table.shape[1]
    if batch == 0 or M % batch:
        raise SnowLLMError("rows are not a whole number of requests")
    return batch, M // batch, table.shape[1]


def _groups(heads, hkv):
    if heads <= 0 or heads % hkv:
        raise SnowLLMError(f"{heads} heads over {hkv} kv heads")


def kv_append(k, v, cos, sin, k_pool, v_pool, table, starts, counts, *, bounds=None, q=None,
              q_out=None, q_gamma=None, k_gamma=None, eps=1e-6):
    """Write counts[b] rows of request b into its pages at positions starts[b], starts[b] + 1, ..

    k, v [batch*tokens, Hkv, d] and q [batch*tokens, Hq, d] bf16, rows at any pitch (views of a
    projection); cos, sin [batch*tokens, half] f32, half % 8 == 0; starts, counts int32 [batch].
    K (and q, into q_out) is normalised per head where its gamma [d] is given, its first 2 half
    elements rotated in the pairs (i, i + half), and rounded once. bounds: those of the pages
    written, over their keys up to the last one written. Rows past a request's count are left as
    they were, in q_out too. Requests must not share the pages they write.
    """
    blocks, hkv, d = _pool(k_pool, "K pool")
    M = k.shape[0]
    batch, tokens, width = _requests(table, M)
    _need(v_pool, "V pool", torch.bfloat16, (blocks, hkv, PAGE // 4, d, 4))
    ks, vs = _rows(k, "k", M, hkv, d), _rows(v, "v", M, hkv, d)
    half = cos.shape[1] if cos.dim() == 2 else -1
    if half < 0 or half % 8 or 2 * half > d:
        raise SnowLLMError(f"cos: expected [rows, half] with half a multiple of 8 up to {d // 2}, "
                           f"got {tuple(cos.shape)}")
    _need(cos, "cos", torch.float32, (M, half))
    _need(sin, "sin", torch.float32, (M, half))
    _need(starts, "starts", torch.int32, (batch,))
    _need(counts, "counts", torch.int32, (batch,))
    if bounds is not None:
        _need(bounds, "bounds", torch.bfloat16, (blocks, hkv, 2, d))
    for t, name in ((q_gamma, "q gamma"), (k_gamma, "k gamma")):
        if t is not None:
            _need(t, name, torch.bfloat16, (d,))
    heads, qs = hkv, 0
    if (q is None) != (q_out is None):
        raise SnowLLMError("q and q_out must be given together")
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        _groups(heads, hkv)
        qs = _rows(q, "q", M, heads, d)
        _need(q_out, "q_out", torch.bfloat16, (M, heads, d))
    stream = _one_device(k, v, q, q_out, cos, sin, k_pool, v_pool, table, starts, counts, bounds,
                         q_gamma, k_gamma)
    check(lib.snowverify_kv_append(k.data_ptr(), ks, v.data_ptr(), vs, _p(q), qs, cos.data_ptr(),
                                   sin.data_ptr(), half, half, _p(q_gamma), _p(k_gamma), eps,
                                   k_pool.data_ptr(), v_pool.data_ptr(), _p(bounds), _p(q_out),
                                   table.data_ptr(), starts.data_ptr(), counts.data_ptr(), batch,
                                   tokens, heads, hkv, d, width, blocks, stream), "kv_append")


def page_bounds(k_pool, bounds, table, starts, counts, tokens):
    """The bounds of the pages that hold positions starts[b] .. starts[b] + counts[b] - 1, over
    their keys up to the last of these, from the K pool: for pages that another writer filled
    (attention.qk_norm_rope_cache, paged_attention_qk, a restored cache). tokens: the most that
    any counts[b] is."""
    blocks, hkv, d = _pool(k_pool, "K pool")
    batch, _, width = _requests(table, table.shape[0])
    _need(bounds, "bounds", torch.bfloat16, (blocks, hkv, 2, d))
    _need(starts, "starts", torch.int32, (batch,))
    _need(counts, "counts", torch.int32, (batch,))
    stream = _one_device(k_pool, bounds, table, starts, counts)
    check(lib.snowverify_page_bounds(k_pool.data_ptr(), bounds.data_ptr(), table.data_ptr(),
                                     starts.data_ptr(), counts.data_ptr(), batch, tokens, hkv, d,
                                     width, blocks, stream), "page_bounds")


def page_select_scratch_bytes(batch, tokens, num_heads, num_kv_heads, head_size, width) -> int:
    """width: pages per request (the table's second dimension)."""
    return int(lib.snowverify_page_select_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                        head_size, width))


def page_select(q, bounds, table, positions, pages, scratch, *, sink=1, recent=2):
    """pages [batch*tokens, Hkv, budget] int32: the pages row m reads, ascending, -1 behind the last.

    q [batch*tokens, Hq, d]; positions int32 [batch*tokens], the last position a row sees (negative:
    a padding row, all -1). Every page where there are at most budget; else the first `sink`, the
    last `recent` (at least 1) and, of the others, those with the largest sum over the kv head's q
    heads and the elements of max(q low, q high), the most that a key within the bounds could
    score; taken in 64 bits, the lowest page first among equals, NaN as -inf.
    """
    if q.dim() != 3 or pages.dim() != 3 or bounds.dim() != 4:
        raise SnowLLMError("expected q [rows, Hq, d], pages [rows, Hkv, budget] and bounds [blocks, Hkv, 2, d]")
    M, heads, d = q.shape
    blocks, hkv = bounds.shape[:2]
    if d not in HEAD_SIZES:
        raise SnowLLMError(f"head size {d} is none of {HEAD_SIZES}")
    batch, tokens, width = _requests(table, M)
    _need(q, "q", torch.bfloat16)
    _need(bounds, "bounds", torch.bfloat16, (blocks, hkv, 2, d))
    _groups(heads, hkv)
    _need(positions, "positions", torch.int32, (M,))
    budget = pages.shape[2]
    _need(pages, "pages", torch.int32, (M, hkv, budget))
    if sink < 0 or recent < 1 or sink + recent > budget:
        raise SnowLLMError(f"a budget of {budget} pages holds {sink} first and {recent} last pages "
                           f"(at least one last)")
    need = page_select_scratch_bytes(batch, tokens, heads, hkv, d, width)
    if need and (scratch is None or scratch.nbytes < need):
        raise SnowLLMError(f"page select needs {need} scratch bytes")
    stream = _one_device(q, bounds, table, positions, pages, scratch)
    check(lib.snowverify_page_select(q.data_ptr(), bounds.data_ptr(), table.data_ptr(),
                                     positions.data_ptr(), pages.data_ptr(), batch, tokens, heads,
                                     hkv, d, width, blocks, budget, sink, recent, _p(scratch),
                                     scratch.nbytes if scratch is not None else 0, stream),
          "page_select")


def sparse_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads, head_size, budget) -> int:
    return int(lib.snowverify_sparse_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                             head_size, budget))


def sparse_attention(q, k_pool, v_pool, out, table, positions, pages, scale, scratch=None):
    """out[m, h] = softmax(scale q k^T) v over the keys at positions <= positions[m] of the pages
    listed for row m and head h's kv head.

    q, out [batch*tokens, Hq, d]; positions int32 [batch*tokens]; pages int32 [batch*tokens, Hkv,
    budget] as page_select gives them, or any other: -1, pages past the row's position and pages
    outside the table are passed over, a page counts as often as it is listed, order is free. A
    row that sees no key gets zeros. scratch: sparse_attention_scratch_bytes (may be 0: None).
    """
    blocks, hkv, d = _pool(k_pool, "K pool")
    if q.dim() != 3 or pages.dim() != 3:
        raise SnowLLMError("expected q [rows, Hq, d] and pages [rows, Hkv, budget]")
    M, heads = q.shape[:2]
    batch, tokens, width = _requests(table, M)
    _need(q, "q", torch.bfloat16, (M, heads, d))
    _need(out, "out", torch.bfloat16, (M, heads, d))
    _groups(heads, hkv)
    _need(v_pool, "V pool", torch.bfloat16, (blocks, hkv, PAGE // 4, d, 4))
    _need(positions, "positions", torch.int32, (M,))
    budget = pages.shape[2]
    _need(pages, "pages", torch.int32, (M, hkv, budget))
    need = sparse_attention_scratch_bytes(batch, tokens, heads, hkv, d, budget)
    if need and (scratch is None or scratch.nbytes < need):
        raise SnowLLMError(f"sparse attention needs {need} scratch bytes")
    stream = _one_device(q, k_pool, v_pool, out, table, positions, pages, scratch)
    check(lib.snowverify_sparse_attention(q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                                          out.data_ptr(), table.data_ptr(), positions.data_ptr(),
                                          pages.data_ptr(), batch, tokens, heads, hkv, d, width,
                                          blocks, budget, float(scale), _p(scratch),
                                          scratch.nbytes if scratch is not None else 0, stream),
          "sparse_attention")
