"""The verify step over a cache in 8 bits (VerifyConfig.kv8) with one position axis and with several:
each layer's attention against oracle/kv8.py on the step's own queries and cache, the rows that the
cache got, a captured step, a checkpoint, refusals."""
from dataclasses import replace

import pytest
import torch

from oracle import kv8 as R
from oracle import sparse as RS
from tests.test_gpu_batch import tiny
from tests.test_gpu_kv8 import U, check_attention, check_code

pytestmark = pytest.mark.gpu


def check_layers(m, contexts, lengths):
    c, T = m.cfg, m.cfg.block
    starts = torch.tensor(contexts, dtype=torch.int32)
    counts = torch.tensor(lengths, dtype=torch.int32)
    for layer in range(c.layers):
        m.attn.fill_(3.0)
        m.forward(upto_layer=layer + 1)
        torch.cuda.synchronize()
        table, cache = m.table.cpu(), tuple(x.cpu() for x in m.caches[layer])
        tree = None if m.tree is None else m.tree.cpu()
        check_attention(m.attn, *R.attention(m.q.cpu(), cache, table, starts, counts, c.head_dim ** -0.5, T, tree))
        # the block's keys: the projection's, normalised, rotated by the step's angles and quantised
        nq, nk = c.heads * c.head_dim, c.kv_heads * c.head_dim
        k = m.proj.cpu()[:, nq:nq + nk].unflatten(1, (c.kv_heads, c.head_dim))
        y, size = RS.norm_rotate(k, m.layers[layer].k_norm.cpu(), m.cos.cpu(), m.sin.cpu(), c.eps)
        for row, blk, off in RS.slots(table, starts, counts, T, m.blocks):
            code, _, scale, _ = R.code_of(cache, blk, off)
            check_code(code, scale, y[row], (c.head_dim + 12) * U * size[row], "K")


@pytest.mark.parametrize("kind", ["moe", "dense"])
def test_step_over_the_cache_in_8_bits(gpu, kind):
    """Two requests, one of them shorter than the block; the blocks cross pages, and a second block
    overwrites rejected rows of the first."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny(kind), kv8=True)
    print("kv8 step", kind, flush=True)
    m = VerifyModel(cfg, seed=5, batch=2)
    g = torch.Generator().manual_seed(1)
    for contexts, lengths in (([250, 90], [9, 4]), ([253, 94], [9, 9])):
        m.set_batch(torch.randint(0, cfg.vocab, (2, cfg.block), generator=g), contexts, lengths)
        check_layers(m, contexts, lengths)
        logits = m.forward().view(2, cfg.block, -1)
        assert all(logits[b, :n].isfinite().all() for b, n in enumerate(lengths))


def test_tree_with_several_axes(gpu):
    """A tree whose rows have positions of their own on three axes."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny("dense"), kv8=True, tree_parents=(-1, 0, 0, 1, 1, 2, 2, 3, 3),
                  rope_sections=(24, 20, 20), rope_interleaved=True)
    m = VerifyModel(cfg, seed=6)
    ids = torch.arange(cfg.block).view(1, -1) * 5
    m.set_batch(ids, [200])
    text = m.positions.clone()
    assert (text == text[0]).all() and text[0].tolist() == [200, 201, 201, 202, 202, 202, 202, 203, 203]
    at = text.cpu() + torch.tensor([[0], [3], [40]])
    m.set_batch(ids, [200], positions=at.view(3, 1, -1))
    check_layers(m, [200], [9])
    want = R.angles(at, m.inv_freq.cpu(), cfg.rope_sections, True)
    assert ((m.cos.cpu() - want.cos()).abs() <= 8 * U).all() and ((m.sin.cpu() - want.sin()).abs() <= 8 * U).all()


def test_step_in_a_graph(gpu):
    """Captured once, replayed at other contexts between eager steps."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny("moe"), kv8=True, rope_sections=(12, 10, 10))
    m = VerifyModel(cfg, seed=2)
    ids = torch.arange(cfg.block) * 11 % cfg.vocab
    m.set_block(ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.forward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.forward()
    for context in (300, 31, 160, 300):
        m.set_block(ids, context)
        want = m.forward().clone()
        torch.cuda.synchronize()
        m.logits.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(m.logits, want), context


def test_checkpoint_with_the_cache_in_8_bits(gpu, tmp_path):
    from snowllm_amd.checkpoint import load_gguf, model_tensors, save_gguf
    from snowllm_amd.verify import VerifyModel
    m = VerifyModel(replace(tiny("dense"), kv8=True), seed=4, keep_raw=True)
    path = save_gguf(tmp_path / "m.gguf", m.cfg, model_tensors(m))
    n = load_gguf(path, context=120, block=5, kv8=True)
    assert n.cfg.kv8
    n.set_block(torch.arange(5))
    check_layers(n, [120], [5])


def test_refusals(gpu):
    from snowllm_amd.errors import SnowLLMError
    from snowllm_amd.verify import VerifyModel
    cfg = tiny("dense")
    with pytest.raises(SnowLLMError, match="takes the bf16 cache"):
        VerifyModel(replace(cfg, kv8=True, sparse_pages=8))
    with pytest.raises(SnowLLMError, match="do not share"):
        VerifyModel(replace(cfg, rope_sections=(20, 20, 20)))
    with pytest.raises(SnowLLMError, match="four axes"):
        VerifyModel(replace(cfg, rope_sections=(8, 8, 8, 8, 0)))
    with pytest.raises(SnowLLMError, match="take turns"):
        VerifyModel(replace(cfg, rope_sections=(0, cfg.rot_half), rope_interleaved=True))
    m = VerifyModel(replace(cfg, kv8=True), seed=1)
    with pytest.raises(SnowLLMError, match="pages of 16"):
        VerifyModel(replace(cfg, kv8=True, page=32))
    with pytest.raises(SnowLLMError, match="rope_sections"):
        m.set_batch(torch.zeros(1, 9), [10], positions=torch.zeros(3, 1, 9))
    n = VerifyModel(replace(cfg, kv8=True, rope_sections=(cfg.rot_half - 8, 4, 4)), seed=1)
    n.set_block(torch.arange(9))
    kept = n.ids.clone(), n.positions.clone()
    for wrong in ((1, 1, 9), (3, 9), (3, 1, 8)):
        with pytest.raises(SnowLLMError, match="axes of rope_sections"):
            n.set_batch(torch.ones(1, 9), [10], positions=torch.zeros(wrong))
    assert torch.equal(kept[0], n.ids) and torch.equal(kept[1], n.positions)   # nothing was staged
