"""The verify step over selected pages (VerifyConfig.sparse_pages): its layers' choice of pages and
attention against oracle/sparse.py on the step's own queries and cache, the step with every page
against the dense step, and a captured step."""
from dataclasses import replace

import pytest
import torch

from oracle import sparse as R
from tests.test_gpu_batch import tiny
from tests.test_gpu_sparse import check_attend

pytestmark = pytest.mark.gpu


def check_layers(m, contexts, lengths):
    c, T = m.cfg, m.cfg.block
    for layer in range(c.layers):
        m.forward(upto_layer=layer + 1)
        torch.cuda.synchronize()
        q, table, pos = m.q.cpu(), m.table.cpu(), m.row_positions.cpu()
        kp, vp, bounds = (x[layer].cpu() for x in (m.k_pools, m.v_pools, m.bounds))
        q[pos < 0] = 0
        zero = torch.zeros(m.batch, dtype=torch.int32)
        ends = torch.tensor([x + n for x, n in zip(contexts, lengths)], dtype=torch.int32)
        want = R.page_limits(kp, bounds, table, zero, ends, int(ends.max()))
        assert torch.equal(bounds.float(), want.float())
        pages = R.select(q, bounds, table, pos, c.sparse_pages, c.sparse_sink, c.sparse_recent)
        assert torch.equal(m.row_pages.cpu(), pages)
        check_attend(m.attn.cpu(), q, kp, vp, table, pos, pages, c.head_dim ** -0.5)
        for b, n in enumerate(lengths):
            assert (m.attn[b * T + n:(b + 1) * T] == 0).all()


@pytest.mark.parametrize("kind", ["moe", "dense"])
def test_step_over_selected_pages(gpu, kind):
    """Two requests, one of them shorter than the block; the blocks cross pages, and a second block
    overwrites rejected rows of the first."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny(kind), sparse_pages=7)
    print("sparse step", kind, flush=True)
    m = VerifyModel(cfg, seed=5, batch=2)
    g = torch.Generator().manual_seed(1)
    for contexts, lengths in (([250, 90], [9, 4]), ([253, 94], [9, 9])):
        m.set_batch(torch.randint(0, cfg.vocab, (2, cfg.block), generator=g), contexts, lengths)
        check_layers(m, contexts, lengths)
        assert m.forward().isfinite().all()


def test_step_with_every_page_is_the_dense_step(gpu):
    """A budget of all pages: the dense step's attention output to its tolerance, layer by layer
    until the first one's difference feeds the next."""
    from snowllm_amd.verify import VerifyModel
    cfg = tiny("dense")
    ids = torch.arange(cfg.block) * 7
    outs = []
    for pages in (0, 64):
        m = VerifyModel(replace(cfg, sparse_pages=pages), seed=3)
        m.set_block(ids)
        m.forward(upto_layer=1)
        torch.cuda.synchronize()
        outs.append(m.attn.double().cpu())
    # each holds the definition to 2e-3 of its norm
    assert ((outs[0] - outs[1]).norm() / outs[0].norm()).item() < 4e-3


def test_step_in_a_graph(gpu):
    """Captured once, replayed at other contexts between eager steps."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny("moe"), sparse_pages=6)
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


def test_refusals(gpu):
    from snowllm_amd.errors import SnowLLMError
    from snowllm_amd.verify import VerifyModel
    cfg = tiny("dense")
    with pytest.raises(SnowLLMError, match="trees"):
        VerifyModel(replace(cfg, sparse_pages=8, tree_parents=(-1, 0, 0, 1, 2, 3, 4, 5, 6)))
    for bad in (dict(sparse_pages=2), dict(sparse_pages=8, sparse_recent=0), dict(sparse_pages=8, sparse_sink=-1)):
        with pytest.raises(SnowLLMError, match="hold"):
            VerifyModel(replace(cfg, **bad))
