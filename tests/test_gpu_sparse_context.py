"""The verify step over selected pages at contexts that move back and forth: every step chooses by
bounds that hold all keys of the pages before its block, whatever earlier blocks ended in them."""
from dataclasses import replace

import pytest
import torch

from tests.test_gpu_batch import tiny
from tests.test_gpu_sparse_step import check_layers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["moe", "dense"])
def test_contexts_back_and_forth(gpu, kind):
    """Back and on again behind a page that a block ended in, twice into the same page, and over
    several such pages at once; one of the requests shorter than the block."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny(kind), sparse_pages=6)
    m = VerifyModel(cfg, seed=4, batch=2)
    g = torch.Generator().manual_seed(3)
    for contexts, lengths in (([200, 90], [9, 4]), ([31, 150], [9, 9]), ([160, 17], [9, 2]),
                              ([33, 18], [3, 9]), ([70, 22], [9, 9]), ([250, 240], [5, 9])):
        print("contexts", kind, contexts, lengths, flush=True)
        m.set_batch(torch.randint(0, cfg.vocab, (2, cfg.block), generator=g), contexts, lengths)
        check_layers(m, contexts, lengths)


def test_staged_blocks_that_do_not_run(gpu):
    """Blocks that are staged and left, which would have written the pages again."""
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny("dense"), sparse_pages=6)
    m = VerifyModel(cfg, seed=4)
    ids = torch.arange(cfg.block)
    for context, left in ((31, 39), (140, 36), (250, 133)):
        m.set_block(ids, context)
        check_layers(m, [context], [cfg.block])
        m.set_block(ids, left)


def test_contexts_back_and_forth_in_a_graph(gpu):
    """The same through a captured step, whose bounds are those of the cache after each replay."""
    from oracle import sparse as R
    from snowllm_amd.verify import VerifyModel
    cfg = replace(tiny("dense"), sparse_pages=6)
    m = VerifyModel(cfg, seed=4)
    ids = torch.arange(cfg.block) * 5 % cfg.vocab
    m.set_block(ids)
    m.forward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.forward()
    for context in (31, 160, 40, 230, 31, 250):
        m.set_block(ids, context)
        want = m.forward().clone()
        torch.cuda.synchronize()
        m.logits.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(m.logits, want), context
        zero, end = torch.zeros(1, dtype=torch.int32), torch.tensor([context + cfg.block], dtype=torch.int32)
        for kp, bounds in zip(m.k_pools, m.bounds):
            kp, bounds = kp.cpu(), bounds.cpu()
            limits = R.page_limits(kp, bounds, m.table.cpu(), zero, end, int(end))
            assert torch.equal(bounds.float(), limits.float()), context
