"""Refusals of the operators over selected pages, without a GPU: the wrappers' checks come before
any launch, and the C entry points return hipErrorInvalidValue for sizes they do not take."""
import pytest
import torch

from oracle import sparse as R

BF, I32 = torch.bfloat16, torch.int32


def entry():
    from snowllm_amd import ops, sparse
    from snowllm_amd._capi import lib
    from snowllm_amd.errors import SnowLLMError
    return ops, sparse, lib, SnowLLMError


def test_wrappers_refuse_host_tensors():
    ops, _, _, Err = entry()
    kp, vp = torch.zeros(4, 2, 4, 16, 16, dtype=BF), torch.zeros(4, 2, 4, 64, 4, dtype=BF)
    k, cs = torch.zeros(2, 2, 64, dtype=BF), torch.zeros(2, 32)
    table, n = torch.zeros(1, 4, dtype=I32), torch.zeros(1, dtype=I32)
    pages, pos = torch.zeros(2, 2, 4, dtype=I32), torch.zeros(2, dtype=I32)
    bounds = torch.zeros(4, 2, 2, 64, dtype=BF)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.kv_append(k, k, cs, cs, kp, vp, table, n, n)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.page_bounds(kp, bounds, table, n, n, 1)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.page_select(k, bounds, table, pos, pages, None)
    with pytest.raises(Err, match="expected a CUDA tensor"):
        ops.sparse_attention(k, kp, vp, k, table, pos, pages, 1.0)


def test_checks_of_shapes_and_strides():
    _, sparse, _, Err = entry()
    with pytest.raises(Err, match="expected .blocks"):
        sparse._pool(torch.zeros(4, 2, 64, 16, dtype=BF), "K pool")
    with pytest.raises(Err, match="expected .blocks"):
        sparse._pool(torch.zeros(4, 2, 6, 16, 16, dtype=BF), "K pool")       # head size 96
    for heads in (0, 3):
        with pytest.raises(Err, match="heads"):
            sparse._groups(heads, 2)

    class Fake:
        """A device tensor's attributes on the host."""

        def __init__(self, shape, stride, dtype=BF, ptr=0, cuda=True):
            self.shape, self._s, self.dtype, self._p = torch.Size(shape), stride, dtype, ptr
            self.is_cuda, self.device = cuda, "cuda:0"

        def stride(self):
            return self._s

        def data_ptr(self):
            return self._p

        def get_device(self):
            return 0 if self.is_cuda else -1

        def is_contiguous(self):
            return True

    rows = (3, 2, 64)
    assert sparse._rows(Fake(rows, (200, 64, 1), ptr=32), "k", rows, 0) == (32, 200)
    assert sparse._rows(Fake((1, 2, 64), (7, 64, 1)), "k", (1, 2, 64), 0) == (0, 128)
    assert sparse._rows(Fake((3, 1, 64), (64, 5, 1)), "k", (3, 1, 64), 0) == (0, 64)
    for shape, stride, ptr, dtype in (((3, 2, 64), (200, 64, 2), 0, BF), ((3, 2, 64), (200, 72, 1), 0, BF),
                                      ((3, 2, 64), (129, 64, 1), 0, BF), ((3, 2, 64), (64, 64, 1), 0, BF),
                                      ((3, 2, 64), (200, 64, 1), 8, BF),
                                      ((3, 2, 64), (200, 64, 1), 0, torch.float16),
                                      ((4, 2, 64), (200, 64, 1), 0, BF)):
        with pytest.raises(Err):
            sparse._rows(Fake(shape, stride, dtype, ptr), "k", rows, 0)
    with pytest.raises(Err, match="on cuda:1"):
        sparse._rows(Fake(rows, (200, 64, 1)), "k", rows, 1)
    with pytest.raises(Err, match="on cuda:1"):
        sparse._need(Fake((3,), (1,), I32), "x", I32, (3,), 1)
    with pytest.raises(Err, match="16-byte"):
        sparse._need(Fake((3,), (1,), BF, 8), "x", BF, (3,), 0)
    assert sparse._need(Fake((3,), (1,), I32, 4), "x", I32, (3,), 0) == 4      # a slice of positions
    with pytest.raises(Err, match="shape"):
        sparse._need(Fake((3,), (1,), I32), "x", I32, (4,), 0)
    with pytest.raises(Err, match="whole number"):
        sparse._requests(Fake((2, 5), (5, 1), I32), 3, 0)
    with pytest.raises(Err, match="whole number"):
        sparse._requests(Fake((0, 5), (5, 1), I32), 3, 0)
    with pytest.raises(Err, match="batch, pages"):
        sparse._requests(Fake((5,), (1,), I32), 5, 0)
    with pytest.raises(Err, match="scratch bytes"):
        sparse._scratch(None, 8, "x", 0)


EINVAL = 1


def test_entry_points_refuse_sizes():
    """Only sizes are looked at: every pointer is null or an address no kernel gets to see."""
    _, _, lib, _ = entry()

    def append(half=32, d=64, T=4, B=1, Hq=4, Hkv=2, ks=128, q=0, qo=0, kp=16):
        return lib.snowverify_kv_append(16, ks, 16, ks, q, ks, 16, 16, half, half, 0, 0, 1e-6, kp, 16, 0,
                                        qo, 16, 16, 16, B, T, Hq, Hkv, d, 4, 4, 0)
    assert append(T=0) == 0 and append(B=0) == 0
    for bad in (dict(half=4), dict(half=40), dict(half=-8), dict(d=96), dict(T=-1), dict(Hq=3),
                dict(Hkv=0), dict(ks=129), dict(q=16), dict(kp=0), dict(T=1 << 40),
                dict(T=1 << 23, Hq=4096, Hkv=4096, q=16, qo=16)):
        assert append(**bad) == EINVAL, bad

    def bounds(B=1, T=4, Hkv=2, d=64, kp=16):
        return lib.snowverify_page_bounds(kp, 16, 16, 16, 16, B, T, Hkv, d, 4, 4, 0)
    assert bounds(B=0) == 0 and bounds(T=0) == 0
    for bad in (dict(d=32), dict(Hkv=0), dict(T=-1), dict(T=1 << 40), dict(kp=0), dict(B=-1),
                dict(B=1 << 24, T=1 << 30)):
        assert bounds(**bad) == EINVAL, bad

    def select(budget=8, sink=1, recent=2, T=1, B=1, width=64, d=64, Hq=4, Hkv=2, blocks=9, scratch=16,
               nbytes=1 << 40, q=16):
        return lib.snowverify_page_select(q, 16, 16, 16, 16, B, T, Hq, Hkv, d, width, blocks, budget,
                                          sink, recent, scratch, nbytes, 0)
    assert select(T=0) == 0
    for bad in (dict(budget=0), dict(sink=-1), dict(recent=0), dict(sink=7, recent=2), dict(d=80),
                dict(width=(1 << 17) + 1), dict(blocks=0), dict(scratch=0), dict(nbytes=100), dict(q=0),
                dict(Hq=5), dict(sink=1 << 62, recent=1 << 62), dict(budget=1 << 40)):
        assert select(**bad) == EINVAL, bad

    def attend(budget=8, T=1, B=1, d=64, Hq=4, Hkv=2, q=16, out=32, pages=16, scratch=16, nbytes=1 << 40):
        return lib.snowverify_sparse_attention(q, 16, 16, out, 16, 16, pages, B, T, Hq, Hkv, d, 64, 9,
                                               budget, 1.0, scratch, nbytes, 0)
    assert attend(B=0) == 0
    for bad in (dict(budget=-1), dict(d=48), dict(Hq=0), dict(q=0), dict(out=16), dict(pages=0), dict(T=1 << 30),
                dict(budget=1000, nbytes=0), dict(budget=1000, scratch=0), dict(budget=1 << 30),
                dict(T=1 << 23, Hq=4096, Hkv=4096)):
        assert attend(**bad) == EINVAL, bad


def test_scratch_queries():
    ops, _, _, _ = entry()
    assert ops.page_select_scratch_bytes(1, 9, 16, 2, 256, 513) >= 9 * 2 * 513 * 4
    assert ops.page_select_scratch_bytes(1, 9, 16, 2, 256, 0) == 0
    # bounded, however many rows
    assert ops.page_select_scratch_bytes(1, 100000, 16, 2, 256, 13751) <= 512 << 20
    assert ops.sparse_attention_scratch_bytes(4, 1000, 16, 2, 256, 64) == 0      # many rows: no splits
    assert ops.sparse_attention_scratch_bytes(1, 1, 16, 2, 256, 64) > 0
    for bad in (dict(d=96), dict(Hq=5)):
        a = dict(B=1, T=1, Hq=4, Hkv=2, d=64) | bad
        assert ops.page_select_scratch_bytes(*a.values(), 64) == 0
        assert ops.sparse_attention_scratch_bytes(*a.values(), 64) == 0


def test_oracle_bounds_hold_the_scores():
    """The page score is an upper bound of the group's summed scores of every key in the page."""
    g = torch.Generator().manual_seed(0)
    Hq, hkv, d, blocks = 6, 2, 64, 5
    kp = torch.randn(blocks, hkv, d // 16, 16, 16, generator=g).to(BF)
    table = torch.tensor([[4, 0, 2]], dtype=I32)
    n = torch.tensor([40], dtype=I32)
    bounds = R.page_limits(kp, torch.zeros(blocks, hkv, 2, d, dtype=BF), table, 0 * n, n, 40)
    q = torch.randn(Hq, d, generator=g).to(BF)
    for h in range(hkv):
        s = R.scores(q, bounds, table, 0, h, hkv)
        for pos in range(40):
            key = R.key(kp, int(table[0, pos // 16]), pos % 16)[h].double()
            assert (q[3 * h:3 * h + 3].double() @ key).sum() <= s[pos // 16] + 1e-9
