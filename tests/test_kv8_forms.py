"""Which of its two forms the attention over the cache in 8 bits takes for the cases of test_gpu_kv8.py and
test_gpu_kv8_corners.py, without a GPU: every case of several tiles of rows runs in both."""
import pytest
import torch

from tests.test_gpu_kv8 import ATTEND, FORMS, PAGE, form_tables


def form_of(batch, T, Hq, Hkv, d, width):
    from snowllm_amd._capi import lib
    return lib.snowverify_kv8_attention_form(batch, T, Hq, Hkv, d, width)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,d,T,starts,counts,tree", ATTEND)
def test_forms_of_the_attention_cases(Hq, Hkv, d, T, starts, counts, tree, form):
    B = len(starts)
    width = max(max(s, 0) + T for s in starts) // PAGE + 1
    table = form_tables(torch.zeros(B, width, dtype=torch.int32), form, Hq, Hkv, d, T)
    one_tile = T * (Hq // Hkv) <= 16
    many_short_prompts = B == 16     # these share their tiles' keys at any width
    want = 0 if one_tile else 1 if many_short_prompts else FORMS.index(form)
    assert form_of(B, T, Hq, Hkv, d, table.shape[1]) == want


def test_forms_of_the_other_cases():
    """The cases that say which form they are for; those of one tile have only the first."""
    cases = [(16, 2, 128, 4, 3, 5), (8, 2, 64, 9, 1, 30), (8, 2, 64, 9, 1, 45), (16, 2, 128, 5, 1, 20), (16, 2, 256, 9, 1, 95),
             (8, 1, 64, 9, 1, 189), (32, 8, 128, 4, 2, 44), (8, 2, 128, 70, 1, 30), (64, 8, 64, 9, 1, 376),
             (16, 2, 256, 8, 1, 1), (8, 1, 128, 8, 1, 20)]
    for Hq, Hkv, d, T, B, width in cases:
        for form in FORMS:
            table = form_tables(torch.zeros(B, width, dtype=torch.int32), form, Hq, Hkv, d, T)
            want = 0 if T * (Hq // Hkv) <= 16 else FORMS.index(form)
            assert form_of(B, T, Hq, Hkv, d, table.shape[1]) == want, (Hq, Hkv, d, T, B, form)


def test_no_such_shape():
    assert form_of(1, 9, 16, 2, 256, 100) == 0
    for wrong in ((1, 9, 16, 3, 256, 100), (1, 9, 16, 2, 96, 100), (0, 9, 16, 2, 256, 100), (1, 0, 16, 2, 256, 100),
                  (1, 9, 16, 2, 256, -1), (1, 9, 16, 2, 256, (1 << 26) + 1)):
        assert form_of(*wrong) == -1
