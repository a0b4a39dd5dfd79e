"""The attention over the cache in 8 bits at the ends of its range of values. Tolerances are those of
test_gpu_kv8.py and of the oracle (oracle/kv8.py)."""
import pytest
import torch

from oracle import kv8 as R
from tests.test_gpu_kv8 import FORMS, check_attention, form_tables, ints, on_gpu, random_cache, run_attention, say, tables

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
