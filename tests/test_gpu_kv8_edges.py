"""The 8-bit paged cache where its kernels' own limits lie, against its definition in 64 bits
(tests/kv8_testlib.py)."""
import numpy as np
import pytest

from gdn_testlib import say
from test_gpu_kv8 import Pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,dim,cached,new,window", [
    (1, 128, 1000, 1537, 1900), (1, 256, 258, 769, 856), (1, 64, 1, 1025, 896),
    (3, 64, 266, 806, 933), (5, 128, 214, 868, 948), (6, 256, 225, 861, 948)])
def test_windows_on_prompts_in_pieces(gpu, hq, dim, cached, new, window):
    """A tile between the first, which starts below its window, and the last, which has few
    tokens, sees more pages than both: every one of its keys counts. (hq query heads on one.)"""
    rng = np.random.default_rng(cached)
    p = Pair(2, 50, 48, hq=hq, hk=1, dim=dim, tokens=1600)
    say("kv8 window on pieces", hq, dim, cached, new, window)
    p.step([1], [0], [cached])
    p.append(rng)
    p.step([1], [cached], [new])
    p.append(rng)
    p.attention(rng, label=f"window {window}", window=window)
    p.kv.close()
