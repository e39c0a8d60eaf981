"""A window of 0 for several new tokens a sequence (qvx_attn_window): none of them sees itself or another, so what the cache holds
for them, NaN here, is not read; first tokens alone, or zeros.  Reference and tolerance are test_gpu_window.py's."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx
from test_gpu_attention import CACHE_TYPES, Cache
from test_gpu_window import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("q_same", (True, False))
@pytest.mark.parametrize("group,new", [(1, 3), (4, 2), (4, 12), (2, 64), (7, 40)])
@pytest.mark.parametrize("sinks", [0, 1, 17, 100])
def test_new_tokens_are_not_read(cuda, t, q_same, group, new, sinks):
    q_type = t if q_same and t in (qvx.F16, qvx.BF16) else qvx.F32
    for page in (16, 24):
        lens = (new + 130, new, new + 5)
        check(cuda, Cache(cuda, t, lens, page, 2, 64, seed=new), 2 * group, [new] * 3, 0, sinks, q_type, bad=True, equal=True)
        check(cuda, Cache(cuda, t, lens, page, 2, 64, seed=new), 2 * group, [new, new // 2, new], 0, sinks, q_type, bad=True, pad=0)
