"""CPU tests of windows and first tokens past 32 bits: as many as a sequence may hold, not what is left of them in 32 bits."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx
from test_attention_api import cache
from test_masked_api import window


@pytest.mark.parametrize("w", [2 ** 31, 2 ** 32, 2 ** 33 + 5, 10 ** 20])
def test_all_of_the_past(w):
    need = qvx.attn_window_ws(cache(), 0, 4, 3, 3, 800, 2 ** 31 - 1, 0)
    assert need > 0 and qvx.attn_window_ws(cache(), 0, 4, 3, 3, 800, w, 0) == need
    assert qvx.attn_window_ws(cache(), 0, 4, 3, 3, 800, 0, w) == qvx.attn_window_ws(cache(), 0, 4, 3, 3, 800, 0, 2 ** 31 - 1) > 0
    for kw in (dict(w=w, sinks=0), dict(w=0, sinks=w)):
        assert window(width=800, n_q=3, ws=0, **kw) == qvx.E_NULL  # of the workspace
    assert window(w=-w) == qvx.E_SHAPE and window(sinks=-w) == qvx.E_SHAPE
