"""CPU tests of the argument checks of qvx_attn_window and qvx_attn_shared: every call here is refused, or has nothing to do,
before any device work."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx
from test_attention_api import BAD_CACHES, P, cache


def window(c=None, out=P, out_stride=256, q=P + 1024, q_stride=256, q_type=qvx.F32, heads=4, offsets=P, n_q=6, table=P, width=8,
           lens=P, n=3, w=64, sinks=4, ws=P, ws_bytes=1 << 40):
    return qvx.attn_window(out, out_stride, q, q_stride, q_type, heads, offsets, n_q, cache() if c is None else c, table, width,
                           lens, n, w, sinks, 0.125, ws, ws_bytes)


def shared(c=None, out=P, out_stride=256, q=P + 1024, q_stride=256, q_type=qvx.F32, heads=4, table=P, width=8, lens=P, n=3,
           groups=P, shared=P, n_groups=2, ws=P, ws_bytes=1 << 40):
    return qvx.attn_shared(out, out_stride, q, q_stride, q_type, heads, cache() if c is None else c, table, width, lens, n, groups,
                           shared, n_groups, 0.125, ws, ws_bytes)


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_bad_caches(kw, rc):
    assert window(cache(**kw)) == rc and shared(cache(**kw)) == rc
    assert qvx.attn_window_ws(cache(**kw), 0, 4, 6, 3, 8, 64, 4) == 0 and qvx.attn_shared_ws(cache(**kw), 0, 4, 3, 8, 1) == 0


@pytest.mark.parametrize("call", [window, shared])
def test_refusals_of_both(call):
    assert call(n=0) == qvx.E_NVEC and call(n=-1) == qvx.E_NVEC
    assert call(heads=3) == qvx.E_SHAPE and call(heads=0) == qvx.E_SHAPE and call(width=0) == qvx.E_SHAPE
    assert call(q_type=qvx.Q8_0) == qvx.E_TYPE and call(q_type=99) == qvx.E_TYPE
    assert call(out_stride=255) == qvx.E_SHAPE and call(q_stride=-1) == qvx.E_SHAPE
    for name in ("out", "q", "table", "lens"):
        assert call(**{name: 0}) == qvx.E_NULL, name
    assert call(n=70000) == qvx.E_RANGE and call(width=1 << 28) == qvx.E_RANGE
    assert call(ws=P + 4) == qvx.E_RANGE and call(out=P, q=P, q_stride=512) == qvx.E_RANGE
    assert call(out=P + 2) == qvx.E_RANGE and call(q=P + 1, q_type=qvx.F16) == qvx.E_RANGE


def test_window_refusals():
    assert window(n_q=-1) == qvx.E_SHAPE and window(offsets=0, n_q=7) == qvx.E_SHAPE
    assert window(w=-1) == qvx.E_SHAPE and window(sinks=-1) == qvx.E_SHAPE
    assert window(n_q=1 << 30) == qvx.E_RANGE
    assert window(n_q=0) == qvx.OK  # nothing to do
    need = qvx.attn_window_ws(cache(), 0, 4, 3, 3, 800, 1 << 20, 0)
    big = dict(width=800, n_q=3, w=1 << 20, sinks=0)
    assert need > 0 and window(**big, ws=0) == qvx.E_NULL and window(**big, ws_bytes=need - 1) == qvx.E_RANGE
    assert qvx.attn_window_ws(cache(), 0, 4, 3, 3, 800, 64, 4) == 0  # a short window is not split, however long the table
    assert qvx.lib().qvx_attn_window(P, 256, P, 256, 0, 4, P, 6, None, P, 8, P, 3, 64, 4, 0.1, P, 1 << 20, None) == qvx.E_NULL


def test_shared_refusals():
    assert shared(n_groups=0) == qvx.E_SHAPE and shared(n_groups=4) == qvx.E_RANGE
    assert shared(groups=0) == qvx.E_NULL and shared(shared=0) == qvx.E_NULL and shared(ws=0) == qvx.E_NULL
    need = qvx.attn_shared_ws(cache(), 0, 4, 3, 8, 2)
    assert need > 0 and shared(ws_bytes=need - 1) == qvx.E_RANGE
    assert qvx.attn_shared_ws(cache(), 0, 4, 3, 8, 4) == 0
    assert qvx.lib().qvx_attn_shared(P, 256, P, 256, 0, 4, None, P, 8, P, 3, P, P, 2, 0.1, P, 1 << 20, None) == qvx.E_NULL


@pytest.mark.parametrize("t", [qvx.F16, qvx.Q8_0])
def test_workspaces_are_bounded(t):
    """Whatever the batch: a few chunks a workgroup, and for a shared prefix a part a row tile beside them."""
    c = cache(type=t, kv_heads=8, head_dim=128)
    assert qvx.attn_window_ws(c, 0, 32, 4096, 64, 1 << 16, 1 << 30, 0) < 64 << 20
    assert qvx.attn_shared_ws(c, 0, 32, 256, 1 << 13, 1) < 96 << 20


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(sinks=1), dict(window=4, sinks=-1), dict(shared_groups=2),
                                dict(shared_groups=-1), dict(window=4, shared_groups=1)])
def test_a_step_refuses_masks_that_are_none(kw):
    from test_decode import _paged_model, _paged_step
    with pytest.raises(ValueError, match="PagedDecodeStep: a window"):
        _paged_step(_paged_model(), **kw)


def test_a_step_refuses_norms_that_are_not_a_heads():
    import torch
    from test_decode import _paged_model, _paged_step
    for k, size in (("q_norm", 32), ("k_norm", 512)):
        m = _paged_model()
        m.norms[1][k] = torch.ones(size)
        with pytest.raises(ValueError, match="layer 1 are of 64 values"):
            _paged_step(m)
