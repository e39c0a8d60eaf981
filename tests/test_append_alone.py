"""CPU tests of appends without queries (qvx_norm_rope_kv with q_heads = 0): the queries' pointers, both NULL, are not rows in place.
Each call is refused by a check behind those of the rows, before any device work."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx
from test_pages_api import turn


@pytest.mark.parametrize("q_type", (qvx.F32, qvx.F16, qvx.BF16))
@pytest.mark.parametrize("strides", [(0, 0), (256, 256), (512, 256)])
def test_rows_that_are_none_are_not_in_place(q_type, strides):
    kw = dict(heads=0, q=0, q_out=0, q_type=q_type, q_stride=strides[0], q_out_stride=strides[1])
    assert turn(w_stride=63, **kw) == qvx.E_SHAPE  # of the norms: all before was taken
    assert turn(eps=-1.0, **kw) == qvx.E_RANGE and turn(k=0, **kw) == qvx.E_NULL
