"""CPU tests of a file's sliding window: read from its key, carried through the fused forms, and no step over it without one."""
from __future__ import annotations

import pytest

from qorvix_amd import decode
from test_decode import _paged_model, _paged_step


@pytest.mark.parametrize("value,want", [(None, None), (0, None), (4096, 4096), ([0, 1024, 512], 512), ([0, 0], None), ("64", None)])
def test_of_a_file(value, want):
    from gguf_build import U32, GgufBuilder
    from qorvix_amd.gguf import GgufFile
    b, key = GgufBuilder(3).str("general.architecture", "llama"), "llama.attention.sliding_window"
    if isinstance(value, list):
        b = b.array(key, U32, value)
    elif value is not None:
        b = b.str(key, value) if isinstance(value, str) else b.u32(key, value)
    assert decode.Model.window_of(GgufFile.parse(b.build(32))) == want


def test_a_step_of_more_tokens_needs_a_window():
    model = _paged_model()
    model.sliding_window = 31
    with pytest.raises(ValueError, match="see 31 tokens, the table holds 32"):  # two pages of sixteen
        _paged_step(model)
    with pytest.raises(ValueError, match="see 31 tokens"):
        _paged_step(model, shared_groups=1)
    for kw in (dict(window=31), dict(window=32), dict(max_pages=1)):
        with pytest.raises(ValueError, match="KvCache.of"):  # it comes as far as the device's memory
            _paged_step(model, **kw)
    for size in (32, None):
        model.sliding_window = size
        with pytest.raises(ValueError, match="KvCache.of"):
            _paged_step(model)


def test_fused_forms_carry_it():
    model = decode.Model(sliding_window=7)
    assert model.fused().sliding_window == 7 and model.fused_ops().sliding_window == 7
