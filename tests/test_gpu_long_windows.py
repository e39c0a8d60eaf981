"""Windows and first tokens past 32 bits on the GPU: the same as 2^31 - 1 of them, in the calls and in decode.PagedDecodeStep."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx
from qorvix_amd import decode
from test_gpu_attention import Cache
from test_gpu_serving import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("w", [2 ** 31, 2 ** 32, 10 ** 20])
def test_all_of_the_past(cuda, w):
    torch = cuda
    c = Cache(torch, qvx.F16, (300, 40), 16, 2, 64, seed=1)
    q = torch.randn((2, 8, 64), device="cuda")
    want = qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 2 ** 31 - 1)
    assert torch.equal(qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, w), want)
    want = qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 5, 2 ** 31 - 1)
    assert torch.equal(qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 5, w), want)


@pytest.mark.parametrize("window,sinks", [(2 ** 33, 0), (4, 2 ** 33)])
def test_a_step(cuda, window, sinks):
    torch = cuda
    torch.manual_seed(1)
    model = _model(torch, layers=1)
    steps = [decode.PagedDecodeStep(model, 2, heads=8, kv_heads=2, n_pages=12, max_pages=6, page_size=3, window=w, sinks=s)
             for w, s in ((window, sinks), (100, 0))]
    for _ in range(12):
        x = torch.randn((2, 512), device="cuda")
        for step in steps:
            step.x.copy_(x)
            step.run(torch.cuda.current_stream().cuda_stream)
            step.trim()
        assert torch.equal(steps[0].table, steps[1].table) and (steps[0].logits - steps[1].logits).abs().max() < 1e-4
