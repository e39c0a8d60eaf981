"""Appends of k and v without queries (qvx_norm_rope_kv with q_heads = 0) on the GPU: the cache as the call with queries leaves it."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", (qvx.F32, qvx.F16, qvx.BF16, qvx.Q8_0))
@pytest.mark.parametrize("dtype", ("float32", "float16", "bfloat16"))
def test_the_cache_is_the_same(cuda, t, dtype):
    torch = cuda
    n, hk, d, page = 21, 2, 64, 8
    q, k, v = (torch.randn((n, h, d), device="cuda") for h in (4, hk, hk))
    w = torch.rand(d, device="cuda")
    norm = qvx.QkNorm.of(w, w)
    rope = qvx.Rope.of(10000.0 ** -(torch.arange(d // 2, dtype=torch.float64, device="cuda") / 32))
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    pools = []
    for x in (q, q[:, :0]):
        pages = torch.zeros((2, 3, qvx.kv_page_bytes(t, hk, page, d)), dtype=torch.uint8, device="cuda")
        out = qvx.norm_rope_kv_t(x, k, v, at, norm, rope, qvx.KvCache.of(pages[0], pages[1], t, page, hk, d), at,
                                 dtype=getattr(torch, dtype))
        assert out.shape == x.shape
        pools.append(pages)
    assert torch.equal(*pools) and bool(pools[0].any())
