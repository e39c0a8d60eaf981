"""The scale down to which queries of the cache's own 16-bit type keep their weights in it (qvx_attn_window, more than 16 rows): below
1e-30 they go in parts, whose weights are off by 2^-18 at most.  Tolerance otherwise as in test_gpu_window.py."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import U, Cache
from test_gpu_window import HALF, attend, seen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.7e-30, 0.9e-30, 0.99e-30])
def test_below_it_weights_go_in_parts(cuda, scale):
    torch = cuda
    c = Cache(torch, qvx.BF16, (400, 300), 16, 1, 64, seed=2)
    new, d = 40, c.d
    q = torch.from_numpy(np.random.default_rng(1).standard_normal((2 * new, 1, d)) * 1e30 / 8).bfloat16().cuda()
    got = qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 1 << 20, scale=scale).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    for b, n in enumerate(c.lens):
        rows = slice(b * new, (b + 1) * new)
        want, most = attend(qh[rows, 0], c.rows(b, 0)[0], c.rows(b, 1)[0], seen(n, new, 1 << 20, 0), scale)
        vmax = float(np.abs(c.rows(b, 1)).max())
        bar = (2 * U * ((d + 3) * most + n + 8) + 2.0 ** -18) * vmax + HALF[qvx.BF16] * np.abs(want)
        assert (np.abs(got[rows, 0] - want) <= bar).all()
