"""17 to 64 rows a sequence behind short windows (qvx_attn_window): row tiles of 64 rows, in which two groups of waves take the
first and the second 32 keys of every 64.  With one or two heads a group a row tile spans so many queries that the later
ones see keys of the second group alone, or of the first.  Reference and tolerance are test_gpu_window.py's."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import U, Cache, _torch_type
from test_gpu_window import HALF, attend, check, seen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("q_same", (True, False))
@pytest.mark.parametrize("hq,new", [(1, 18), (1, 32), (1, 40), (1, 64), (2, 9), (2, 20), (2, 32)])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 32, 33])
def test_keys_of_one_group_of_waves(cuda, t, q_same, hq, new, window):
    """The first visible key at every fourth place of its tile, equal and ragged pieces, one of them a whole prompt."""
    q_type = t if q_same else qvx.F32
    for past in (0, 5, 10, 15, 32, 47):
        c = Cache(cuda, t, [past + window + new, new, 200 + past], 16, 1, 64, seed=past)
        check(cuda, c, hq, [new] * 3, window, 0, q_type, equal=True)
    check(cuda, c, hq, [new - 2, new, new + 2], window, 0, q_type)
    check(cuda, c, hq, [new - 2, new, new + 2], window, 3, q_type)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("d", [32, 96, 128, 160, 256])
@pytest.mark.parametrize("q_same", (True, False))
def test_head_sizes(cuda, t, d, q_same):
    for window in (1, 17, 32):
        check(cuda, Cache(cuda, t, (100, 70, 64), 24, 2, d, seed=d), 2, [60, 64, 64], window, 0, t if q_same else qvx.F32)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("missing", [0, 1, 2, 3])
@pytest.mark.parametrize("window", [20, 40, 1 << 20])
def test_pages_that_are_not_held(cuda, t, missing, window):
    """A page of 32 keys, as many as a group of waves takes, is not held: rows that see it alone are zeros, the others theirs."""
    torch = cuda
    c = Cache(torch, t, (128, 110), 32, 1, 64, seed=missing)
    new, d = 64, c.d
    q = torch.from_numpy(np.random.default_rng(3).standard_normal((2 * new, 1, d)).astype(np.float32)).to(_torch_type(torch, t)).cuda()
    table = c.dev_table.clone()
    table[:, missing] = -1
    got = qvx.attn_window_t(q, c.desc, table, c.dev_lens, window).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    for b, n in enumerate(c.lens):
        held = np.arange(n) // 32 != missing
        see = seen(n, new, window, 0) & held[None]
        want, most = attend(qh[b * new: (b + 1) * new, 0], c.rows(b, 0)[0], c.rows(b, 1)[0], see, d ** -0.5)
        vmax = float(np.abs(c.rows(b, 1)).max())
        bar = 2 * U * ((d + 3) * most + n + 8) * vmax + HALF[t] * vmax + HALF[t] * np.abs(want)
        assert (np.abs(got[b * new: (b + 1) * new, 0] - want) <= bar).all()
