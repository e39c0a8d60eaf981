"""Groups whose sequences are shorter than the tokens they are said to share (qvx_attn_shared), against the formula in 64 bits on
the CPU; what stands behind a sequence's tokens is NaN.  Tolerances as in test_gpu_shared.py."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import CACHE_TYPES, U, Cache, _torch_type
from test_gpu_window import HALF, attend

pytestmark = pytest.mark.gpu


def check(torch, c, hq, groups, shared, leads, q_type=qvx.F32, wide=False):
    """leads: the sequence whose pages hold each group's shared tokens."""
    d, n, grp = c.d, len(c.lens), hq // c.hk
    table = c.table.copy()
    for g, lead in enumerate(leads):  # the others hold its full pages too, and other values on the last one
        for b in range(groups[g], groups[g + 1]):
            full = min(shared[g], c.lens[b], c.lens[lead]) // c.page
            table[b, :full] = table[lead, :full]
    c.table = table
    if wide:  # past what is read whole
        token = qvx.kv_page_bytes(c.t, c.hk, c.page, c.d) * 2 // c.page * n
        table = np.concatenate([table, np.full((n, (257 << 20) // token // c.page), -1, table.dtype)], 1)
    q = torch.from_numpy(np.random.default_rng(1).standard_normal((n, hq, d)).astype(np.float32) * 1.5)
    q = q.to(_torch_type(torch, q_type)).cuda()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = qvx.attn_shared_t(q, c.desc, torch.from_numpy(table).cuda(), c.dev_lens, ints(shared), ints(groups))
    got, qh = out.double().cpu().numpy(), q.double().cpu().numpy()
    want, most, vmax = np.zeros((n, hq, d)), 0.0, 0.0
    for g, lead in enumerate(leads):
        for b in range(groups[g], groups[g + 1]):
            if not c.lens[b]:
                continue
            m = min(shared[g], c.lens[b])
            k, v = (np.concatenate([c.rows(lead, i)[:, :m], c.rows(b, i)[:, m:]], 1) for i in range(2))
            for h in range(hq):
                y, s = attend(qh[b, h: h + 1], k[h // grp], v[h // grp], np.ones((1, c.lens[b]), bool), d ** -0.5)
                want[b, h] = y[0]
                most = max(most, s)
            vmax = max(vmax, float(np.abs(v).max()))
    tol = 2 * U * ((d + 3) * most + max(c.lens) + 10) * vmax
    if q_type != qvx.F32 and q_type == c.t and n * grp / len(shared) > 16:
        tol += HALF[q_type] * vmax
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol + HALF[q_type] * np.abs(want)).all(), float((np.abs(got - want) - tol).max())


@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("shared,lens", [(64, (40, 30, 5)), (300, (290, 7, 130, 0)), (300, (16, 16, 15)), (2000, (1999, 3, 900)), (50, (0, 0))])
def test_all_are_shorter_than_the_shared_tokens(cuda, t, wide, shared, lens):
    check(cuda, Cache(cuda, t, lens, 16, 2, 64, seed=shared), 8, [0, len(lens)], [shared], [0], wide=wide)


@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("q_same", (True, False))
@pytest.mark.parametrize("n", [6, 16, 40])
def test_groups_of_many_rows(cuda, t, q_same, wide, n):
    """Row tiles of 64 and of 128 rows, of which one may hold short sequences alone."""
    for shared, longest in ((100, 90), (1500, 1401), (70, 1)):
        lens = [longest] + [max(longest - 7 * i, 0) for i in range(1, n)]
        check(cuda, Cache(cuda, t, lens, 16, 1, 128, seed=n), 4, [0, n], [shared], [0], t if q_same else qvx.F32, wide)
