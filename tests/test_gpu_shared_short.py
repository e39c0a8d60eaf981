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


def holders(lens, groups, shared):
    """The first sequence of each group that holds most of its shared tokens."""
    return [max(range(groups[g], groups[g + 1]), key=lambda b: min(lens[b], shared[g])) for g in range(len(shared))]


@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("groups,shared,lens", [
    ([0, 4], [64], (0, 100, 64, 70)), ([0, 4], [64], (3, 0, 17, 90)), ([0, 5], [300], (10, 200, 250, 40, 250)),
    ([0, 2, 3, 6], [33, 20, 900], (5, 40, 0, 899, 900, 1000)), ([0, 3, 5], [48, 0], (0, 0, 0, 9, 0))])
def test_the_first_sequence_is_shorter(cuda, t, wide, groups, shared, lens):
    """Released and refilled first sequences: the others' tokens are read from one that holds them."""
    check(cuda, Cache(cuda, t, lens, 16, 2, 64, seed=len(lens)), 8, groups, shared, holders(lens, groups, shared), wide=wide)


@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("t,q_type", [(qvx.F16, qvx.F16), (qvx.BF16, qvx.F32), (qvx.Q8_0, qvx.F32)])
@pytest.mark.parametrize("n,at", [(20, 3), (100, 70), (300, 299)])
def test_a_holder_far_behind(cuda, t, q_type, wide, n, at):
    """Past a wave's lanes, and a workgroup's threads; in a group that begins at 0, and behind another."""
    r = np.random.default_rng(n)
    for cut in (0, 2):
        lens = [int(x) for x in r.integers(0, 50, n)]
        lens[at] = 200
        groups, shared = ([0, 2, n], [10, 190]) if cut else ([0, n], [190])
        check(cuda, Cache(cuda, t, lens, 16, 1, 32, seed=n), 4, groups, shared, holders(lens, groups, shared), q_type, wide)
