"""Attention over shared prefixes on the GPU (qvx_attn_shared) against the formula in 64 bits on the CPU.

Tolerances as in test_gpu_window.py: the joined parts' weights carry one factor more, 2 u of the sum."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import CACHE_TYPES, U, Cache, _torch_type
from test_gpu_window import HALF, attend

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["narrow", "wide"])
def wide(request):
    """Short tables of few sequences run as one launch, in which each reads the shared keys for itself: the second time round
    tables are so wide that the sequences could pass that."""
    global WIDE
    WIDE = request.param == "wide"


def share(torch, c, groups, shared):
    """Every sequence of a group is given its first one's pages for the shared tokens; a page that ends behind them stays
    its own, and holds other values for them, which must not count."""
    for g in range(len(shared)):
        lead = groups[g]
        for b in range(groups[g], groups[g + 1]):
            full = min(shared[g], c.lens[b]) // c.page
            c.table[b, :full] = c.table[lead, :full]
    if WIDE:
        token = qvx.kv_page_bytes(c.t, c.hk, c.page, c.d) * 2 // c.page * len(c.lens)
        more = (257 << 20) // token // c.page
        c.table = np.concatenate([c.table, np.full((len(c.lens), more), -1, c.table.dtype)], 1)
    c.dev_table = torch.from_numpy(c.table).cuda()


def check(torch, c, hq, groups, shared, q_type=qvx.F32, scale=None, seed=1, one=False):
    d, n = c.d, len(c.lens)
    scale = d ** -0.5 if scale is None else scale
    share(torch, c, groups, shared)
    q = torch.from_numpy(np.random.default_rng(seed).standard_normal((n, hq, d)).astype(np.float32) * 1.5)
    q = q.to(_torch_type(torch, q_type)).cuda()
    out = torch.full_like(q, 7.0)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    qvx.attn_shared_t(q, c.desc, c.dev_table, c.dev_lens, ints(shared), None if one else ints(groups), scale, out=out)
    torch.cuda.synchronize()
    got, qh = out.double().cpu().numpy(), q.double().cpu().numpy()
    grp = hq // c.hk
    want, most, vmax = np.zeros((n, hq, d)), 0.0, 0.0
    for g in range(len(shared)):
        lead = groups[g]
        for b in range(groups[g], groups[g + 1]):
            if not c.lens[b]:
                continue
            m = min(shared[g], c.lens[b])
            k, v = (np.concatenate([c.rows(lead, i)[:, :m], c.rows(b, i)[:, m:]], 1) for i in range(2))
            for h in range(hq):
                y, s = attend(qh[b, h: h + 1], k[h // grp], v[h // grp], np.ones((1, c.lens[b]), bool), scale)
                want[b, h] = y[0]
                most = max(most, s)
            vmax = max(vmax, float(np.abs(v).max()))
    tol = 2 * U * ((d + 3) * most + max(c.lens) + 10) * vmax
    if q_type != qvx.F32 and q_type == c.t and n * grp / len(shared) > 16:
        tol += HALF[q_type] * vmax
    assert np.isfinite(got).all()
    bar = tol + HALF[q_type] * np.abs(want)
    assert (np.abs(got - want) <= bar).all(), float((np.abs(got - want) - bar).max())
    return q, out


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("shared,lens", [(64, (70, 100, 64, 65)), (0, (3, 40, 0, 700)), (33, (40, 100, 33, 20)), (500, (600, 501, 900, 0)),
                                         (2000, (2010, 2000, 2100, 1999)), (1, (1, 2, 3, 1))])
def test_one_group(cuda, t, shared, lens):
    """Prefixes that end inside a page, sequences that end inside the prefix, empty ones, no prefix at all."""
    lens = (max(lens[0], shared),) + lens[1:]
    check(cuda, Cache(cuda, t, lens, 16, 2, 64, seed=shared), 8, [0, 4], [shared], one=True)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 5), (7, 1), (17, 1), (32, 8)])
@pytest.mark.parametrize("d", [32, 128, 256])
def test_heads(cuda, t, hq, hk, d):
    check(cuda, Cache(cuda, t, (200, 130, 290, 128, 131), 16, hk, d, seed=d + hq), hq, [0, 5], [128])


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32, qvx.BF16))
@pytest.mark.parametrize("d", [8, 40, 72, 136, 248])
def test_odd_head_sizes(cuda, t, d):
    check(cuda, Cache(cuda, t, (100, 90, 290) * 8, 32, 2, d, seed=d), 4, [0, 24], [80])


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 256])
@pytest.mark.parametrize("t", CACHE_TYPES)
def test_page_sizes(cuda, t, page):
    check(cuda, Cache(cuda, t, (333, 300, 400, 301, 299), page, 2, 64, seed=page), 4, [0, 5], [300])


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("q_type", (qvx.F32, qvx.F16, qvx.BF16))
def test_groups(cuda, t, q_type):
    """Groups of all sizes, one of a sequence alone, one without a prefix."""
    lens = [300, 310, 400, 80, 90, 1000, 1010, 1020, 1000, 1500, 60, 0, 7, 8, 9, 2, 1, 44]
    c = Cache(cuda, t, lens, 16, 2, 64, seed=6)
    check(cuda, c, 8, [0, 3, 5, 10, 12, 18], [290, 64, 999, 50, 0], q_type)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("n", [20, 70, 300])
def test_many_sequences(cuda, t, n):
    """Wave-wide and workgroup-wide partitions over groups and sequences, a prefix longer than one chunk."""
    r = np.random.default_rng(n)
    for n_groups in (1, 3, min(n, 66)):
        cuts = [0] + sorted(int(x) for x in r.choice(np.arange(1, n), n_groups - 1, replace=False)) + [n]
        shared = [int(x) for x in r.integers(0, 700, n_groups)]
        lens = [0] * n
        for g in range(n_groups):
            for b in range(cuts[g], cuts[g + 1]):
                lens[b] = shared[g] + int(r.integers(0, 60))
        lens[n - 1] += 500
        check(cuda, Cache(cuda, t, lens, 16, 1, 32, seed=n), 4, cuts, shared)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16, qvx.Q8_0))
@pytest.mark.parametrize("q_same", (True, False))
def test_a_long_prefix(cuda, t, q_same):
    lens = [9000 + 13 * i for i in range(40)]
    c = Cache(cuda, t, lens, 16, 2, 64, seed=2)
    check(cuda, c, 8, [0, 40], [8990], t if q_same and t != qvx.Q8_0 else qvx.F32)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("d", [24, 64, 96, 128, 152, 256])
@pytest.mark.parametrize("n", [5, 9, 16])
def test_groups_of_up_to_64_rows(cuda, t, d, n):
    """20 to 64 rows of 16-bit and fp32 queries: waves on other keys of the same rows, prefixes that end in either's."""
    for shared in (15, 40, 333, 2100):
        lens = [shared + 5 * i for i in range(n)]
        lens[1] = max(shared - 20, 0)
        for q_type in (t, qvx.F32):
            check(cuda, Cache(cuda, t, lens, 16, 2, d, seed=n), 8, [0, n], [shared], q_type)


def test_sharp_logits(cuda):
    """Nearly all the weight on one key, in the prefix or in the rest."""
    for t in CACHE_TYPES:
        c = Cache(cuda, t, (600, 500, 700, 460, 450, 800), 16, 1, 64, seed=2)
        for scale in (3.0, 0.0, -0.5):
            check(cuda, c, 16, [0, 6], [450], scale=scale)


def test_it_agrees_with_paged_attention(cuda):
    torch = cuda
    for t in CACHE_TYPES:
        c = Cache(torch, t, (700, 650, 641, 900), 16, 2, 128, seed=9)
        share(torch, c, [0, 4], [640])
        q = torch.randn((4, 8, 128), device="cuda")
        want = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
        shared = torch.tensor([640], dtype=torch.int32, device="cuda")
        got = qvx.attn_shared_t(q, c.desc, c.dev_table, c.dev_lens, shared)
        assert (got - want).abs().max() < 1e-5
        again = qvx.attn_shared_t(q, c.desc, c.dev_table, c.dev_lens, shared)
        assert torch.equal(got, again)
        qvx.attn_shared_t(q, c.desc, c.dev_table, c.dev_lens, shared, out=q)
        assert torch.equal(q, got)


def test_groups_that_are_none(cuda):
    """Groups that do not rise or pass the batch, shared lengths past the table: nothing out of range."""
    torch = cuda
    c = Cache(torch, qvx.F16, (160, 90, 100, 40), 16, 1, 64, seed=11)
    q = torch.randn((4, 4, 64), device="cuda")
    table = c.dev_table.clone()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ws = torch.full((qvx.attn_shared_ws(c.desc, torch.float32, 4, 4, table.shape[1], 3),), 255, dtype=torch.uint8, device="cuda")
    for groups in ([0, 3, 1, 4], [0, -7, 900, 4], [9, 9, 9, 9], [0, 1 << 30, 2, 4]):
        for shared in ([30, 1 << 30, -5], [40, 0, 40]):
            ws.random_(0, 256)
            qvx.attn_shared_t(q, c.desc, table, c.dev_lens, ints(shared), ints(groups), ws=ws)
            torch.cuda.synchronize()


@pytest.mark.parametrize("q_type", (qvx.F32, qvx.F16))
def test_captured(cuda, q_type):
    torch = cuda
    n = 24
    c = Cache(torch, qvx.F16, [3000 + 5 * i for i in range(n)], 16, 2, 64, seed=13)
    groups, shared = [0, 16, n], [2990, 1000]
    share(torch, c, groups, shared)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn((n, 8, 64), device="cuda").to(_torch_type(torch, q_type))
    out, gd, sd, lens = torch.zeros_like(q), ints(groups), ints(shared), c.dev_lens.clone()
    qvx.attn_shared_t(q, c.desc, c.dev_table, lens, sd, gd, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qvx.attn_shared_t(q, c.desc, c.dev_table, lens, sd, gd, out=out)
    for s, cut in (([2990, 1000], 0), ([16, 0], 500), ([2000, 640], 900)):
        sd.copy_(ints(s))
        lens.copy_(c.dev_lens - cut)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, qvx.attn_shared_t(q, c.desc, c.dev_table, lens, sd, gd))
