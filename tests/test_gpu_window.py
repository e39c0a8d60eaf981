"""Attention with a window and first tokens on the GPU (qvx_attn_window) against the formula in 64 bits on the CPU.

Tolerances as in test_gpu_attention.py: |error| <= 2 u ((d + 3) S + n + 8) max |v|, S the largest sum |q_i k_i| scale, n the
keys, u = 2^-24; a 16-bit output adds half a step of its own value, and where the weights are rounded to 16 bits (queries and
cache of one 16-bit type, more than 16 rows a sequence) half a step of every weight: that part of max |v|."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import CACHE_TYPES, U, Cache, _torch_type

pytestmark = pytest.mark.gpu

HALF = {qvx.F32: 2.0 ** -24, qvx.F16: 2.0 ** -11, qvx.BF16: 2.0 ** -8}


def attend(q, k, v, see, scale):
    """q [rows, d], k, v [keys, d], see [rows, keys]: zeros for rows that see nothing, and the largest sum |q k| scale."""
    out = np.zeros((q.shape[0], v.shape[1]))
    s = (q @ k.T) * scale
    any_ = see.any(1)
    if any_.any():
        s = np.where(see, s, -np.inf)[any_]
        w = np.exp(s - s.max(1, keepdims=True))
        out[any_] = (w @ np.where(see.any(0)[:, None], v, 0)) / w.sum(1, keepdims=True)
    used = see.any(0)
    most = float((np.abs(q) @ np.abs(k[used]).T).max() * abs(scale)) if used.any() and q.size else 0.0
    return out, most


def seen(n, new, window, sinks):
    """[new, n]: what the last `new` of n tokens see."""
    p = n - new + np.arange(new)[:, None]
    j = np.arange(n)[None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def poison(torch, c, b, hidden):
    """NaN (Q8_0: NaN scales) in the tokens `hidden` of sequence b."""
    for x in c.desc.tensors:
        raw = x
        for j in np.flatnonzero(hidden):
            p, o = int(c.table[b, j // c.page]), int(j % c.page)
            if c.t == qvx.Q8_0:
                at = c.hk * c.page * c.d
                raw[p, at: at * 17 // 16].view(c.hk, c.page, c.d // 16)[:, o] = 255
            else:
                es = 4 if c.t == qvx.F32 else 2
                raw[p, : c.hk * c.page * c.d * es].view(c.hk, c.page, c.d * es)[:, o] = 255


def check(torch, c, hq, new, window, sinks, q_type=qvx.F32, scale=None, seed=1, free=False, equal=False, pad=3, bad=False):
    d, n = c.d, len(c.lens)
    scale = d ** -0.5 if scale is None else scale
    rows = sum(new)
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = torch.from_numpy(np.random.default_rng(seed).standard_normal((rows + (0 if equal else pad), hq, d)).astype(np.float32) * 1.5)
    q = q.to(_torch_type(torch, q_type)).cuda()
    table = c.dev_table.clone()
    views = [seen(m, min(k, m), window, sinks) for m, k in zip(c.lens, new)]
    for b, see in enumerate(views):
        hidden = ~see.any(0)
        if bad and hidden.any():
            poison(torch, c, b, hidden)
        if free:
            for p in range(-(-c.lens[b] // c.page)):
                if hidden[p * c.page: (p + 1) * c.page].all():
                    table[b, p] = -1
    out = torch.full_like(q, 7.0)
    dev = None if equal else torch.from_numpy(offsets).cuda()
    qvx.attn_window_t(q, c.desc, table, c.dev_lens, window, sinks, dev, scale, out=out)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    qh = q.double().cpu().numpy()
    g = hq // c.hk
    most = vmax = 0.0
    want = np.zeros((rows, hq, d))
    for b, see in enumerate(views):
        if not c.lens[b] or not new[b]:
            continue
        k, v = c.rows(b, 0), c.rows(b, 1)
        first = offsets[b + 1] - see.shape[0]  # rows at positions below 0 see nothing
        for h in range(hq):
            want[first: offsets[b + 1], h], s = attend(qh[first: offsets[b + 1], h], k[h // g], v[h // g], see, scale)
            most = max(most, s)
        vmax = max(vmax, float(np.abs(v).max()))
    mean = rows * g / n
    tol = 2 * U * ((d + 3) * most + max(c.lens) + 8) * vmax
    if q_type != qvx.F32 and q_type == c.t and mean > 16:
        tol += HALF[q_type] * vmax
    tol = tol + HALF[q_type] * np.abs(want)
    assert np.isfinite(got).all()
    assert (np.abs(got[:rows] - want) <= tol).all(), float((np.abs(got[:rows] - want) - tol).max())
    assert (got[rows:] == 7.0).all()
    return q, out


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (16, 4), (33, 1), (100, 20), (128, 130), (1000, 0), (2 ** 31 - 1, 3)])
def test_one_token(cuda, t, window, sinks):
    c = Cache(cuda, t, (1, 17, 300, 0, 129, 16, 700), 16, 2, 64, seed=window % 1000)
    check(cuda, c, 8, [1, 1, 1, 1, 1, 1, 1], window, sinks, bad=True, equal=True)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 256])
def test_pages_that_end_inside_a_tile(cuda, t, page):
    c = Cache(cuda, t, (1, 100, 333, page, 500), page, 2, 64, seed=page)
    check(cuda, c, 4, [1] * 5, 70, 5, bad=True, free=True, equal=True)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 1), (8, 1), (17, 1), (40, 2)])
@pytest.mark.parametrize("d", [32, 128, 256])
def test_heads(cuda, t, hq, hk, d):
    c = Cache(cuda, t, (5, 290, 77), 16, hk, d, seed=d + hq)
    check(cuda, c, hq, [1, 1, 1], 100, 3, bad=True, equal=True)


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32))
@pytest.mark.parametrize("d", [8, 40, 72, 136, 248])
def test_odd_head_sizes(cuda, t, d):
    c = Cache(cuda, t, (5, 0, 290), 32, 2, d, seed=d)
    check(cuda, c, 4, [1, 1, 1], 64, 2, bad=True, equal=True)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("q_type", (qvx.F32, qvx.BF16, qvx.F16))
@pytest.mark.parametrize("new", [(2, 1, 3, 0, 4), (5, 17, 40, 1, 0), (130, 64, 33, 200, 7)])
def test_pieces_of_prompts(cuda, t, q_type, new):
    """Several new tokens a sequence, ragged, none among them; whole prompts (as many as the sequence holds)."""
    c = Cache(cuda, t, (2, 100, 300, 200, 60), 16, 2, 64, seed=sum(new))
    new = [min(a, b) for a, b in zip(new, c.lens)]
    for window, sinks in ((1, 0), (20, 4), (90, 0), (5000, 0)):
        check(cuda, c, 8, new, window, sinks, q_type)
    check(cuda, c, 8, new, 20, 40, q_type, free=True, bad=True)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("q_same", (True, False))
@pytest.mark.parametrize("d", [32, 40, 96, 128, 160, 256])
def test_prompts_of_16_bits(cuda, t, q_same, d):
    c = Cache(cuda, t, (513, 40, 129, 260), 24, 2, d, seed=d)
    check(cuda, c, 6, [513, 33, 100, 256], 100, 5, t if q_same else qvx.F32)
    check(cuda, c, 6, [300, 40, 129, 1], 1 << 20, 0, t if q_same else qvx.F32)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("q_same", (True, False))
def test_a_long_past(cuda, t, q_same):
    """Few new tokens on many keys: the keys are split, with and without a window, some chunks without a key."""
    c = Cache(cuda, t, (9000, 70, 4000), 16, 2, 64, seed=3)
    for new in ([20, 20, 20], [64, 70, 10], [300, 1, 0]):
        for window, sinks in ((1 << 30, 0), (3000, 17), (40, 100)):
            check(cuda, c, 8, new, window, sinks, t if q_same else qvx.F32)


@pytest.mark.parametrize("t", (qvx.F16, qvx.Q8_0))
@pytest.mark.parametrize("window,sinks", [(4096, 4), (300, 300), (20000, 0)])
def test_long_windows_of_many_sequences(cuda, t, window, sinks):
    r = np.random.default_rng(5)
    lens = [int(x) for x in np.exp(r.uniform(0, np.log(9000), 70))]
    lens[3], lens[60] = 9001, 0
    c = Cache(cuda, t, lens, 16, 2, 32, seed=7)
    check(cuda, c, 8, [1] * 70, window, sinks, free=True, equal=True)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("group", [1, 4, 8, 16])
def test_rows_that_see_nothing(cuda, t, group):
    """A window of 0, alone and beside sinks; more new tokens than the sequence holds: positions below 0."""
    c = Cache(cuda, t, (40, 300, 3), 16, 1, 64, seed=group)
    check(cuda, c, group, [1, 1, 1], 0, 0, equal=True)
    check(cuda, c, group, [1, 1, 1], 0, 5, equal=True, bad=True)
    torch = cuda
    q = torch.randn((12, group, 64), device="cuda")
    lens = torch.tensor([4, 0, 3], dtype=torch.int32, device="cuda")
    table = c.dev_table.clone()
    out = qvx.attn_window_t(q, c.desc, table, lens, 10, 0)  # four each
    assert (out[4:9] == 0).all() and torch.isfinite(out).all()
    alone = qvx.attn_window_t(q[9:].contiguous(), c.desc, table[2:].contiguous(), lens[2:], 10, 0)
    # Two calls of other sizes may run on other kernels, each within the bar above of the formula; the one of many rows takes
    # weights in two 16-bit parts, which leave 2^-18 of a weight (bf16), so at most that part of max |v|.
    k, v = c.rows(2, 0), c.rows(2, 1)
    most = float((np.abs(q[9:].cpu().double().numpy().reshape(-1, 64)) @ np.abs(k[0]).T).max()) / 8
    bar = (2 * 2 * U * (67 * most + 3 + 8) + 2.0 ** -18) * float(np.abs(v).max())
    assert float((out[9:] - alone).abs().max()) <= bar
    table[0, :] = -1
    assert (qvx.attn_window_t(q, c.desc, table, lens, 10, 0)[:4] == 0).all()


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32))
def test_scales(cuda, t):
    for scale in (0.0, -0.4, 3.0):
        c = Cache(cuda, t, (37, 1, 500), 24, 1, 64, seed=16)
        check(cuda, c, 4, [1, 1, 1], 50, 3, scale=scale, equal=True)
        check(cuda, c, 4, [30, 1, 200], 50, 3, scale=scale)
        if t == qvx.F16:
            check(cuda, c, 4, [30, 1, 200], 50, 3, scale=scale, q_type=qvx.F16)


def test_a_window_over_all_is_paged_attention(cuda):
    torch = cuda
    for t in CACHE_TYPES:
        c = Cache(torch, t, (1200, 5, 0, 333), 16, 2, 128, seed=9)
        q = torch.randn((4, 8, 128), device="cuda")
        want = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
        got = qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 1 << 30)
        assert (got - want).abs().max() < 1e-5
        qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 1 << 30, out=q)
        assert torch.equal(q, got)


@pytest.mark.parametrize("q_type", (qvx.F32, qvx.F16))
def test_strided_rows_in_place_and_repeatable(cuda, q_type):
    torch = cuda
    c = Cache(torch, qvx.F16, (50, 0, 777), 16, 2, 64, seed=8, pad=48)
    wide = torch.randn((60, 1000), device="cuda").to(_torch_type(torch, q_type))
    new = torch.tensor([0, 20, 20, 57], dtype=torch.int32, device="cuda")
    q = wide[:, 101:101 + 8 * 64].unflatten(1, (8, 64))
    dst = torch.full((60, 701), 5.0, device="cuda", dtype=q.dtype)
    out = dst[:, 61:61 + 8 * 64].unflatten(1, (8, 64))
    first = qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 100, 4, new)
    qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 100, 4, new, out=out)
    assert torch.equal(out[:57], first[:57]) and (out[57:] == 5.0).all() and (first[57:] == 0).all()
    assert (dst[:, :61] == 5.0).all() and (dst[:, 61 + 512:] == 5.0).all()
    again = qvx.attn_window_t(q.contiguous(), c.desc, c.dev_table, c.dev_lens, 100, 4, new)
    assert torch.equal(first, again)
    keep = wide.clone()
    qvx.attn_window_t(q, c.desc, c.dev_table, c.dev_lens, 100, 4, new, out=q)
    assert torch.equal(q[:57], first[:57]) and torch.equal(wide[57:], keep[57:])


def test_offsets_and_lengths_that_are_none(cuda):
    """Offsets that do not rise, past the rows or below 0, lengths past the table: nothing out of range, the good rows right."""
    torch = cuda
    c = Cache(torch, qvx.F16, (160, 90), 16, 1, 64, seed=11)
    q = torch.randn((10, 2, 64), device="cuda")
    for off in ([0, 7, 3], [-4, 900, 2], [5, 5, 1 << 30], [9, -9, 9], [0, 1 << 30, 1 << 30]):
        for lens in ([160, 90], [1 << 30, -5], [0, 0]):
            out = qvx.attn_window_t(q, c.desc, c.dev_table[:, :10].contiguous(),
                                    torch.tensor(lens, dtype=torch.int32, device="cuda"), 30, 2,
                                    torch.tensor(off, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            assert out.shape == q.shape


def test_captured_replays_follow_the_lengths(cuda):
    torch = cuda
    c = Cache(torch, qvx.F16, (5000, 400), 16, 2, 64, seed=13)
    lens = torch.tensor([5000, 400], dtype=torch.int32, device="cuda")
    calls = []
    for q_type, n_q in ((torch.float32, 2), (torch.float16, 64)):
        q = torch.randn((n_q, 4, 64), device="cuda").to(q_type)
        out = torch.zeros_like(q)
        calls.append((q, out))
        qvx.attn_window_t(q, c.desc, c.dev_table, lens, 2000, 4, out=out)
    torch.cuda.synchronize()
    graphs = []
    for q, out in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qvx.attn_window_t(q, c.desc, c.dev_table, lens, 2000, 4, out=out)
        graphs.append(graph)
    for a, b in ((5000, 400), (1, 0), (2513, 39), (4999, 16)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for q, out in calls:
            assert torch.equal(out, qvx.attn_window_t(q, c.desc, c.dev_table, lens, 2000, 4))
