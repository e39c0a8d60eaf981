"""The paged cache's upkeep on the GPU: page tables and slots (qvx_kv_map), exact, against loops over sequences; and
rotary positions with the append (qvx_rope_kv) against the formula in 64 bits.

Tolerances of the rotation, u = 2^-24: the reduced angle is rounded once (at most pi u relative to a half turn), sine
and cosine are off by at most 2 ulp, each product and the sum by one rounding; so |error| <= (pi + 2 * 2 + 3) u * 2 max(|a|,
|b|) |scale|, 32 u max |x| |scale| in whole.  A 16-bit cache adds half a step of the value, Q8_0 half a step of its
block's scale and what rounding the scale adds to 127 of them."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _map_reference(held, new, table, page, free, taken, max_tokens):
    n = len(held)
    table = table.copy()
    rows = [(-1, 0, -1)] * max_tokens
    status = 0
    if taken < 0 or min(held) < 0 or min(new) < 0:
        status |= qvx.MAP_NEGATIVE
    good = [(h, k) for h, k in zip(held, new) if h >= 0 and k >= 0]
    need = sum(-(-(h + k) // page) - -(-h // page) for h, k in good)
    if any(h + k > table.shape[1] * page for h, k in good):
        status |= qvx.MAP_COLUMNS
    if sum(k for _, k in good) > max_tokens:
        status |= qvx.MAP_ROWS
    if taken >= 0 and taken + need > len(free):
        status |= qvx.MAP_PAGES
    if status:
        return table, list(held), [0] * (n + 1), rows, [taken, status]
    at, t, offsets = taken, 0, [0]
    for b in range(n):
        for column in range(-(-held[b] // page), -(-(held[b] + new[b]) // page)):
            table[b, column] = free[at]
            at += 1
        for p in range(held[b], held[b] + new[b]):
            page_id = int(table[b, p // page])
            slot = page_id * page + p % page
            rows[t] = (slot if page_id >= 0 and slot < 1 << 31 else -1, p, b)
            t += 1
        offsets.append(t)
    return table, [h + k for h, k in zip(held, new)], offsets, rows, [at, 0]


def _map_case(seed, n, most_held, most_new, page):
    r = np.random.default_rng(seed)
    held = [int(x) for x in r.integers(0, most_held + 1, n)]
    new = [int(x) for x in r.integers(0, most_new + 1, n)]
    width = -(-(most_held + most_new) // page) + 1
    table = np.full((n, width), -1, np.int32)
    for b in range(n):
        k = -(-held[b] // page)
        table[b, :k] = r.integers(0, 5000, k)
    need = sum(-(-(h + k) // page) - -(-h // page) for h, k in zip(held, new))
    free = r.permutation(need + 9).astype(np.int32)
    return held, new, table, free, need


def _run_map(torch, held, new, table, page, free, taken, max_tokens, in_place=False):
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    h, k, tab, fr, tk = i32(held), i32(new), i32(table), i32(free), i32([taken, 77])
    if not in_place:
        lens, offsets, slots, pos, seq, out = qvx.kv_map_t(h, k, tab, page, fr, tk, max_tokens)
    else:
        lens, out = h, tk
        offsets = torch.full((len(held) + 1,), 9, dtype=torch.int32, device="cuda")
        slots, pos, seq = (torch.full((max(max_tokens, 1),), 9, dtype=torch.int32, device="cuda") for _ in range(3))
        rc = qvx.kv_map(h.data_ptr(), k.data_ptr(), len(held), tab.data_ptr(), tab.shape[1], page, fr.data_ptr(),
                        fr.shape[0], tk.data_ptr(), tk.data_ptr(), h.data_ptr(), offsets.data_ptr(), slots.data_ptr(),
                        pos.data_ptr(), seq.data_ptr(), max_tokens, torch.cuda.current_stream().cuda_stream)
        assert rc == qvx.OK
        slots, pos, seq = slots[:max_tokens], pos[:max_tokens], seq[:max_tokens]
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (tab, lens, offsets, slots, pos, seq, out)]


def _check_map(torch, held, new, table, page, free, taken, max_tokens, in_place=False):
    got = _run_map(torch, held, new, table, page, free, taken, max_tokens, in_place)
    table, lens, offsets, rows, out = _map_reference(held, new, table, page, free, taken, max_tokens)
    rows = np.array(rows, np.int64).reshape(-1, 3)
    for g, w in zip(got, (table, lens, offsets, rows[:, 0], rows[:, 1], rows[:, 2], out)):
        np.testing.assert_array_equal(g, np.asarray(w))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,held,new,page", [(1, 0, 1, 16), (1, 40, 0, 16), (7, 100, 5, 1), (64, 300, 1, 16), (65, 10, 90, 24),
                                             (1000, 50, 3, 8), (1025, 20, 12, 16), (5000, 6, 2, 4), (3, 5, 9000, 256)])
def test_map_matches_the_loops(cuda, n, held, new, page, in_place):
    held, new, table, free, need = _map_case(n + page, n, held, new, page)
    _check_map(cuda, held, new, table, page, free, 4, sum(new) + 6, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_map_refusals_change_nothing(cuda, in_place):
    held, new, table, free, need = _map_case(3, 20, 60, 30, 16)
    total = sum(new)
    for status, args in ((qvx.MAP_PAGES, (free[: need + 3], 4, total)), (qvx.MAP_ROWS, (free, 4, total - 1)),
                         (qvx.MAP_NEGATIVE, (free, -1, total))):
        fr, taken, rows = args
        got = _run_map(cuda, held, new, table, 16, fr, taken, rows, in_place)
        assert got[-1].tolist() == [taken, status]
        _check_map(cuda, held, new, table, 16, fr, taken, rows, in_place)
    bad = list(new)
    bad[3] = -1
    _check_map(cuda, held, bad, table, 16, free, 4, total, in_place)
    bad = list(held)
    bad[19] = 1 << 30
    got = _run_map(cuda, bad, new, table, 16, free, 4, total, in_place)
    assert got[-1].tolist()[1] & qvx.MAP_COLUMNS
    big = [2 ** 31 - 1] * 3
    got = _run_map(cuda, big, big, np.zeros((3, 4), np.int32), 16, free, 0, 10, in_place)
    assert got[-1].tolist()[0] == 0 and got[-1].tolist()[1] & qvx.MAP_ROWS
    assert got[1].tolist() == big and (got[3] == -1).all()


def test_map_captured_steps_in_place(cuda):
    """A captured in-place step replayed as decoding goes on: lengths and the pages taken carry over."""
    torch = cuda
    n, page, steps = 9, 4, 10
    held = [3, 0, 4, 7, 8, 1, 2, 15, 11]
    table = np.full((n, 8), -1, np.int32)
    ids = iter(range(100, 200))
    for b, h in enumerate(held):
        for p in range(-(-h // page)):
            table[b, p] = next(ids)
    free = np.arange(40, dtype=np.int32)[::-1].copy()
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    lens, new, tab, fr, tk = i32(held), i32([1] * n), i32(table), i32(free), i32([0, 0])
    offsets, slots, pos, seq = i32([0] * (n + 1)), i32([0] * 12), i32([0] * 12), i32([0] * 12)

    def step():
        return qvx.kv_map(lens.data_ptr(), new.data_ptr(), n, tab.data_ptr(), 8, page, fr.data_ptr(), 40, tk.data_ptr(),
                          tk.data_ptr(), lens.data_ptr(), offsets.data_ptr(), slots.data_ptr(), pos.data_ptr(),
                          seq.data_ptr(), 12, torch.cuda.current_stream().cuda_stream)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert step() == qvx.OK
    taken = 0
    for _ in range(steps):
        g.replay()
        torch.cuda.synchronize()
        table, held, want, rows, out = _map_reference(held, [1] * n, table, page, free, taken, 12)
        taken = out[0]
        assert tk.tolist() == out and lens.tolist() == held and offsets.tolist() == want
        np.testing.assert_array_equal(tab.cpu().numpy(), table)
        assert slots.tolist() == [r[0] for r in rows] and pos.tolist() == [r[1] for r in rows]


# ---- rotary positions and the append ------------------------------------------------------------------------

def _turn(x, angle, rot, pairing, scale):
    """x [tokens, heads, d] in float64, angle [tokens, rot / 2]."""
    y = x.copy()
    c, s = (scale * f(angle)[:, None, :] for f in (np.cos, np.sin))
    if rot:
        if pairing == qvx.ROPE_HALVES:
            a, b = x[..., : rot // 2], x[..., rot // 2: rot]
            y[..., : rot // 2], y[..., rot // 2: rot] = a * c - b * s, a * s + b * c
        else:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    return y


def _check_rope(torch, t, n, hq, hk, d, page, rot=None, axes=1, pairing=qvx.ROPE_HALVES, scale=1.0, far=1 << 20, seed=0,
                shift=0, in_place=False, pad=0):
    r = np.random.default_rng(seed)
    rot = d if rot is None else rot
    half = rot // 2
    pages = -(-n // page) + 2
    slots = r.permutation(pages * page)[:n].astype(np.int32)
    padding = r.random(n) < 0.2 if n > 3 else np.zeros(n, bool)
    dev_slots = np.where(padding, np.where(r.random(n) < 0.5, -1, pages * page), slots).astype(np.int32)
    pos = r.integers(0, far, (axes, n)).astype(np.int32)
    freq = 10000.0 ** (-np.arange(half) / max(half, 1))
    axis = r.integers(0, axes, half).astype(np.uint8)
    wide = torch.from_numpy(r.standard_normal((n, shift + (hq + 2 * hk) * d + 3 * shift)).astype(np.float32)).cuda()
    q, k, v = (wide[:, shift + a * d: shift + b * d].unflatten(1, (b - a, d)) for a, b in
               ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
    before = [x.cpu().double().numpy() for x in (q, k, v)]
    size = qvx.kv_page_bytes(t, hk, page, d)
    caches = [torch.from_numpy(r.integers(0, 120, (pages, size + pad)).astype(np.uint8)).cuda() for _ in range(2)]
    old = [c.cpu().numpy().copy() for c in caches]
    desc = qvx.KvCache(caches[0].data_ptr(), caches[1].data_ptr(), size + pad, t, pages, page, hk, d)
    rope = qvx.Rope.of(torch.from_numpy(freq).cuda(), torch.from_numpy(axis).cuda() if axes > 1 else None, axes, pairing, scale)
    out = q if in_place else torch.full((n, hq, d), 9.0, device="cuda")
    qvx.rope_kv_t(q, k, v, torch.from_numpy(pos).cuda(), rope, desc, torch.from_numpy(dev_slots).cuda(), out=out)
    torch.cuda.synchronize()
    angle = pos[axis if axes > 1 else np.zeros(half, int)].T * freq[None, :]
    want = [_turn(x, angle, rot, pairing, scale) for x in before[:2]] + [before[2]]
    got = out.cpu().double().numpy()
    top = max(np.abs(x).max() for x in before)
    tol = 32 * U * top * max(1.0, abs(scale))
    kept = before[0] if in_place else np.full_like(got, 9.0)
    assert np.abs(got[~padding] - want[0][~padding]).max(initial=0.0) <= tol
    np.testing.assert_array_equal(got[padding], kept[padding])
    for cache, was, w in zip(caches, old, want[1:]):
        raw = cache.cpu().numpy()
        live = np.zeros((pages, page), bool)
        live[slots[~padding] // page, slots[~padding] % page] = True
        if t == qvx.Q8_0:
            cut = hk * page * d
            quant = raw[:, :cut].view(np.int8).reshape(pages, hk, page, d)
            steps = raw[:, cut: cut + cut // 16].copy().view(np.float16).reshape(pages, hk, page, d // 32).astype(np.float64)
            vals = quant * np.repeat(steps, 32, -1)
            for i in np.flatnonzero(~padding):
                p, o = slots[i] // page, slots[i] % page
                blocks = np.abs(w[i]).reshape(hk, d // 32, 32).max(-1)
                np.testing.assert_allclose(steps[p, :, o], blocks / 127, rtol=2.0 ** -11 + 1e-5)
                half_step = np.repeat(steps[p, :, o], 32, -1) * (0.5 + 127 * 2.0 ** -11)
                assert (np.abs(vals[p, :, o] - w[i]) <= half_step + tol).all()
            raw_rows, was_rows = quant, was[:, :cut].view(np.int8).reshape(pages, hk, page, d)
        else:
            es = 4 if t == qvx.F32 else 2
            x = torch.from_numpy(raw[:, : hk * page * d * es].copy()).view({qvx.F32: torch.float32, qvx.F16: torch.float16,
                                                                            qvx.BF16: torch.bfloat16}[t])
            vals = x.double().numpy().reshape(pages, hk, page, d)
            step = {qvx.F32: 2.0 ** -24, qvx.F16: 2.0 ** -11, qvx.BF16: 2.0 ** -8}[t]
            for i in np.flatnonzero(~padding):
                got = vals[slots[i] // page, :, slots[i] % page]
                assert (np.abs(got - w[i]) <= tol + (np.abs(w[i]) + tol) * step + 2.0 ** -25).all()
            raw_rows = raw[:, : hk * page * d * es].reshape(pages, hk, page, d * es)
            was_rows = was[:, : hk * page * d * es].reshape(pages, hk, page, d * es)
        dead = np.broadcast_to(~live[:, None, :, None], raw_rows.shape)
        np.testing.assert_array_equal(raw_rows[dead], was_rows[dead])
        if pad:
            np.testing.assert_array_equal(raw[:, size:], was[:, size:])


CACHE_TYPES = (qvx.F16, qvx.BF16, qvx.F32, qvx.Q8_0)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("n", [1, 2, 37, 600, 2100])
def test_rope_tokens(cuda, t, n):
    _check_rope(cuda, t, n, 4, 2, 64, 16, seed=n)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("pairing", [qvx.ROPE_HALVES, qvx.ROPE_PAIRS])
@pytest.mark.parametrize("d,rot", [(32, 32), (96, 96), (128, 64), (128, 24), (256, 256), (64, 0), (64, 8)])
def test_rope_sizes(cuda, t, pairing, d, rot):
    _check_rope(cuda, t, 21, 3, 1, d, 8, rot=rot, pairing=pairing, scale=0.75, seed=d + rot)


@pytest.mark.parametrize("d", [8, 40, 72, 80])
def test_rope_odd_sizes(cuda, d):
    for pairing in (qvx.ROPE_HALVES, qvx.ROPE_PAIRS):
        _check_rope(cuda, qvx.F16, 30, 5, 5, d, 24, pairing=pairing, seed=d)


@pytest.mark.parametrize("axes", [2, 3, 4])
def test_rope_axes(cuda, axes):
    _check_rope(cuda, qvx.BF16, 50, 8, 2, 128, 32, axes=axes, seed=axes)


def test_rope_far_positions(cuda):
    _check_rope(cuda, qvx.F32, 64, 2, 2, 64, 16, far=2 ** 31 - 1, seed=1)


@pytest.mark.parametrize("shift", [0, 4, 1])
def test_rope_strides_and_alignment(cuda, shift):
    """Rows inside a wider product: 16-byte-aligned ones, and ones that are only 4-byte aligned."""
    for t in (qvx.F16, qvx.Q8_0):
        _check_rope(cuda, t, 40, 4, 2, 64, 16, seed=shift, shift=shift)
        _check_rope(cuda, t, 40, 4, 2, 64, 16, seed=shift, shift=shift, in_place=True, pad=32)


def test_rope_without_a_cache(cuda):
    torch = cuda
    r = np.random.default_rng(2)
    q = torch.from_numpy(r.standard_normal((33, 5, 80)).astype(np.float32)).cuda()
    freq = 10000.0 ** (-np.arange(40) / 40)
    pos = r.integers(0, 90, (2, 33)).astype(np.int32)
    axis = (np.arange(40) % 2).astype(np.uint8)
    rope = qvx.Rope.of(torch.from_numpy(freq).cuda(), torch.from_numpy(axis).cuda(), 2)
    got = qvx.rope_kv_t(q, None, None, torch.from_numpy(pos).cuda(), rope)
    torch.cuda.synchronize()
    x = q.cpu().double().numpy()
    want = _turn(x, pos[axis].T * freq, 80, qvx.ROPE_HALVES, 1.0)
    assert np.abs(got.cpu().double().numpy() - want).max() <= 32 * U * np.abs(x).max()


def test_rope_non_finite_values(cuda):
    """A NaN stays in its pair; a Q8_0 block that holds one stands for NaN as a whole."""
    torch = cuda
    for t in (qvx.F16, qvx.Q8_0):
        k = torch.ones((1, 1, 64), device="cuda")
        k[0, 0, 3] = float("nan")
        v = torch.ones((1, 1, 64), device="cuda")
        size = qvx.kv_page_bytes(t, 1, 16, 64)
        caches = [torch.zeros((2, size), dtype=torch.uint8, device="cuda") for _ in range(2)]
        desc = qvx.KvCache.of(*caches, t, 16, 1, 64)
        rope = qvx.Rope.of(torch.zeros(32, dtype=torch.float64, device="cuda"))
        one = torch.zeros(1, dtype=torch.int32, device="cuda")
        qvx.rope_kv_t(torch.ones((1, 1, 64), device="cuda"), k, v, one, rope, desc, one)
        raw = caches[0].cpu()
        if t == qvx.F16:
            row = raw.view(torch.float16).view(2, 16, 64)[0, 0]
            nan = torch.isnan(row)
            assert bool(nan[3]) and bool(nan[35]) and int(nan.sum()) == 2
        else:
            scales = raw[0, 16 * 64:].view(torch.float16).view(16, 2)[0]
            assert bool(torch.isnan(scales).all())  # pairs 3 and 35: one in each block


def test_rope_captured(cuda):
    torch = cuda
    n, hq, hk, d = 5, 4, 2, 64
    q, k, v = (torch.randn((n, h, d), device="cuda") for h in (hq, hk, hk))
    caches = [torch.zeros((4, qvx.kv_page_bytes(qvx.F16, hk, 16, d)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    desc = qvx.KvCache.of(*caches, qvx.F16, 16, hk, d)
    rope = qvx.Rope.of(torch.from_numpy(10000.0 ** (-np.arange(32) / 32)).cuda())
    pos, slots = torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    qvx.rope_kv_t(q, k, v, pos, rope, desc, slots, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qvx.rope_kv_t(q, k, v, pos, rope, desc, slots, out=out)
    for step in range(3):
        pos.add_(7)
        slots.add_(11)
        q.normal_()
        g.replay()
        torch.cuda.synchronize()
        got, kept = out.clone(), [c.clone() for c in caches]
        want = qvx.rope_kv_t(q, k, v, pos, rope, desc, slots)
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(kept, caches))


def test_rope_leaves_zeros_in_padding_rows_of_its_own_output(cuda):
    """Rows of a token without a slot in the tensor that the call makes: zeros, not what its memory held before."""
    torch = cuda
    n, hq, hk, d = 6, 4, 2, 64
    q, k, v = (torch.randn((n, h, d), device="cuda") for h in (hq, hk, hk))
    caches = [torch.zeros((4, qvx.kv_page_bytes(qvx.F16, hk, 16, d)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    desc = qvx.KvCache.of(*caches, qvx.F16, 16, hk, d)
    rope = qvx.Rope.of(torch.ones(32, dtype=torch.float64, device="cuda"))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = torch.tensor([3, -1, 64, 5, -1, 0], dtype=torch.int32, device="cuda")
    held = [torch.full((n, hq, d), float("nan"), device="cuda") for _ in range(8)]
    del held
    got = qvx.rope_kv_t(q, k, v, pos, rope, desc, slots)
    dead = torch.tensor([1, 2, 4], device="cuda")
    assert bool((got[dead] == 0).all())
    want = qvx.rope_kv_t(q, k, v, pos, rope, desc, slots, out=torch.full_like(q, 2.0))
    live = torch.tensor([0, 3, 5], device="cuda")
    assert torch.equal(got[live], want[live]) and bool((want[dead] == 2.0).all())


@pytest.mark.parametrize("in_place", [False, True])
def test_map_of_as_many_sequences_as_a_call_takes(cuda, in_place):
    held, new, table, free, need = _map_case(3, 16384, 30, 4, 8)
    _check_map(cuda, held, new, table, 8, free, 2, sum(new) + 3, in_place)
