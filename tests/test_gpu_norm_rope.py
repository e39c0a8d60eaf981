"""Norms of q and k heads with rotation and append on the GPU (qvx_norm_rope_kv) against the formula in 64 bits.

Tolerance.  u = 2^-24, a and b the normed values of a pair in 64 bits.  The squares are summed in 64 bits; mean, root and
quotient are rounded once each in fp32 (2.5 u, the root halving the mean's), as are the products with the scale and the weight: 4.5 u
of a value.  A cosine or sine is off by pi / 2 u for the angle's rounding to fp32 half turns and 2 u of its own.  Two products and
their sum add 2 u.  So |error| <= 12 u (|a| + |b|), and for the output's type half a step of the value.  Q8_0 rounds to half
a step of its block, and to what a scale rounded down leaves of the largest: 127 half steps of fp16."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def half_step(t):
    return {qvx.F32: 2.0 ** -24, qvx.F16: 2.0 ** -11, qvx.BF16: 2.0 ** -8}[t]


def torch_type(torch, t):
    return {qvx.F32: torch.float32, qvx.F16: torch.float16, qvx.BF16: torch.bfloat16}[t]


def turned(x, w, eps, angle, rot, pairing, scale):
    """x [tokens, heads, d] in float64, w [heads or 1, d] or None, angle [tokens, rot / 2]: values and |a| + |b|."""
    y = x.copy()
    if w is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    size = np.abs(y)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if pairing == qvx.ROPE_PAIRS else (i, i + rot // 2)
    out = y.copy()
    c, s = (f(angle)[:, None] * scale for f in (np.cos, np.sin))
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    both = (size[..., a] + size[..., b]) * max(1.0, abs(scale))
    size[..., a], size[..., b] = both, both
    return out, size


def check(torch, t, d, rot, pairing, hq, hk, n, each=False, q_type=qvx.F32, page=16, axes=1, shift=0, inplace=False,
          q_norm=True, k_norm=True, mul=1.0, eps=1e-6, seed=0, scale=1.0, pad_rows=()):
    r = np.random.default_rng(seed)
    width = (hq + hk) * d
    flat = torch.zeros(n * width + 8, device="cuda")
    qk = flat[shift: shift + n * width].view(n, width)
    host = (r.standard_normal((n, width)) * mul).astype(np.float32)
    qk.copy_(torch.from_numpy(host))
    v = torch.from_numpy(r.standard_normal((n, hk, d)).astype(np.float32)).cuda()
    w = [(1 + 0.3 * r.standard_normal((h, d) if each else (1, d))).astype(np.float32) for h in (hq, hk)]
    wt = [torch.from_numpy(x if each else x[0]).cuda() for x in w]
    norm = qvx.QkNorm.of(wt[0] if q_norm else None, wt[1] if k_norm else None, eps)
    freq = 10000.0 ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))
    axis = r.integers(0, axes, rot // 2).astype(np.uint8)
    pos = r.integers(0, 200000, (axes, n)).astype(np.int32)
    rope = qvx.Rope.of(torch.from_numpy(freq).cuda(), torch.from_numpy(axis).cuda(), axes, pairing, scale)
    pages = -(-n // page) + 2
    size = qvx.kv_page_bytes(t, hk, page, d)
    raw = [torch.full((pages, size), 7, dtype=torch.uint8, device="cuda") for _ in range(2)]
    before = [x.cpu().numpy() for x in raw]
    cache = qvx.KvCache.of(*raw, t, page, hk, d)
    slots = r.permutation(pages * page)[:n].astype(np.int32)
    for i, bad in pad_rows:
        slots[i] = bad
    q = qk[:, : hq * d].unflatten(1, (hq, d))
    k = qk[:, hq * d:].unflatten(1, (hk, d))
    out = q if inplace else torch.full((n, hq, d), 3.0, dtype=torch_type(torch, q_type), device="cuda")
    qvx.norm_rope_kv_t(q, k, v, torch.from_numpy(pos).cuda(), norm, rope, cache, torch.from_numpy(slots).cuda(), out=out)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < pages * page)
    angle = pos.astype(np.float64)[axis].T * freq
    x = host.astype(np.float64).reshape(n, hq + hk, d)
    want, mag = turned(x[:, :hq], w[0].astype(np.float64) if q_norm else None, eps, angle, rot, pairing, scale)
    got = out.double().cpu().numpy()
    bar = 12 * U * mag + half_step(q_type) * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want)[live] <= bar[live]).all()
    assert np.array_equal(got[~live], (x[:, :hq] if inplace else np.full_like(got, 3.0))[~live])

    wk, magk = turned(x[:, hq:], w[1].astype(np.float64) if k_norm else None, eps, angle, rot, pairing, scale)
    for raw_i, old, want, mag in ((raw[0], before[0], wk, magk), (raw[1], before[1], v.double().cpu().numpy(), np.zeros((n, hk, d)))):
        bytes_ = raw_i.cpu().numpy()
        touched = np.zeros(pages * page, bool)
        touched[slots[live]] = True
        if t == qvx.Q8_0:
            quant = bytes_[:, : hk * page * d].view(np.int8).reshape(pages, hk, page, d)
            steps = bytes_[:, hk * page * d: hk * page * d * 17 // 16].copy().view(np.float16).reshape(pages, hk, page, d // 32)
            vals = quant.astype(np.float64) * np.repeat(steps.astype(np.float64), 32, -1)
        else:
            vals = torch.from_numpy(bytes_[:, : hk * page * d * (4 if t == qvx.F32 else 2)].copy()).view(
                torch_type(torch, t)).double().numpy().reshape(pages, hk, page, d)
        for i in np.flatnonzero(live):
            p, o = divmod(int(slots[i]), page)
            bar = 12 * U * mag[i] + 2.0 ** -25
            if t == qvx.Q8_0:
                top = np.repeat(np.abs(want[i]).reshape(hk, d // 32, 32).max(-1), 32, -1).reshape(hk, d)
                bar = bar + (0.5 + 127 * 2.0 ** -11) * top / 127 * (1 + 2.0 ** -10)
            else:
                bar = bar + half_step(t) * np.abs(want[i])
            assert (np.abs(vals[p, :, o] - want[i]) <= bar).all(), i
        # what no token's slot names stays as it was
        if t != qvx.Q8_0:
            es = d * (4 if t == qvx.F32 else 2)
            same = (bytes_[:, : hk * page * es] == old[:, : hk * page * es]).reshape(pages, hk, page, es)
            assert same.transpose(0, 2, 1, 3).reshape(pages * page, -1)[~touched].all()


@pytest.mark.parametrize("t", [qvx.F32, qvx.F16, qvx.BF16, qvx.Q8_0])
@pytest.mark.parametrize("d,rot,pairing,hq,hk,n,each", [
    (128, 128, qvx.ROPE_HALVES, 32, 8, 1, False), (128, 64, qvx.ROPE_HALVES, 4, 2, 37, True),
    (64, 64, qvx.ROPE_PAIRS, 6, 3, 129, False), (96, 48, qvx.ROPE_PAIRS, 16, 4, 19, True),
    (96, 24, qvx.ROPE_HALVES, 2, 1, 5, False), (32, 8, qvx.ROPE_HALVES, 3, 3, 700, True),
    (256, 256, qvx.ROPE_HALVES, 4, 2, 33, False), (160, 0, qvx.ROPE_HALVES, 2, 2, 3, False)])
def test_types_and_heads(cuda, t, d, rot, pairing, hq, hk, n, each):
    check(cuda, t, d, rot, pairing, hq, hk, n, each)


@pytest.mark.parametrize("d,rot,hk", [(8, 8, 1), (16, 8, 5), (24, 16, 2), (40, 40, 4), (80, 40, 2), (112, 112, 1), (248, 24, 2)])
@pytest.mark.parametrize("pairing", [qvx.ROPE_HALVES, qvx.ROPE_PAIRS])
def test_odd_head_sizes(cuda, d, rot, hk, pairing):
    check(cuda, qvx.F16, d, rot, pairing, 3 * hk, hk, 21, each=True, q_type=qvx.BF16, page=5)


@pytest.mark.parametrize("q_type", [qvx.F16, qvx.BF16])
@pytest.mark.parametrize("shift", [0, 1])
def test_rounded_queries(cuda, q_type, shift):
    check(cuda, qvx.BF16, 128, 128, qvx.ROPE_HALVES, 8, 2, 300, q_type=q_type, shift=shift)


@pytest.mark.parametrize("kw", [dict(shift=1), dict(inplace=True), dict(axes=3), dict(q_norm=False), dict(k_norm=False),
                                dict(q_norm=False, k_norm=False), dict(mul=1e22), dict(mul=1e-22, eps=0.0), dict(scale=1.25),
                                dict(pad_rows=((0, -1), (5, 1 << 30), (6, -7)))])
@pytest.mark.parametrize("t", [qvx.F32, qvx.Q8_0])
def test_forms(cuda, t, kw):
    if kw.get("mul") == 1e22 and t == qvx.Q8_0:
        kw = dict(kw, k_norm=True)
    check(cuda, t, 64, 64, qvx.ROPE_HALVES, 4, 2, 40, **kw)


def test_without_a_cache(cuda):
    torch = cuda
    r = np.random.default_rng(1)
    x = r.standard_normal((9, 5, 48)).astype(np.float32)
    w = (1 + r.random(48)).astype(np.float32)
    pos = r.integers(0, 4096, 9).astype(np.int32)
    freq = 10000.0 ** (-np.arange(24) / 24.0)
    rope = qvx.Rope.of(torch.from_numpy(freq).cuda())
    q = torch.from_numpy(x).cuda()
    got = qvx.norm_rope_kv_t(q, None, None, torch.from_numpy(pos).cuda(), qvx.QkNorm.of(torch.from_numpy(w).cuda(), eps=1e-5), rope)
    want, mag = turned(x.astype(np.float64), w.astype(np.float64)[None], np.float64(np.float32(1e-5)),
                       pos[:, None].astype(np.float64) * freq, 48, qvx.ROPE_HALVES, 1.0)
    assert (np.abs(got.double().cpu().numpy() - want) <= 13 * U * mag).all()


def test_rows_of_zeros_nan_and_infinity(cuda):
    """A row of zeros stays one with an eps; what a row holds of NaN or infinity stays in it."""
    torch = cuda
    q = torch.ones((4, 3, 64), device="cuda")
    q[0, 1] = 0
    q[1, 2, 5] = float("nan")
    q[2, 0, 63] = float("inf")
    rope = qvx.Rope.of(torch.ones(32, dtype=torch.float64, device="cuda"))
    out = qvx.norm_rope_kv_t(q, None, None, torch.zeros(4, dtype=torch.int32, device="cuda"),
                             qvx.QkNorm.of(torch.ones(64, device="cuda")), rope)
    assert (out[0, 1] == 0).all() and torch.isnan(out[1, 2]).all() and not torch.isfinite(out[2, 0, 63])
    rest = torch.ones((4, 3), dtype=torch.bool)
    rest[0, 1] = rest[1, 2] = rest[2, 0] = False
    assert (out.cpu()[rest] - 1).abs().max() < 1e-5


def test_captured(cuda):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(3)
    n, hq, hk, d, page = 7, 8, 2, 128, 16
    q, k, v = (torch.randn((n, h, d), generator=g, device="cuda") for h in (hq, hk, hk))
    pages = torch.zeros((2, 3, qvx.kv_page_bytes(qvx.F16, hk, page, d)), dtype=torch.uint8, device="cuda")
    cache = qvx.KvCache.of(pages[0], pages[1], qvx.F16, page, hk, d)
    w = torch.rand(d, generator=g, device="cuda") + 0.5
    norm, rope = qvx.QkNorm.of(w, w, 1e-6), qvx.Rope.of(torch.rand(d // 2, dtype=torch.float64, generator=g, device="cuda"))
    pos, slots = torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    out = torch.zeros((n, hq, d), dtype=torch.float16, device="cuda")

    def call():
        qvx.norm_rope_kv_t(q, k, v, pos, norm, rope, cache, slots, out=out)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        q.normal_(generator=g)
        k.normal_(generator=g)
        pos.add_(5)
        slots.add_(3)
        pages.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [out.clone(), pages.clone()]
        pages.zero_()
        out.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], pages), i
