"""The attention calls on the GPU (qvx_attn_paged, qvx_attn_cross) against the formula in 64 bits on the CPU.

Tolerances.  u = 2^-24.  A logit is a sum of d products: its error is at most (d + 3) u sum |q_i k_i| scale, which
moves a weight by that much relative to itself; the hardware's power of two adds 2 u, the sum of n weights and that
of n products n u each at worst, and numerator and denominator both carry them.  So |error| <= 2 u ((d + 3) S + n + 8)
max |v|, S the largest sum |q_i k_i| scale of the call.  A 16-bit output adds half a step of its own value; where the
weights are rounded to 16 bits, half a step of every weight: at most that part of max |v|."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _torch_type(torch, t):
    return {qvx.F32: torch.float32, qvx.F16: torch.float16, qvx.BF16: torch.bfloat16}[t]


def _attend(q, k, v, scale):
    """q [rows, d], k and v [keys, d] in float64: (softmax(scale q k^T) v, the largest sum |q k| scale)."""
    s = (q @ k.T) * scale
    w = np.exp(s - s.max(axis=-1, keepdims=True))
    return (w @ v) / w.sum(-1, keepdims=True), float((np.abs(q) @ np.abs(k).T).max() * abs(scale))


class Cache:
    """A paged cache on the GPU, its values in float64 on the host, and NaN wherever no sequence lives."""

    def __init__(self, torch, t, lens, page, kv_heads, d, seed=0, spare=3, pad=0):
        r = np.random.default_rng(seed)
        self.t, self.page, self.hk, self.d = t, page, kv_heads, d
        self.lens = list(lens)
        used = [-(-n // page) for n in lens]
        self.width = max(max(used), 1) + 1
        ids = r.permutation(sum(used) + spare)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.n_pages = sum(used) + spare
        self.host, tensors = [], []
        stride = qvx.kv_page_bytes(t, kv_heads, page, d) + pad
        both = torch.full((self.n_pages, 2 * stride if pad else stride), 255, dtype=torch.uint8)  # NaN, or quants of -1
        for i in range(2):
            vals = r.standard_normal((self.n_pages, kv_heads, page, d)).astype(np.float32)
            live = np.zeros((self.n_pages, page), bool)
            for b, n in enumerate(lens):
                for p in range(used[b]):
                    live[self.table[b, p], : min(page, n - p * page)] = True
            if t == qvx.Q8_0:
                scale = (r.random((self.n_pages, kv_heads, page, d // 32)).astype(np.float32) * 0.02 + 0.001).astype(np.float16)
                quant = r.integers(-127, 128, vals.shape).astype(np.int8)
                mask = np.broadcast_to(live[:, None, :, None], scale.shape)
                scale = np.where(mask, scale, np.float16(np.nan))
                host = quant.astype(np.float64) * np.repeat(scale.astype(np.float64), 32, axis=-1)
                raw = np.concatenate([quant.reshape(self.n_pages, -1).view(np.uint8),
                                      scale.reshape(self.n_pages, -1).view(np.uint8)], 1)
                raw = torch.from_numpy(raw)
            else:
                vals = np.where(live[:, None, :, None], vals, np.float32(np.nan))
                x = torch.from_numpy(vals).to(_torch_type(torch, t))
                host = x.double().numpy()
                raw = x.reshape(self.n_pages, -1).view(torch.uint8)
            self.host.append(host)
            if pad:  # K and V in one allocation, with a gap
                both[:, i * stride: i * stride + raw.shape[1]] = raw
            else:
                tensors.append(torch.nn.functional.pad(raw, (0, stride - raw.shape[1])).cuda())
        if pad:
            both = both.cuda()
            tensors = [both[:, :stride], both[:, stride:]]
            self.desc = qvx.KvCache(tensors[0].data_ptr(), tensors[1].data_ptr(), 2 * stride, t, self.n_pages, page,
                                    kv_heads, d)
            self.desc.tensors = tensors
        else:
            self.desc = qvx.KvCache(tensors[0].data_ptr(), tensors[1].data_ptr(), 0, t, self.n_pages, page, kv_heads, d)
            self.desc.tensors = tensors
        self.dev_table = torch.from_numpy(self.table).cuda()
        self.dev_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def rows(self, b, i):
        """K (i = 0) or V of sequence b: [heads, tokens, d]."""
        n = self.lens[b]
        pages = self.host[i][self.table[b, : -(-n // self.page)]]
        return pages.transpose(1, 0, 2, 3).reshape(self.hk, -1, self.d)[:, :n]


def _paged_reference(c, q, scale):
    n, hq, d = q.shape
    g = hq // c.hk
    out, most = np.zeros((n, hq, d)), 0.0
    for b in range(n):
        if not c.lens[b]:
            continue
        k, v = c.rows(b, 0), c.rows(b, 1)
        for h in range(c.hk):
            out[b, h * g:(h + 1) * g], s = _attend(q[b, h * g:(h + 1) * g].astype(np.float64), k[h], v[h], scale)
            most = max(most, s)
    vmax = max((float(np.abs(c.rows(b, 1)).max()) for b in range(n) if c.lens[b]), default=0.0)
    return out, 2 * U * ((d + 3) * most + max(c.lens) + 8) * vmax


def _check_paged(torch, c, hq, seed=1, scale=None):
    q = torch.from_numpy(np.random.default_rng(seed).standard_normal((len(c.lens), hq, c.d)).astype(np.float32) * 1.5).cuda()
    out = torch.full_like(q, 7.0)
    qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens, scale=scale, out=out)
    torch.cuda.synchronize()
    want, tol = _paged_reference(c, q.cpu().numpy(), c.d ** -0.5 if scale is None else scale)
    got = out.cpu().double().numpy()
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= tol, (np.abs(got - want).max(), tol)
    return q, out


CACHE_TYPES = (qvx.F16, qvx.BF16, qvx.F32, qvx.Q8_0)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("lens", [(1,), (16,), (17, 1, 0, 33), (127, 128, 129), (700,), (1500, 3, 0, 260)])
def test_paged_lengths(cuda, t, lens):
    _check_paged(cuda, Cache(cuda, t, lens, 16, 2, 128, seed=sum(lens)), 8)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 256])
def test_paged_head_sizes(cuda, t, d):
    _check_paged(cuda, Cache(cuda, t, (5, 0, 290), 32, 2, d, seed=d), 6)


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32))
@pytest.mark.parametrize("d", [8, 40, 72, 80, 136, 248])
def test_paged_odd_head_sizes(cuda, t, d):
    _check_paged(cuda, Cache(cuda, t, (5, 0, 290), 32, 2, d, seed=d), 4)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 40, 64, 256])
@pytest.mark.parametrize("t", (qvx.BF16, qvx.Q8_0))
def test_paged_page_sizes(cuda, t, page):
    """Pages that end inside a tile of 16 keys, and pages of many tiles."""
    _check_paged(cuda, Cache(cuda, t, (1, 100, 333, page), page, 2, 64, seed=page), 4)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 5), (7, 1), (16, 1), (17, 1), (40, 1), (24, 2), (64, 4)])
def test_paged_head_layouts(cuda, hq, hk):
    """A head each, groups, one key head for more query heads than a row tile holds."""
    _check_paged(cuda, Cache(cuda, qvx.F16, (400, 9), 16, hk, 64, seed=hq), hq)


@pytest.mark.parametrize("n", [64, 65, 300, 1030])
def test_paged_many_sequences(cuda, n):
    """Wave-wide and workgroup-wide partitions, most sequences short, some split."""
    lens = [int(x) for x in np.random.default_rng(n).integers(0, 40, n)]
    lens[n // 2] = 900
    lens[-1] = 411
    _check_paged(cuda, Cache(cuda, qvx.F16, lens, 16, 1, 64, seed=n), 2)


@pytest.mark.parametrize("n,longest", [(60, 3000), (64, 200), (150, 2500)])
@pytest.mark.parametrize("t", (qvx.F16, qvx.Q8_0))
def test_paged_lengths_of_every_kind(cuda, t, n, longest):
    """More chunks and rests than the card has places, of all lengths, in no order, empty sequences among them."""
    r = np.random.default_rng(n)
    lens = [int(x) for x in np.exp(r.uniform(0, np.log(longest), n))]
    lens[n // 2], lens[n // 3], lens[7] = longest, 0, longest // 2 + 1
    _check_paged(cuda, Cache(cuda, t, lens, 16, 8, 32, seed=n), 16)


def test_paged_long_sequence(cuda):
    """Many chunks a sequence, several tiles a wave: lengths around 40000 tokens."""
    _check_paged(cuda, Cache(cuda, qvx.BF16, (40007, 39999), 64, 2, 64, seed=4), 4)


def test_paged_sharp_and_rising_logits(cuda):
    """One key carries nearly all the weight, and logits that rise along the sequence by more than the kernel's slack."""
    torch = cuda
    c = Cache(torch, qvx.F16, (600,), 16, 1, 64, seed=2)
    _check_paged(torch, c, 4, scale=3.0)
    r = np.random.default_rng(5)
    c = Cache(torch, qvx.F32, (640,), 16, 1, 64, seed=5)
    q = r.standard_normal((1, 4, 64)).astype(np.float32)
    for p in range(40):  # logits of head 0 from about -160 to 160
        for o in range(16):
            j = 16 * p + o
            c.host[0][c.table[0, p], 0, o] = q[0, 0] * (j - 320) / 2 / 64
    k = torch.from_numpy(c.host[0].astype(np.float32)).reshape(c.n_pages, -1).view(torch.uint8).cuda()
    c.host[0] = c.host[0].astype(np.float32).astype(np.float64)
    c.desc.d_k = k.data_ptr()
    qd = torch.from_numpy(q).cuda()
    out = qvx.attn_paged_t(qd, c.desc, c.dev_table, c.dev_lens, scale=1.0)
    torch.cuda.synchronize()
    want, tol = _paged_reference(c, q, 1.0)
    assert np.abs(out.cpu().double().numpy() - want).max() <= tol


def test_paged_interleaved_pages_and_strided_rows(cuda):
    """K and V in one allocation (a page stride), q rows out of a wider product, out rows into one."""
    torch = cuda
    c = Cache(torch, qvx.F16, (50, 0, 777), 16, 2, 64, seed=8, pad=48)
    wide = torch.randn((3, 1000), device="cuda")
    q = wide[:, 100:100 + 8 * 64].unflatten(1, (8, 64))
    dst = torch.full((3, 700), 5.0, device="cuda")
    out = dst[:, 60:60 + 8 * 64].unflatten(1, (8, 64))
    qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens, out=out)
    torch.cuda.synchronize()
    want, tol = _paged_reference(c, q.cpu().numpy(), 64 ** -0.5)
    assert np.abs(out.cpu().double().numpy() - want).max() <= tol
    assert bool((dst[:, :60] == 5.0).all()) and bool((dst[:, 60 + 512:] == 5.0).all())


def test_paged_in_place_and_repeatable(cuda):
    torch = cuda
    c = Cache(torch, qvx.F16, (1200, 5, 0, 333), 16, 2, 128, seed=9)
    q = torch.randn((4, 8, 128), device="cuda")
    first = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
    again = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
    assert torch.equal(first, again)
    qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens, out=q)
    assert torch.equal(first, q)


def test_paged_missing_pages_do_not_count(cuda):
    """Ids outside the cache inside a sequence: its other pages alone are attended."""
    torch = cuda
    c = Cache(torch, qvx.BF16, (96, 64), 16, 1, 64, seed=10)
    q = torch.randn((2, 2, 64), device="cuda")
    bad = c.table.copy()
    bad[0, 1], bad[0, 4], bad[1, :4] = -1, c.n_pages, 1 << 30
    out = qvx.attn_paged_t(q, c.desc, torch.from_numpy(bad).cuda(), c.dev_lens)
    torch.cuda.synchronize()
    k, v = c.rows(0, 0), c.rows(0, 1)
    keep = np.r_[0:16, 32:64, 80:96]
    want, s = _attend(q[0].cpu().double().numpy(), k[0][keep], v[0][keep], 64 ** -0.5)
    assert np.abs(out[0].cpu().double().numpy() - want).max() <= 2 * U * (67 * s + 104) * np.abs(v).max()
    assert bool((out[1] == 0).all())  # none is left: as for a sequence without any


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32))
@pytest.mark.parametrize("n", [20, 2000])
@pytest.mark.parametrize("group", [1, 6, 16])
def test_paged_keys_without_weight(cuda, t, n, group):
    """Logits of -inf weigh nothing; where a row has no other it is 0 / 0, unless its pages are missing: then zeros."""
    torch = cuda
    c = Cache(torch, t, (n, n, n), 16, 1, 64, seed=15)
    k = c.desc.tensors[0].view(_torch_type(torch, t)).view(c.n_pages, 16, 64)
    pages = torch.from_numpy(c.table).cuda().long()
    full = n // 16
    k[pages[0, : full - 1], :, 3] = float("-inf")   # all but the last pages' keys of sequence 0
    k[pages[1, : c.width - 1], :, 3] = float("-inf")  # all of sequence 1
    c.dev_table[2] = -1
    q = torch.randn((3, group, 64), device="cuda")
    q[:, :, 3] = 1.0
    out = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
    kept = np.arange(16 * (full - 1), n)
    kk, vv = c.rows(0, 0)[0][kept], c.rows(0, 1)[0][kept]
    want, s = _attend(q[0].cpu().double().numpy(), kk, vv, 64 ** -0.5)
    if t == qvx.F32:  # of a 16-bit cache the query is multiplied in parts, 0 times an infinite key among them
        assert np.abs(out[0].cpu().double().numpy() - want).max() <= 2 * U * (67 * s + n + 8) * np.abs(c.rows(0, 1)).max()
    assert bool(torch.isnan(out[1]).all()) and bool((out[2] == 0).all())


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("group", [1, 8, 16])
def test_paged_scale_of_zero_and_below(cuda, t, group):
    """Equal weights, whatever the masked tail of a tile holds; and the smallest key the heaviest."""
    for scale in (0.0, -0.3):
        c = Cache(cuda, t, (37, 1, 500), 24, 1, 64, seed=16)
        _check_paged(cuda, c, group, scale=scale)


@pytest.mark.parametrize("t,n", [(qvx.F16, 8), (qvx.Q8_0, 16)])
def test_paged_past_half_the_memory_side_cache(cuda, t, n):
    """More than 128 MiB of keys and values (their loads are marked as read once), the smallest sequences beside them."""
    c = Cache(cuda, t, (8191,) * n + (1, 0), 32, 8, 64 if t == qvx.F16 else 64, seed=17)
    _check_paged(cuda, c, 8)


def test_paged_lengths_past_the_table(cuda):
    torch = cuda
    c = Cache(torch, qvx.F16, (160,), 16, 1, 64, seed=11)
    q = torch.randn((1, 2, 64), device="cuda")
    full = qvx.attn_paged_t(q, c.desc, c.dev_table[:, :10].contiguous(), c.dev_lens)
    cut = qvx.attn_paged_t(q, c.desc, c.dev_table[:, :10].contiguous(), torch.tensor([1 << 30], dtype=torch.int32, device="cuda"))
    below = qvx.attn_paged_t(q, c.desc, c.dev_table, torch.tensor([-5], dtype=torch.int32, device="cuda"))
    assert torch.equal(full, cut) and bool((below == 0).all())


def test_paged_non_finite_values_stay_in_their_rows(cuda):
    """A NaN query makes its own head NaN, an infinite logit its own row; the neighbours keep their bits."""
    torch = cuda
    c = Cache(torch, qvx.F16, (300, 200), 16, 2, 64, seed=12)
    q = torch.randn((2, 4, 64), device="cuda")
    clean = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
    q[0, 1, 5] = float("nan")
    q[1, 2, 7] = float("inf")
    got = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
    assert bool(torch.isnan(got[0, 1]).all()) and bool(torch.isnan(got[1, 2]).all())
    keep = torch.ones((2, 4), dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[1, 2] = False
    assert torch.equal(got[keep], clean[keep])


def test_paged_captured_replays_follow_the_lengths(cuda):
    """One captured call over growing lengths; a second graph with its own workspace between the replays."""
    torch = cuda
    c = Cache(torch, qvx.F16, (900, 40), 16, 2, 64, seed=13)
    q = torch.randn((2, 4, 64), device="cuda")
    q2 = torch.randn((2, 4, 64), device="cuda")
    lens = torch.tensor([900, 40], dtype=torch.int32, device="cuda")
    qvx.attn_paged_t(q, c.desc, c.dev_table, lens)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        out = torch.empty_like(x)
        with torch.cuda.graph(g):
            qvx.attn_paged_t(x, c.desc, c.dev_table, lens, out=out)
        graphs.append(g)
        outs.append(out)
    for a, b in ((900, 40), (1, 0), (513, 39), (900, 16)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        for g in graphs:
            g.replay()
        for x, out in zip((q, q2), outs):
            assert torch.equal(out, qvx.attn_paged_t(x, c.desc, c.dev_table, lens))
        torch.cuda.synchronize()


def test_paged_on_another_stream(cuda):
    torch = cuda
    c = Cache(torch, qvx.F16, (2000, 17), 16, 2, 64, seed=14)
    q = torch.randn((2, 4, 64), device="cuda")
    want = qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (s1, s2, s1, s2):
        with torch.cuda.stream(s):
            outs.append(qvx.attn_paged_t(q, c.desc, c.dev_table, c.dev_lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---- cross attention --------------------------------------------------------------------------------------

def _check_cross(torch, q_type, kv_type, nq, ns, hq, hk, d, seed=0, stacked=True, equal=False, tail=3, scale=None, pads=None):
    """pads: elements before q's and out's first row, and behind each of their rows."""
    r = np.random.default_rng(seed)
    qt, kt = _torch_type(torch, q_type), _torch_type(torch, kv_type)
    n, most = len(nq), max(max(ns), 1)
    rows = sum(nq) + (0 if equal else tail)
    q = torch.from_numpy(r.standard_normal((rows, hq, d)).astype(np.float32) * 1.5).to(qt)
    kv = torch.from_numpy(r.standard_normal((n, most, 2, hk, d)).astype(np.float32)).to(kt)
    for b, s in enumerate(ns):
        kv[b, s:] = float("nan")
    dev = kv.cuda()
    if stacked:
        k, v = dev[:, :, 0], dev[:, :, 1]
    else:  # head by head
        k, v = (dev[:, :, i].transpose(1, 2).contiguous().transpose(1, 2) for i in range(2))
    place = lambda x, pad, gap: torch.cat([x.flatten(1), torch.full((rows, gap), 5.0, dtype=qt)], 1).flatten()  # noqa: E731
    view = lambda x, pad, gap: x[pad:].view(rows, -1)[:, : hq * d].unflatten(1, (hq, d))  # noqa: E731
    out = torch.full((rows, hq, d), 3.0, dtype=qt, device="cuda")
    qdev = q.cuda()
    if pads:
        qdev, out = (view(torch.nn.functional.pad(place(x.cpu(), *p), (p[0], 0)).cuda(), *p) for x, p in zip((q, out), pads))
    offsets = None if equal else torch.tensor(np.r_[0, np.cumsum(nq)], dtype=torch.int32, device="cuda")
    lens = None if equal and len(set(ns)) == 1 else torch.tensor(ns, dtype=torch.int32, device="cuda")
    qvx.attn_cross_t(qdev, qvx.KvStates.of(k, v), lens=lens, offsets=offsets, out=out, scale=scale)
    torch.cuda.synchronize()
    got = out.cpu().double().numpy()
    qn, kvn = q.double().numpy(), kv.double().numpy()
    g, at, scale = hq // hk, 0, d ** -0.5 if scale is None else scale
    half = {qvx.F32: 0.0, qvx.F16: 2.0 ** -11, qvx.BF16: 2.0 ** -8}[q_type]
    for b in range(n):
        mine = got[at:at + nq[b]]
        if ns[b] == 0:
            assert (mine == 0).all()
        for h in range(hq if ns[b] and nq[b] else 0):
            k1, v1 = kvn[b, :ns[b], 0, h // g], kvn[b, :ns[b], 1, h // g]
            want, s = _attend(qn[at:at + nq[b], h], k1, v1, scale)
            tol = 2 * U * ((d + 3) * s + ns[b] + 8) * np.abs(v1).max() + half * (np.abs(want) + np.abs(v1).max())
            assert (np.abs(mine[:, h] - want) <= tol).all(), (b, h, np.abs(mine[:, h] - want).max())
        at += nq[b]
    assert (got[at:] == 3.0).all()  # rows behind the last sequence


TYPES16 = ((qvx.F16, qvx.F16), (qvx.BF16, qvx.BF16))
MIXED = ((qvx.F32, qvx.F16), (qvx.F32, qvx.BF16), (qvx.F32, qvx.F32), (qvx.F16, qvx.F32), (qvx.BF16, qvx.F16))


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED)
@pytest.mark.parametrize("nq,ns", [((1,), (1,)), ((1, 1, 1), (1500, 77, 0)), ((5, 0, 33), (40, 9, 129)),
                                   ((70, 129), (300, 64))])
def test_cross_lengths(cuda, q_type, kv_type, nq, ns):
    _check_cross(cuda, q_type, kv_type, nq, ns, 4, 4, 64, seed=sum(ns))


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 80, 96, 128, 160, 200, 256])
def test_cross_head_sizes(cuda, q_type, kv_type, d):
    _check_cross(cuda, q_type, kv_type, (150, 20), (77, 200), 2, 2, d, seed=d)


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 2), (12, 12), (20, 1)])
def test_cross_head_layouts(cuda, q_type, kv_type, hq, hk):
    _check_cross(cuda, q_type, kv_type, (260, 3), (150, 90), hq, hk, 64, seed=hq, stacked=False)


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
def test_cross_equal_parts(cuda, q_type, kv_type):
    _check_cross(cuda, q_type, kv_type, (300, 300), (77, 77), 4, 4, 40, seed=1, equal=True)
    _check_cross(cuda, q_type, kv_type, (1,) * 5, (1500,) * 5, 4, 4, 64, seed=2, equal=True)
    _check_cross(cuda, q_type, kv_type, (64, 64, 64), (130, 0, 64), 2, 2, 64, seed=3, equal=True)


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
def test_cross_many_sequences(cuda, q_type, kv_type):
    r = np.random.default_rng(3)
    nq, ns = [int(x) for x in r.integers(0, 40, 90)], [int(x) for x in r.integers(0, 60, 90)]
    _check_cross(cuda, q_type, kv_type, nq, ns, 2, 2, 64, seed=5)


# ---- cross attention on the 16-bit matrix cores: its split, its fallbacks and its callers ------------------

@pytest.mark.parametrize("q_type,kv_type", TYPES16)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("nq,ns", [((40,), (1500,)), ((129, 33, 0, 32), (700, 255, 90, 0)), ((64, 200), (257, 4100))])
def test_cross_few_rows_on_many_states(cuda, q_type, kv_type, d, nq, ns):
    """Too few row tiles for the card: their states are split over workgroups."""
    _check_cross(cuda, q_type, kv_type, nq, ns, 2, 1, d, seed=d + len(nq))


@pytest.mark.parametrize("q_type,kv_type", TYPES16)
def test_cross_split_of_many_sequences(cuda, q_type, kv_type):
    """More sequences than a wave has lanes, some long enough for a split."""
    r = np.random.default_rng(18)
    nq = [int(x) for x in r.integers(20, 60, 70)]
    ns = [int(x) for x in r.integers(0, 40, 70)]
    ns[3], ns[68] = 1300, 900
    _check_cross(cuda, q_type, kv_type, nq, ns, 1, 1, 40, seed=6)


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
@pytest.mark.parametrize("scale", [0.0, 1e-38, 2e-30, -0.2, 1.0])
def test_cross_scales(cuda, q_type, kv_type, scale):
    """Odd states in the last tile: masked ones stay masked at every scale."""
    _check_cross(cuda, q_type, kv_type, (50, 33), (45, 70), 2, 2, 64, seed=7, scale=scale)
    _check_cross(cuda, q_type, kv_type, (40,), (800,), 1, 1, 64, seed=8, scale=scale)


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED)
@pytest.mark.parametrize("pads", [((8, 8), (4, 4)), ((1, 0), (0, 3)), ((0, 5), (1, 8)), ((3, 7), (2, 2))])
def test_cross_alignment(cuda, q_type, kv_type, pads):
    """Rows of q and out on any element."""
    _check_cross(cuda, q_type, kv_type, (50, 33), (45, 70), 2, 2, 40, seed=9, pads=pads)


@pytest.mark.parametrize("q_type,kv_type", TYPES16)
def test_cross_wide_pitch(cuda, q_type, kv_type):
    """States 20 MiB apart: a tile of 64 would pass 32-bit offsets."""
    torch = cuda
    pitch, d = 10 << 20, 64
    kt = _torch_type(torch, kv_type)
    held = torch.zeros(3 * pitch, dtype=kt, device="cuda")
    k, v = (held[i * 64:].as_strided((1, 3, 1, d), (0, pitch, 0, 1)) for i in (0, 1))
    k.copy_(torch.randn((1, 3, 1, d), device="cuda"))
    v.copy_(torch.randn((1, 3, 1, d), device="cuda"))
    q = torch.randn((40, 1, d), device="cuda").to(kt)
    got = qvx.attn_cross_t(q, qvx.KvStates.of(k, v))
    packed = qvx.attn_cross_t(q.float(), qvx.KvStates.of(k.contiguous(), v.contiguous()))
    half = 2.0 ** -11 if kv_type == qvx.F16 else 2.0 ** -8
    s = float((q.float()[:, 0].abs() @ k.float()[0, :, 0].abs().T).max()) / 8
    tol = 2 * 2 * U * ((d + 3) * s + 11) * float(v.abs().max()) + half * packed.abs()
    assert bool(((got.float() - packed).abs() <= tol).all())


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
def test_cross_in_place_and_repeatable(cuda, q_type, kv_type):
    torch = cuda
    q = torch.randn((60, 2, 64), device="cuda").to(_torch_type(torch, q_type))
    k, v = (torch.randn((2, 1100, 2, 64), device="cuda").to(_torch_type(torch, kv_type)) for _ in range(2))
    offsets = torch.tensor([0, 50, 58], dtype=torch.int32, device="cuda")
    st = qvx.KvStates.of(k, v)
    first = qvx.attn_cross_t(q, st, offsets=offsets)
    assert torch.equal(first[:58], qvx.attn_cross_t(q, st, offsets=offsets)[:58])
    behind = q[58:].clone()
    qvx.attn_cross_t(q, st, offsets=offsets, out=q)
    assert torch.equal(first[:58], q[:58]) and torch.equal(behind, q[58:])


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
def test_cross_captured_replays_follow_the_lengths(cuda, q_type, kv_type):
    """Lengths and offsets change between replays, in two graphs with workspaces of their own."""
    torch = cuda
    kt = _torch_type(torch, kv_type)
    k, v = (torch.randn((3, 1500, 2, 64), device="cuda").to(kt) for _ in range(2))
    st = qvx.KvStates.of(k, v)
    qs = [torch.randn((120, 2, 64), device="cuda").to(_torch_type(torch, q_type)) for _ in range(2)]
    lens = torch.tensor([1500, 3, 700], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 40, 41, 120], dtype=torch.int32, device="cuda")
    qvx.attn_cross_t(qs[0], st, lens=lens, offsets=offsets)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        out = torch.empty_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qvx.attn_cross_t(q, st, lens=lens, offsets=offsets, out=out)
        graphs.append(g)
        outs.append(out)
    for n, o in (([1500, 3, 700], [0, 40, 41, 120]), ([0, 1500, 1], [0, 1, 119, 120]), ([17, 16, 15], [0, 0, 0, 120]),
                 ([1500, 1500, 1500], [0, 100, 110, 120])):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        offsets.copy_(torch.tensor(o, dtype=torch.int32))
        for g in graphs:
            g.replay()
        for q, out in zip(qs, outs):
            assert torch.equal(out, qvx.attn_cross_t(q, st, lens=lens, offsets=offsets))
        torch.cuda.synchronize()


@pytest.mark.parametrize("q_type,kv_type", TYPES16)
def test_cross_many_small_weights(cuda, q_type, kv_type):
    """One heavy state and thousands whose weights lie among fp16's subnormal numbers, which together weigh as much."""
    torch = cuda
    n, d = 4096, 64
    kt = _torch_type(torch, kv_type)
    k = torch.zeros((1, n, 1, d), device="cuda")
    k[0, 5, 0, 0] = 8.0  # logit 64 / 8 = 8: the others weigh e^-8 of it, and 4095 e^-8 = 1.37 of it in all
    v = torch.ones((1, n, 1, d), device="cuda")
    v[0, 5] = 0.0
    q = torch.zeros((64, 1, d), device="cuda")
    q[:, 0, 0] = 8.0
    got = qvx.attn_cross_t(q.to(kt), qvx.KvStates.of(k.to(kt), v.to(kt)), scale=0.125).float()
    rest = (n - 1) * np.exp(-8.0)
    want = rest / (1 + rest)
    # Two roundings to 16 bits (the weights', the output's) of half a step each; the power of two and the sums as ever.
    half = 2.0 ** -11 if kv_type == qvx.F16 else 2.0 ** -8
    assert float((got - want).abs().max()) <= (2 * half + 2 * U * (67 * 8 + n + 8)) * 1.0


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
def test_cross_without_queries_or_states(cuda, q_type, kv_type):
    torch = cuda
    qt, kt = _torch_type(torch, q_type), _torch_type(torch, kv_type)
    k = torch.randn((2, 9, 2, 64), device="cuda").to(kt)
    none = qvx.attn_cross_t(torch.empty((0, 2, 64), dtype=qt, device="cuda"), qvx.KvStates.of(k, k))
    assert none.shape == (0, 2, 64)
    empty = torch.empty((2, 0, 2, 64), dtype=kt, device="cuda")
    for rows in (2, 80):
        out = qvx.attn_cross_t(torch.randn((rows, 2, 64), device="cuda").to(qt), qvx.KvStates.of(empty, empty))
        assert bool((out == 0).all())


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + MIXED[:1])
def test_cross_offsets_that_are_no_running_sums(cuda, q_type, kv_type):
    """Decreasing and far offsets: nothing outside the rows is written, whatever the workspace holds, and the next call
    with good ones is right."""
    torch = cuda
    qt, kt = _torch_type(torch, q_type), _torch_type(torch, kv_type)
    k, v = (torch.randn((6, 1400, 2, 64), device="cuda").to(kt) for _ in range(2))
    st = qvx.KvStates.of(k, v)
    q = torch.randn((40, 2, 64), device="cuda").to(qt)
    whole = torch.full((60, 2, 64), 5.0, dtype=qt, device="cuda")
    good = torch.tensor([0, 3, 3, 10, 20, 38, 40], dtype=torch.int32, device="cuda")
    ws = torch.full((qvx.attn_cross_ws(st, q.dtype, 2, 40, 6),), 255, dtype=torch.uint8, device="cuda")
    want = qvx.attn_cross_t(q, st, offsets=good)
    for bad in ([40, 0, 40, 0, 40, 0, 40], [0, 40, 0, 40, 0, 40, 0], [-7, 1 << 30, -(1 << 31), 5, 2000000000, 1, 40]):
        qvx.attn_cross_t(q, st, offsets=torch.tensor(bad, dtype=torch.int32, device="cuda"), out=whole[10:50], ws=ws)
        torch.cuda.synchronize()
        assert bool((whole[:10] == 5.0).all()) and bool((whole[50:] == 5.0).all())
        assert torch.equal(qvx.attn_cross_t(q, st, offsets=good, ws=ws), want)


@pytest.mark.parametrize("t", (qvx.BF16, qvx.Q8_0))
def test_pages_past_four_gib(cuda, t):
    """Append and attention on pages whose byte offsets pass 32 bits, beside one at the start."""
    torch = cuda
    page, hk, d, n = 128, 8, 128, 1000
    size = qvx.kv_page_bytes(t, hk, page, d)
    n_pages = (5 << 30) // size
    k, v = (torch.empty((n_pages, size), dtype=torch.uint8, device="cuda") for _ in range(2))
    far = qvx.KvCache.of(k, v, t, page, hk, d)
    near_k, near_v = (torch.empty((9, size), dtype=torch.uint8, device="cuda") for _ in range(2))
    near = qvx.KvCache.of(near_k, near_v, t, page, hk, d)
    ids = torch.tensor([0, n_pages - 1, n_pages - 5, 3, n_pages - 9, n_pages // 2, n_pages - 2, n_pages - 3], dtype=torch.int32,
                       device="cuda")
    here = torch.tensor([8, 1, 2, 3, 4, 5, 6, 7], dtype=torch.int32, device="cuda")
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    q, kk, vv = (torch.randn((n, h, d), device="cuda") for h in (16, hk, hk))
    rope = qvx.Rope.of(10000.0 ** -(torch.arange(64, dtype=torch.float64, device="cuda") / 64))
    outs = []
    for c, p in ((far, ids), (near, here)):
        turned = qvx.rope_kv_t(q, kk, vv, at, rope, cache=c, slots=p[(at // page).long()] * page + at % page)
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        outs.append((turned, qvx.attn_paged_t(turned[-1:], c, p[None], lens)))
    assert torch.equal(k[ids.long()][:, :64], near_k[here.long()][:, :64])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
