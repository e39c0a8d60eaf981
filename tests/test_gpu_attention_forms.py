"""Every form of the attention kernels (types, padded head sizes, row tiles, whole and split sequences, few and many of
them) on inputs that show each key.

Queries.  A row is zero or has one value, so its logits are zeros or single products: the error of a logit S is at most
8 u S (the query times the scale, its 16-bit parts 2 u, their sum, a block's scale, the exponent's fma).  A row of
zeros weighs all keys alike and exactly, so its output is their mean value, and a key that is lost or counted twice
moves it by what it is: each check also leaves one tile of 16 keys out of the reference and asks that the bar sees it.

Bars.  u = 2^-24.  Weights: 8 u S (above, and the exponent's own rounding: at most S log2(e) from the reference on
either side), nothing where S = 0; the hardware's power of two and the factors of the joins 8 u in all.  Sums: `depth`
additions on any path, at most 16 a tile for the tiles of a chunk that a wave takes (every fourth), four waves and the chunks of the sequence; so
|error| <= 2 u (8 S + depth + 8) max |v|, numerator and denominator both.  On the 16-bit matrix cores the
weights are powers of two from 1 to 2^-7 of the largest, so rounding them changes nothing and only the output is rounded: half
a step more."""
from __future__ import annotations

import math

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import CACHE_TYPES, TYPES16, U, Cache, _check_cross, _check_paged, _torch_type

pytestmark = pytest.mark.gpu


def _ceil(a, b):
    return -(-a // b)


def _chunk_tiles(tiles, rows, heads, least, wgs):
    """Tiles of a chunk of a split call: `tiles` and `rows` row tiles of each sequence, `least` of a chunk, `wgs` aimed at."""
    total = sum(t * r for t, r in zip(tiles, rows))
    return max(least, _ceil(_ceil(total, max(1, wgs // heads)), 4) * 4)


def _paged_chunks(c, hq):
    """(tiles of each sequence, tiles of a chunk) of a paged call."""
    group = hq // c.hk
    r = 4 if group <= 4 else 8 if group <= 8 else 16
    page_tiles = _ceil(c.page, 16)
    tiles = [n // c.page * page_tiles + _ceil(n % c.page, 16) for n in c.lens]
    split = qvx.attn_paged_ws(c.desc, hq, len(c.lens), c.width) > 0
    return tiles, _chunk_tiles(tiles, [_ceil(group, r)] * len(tiles), c.hk, 8, 512) if split else max(tiles + [1])


def _mean(q, k, v, scale):
    """softmax(scale q k^T) v and the largest |logit| of each row, in 64 bits."""
    s = (q @ k.T) * scale
    w = np.exp(s - s.max(-1, keepdims=True))
    return (w @ v) / w.sum(-1, keepdims=True), np.abs(s).max(-1)


def _bar(s, depth, top):
    return 2 * U * (8 * s + depth + 8) * top


def _sharp_queries(n, heads, d, value, seed):
    """Rows with one value, every third of zeros."""
    r = np.random.default_rng(seed)
    q = np.zeros((n, heads, d), np.float32)
    for b in range(n):
        for h in range(heads):
            if (b + h) % 3:
                q[b, h, r.integers(0, d)] = value * r.choice([-1, 1])
    return q


def _sharp_paged(torch, c, hq, seed=0):
    tiles, chunk = _paged_chunks(c, hq)
    q = _sharp_queries(len(c.lens), hq, c.d, 2.0, seed)
    out = qvx.attn_paged_t(torch.from_numpy(q).cuda(), c.desc, c.dev_table, c.dev_lens, scale=1.0)
    torch.cuda.synchronize()
    got, group = out.cpu().double().numpy(), hq // c.hk
    for b, n in enumerate(c.lens):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        depth = 4 * min(chunk, tiles[b]) + _ceil(tiles[b], chunk) + 8
        k, v = c.rows(b, 0), c.rows(b, 1)
        seen = n < 48
        for h in range(c.hk):
            rows = slice(h * group, (h + 1) * group)
            x = q[b, rows].astype(np.float64)
            want, s = _mean(x, k[h], v[h], 1.0)
            bar = _bar(s, depth, np.abs(v[h]).max())[:, None]
            assert (np.abs(got[b, rows] - want) <= bar).all(), (b, h, n, np.abs(got[b, rows] - want).max(), bar.max())
            if n >= 48 and not seen:  # the bar sees a tile that is left out
                at = 16 * (n // 32)
                less, _ = _mean(x, np.delete(k[h], np.s_[at:at + 16], 0), np.delete(v[h], np.s_[at:at + 16], 0), 1.0)
                seen = seen or bool((np.abs(less - want) > 2 * bar).any())
        assert seen, (b, n)


# ---- paged: every instance ----------------------------------------------------------------------------------

@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("group", [1, 4, 5, 7, 8, 9, 16, 24])
def test_paged_forms_split(cuda, t, d, group):
    """One sequence of several chunks beside short, empty and middling ones, for every row tile."""
    c = Cache(cuda, t, (9, 2500, 0, 333, 16), 16, 1, d, seed=d + group, spare=2)
    assert qvx.attn_paged_ws(c.desc, group, 5, c.width) > 0
    _sharp_paged(cuda, c, group)
    _check_paged(cuda, c, group)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 160, 256])
@pytest.mark.parametrize("group", [1, 4, 6, 8, 16])
def test_paged_forms_whole(cuda, t, d, group):
    """As many keys as one workgroup takes: several tiles a wave, the last of them ragged, on pages of every size."""
    page, key_bytes = 40, {qvx.F32: 4 * d, qvx.Q8_0: d + d // 16}.get(t, 2 * d)  # a page holds three tiles
    most = ((320 << 10) // (2 * 16 * key_bytes) // 3 - 1) * page
    c = Cache(cuda, t, (most - 5, 70, 1, most // 2), page, 2, d, seed=d + group)
    assert qvx.attn_paged_ws(c.desc, 2 * group, 4, c.width) == 0
    _sharp_paged(cuda, c, 2 * group)
    _check_paged(cuda, c, 2 * group)


@pytest.mark.parametrize("d", [40, 80, 136, 248])
@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16, qvx.F32))
@pytest.mark.parametrize("group", [6, 16])
def test_paged_forms_odd_head_sizes(cuda, t, d, group):
    c = Cache(cuda, t, (2600, 31), 40, 1, d, seed=d)
    assert qvx.attn_paged_ws(c.desc, group, 2, c.width) > 0 or d == 40
    _sharp_paged(cuda, c, group)


@pytest.mark.parametrize("t", CACHE_TYPES)
@pytest.mark.parametrize("n,longest,group", [(64, 2600, 2), (65, 2600, 2), (150, 2400, 8), (150, 2400, 16)])
def test_paged_split_of_many_sequences(cuda, t, n, longest, group):
    """Up to 64 sequences (a wave's scan) and more (through LDS), of all lengths in no order, empty ones among them: more
    items than the card has places, so the rests come from long to short."""
    r = np.random.default_rng(n)
    longest += 900 if t == qvx.Q8_0 else 0  # half the bytes a key: longer before it is split
    lens = [int(x) for x in np.exp(r.uniform(0, np.log(longest), n))]
    lens[n // 2], lens[n // 3], lens[7] = longest, 0, longest // 2 + 1
    c = Cache(cuda, t, lens, 16, 8, 64 if t == qvx.F32 else 96, seed=n)
    assert qvx.attn_paged_ws(c.desc, 8 * group, n, c.width) > 0
    tiles, chunk = _paged_chunks(c, 8 * group)
    kinds = [4 - min(3, 4 * (x % chunk) // chunk) for x in tiles if x % chunk]
    assert sum(x > chunk for x in tiles) >= 3 and set(kinds) >= {1, 2, 3, 4}
    _sharp_paged(cuda, c, 8 * group)


@pytest.mark.parametrize("t,lens,hk,d,group", [(qvx.BF16, (40007, 39999), 2, 64, 2), (qvx.BF16, (40007, 39999), 2, 64, 6),
                                               (qvx.F16, (40007, 39999), 2, 64, 16), (qvx.F16, (20011,), 1, 64, 1),
                                               (qvx.Q8_0, (30001,), 1, 64, 8), (qvx.F32, (20011, 5), 1, 64, 16),
                                               (qvx.F16, (20011,), 1, 256, 4), (qvx.BF16, (9001, 17000), 1, 256, 7)])
def test_paged_long_sequences_key_by_key(cuda, t, lens, hk, d, group):
    """Hundreds of chunks a sequence: both of the join's ways to take rows, and more than one round of its loads."""
    c = Cache(cuda, t, lens, 64, hk, d, seed=4)
    tiles, chunk = _paged_chunks(c, hk * group)
    assert max(_ceil(x, chunk) for x in tiles) > 64
    _sharp_paged(cuda, c, hk * group)


def test_paged_graphs_with_workspaces_of_their_own(cuda):
    """Two captured calls whose sequences are split, replayed on two streams at once while the lengths move, against eager
    calls."""
    torch = cuda
    c = Cache(torch, qvx.F16, (4000, 3000, 2000), 16, 2, 128, seed=13)
    need = qvx.attn_paged_ws(c.desc, 8, 3, c.width)
    assert need > 0
    qs = [torch.randn((3, 8, 128), device="cuda") for _ in range(2)]
    lens = torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    ws = [torch.full((need,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    qvx.attn_paged_t(qs[0], c.desc, c.dev_table, lens, ws=ws[0])
    torch.cuda.synchronize()
    graphs, outs = [], [torch.empty_like(q) for q in qs]
    for q, out, w in zip(qs, outs, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qvx.attn_paged_t(q, c.desc, c.dev_table, lens, out=out, ws=w)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for now in ((4000, 3000, 2000), (1, 0, 1999), (4000, 16, 17), (129, 3000, 1), (4000, 3000, 2000)):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        want = [qvx.attn_paged_t(q, c.desc, c.dev_table, lens) for q in qs]
        torch.cuda.synchronize()
        for _ in range(3):
            for out in outs:
                out.fill_(9.0)
            torch.cuda.synchronize()
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- cross attention ------------------------------------------------------------------------------------------

def _sharp_cross(torch, q_type, kv_type, nq, ns, hq, hk, d, seed=0):
    """Ragged queries and states; weights are powers of two (scale ln 2, keys of 0 to -7)."""
    r = np.random.default_rng(seed)
    n, most, rows, group = len(nq), max(ns), sum(nq), hq // hk
    q = _sharp_queries(rows, hq, d, 1.0, seed)
    q = np.abs(q)
    k = -r.integers(0, 8, (n, most, hk, d)).astype(np.float32)
    v = torch.from_numpy(r.standard_normal((n, most, hk, d)).astype(np.float32)).to(_torch_type(torch, kv_type))
    for b, s in enumerate(ns):
        k[b, s:], v[b, s:] = np.nan, float("nan")
    states = qvx.KvStates.of(torch.from_numpy(k).to(_torch_type(torch, kv_type)).cuda(), v.cuda())
    offsets = torch.tensor(np.r_[0, np.cumsum(nq)], dtype=torch.int32, device="cuda")
    lens = torch.tensor(ns, dtype=torch.int32, device="cuda")
    got = qvx.attn_cross_t(torch.from_numpy(q).to(_torch_type(torch, q_type)).cuda(), states, lens=lens, offsets=offsets,
                           scale=math.log(2.0))
    torch.cuda.synchronize()
    got, v = got.cpu().double().numpy(), v.double().numpy()
    half = {qvx.F32: 0.0, qvx.F16: 2.0 ** -11, qvx.BF16: 2.0 ** -8}[q_type]
    at = 0
    for b, s in enumerate(ns):
        mine = slice(at, at + nq[b])
        at += nq[b]
        if not nq[b]:
            continue
        if s == 0:
            assert (got[mine] == 0).all()
            continue
        seen = s < 48
        for h in range(hq):
            kk, vv, x = k[b, :s, h // group].astype(np.float64), v[b, :s, h // group], q[mine, h].astype(np.float64)
            want, size = _mean(x, kk, vv, math.log(2.0))
            # at most 1024 keys on a path, or a chunk, and the chunks' join
            bar = _bar(size, min(s, 1024) / 2 + s / 128 + 8, np.abs(vv).max())[:, None] + half * np.abs(want)
            assert (np.abs(got[mine, h] - want) <= bar).all(), (b, h, s, np.abs(got[mine, h] - want).max())
            if s >= 48 and not seen:
                cut = 16 * (s // 32)
                less, _ = _mean(x, np.delete(kk, np.s_[cut:cut + 16], 0), np.delete(vv, np.s_[cut:cut + 16], 0), math.log(2.0))
                seen = seen or bool((np.abs(less - want) > 2 * bar).any())
        assert seen, (b, s)


def _ws(torch, q_type, kv_type, nq, ns, hq, hk, d):
    st = qvx.KvStates(0x10000, 0x10000, max(ns) * hk * d, hk * d, d, kv_type, max(ns), hk, d)
    return qvx.attn_cross_ws(st, q_type, hq, sum(nq), len(nq))


@pytest.mark.parametrize("q_type,kv_type", TYPES16 + ((qvx.F32, qvx.F16), (qvx.F32, qvx.BF16)))
@pytest.mark.parametrize("d", [40, 128])
def test_cross_split_of_many_long_sequences(cuda, q_type, kv_type, d):
    """More sequences than a wave has lanes, two of them of many chunks: 128-row and 16-row tiles."""
    r = np.random.default_rng(18)
    nq = [int(x) for x in r.integers(20, 60, 70)]
    ns = [int(x) for x in r.integers(0, 40, 70)]
    ns[3], ns[68] = 5000, 2900
    assert 16 * sum(nq) > 16 * 16 * 70 and _ceil(5000, 16) > 40 + (sum(nq) // 128 + 70) / 2  # wide, and split there
    assert _ws(cuda, q_type, kv_type, nq, ns, 1, 1, d) > 0
    _sharp_cross(cuda, q_type, kv_type, nq, ns, 1, 1, d, seed=6)


@pytest.mark.parametrize("q_type,kv_type", TYPES16)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("nq,ns", [((40,), (1500,)), ((129, 33, 0, 32), (700, 255, 90, 0)), ((64, 200), (257, 4100)),
                                   ((300, 260, 500), (90, 65, 64))])
def test_cross_16_bit_state_by_state(cuda, q_type, kv_type, d, nq, ns):
    _sharp_cross(cuda, q_type, kv_type, nq, ns, 2, 1, d, seed=d)


@pytest.mark.parametrize("q_type,kv_type", [(qvx.F32, qvx.F16), (qvx.F32, qvx.BF16), (qvx.F32, qvx.F32), (qvx.F16, qvx.F32),
                                            (qvx.BF16, qvx.F16)])
@pytest.mark.parametrize("d", [96, 128, 200, 256])
@pytest.mark.parametrize("nq", [(5, 8, 7), (3, 0, 4), (16, 15, 20)])
def test_cross_few_rows_at_every_head_size(cuda, q_type, kv_type, d, nq):
    """Five to eight rows a sequence, up to four, and more, at head sizes above 64, whole and split."""
    _sharp_cross(cuda, q_type, kv_type, nq, (300, 41, 77), 2, 2, d, seed=d)
    _sharp_cross(cuda, q_type, kv_type, nq, (300, 3000, 1), 1, 1, d, seed=d)
    _check_cross(cuda, q_type, kv_type, nq, (300, 0, 77), 2, 2, d, seed=d)


# ---- counts at the ends of what the calls take --------------------------------------------------------------------

def test_paged_thousands_of_sequences(cuda):
    """Threads that each look through many sequences, one of them split."""
    r = np.random.default_rng(2)
    lens = [int(x) for x in r.integers(0, 4, 9000)]
    lens[8191], lens[4000] = 4200, 33
    c = Cache(cuda, qvx.F16, lens, 16, 1, 64, seed=2)
    assert qvx.attn_paged_ws(c.desc, 2, len(lens), c.width) > 0
    _sharp_paged(cuda, c, 2)


def test_paged_as_many_sequences_as_a_call_takes(cuda):
    """65536 sequences of no key or one: the key's value, or zeros."""
    torch = cuda
    n, d = 65536, 32
    size = qvx.kv_page_bytes(qvx.F32, 1, 1, d)
    k, v = (torch.randn((n, size // 4), device="cuda") for _ in range(2))
    cache = qvx.KvCache.of(k, v, qvx.F32, 1, 1, d)
    table = torch.randperm(n, device="cuda").to(torch.int32).view(n, 1)
    lens = (torch.arange(n, device="cuda") % 3 != 1).to(torch.int32)
    out = qvx.attn_paged_t(torch.randn((n, 1, d), device="cuda"), cache, table, lens)
    want = v[table[:, 0].long()] * lens[:, None]
    assert bool(((out[:, 0] - want).abs() <= 4 * U * want.abs()).all())
