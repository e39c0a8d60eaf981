"""CPU tests of the argument checks of the page calls and of the norms with rotation: every call here is refused, or has
nothing to do, before any device work."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx

K = 1 << 20
A = [0x1000000 + i * K for i in range(16)]  # addresses apart from each other that nothing reads


def fork(frm=A[0], to=A[1], n=4, table=A[2], rows=8, width=10, page=16, lens=A[3], extra=A[4], pages=50, free=A[5], n_free=50,
         taken=A[6], out=A[7], pairs=A[8], n_pairs=A[9]):
    return qvx.kv_fork(frm, to, n, table, rows, width, page, lens, extra, pages, free, n_free, taken, out, pairs, n_pairs)


def test_fork_refusals():
    assert fork(n=0) == qvx.E_NVEC and fork(n=-1) == qvx.E_NVEC
    for kw in (dict(rows=0), dict(width=0), dict(page=0), dict(pages=0), dict(n_free=-1)):
        assert fork(**kw) == qvx.E_SHAPE
    for kw in (dict(n=16385), dict(width=(1 << 24) + 1), dict(pages=1 << 27, page=16), dict(table=A[0]), dict(pairs=A[8], n_pairs=A[8]),
               dict(taken=A[6], out=A[6] + 4), dict(lens=A[2] + 4 * 79), dict(extra=A[3]), dict(pairs=A[5] + 4), dict(out=A[3]),
               dict(to=A[9], n_pairs=A[9])):
        assert fork(**kw) == qvx.E_RANGE, kw
    for k in ("frm", "to", "table", "lens", "extra", "free", "taken", "out", "pairs", "n_pairs"):
        assert fork(**{k: 0}) == qvx.E_NULL


def free(rows=A[0], begin=0, end=0, n=3, table=A[1], n_rows=8, width=10, lens=A[2], extra=A[3], pages=50, lst=A[4], n_free=50,
         taken=A[5], out=A[6], ws=0, ws_bytes=0):
    return qvx.kv_free(rows, begin, end, n, table, n_rows, width, lens, extra, pages, lst, n_free, taken, out, ws, ws_bytes)


def test_free_refusals():
    assert qvx.kv_free_ws(16384) == 0 and qvx.kv_free_ws(16385) == 16 and qvx.kv_free_ws(0) == 0 and qvx.kv_free_ws(-5) == 0
    assert free(n=0) == qvx.E_NVEC
    for kw in (dict(n_rows=0), dict(width=-1), dict(pages=0), dict(n_free=-1)):
        assert free(**kw) == qvx.E_SHAPE
    for k in ("rows", "table", "lens", "extra", "lst", "taken", "out"):
        assert free(**{k: 0}) == qvx.E_NULL
    assert free(begin=A[7]) == qvx.E_NULL and free(end=A[7]) == qvx.E_NULL  # one without the other
    assert free(pages=20000, ws=0, ws_bytes=64) == qvx.E_NULL
    assert free(pages=20000, ws=A[8], ws_bytes=15) == qvx.E_RANGE and free(pages=20000, ws=A[8] + 2, ws_bytes=64) == qvx.E_RANGE
    for kw in (dict(n=16385), dict(taken=A[5], out=A[5] + 4), dict(lens=A[1] + 316), dict(lst=A[3]), dict(rows=A[4] + 196),
               dict(out=A[0]), dict(begin=A[7], end=A[1]), dict(pages=20000, ws=A[2], ws_bytes=64), dict(width=(1 << 24) + 1)):
        assert free(**kw) == qvx.E_RANGE, kw


def compact(table=A[0], t_out=A[1], rows=8, width=10, extra=A[2], e_out=A[3], pages=50, lst=A[4], l_out=A[5], n_free=50,
            taken=A[6], pairs=A[7], moved=A[8]):
    return qvx.kv_compact(table, t_out, rows, width, extra, e_out, pages, lst, l_out, n_free, taken, pairs, moved)


def test_compact_refusals():
    for kw in (dict(rows=0), dict(width=0), dict(pages=0), dict(n_free=-1)):
        assert compact(**kw) == qvx.E_SHAPE
    for k in ("table", "t_out", "extra", "e_out", "lst", "l_out", "taken", "pairs", "moved"):
        assert compact(**{k: 0}) == qvx.E_NULL
    for kw in (dict(pages=(1 << 20) + 1), dict(t_out=A[0] + 4), dict(e_out=A[0]), dict(l_out=A[4] + 4), dict(pairs=A[2]),
               dict(moved=A[7]), dict(moved=A[6]), dict(t_out=A[1], e_out=A[1] + 316), dict(pairs=A[4])):
        assert compact(**kw) == qvx.E_RANGE, kw


def cache(**kw):
    a = dict(d_k=A[0], d_v=A[1], page_stride=0, type=qvx.F16, n_pages=10, page_size=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return qvx.KvCache(**a)


def test_copy_refusals():
    two = qvx.kv_caches([cache(), cache()])
    assert qvx.kv_copy(qvx.kv_caches([]), A[2], 0, 3) == qvx.E_NVEC
    assert qvx.lib().qvx_kv_copy(two, 0, A[2], None, 3, None) == qvx.E_NVEC
    assert qvx.lib().qvx_kv_copy(None, 2, A[2], None, 3, None) == qvx.E_NULL
    assert qvx.kv_copy(two, A[2], 0, -1) == qvx.E_NVEC
    assert qvx.kv_copy(two, 0, 0, 3) == qvx.E_NULL
    assert qvx.kv_copy(two, A[2], A[3], 0) == qvx.OK  # nothing to copy
    for kw in (dict(type=qvx.BF16), dict(n_pages=11), dict(page_size=8), dict(kv_heads=1), dict(head_dim=128)):
        assert qvx.kv_copy(qvx.kv_caches([cache(), cache(**kw)]), A[2], 0, 3) == qvx.E_SHAPE
    assert qvx.kv_copy(qvx.kv_caches([cache(), cache(d_v=0)]), A[2], 0, 3) == qvx.E_NULL
    assert qvx.kv_copy(qvx.kv_caches([cache(kv_heads=1 << 20, page_size=1 << 10, head_dim=256, n_pages=1)]), A[2], 0, 3) == qvx.E_RANGE


def turn(norm=True, q_out=A[0], q_out_stride=256, q_type=qvx.F32, q=A[1], q_stride=256, heads=4, k=A[2], ks=128, v=A[3], vs=128,
         n=5, d=64, pos=A[4], ps=5, c=True, slots=A[5], eps=1e-6, w_stride=0, **kw):
    a = dict(d_inv_freq=A[6], d_axis=None, rot_dim=64, n_axes=1, pairing=qvx.ROPE_HALVES, scale=1.0)
    a.update(kw)
    w = qvx.QkNorm(A[7], A[8], w_stride, eps)
    return qvx.norm_rope_kv(q_out, q_out_stride, q_type, q, q_stride, heads, k, ks, v, vs, n, d, w, qvx.Rope(**a), pos, ps,
                            cache() if c is True else c, slots)


@pytest.mark.parametrize("kw,rc", [
    (dict(n=0), qvx.E_NVEC), (dict(q_type=qvx.Q8_0), qvx.E_TYPE), (dict(q_type=99), qvx.E_TYPE), (dict(w_stride=63), qvx.E_SHAPE),
    (dict(w_stride=-64), qvx.E_SHAPE), (dict(eps=-1e-9), qvx.E_RANGE), (dict(eps=float("nan")), qvx.E_RANGE),
    (dict(pairing=2), qvx.E_VARIANT), (dict(rot_dim=72), qvx.E_SHAPE), (dict(rot_dim=12), qvx.E_SHAPE), (dict(d=128), qvx.E_SHAPE),
    (dict(n_axes=5), qvx.E_SHAPE), (dict(n_axes=2, ps=4), qvx.E_SHAPE), (dict(q_out_stride=255), qvx.E_SHAPE),
    (dict(q=0), qvx.E_NULL), (dict(k=0), qvx.E_NULL), (dict(v=0), qvx.E_NULL), (dict(slots=0), qvx.E_NULL), (dict(pos=0), qvx.E_NULL),
    (dict(d_inv_freq=None), qvx.E_NULL), (dict(q_out=A[1], q_type=qvx.F16), qvx.E_RANGE), (dict(q_out=A[1], q_stride=300), qvx.E_RANGE),
    (dict(q_out=A[0] + 1, q_type=qvx.BF16), qvx.E_RANGE), (dict(n=1 << 28, ps=1 << 28), qvx.E_RANGE)])
def test_norm_rope_refusals(kw, rc):
    assert turn(**kw) == rc


def test_norm_rope_needs_its_descriptions():
    lib = qvx.lib()
    assert lib.qvx_norm_rope_kv(A[0], 256, 0, A[1], 256, 4, None, 0, None, 0, 5, 64, None, None, A[4], 5, None, None, None) == qvx.E_NULL
