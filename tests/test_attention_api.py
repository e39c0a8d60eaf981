"""CPU tests of the attention calls' argument checks: every call here is refused, or has nothing to do, before any
device work, so the addresses are never dereferenced."""
from __future__ import annotations

import ctypes as C

import pytest

import qorvix_amd as qvx

P = 0x10000  # a 16-byte-aligned address that nothing reads


def cache(**kw):
    a = dict(d_k=P, d_v=P, page_stride=0, type=qvx.F16, n_pages=10, page_size=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return qvx.KvCache(**a)


def states(**kw):
    a = dict(d_k=P, d_v=P, batch_stride=77 * 128, row_stride=128, head_stride=64, type=qvx.F16, max_len=77, kv_heads=2,
             head_dim=64)
    a.update(kw)
    return qvx.KvStates(**a)


def paged(c=None, out=P, out_stride=256, q=P + 16, q_stride=256, heads=4, table=P, width=8, lens=P, n=3, ws=P, ws_bytes=None):
    c = cache() if c is None else c
    ws_bytes = qvx.attn_paged_ws(c, heads, n, width) if ws_bytes is None else ws_bytes
    return qvx.attn_paged(out, out_stride, q, q_stride, heads, c, table, width, lens, n, 0.125, ws, ws_bytes)


BAD_CACHES = [(dict(type=qvx.Q4_0), qvx.E_TYPE), (dict(type=99), qvx.E_TYPE), (dict(head_dim=60), qvx.E_SHAPE),
              (dict(head_dim=264), qvx.E_SHAPE), (dict(head_dim=0), qvx.E_SHAPE),
              (dict(type=qvx.Q8_0, head_dim=40), qvx.E_SHAPE), (dict(n_pages=0), qvx.E_SHAPE),
              (dict(page_size=0), qvx.E_SHAPE), (dict(kv_heads=0), qvx.E_SHAPE), (dict(d_k=0), qvx.E_NULL),
              (dict(d_v=None), qvx.E_NULL), (dict(d_k=P + 8), qvx.E_RANGE), (dict(d_v=P + 2), qvx.E_RANGE),
              (dict(page_stride=4095), qvx.E_RANGE), (dict(page_stride=4080), qvx.E_RANGE),
              (dict(page_stride=4104), qvx.E_RANGE), (dict(n_pages=1 << 30), qvx.E_RANGE)]


def test_page_bytes():
    assert qvx.kv_page_bytes(qvx.F16, 8, 16, 128) == 8 * 16 * 128 * 2
    assert qvx.kv_page_bytes(qvx.F32, 1, 1, 8) == 32
    assert qvx.kv_page_bytes(qvx.Q8_0, 2, 16, 64) == 2 * 16 * 64 * 34 // 32
    assert qvx.kv_page_bytes(qvx.Q8_0, 1, 1, 32) == 48  # 34 bytes, rounded up to a multiple of 16
    assert qvx.kv_page_bytes(qvx.BF16, 1 << 20, 1 << 10, 256) == 1 << 39  # past 32 bits
    for bad in ((qvx.Q4_K, 1, 16, 256), (qvx.F16, 0, 16, 64), (qvx.F16, 1, -1, 64), (qvx.F16, 1, 16, 12),
                (qvx.F16, 1, 16, 512), (qvx.Q8_0, 1, 16, 48)):
        assert qvx.kv_page_bytes(*bad) == 0


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_paged_refuses_caches(kw, rc):
    assert paged(cache(**kw), ws_bytes=1 << 30) == rc
    assert qvx.attn_paged_ws(cache(**kw), 4, 3, 8) == 0


def test_paged_refusals():
    assert paged(n=0) == qvx.E_NVEC and paged(n=-1) == qvx.E_NVEC
    assert paged(heads=3) == qvx.E_SHAPE and paged(heads=0) == qvx.E_SHAPE
    assert paged(width=0) == qvx.E_SHAPE
    assert paged(out_stride=255) == qvx.E_SHAPE and paged(q_stride=-1) == qvx.E_SHAPE
    for name in ("out", "q", "table", "lens"):
        assert paged(**{name: 0}) == qvx.E_NULL
    assert paged(n=70000) == qvx.E_RANGE
    assert paged(width=1 << 28) == qvx.E_RANGE
    need = qvx.attn_paged_ws(cache(), 4, 3, 100)
    assert need > 0
    assert paged(width=100, ws=0) == qvx.E_NULL
    assert paged(width=100, ws_bytes=need - 1) == qvx.E_RANGE
    assert paged(width=100, ws=P + 4) == qvx.E_RANGE
    assert paged(out=P, q=P, q_stride=512) == qvx.E_RANGE  # in place only row by row
    assert qvx.lib().qvx_attn_paged(P, 256, P, 256, 4, None, P, 8, P, 3, 0.1, P, 1 << 20, None) == qvx.E_NULL


def cross(s=None, out=P, out_stride=256, q=P + 16, q_stride=256, q_type=qvx.F32, heads=4, offsets=P, n_q=6, lens=0, n=3,
          ws=P, ws_bytes=1 << 40):
    return qvx.attn_cross(out, out_stride, q, q_stride, q_type, heads, offsets, n_q, states() if s is None else s, lens, n,
                          0.125, ws, ws_bytes)


@pytest.mark.parametrize("kw,rc", [
    (dict(type=qvx.Q8_0), qvx.E_TYPE), (dict(type=12), qvx.E_TYPE), (dict(head_dim=20), qvx.E_SHAPE),
    (dict(head_dim=264), qvx.E_SHAPE), (dict(kv_heads=0), qvx.E_SHAPE), (dict(max_len=-1), qvx.E_SHAPE),
    (dict(row_stride=56), qvx.E_SHAPE), (dict(batch_stride=-8), qvx.E_SHAPE), (dict(head_stride=-8), qvx.E_SHAPE),
    (dict(row_stride=132), qvx.E_RANGE), (dict(head_stride=68), qvx.E_RANGE), (dict(batch_stride=9), qvx.E_RANGE),
    (dict(row_stride=1 << 26), qvx.E_RANGE), (dict(d_k=None), qvx.E_NULL), (dict(d_v=P + 8), qvx.E_RANGE)])
def test_cross_refuses_states(kw, rc):
    assert cross(states(**kw)) == rc
    assert qvx.attn_cross_ws(states(**kw), qvx.F32, 4, 6, 3) == 0


def test_cross_refusals():
    assert cross(n=0) == qvx.E_NVEC
    assert cross(q_type=qvx.Q8_0) == qvx.E_TYPE
    assert cross(heads=3) == qvx.E_SHAPE and cross(n_q=-1) == qvx.E_SHAPE
    assert cross(offsets=0, n_q=7) == qvx.E_SHAPE  # 7 queries are no three equal parts
    assert cross(out_stride=255) == qvx.E_SHAPE and cross(q_stride=-256) == qvx.E_SHAPE
    assert cross(n_q=0) == qvx.OK  # nothing to do
    assert cross(states(d_k=0, d_v=0, max_len=0), n_q=0) == qvx.OK  # no states: no addresses
    assert cross(out=0) == qvx.E_NULL and cross(q=0) == qvx.E_NULL
    assert cross(out=P + 2) == qvx.E_RANGE and cross(q=P + 1, q_type=qvx.F16) == qvx.E_RANGE
    assert cross(out=P, q=P, q_stride=300) == qvx.E_RANGE
    big = states(max_len=1500, batch_stride=1500 * 128)
    need = qvx.attn_cross_ws(big, qvx.F32, 4, 6, 3)
    assert need > 0 and cross(big, ws=0) == qvx.E_NULL and cross(big, ws_bytes=need - 1) == qvx.E_RANGE
    assert qvx.lib().qvx_attn_cross(P, 256, P, 256, 0, 4, P, 6, None, P, 3, 0.1, P, 1 << 20, None) == qvx.E_NULL


def rope(q_out=P, q_out_stride=256, q=P + (1 << 20), q_stride=256, heads=4, k=P, ks=128, v=P, vs=128, n=5, d=64, pos=P, ps=5,
         c=True, slots=P, **kw):
    a = dict(d_inv_freq=P, d_axis=None, rot_dim=64, n_axes=1, pairing=qvx.ROPE_HALVES, scale=1.0)
    a.update(kw)
    c = cache() if c is True else c
    return qvx.rope_kv(q_out, q_out_stride, q, q_stride, heads, k, ks, v, vs, n, d, qvx.Rope(**a), pos, ps, c, slots)


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_rope_refuses_caches(kw, rc):
    c = cache(**kw)
    assert rope(c=c, d=c.head_dim) == rc


def test_rope_refusals():
    assert rope(n=0) == qvx.E_NVEC
    assert rope(pairing=2) == qvx.E_VARIANT
    assert rope(d=128) == qvx.E_SHAPE  # the cache's heads are of 64
    for kw in (dict(rot_dim=72), dict(rot_dim=12), dict(rot_dim=-8), dict(n_axes=0), dict(n_axes=5), dict(heads=-1),
               dict(q_out_stride=255), dict(q_stride=-4), dict(ks=-1), dict(vs=-1), dict(n_axes=3, ps=4), dict(ps=-1)):
        assert rope(**kw) == qvx.E_SHAPE, kw
    for kw in (dict(q=0), dict(q_out=0), dict(k=0), dict(v=0), dict(slots=0), dict(pos=0), dict(d_inv_freq=None)):
        assert rope(**kw) == qvx.E_NULL, kw
    assert rope(q_out=P, q=P, q_stride=300) == qvx.E_RANGE
    assert rope(c=None, heads=0) == qvx.E_SHAPE
    assert qvx.lib().qvx_rope_kv(P, 256, P, 256, 4, P, 128, P, 128, 5, 64, None, P, 5, None, P, None) == qvx.E_NULL


def kv_map(held=P, new=P + 4096, n=8, table=2 * P, width=4, page=16, free=3 * P, n_free=9, t_in=4 * P, t_out=4 * P + 64,
           lens=5 * P, offsets=6 * P, slots=7 * P, pos=8 * P, seq=9 * P, rows=20):
    return qvx.kv_map(held, new, n, table, width, page, free, n_free, t_in, t_out, lens, offsets, slots, pos, seq, rows)


def test_map_refusals():
    assert kv_map(n=0) == qvx.E_NVEC
    for kw in (dict(width=0), dict(page=0), dict(n_free=-1), dict(rows=-1)):
        assert kv_map(**kw) == qvx.E_SHAPE
    assert kv_map(n=16385) == qvx.E_RANGE
    for name in ("held", "new", "table", "free", "t_in", "t_out", "lens", "offsets", "slots"):
        assert kv_map(**{name: 0}) == qvx.E_NULL, name
    # outputs on inputs: the lengths and the count in place, nothing else
    for kw in (dict(lens=P + 4), dict(lens=P + 4096), dict(t_out=4 * P + 4), dict(offsets=P), dict(slots=P + 4096),
               dict(pos=4 * P), dict(seq=P + 28)):
        assert kv_map(**kw) == qvx.E_RANGE, kw


def test_descriptions_of_tensors_are_checked():
    import torch
    cpu = torch.zeros((4, 4096), dtype=torch.uint8)
    with pytest.raises(ValueError):
        qvx.KvCache.of(cpu, cpu, qvx.F16, 16, 2, 64)
    with pytest.raises(ValueError):
        qvx.Rope.of(torch.zeros(32))
    with pytest.raises(ValueError):
        qvx.KvStates.of(torch.zeros((1, 4, 2, 64)), torch.zeros((1, 4, 2, 64)))


def test_descriptions_and_workspaces_lie_beside_the_tensors():
    import torch
    far = torch.empty(1, device="meta")
    q, ints = torch.zeros((3, 4, 64)), torch.zeros(3, dtype=torch.int32)
    c, st, r = cache(), states(), qvx.Rope(P, None, 64, 1, 0, 1.0)
    c.tensors = st.tensors = r.tensors = (far, far)
    with pytest.raises(ValueError, match="cache: on meta"):
        qvx.attn_paged_t(q, c, ints, ints)
    with pytest.raises(ValueError, match="states: on meta"):
        qvx.attn_cross_t(q, st)
    with pytest.raises(ValueError, match="rope: on meta"):
        qvx.rope_kv_t(q, None, None, ints, r)
    r.tensors = (q, None)
    with pytest.raises(ValueError, match="cache: on meta"):
        qvx.rope_kv_t(q, q, q, ints, r, cache=c, slots=ints)


def test_structures_match_the_header():
    """Sizes and offsets as the C compiler lays the descriptions out."""
    import os
    import subprocess
    import tempfile

    from conftest import ROOT
    names = {"qvx_kv_cache": qvx.KvCache, "qvx_rope": qvx.Rope, "qvx_kv_states": qvx.KvStates}
    lines = []
    for c_name, cls in names.items():
        lines.append(f'printf("{c_name} %zu", sizeof({c_name}));')
        lines += [f'printf(" %zu", offsetof({c_name}, {f[0]}));' for f in cls._fields_] + ['printf("\\n");']
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "qvx.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", os.path.join(d, "s")], check=True)
        out = subprocess.run([os.path.join(d, "s")], check=True, capture_output=True, text=True).stdout
    for line in out.splitlines():
        name, size, *offsets = line.split()
        cls = names[name]
        assert C.sizeof(cls) == int(size)
        assert [getattr(cls, f[0]).offset for f in cls._fields_] == [int(o) for o in offsets]


def test_cache_pages_that_overlap_are_refused():
    """An expanded page has a stride of 0, which a description reads as pages side by side: past the one that there is."""
    import torch
    size = qvx.kv_page_bytes(qvx.F16, 2, 16, 64)
    one = torch.zeros((1, size), dtype=torch.uint8)
    for pages in (one.expand(4, size), torch.zeros(4 * size, dtype=torch.uint8).as_strided((4, size), (16, 1))):
        with pytest.raises(ValueError, match="overlap"):
            qvx.KvCache.of(pages, pages, qvx.F16, 16, 2, 64)


def test_lengths_whose_tiles_pass_31_bits_are_refused():
    """A length is rounded up to whole tiles of 16 keys, and a chunk's first tile and length are added, in 32 bits."""
    for n in (0x7ffffff1, 0x7fffffff):
        long = states(max_len=n, batch_stride=1 << 40)
        assert cross(long) == qvx.E_RANGE and qvx.attn_cross_ws(long, qvx.F32, 4, 6, 3) == 0
        one = cache(n_pages=1, page_size=n)
        assert paged(one, width=1, ws_bytes=1 << 40) == qvx.E_RANGE and qvx.attn_paged_ws(one, 4, 3, 1) == 0
    assert qvx.attn_cross_ws(states(max_len=0x7ffffff0, batch_stride=1 << 40), qvx.F32, 4, 6, 3) > 0
    assert qvx.attn_paged_ws(cache(n_pages=1, page_size=0x7ffffff0), 4, 3, 1) > 0
    small = cache(n_pages=0x7fffffff, page_size=1)
    assert paged(small, width=0x7fffffff, ws_bytes=1 << 40) == qvx.E_RANGE
    assert qvx.attn_paged_ws(small, 4, 1, 0x40000000) == 0 and qvx.attn_paged_ws(small, 4, 1, 0x3fffffff) > 0


def test_launches_past_32_bits_of_threads_are_refused():
    """A launch holds fewer than 2^32 threads: 2^24 workgroups of 256."""
    many = cache(kv_heads=256)
    assert paged(many, heads=256, out_stride=256 * 64, q_stride=256 * 64, n=65536, ws_bytes=1 << 40) == qvx.E_RANGE
    assert paged(cache(kv_heads=255), heads=256 * 255, n=65536, ws_bytes=1 << 40) == qvx.E_RANGE  # row tiles count too
    wide = states(kv_heads=256, row_stride=256 * 64, batch_stride=0)
    assert cross(wide, heads=256, out_stride=256 * 64, q_stride=256 * 64, n_q=65536, n=65536) == qvx.E_RANGE
    for c in (True, None):
        assert rope(c=c, n=8 * 0xffffff + 1, ps=1 << 28) == qvx.E_RANGE
