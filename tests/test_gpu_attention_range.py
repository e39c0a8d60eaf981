"""The attention calls at the ends of fp32's and bf16's range: keys and queries of far exponents whose logits are
ordinary, and values so large that only weights of at most 1 keep their sums finite.

Tolerances as in test_gpu_attention.py: powers of two move nothing but the exponents.  A query below 2^-126 loses
half of 2^-149 to its scale, which its key (2^123 at most) and d = 256 of them make 2^-19 of a logit: the (d + 3) u S of
those tests is at least 2^-24 * 67 * 1 = 2^-17.9 for the sums S >= 1 here."""
from __future__ import annotations

import math

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import Cache, U, _attend, _paged_reference, _torch_type

pytestmark = pytest.mark.gpu


def _upload(torch, c, i):
    """The host's values of K (i = 0) or V in the cache again, rounded to its type first."""
    x = torch.from_numpy(c.host[i].astype(np.float32)).to(_torch_type(torch, c.t))
    c.host[i] = x.double().numpy()
    c.desc.tensors[i].copy_(x.reshape(c.n_pages, -1).view(torch.uint8))


def _each_key(c):
    """(page, place in it, position) of every key of sequence 0."""
    for j in range(c.lens[0]):
        yield c.table[0, j // c.page], j % c.page, j


def _compare(torch, c, q, scale):
    out = qvx.attn_paged_t(q.cuda(), c.desc, c.dev_table, c.dev_lens, scale=scale)
    torch.cuda.synchronize()
    want, tol = _paged_reference(c, q.numpy(), scale)
    got = out.cpu().double().numpy()
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= tol, (np.abs(got - want).max(), tol)


@pytest.mark.parametrize("t", (qvx.BF16, qvx.F32))
@pytest.mark.parametrize("shift", [120, 100, -100])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 6, 16])
def test_paged_far_exponents(cuda, t, shift, d, group):
    """Keys 2^shift as large and queries as small: the same logits."""
    torch = cuda
    c = Cache(torch, t, (37, 1, 200), 16, 1, d, seed=d + group)
    c.host[0] = np.ldexp(c.host[0], shift)
    _upload(torch, c, 0)
    q = np.random.default_rng(3).standard_normal((3, group, d)) * 1.5
    _compare(torch, c, torch.from_numpy(np.ldexp(q, -shift).astype(np.float32)), d ** -0.5)


@pytest.mark.parametrize("t", (qvx.BF16, qvx.F32))
@pytest.mark.parametrize("group", [1, 6, 16])
def test_paged_largest_query(cuda, t, group):
    """fp32's largest number, which rounds to infinity in bf16, on keys of 2^-126 and a little more: logits of 2 to 4."""
    torch = cuda
    c = Cache(torch, t, (90,), 16, 1, 64, seed=group)
    c.host[0] = np.zeros_like(c.host[0])
    for p, o, j in _each_key(c):
        c.host[0][p, :, o, 0] = np.ldexp(1.0 + j % 4 / 4, -126)
    _upload(torch, c, 0)
    q = torch.zeros((1, group, 64))
    q[:, :, 0] = torch.finfo(torch.float32).max
    _compare(torch, c, q, 0.5)


@pytest.mark.parametrize("q_type,kv_type", [(qvx.F32, qvx.BF16), (qvx.BF16, qvx.BF16), (qvx.F16, qvx.BF16)])
@pytest.mark.parametrize("rows", [1, 6, 40])
def test_cross_far_exponents(cuda, q_type, kv_type, rows):
    torch = cuda
    d, n, shift = 64, 150, 120 if q_type != qvx.F16 else 8
    r = np.random.default_rng(rows)
    k = torch.from_numpy(np.ldexp(r.standard_normal((1, n, 1, d)), shift).astype(np.float32)).to(_torch_type(torch, kv_type))
    v = torch.from_numpy(r.standard_normal((1, n, 1, d)).astype(np.float32)).to(_torch_type(torch, kv_type))
    q = torch.from_numpy(np.ldexp(r.standard_normal((rows, 1, d)) * 1.5, -shift).astype(np.float32)).to(
        _torch_type(torch, q_type))
    got = qvx.attn_cross_t(q.cuda(), qvx.KvStates.of(k.cuda(), v.cuda())).cpu().double().numpy()[:, 0]
    want, s = _attend(q.double().numpy()[:, 0], k.double().numpy()[0, :, 0], v.double().numpy()[0, :, 0], d ** -0.5)
    half = {qvx.F32: 0.0, qvx.F16: 2.0 ** -11, qvx.BF16: 2.0 ** -8}[q_type]
    top = float(v.double().abs().max())
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2 * U * ((d + 3) * s + n + 8) * top + half * (np.abs(want) + top)).all()


@pytest.mark.parametrize("t", (qvx.BF16, qvx.F32))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 6, 16])
def test_paged_large_values(cuda, t, d, group):
    """Logits that rise by 2^19 behind the first tiles, values of 2^115: their products with weights above 1 overflow."""
    torch = cuda
    n = 150
    c = Cache(torch, t, (n,), 16, 1, d, seed=d)
    c.host[1] = np.ldexp(c.host[1], 115)
    for p, o, j in _each_key(c):
        c.host[0][p, :, o, 0] = 0.0 if j < 64 else 19.0
    _upload(torch, c, 0)
    _upload(torch, c, 1)
    q = torch.zeros((1, group, d))
    q[:, :, 0] = 1.0
    _compare(torch, c, q, math.log(2.0))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_cross_large_values(cuda, d):
    """As above on the 16-bit matrix cores: logits that rise by 2^7, values of 2^122."""
    torch = cuda
    n, rows = 200, 40
    r = np.random.default_rng(d)
    k = torch.zeros((1, n, 1, d), dtype=torch.bfloat16)
    k[0, 64:, 0, 0] = 7.0
    v = torch.from_numpy(np.ldexp(r.standard_normal((1, n, 1, d)), 122).astype(np.float32)).to(torch.bfloat16)
    q = torch.zeros((rows, 1, d), dtype=torch.bfloat16)
    q[:, 0, 0] = 1.0
    got = qvx.attn_cross_t(q.cuda(), qvx.KvStates.of(k.cuda(), v.cuda()), scale=math.log(2.0)).cpu().double().numpy()[:, 0]
    want, s = _attend(q.double().numpy()[:, 0], k.double().numpy()[0, :, 0], v.double().numpy()[0, :, 0], math.log(2.0))
    top = float(v.double().abs().max())
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2 * U * ((d + 3) * s + n + 8) * top + 2.0 ** -8 * (np.abs(want) + top)).all()
