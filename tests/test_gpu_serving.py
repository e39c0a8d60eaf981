"""The attention calls in the steps that use them: a decoder's whole step over a paged cache
(decode.PagedDecodeStep), eager and captured, and a speech decoder's layer with attention to its own tokens
and to an encoder's states.  Each is held against the same step with the engine's own projections and the
rotation, the cache and the attention formed in 64 bits on the host from the tokens' whole history.

Tolerance: the two steps' attention outputs differ by fp32 rounding, far below the 3.1e-5 of its slot's largest
to which a projection holds its activations; a difference can move such a code by one step, which the
projections' own bar of 1e-3 a product covers.  Four products follow one another in a layer: 4e-3 a layer."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from qorvix_amd import decode

pytestmark = pytest.mark.gpu


def _weight(torch, t, rows, cols, seed):
    w = qvx.empty_weight(t, rows, cols)
    qvx.fill_synthetic_t(w, t, rows, cols, seed=seed, scale_mul=3e-3)
    return decode.DevWeight(w, t, rows, cols)


def _model(torch, layers=2, d=512, heads=8, kv_heads=2, hd=64, ffn=1024, vocab=256):
    m = decode.Model()
    for l in range(layers):
        m.layers.append({
            "wq": _weight(torch, qvx.Q4_K, heads * hd, d, 10 * l), "wk": _weight(torch, qvx.Q4_K, kv_heads * hd, d, 10 * l + 1),
            "wv": _weight(torch, qvx.Q6_K, kv_heads * hd, d, 10 * l + 2), "wo": _weight(torch, qvx.Q4_K, d, heads * hd, 10 * l + 3),
            "ffn_gate": _weight(torch, qvx.Q4_K, ffn, d, 10 * l + 4), "ffn_up": _weight(torch, qvx.Q4_K, ffn, d, 10 * l + 5),
            "ffn_down": _weight(torch, qvx.Q6_K, d, ffn, 10 * l + 6)})
        m.norms.append({k: 1.0 + 0.1 * torch.randn(d, device="cuda") for k in ("attn_norm", "ffn_norm")})
    m.lm_head = _weight(torch, qvx.Q6_K, vocab, d, 99)
    m.output_norm = 1.0 + 0.1 * torch.randn(d, device="cuda")
    return m.fused_ops()


class HostStep:
    """The step of decode.PagedDecodeStep with the engine's projections; rotation, cache and attention on the host."""

    def __init__(self, torch, step, cache_dtype):
        self.torch, self.s, self.dtype = torch, step, cache_dtype
        n = len(step.model.layers)
        self.k = [[[] for _ in range(step.m)] for _ in range(n)]
        self.v = [[[] for _ in range(step.m)] for _ in range(n)]
        self.t = [0] * step.m

    def rounded(self, x):
        return self.torch.from_numpy(x.astype(np.float32)).to(self.dtype).double().numpy()

    def turn(self, x, pos):
        hd = self.s.head_dim
        a = pos * 500000.0 ** (-np.arange(hd // 2) * 2 / hd)
        lo, hi = x[:, : hd // 2], x[:, hd // 2:]
        return np.concatenate([lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)], 1)

    def run(self, x):
        torch, s, model = self.torch, self.s, self.s.model
        hd, hk, g = s.head_dim, s.kv_heads, s.heads // s.kv_heads
        x = x.clone()
        for l, w in enumerate(model.layers):
            an, fn = model.norms[l]["attn_norm"], model.norms[l]["ffn_norm"]
            qk = qvx.qmatmul_rmsnorm_t(w["wqk"].data, w["wqk"].type, x, an, model.eps, w["wqk"].rows, w["wqk"].cols)
            v = qvx.qmatmul_rmsnorm_t(w["wv"].data, w["wv"].type, x, an, model.eps, w["wv"].rows, w["wv"].cols)
            qk, v = qk.cpu().double().numpy(), v.cpu().double().numpy()
            attn = np.zeros((s.m, s.heads * hd))
            for b in range(s.m):
                q = self.turn(qk[b, : s.heads * hd].reshape(-1, hd), self.t[b])
                self.k[l][b].append(self.rounded(self.turn(qk[b, s.heads * hd:].reshape(-1, hd), self.t[b])))
                self.v[l][b].append(self.rounded(v[b].reshape(-1, hd)))
                keys, vals = np.stack(self.k[l][b]), np.stack(self.v[l][b])
                for h in range(s.heads):
                    z = keys[:, h // g] @ q[h] * hd ** -0.5
                    p = np.exp(z - z.max())
                    attn[b, h * hd:(h + 1) * hd] = p @ vals[:, h // g] / p.sum()
            a = torch.from_numpy(attn.astype(np.float32)).cuda()
            x += qvx.qmatmul_t(w["wo"].data, w["wo"].type, a, w["wo"].rows, w["wo"].cols)
            gu, down = w["ffn_gateup"], w["ffn_down"]
            h = qvx.qmatmul_swiglu_t(gu.data, gu.type, x, gu.rows // 2, gu.cols, fn, model.eps)
            x += qvx.qmatmul_t(down.data, down.type, h, down.rows, down.cols)
        self.t = [t + 1 for t in self.t]
        lm = model.lm_head
        return x, qvx.qmatmul_rmsnorm_t(lm.data, lm.type, x, model.output_norm, model.eps, lm.rows, lm.cols)


def _near(got, want, tol):
    got, want = got.cpu().double(), want.cpu().double()
    assert bool(got.isfinite().all())
    assert float((got - want).abs().max() / want.abs().max()) <= tol


@pytest.mark.parametrize("m,t", [(1, qvx.F16), (3, qvx.F16), (1, qvx.F32), (3, qvx.F32), (20, qvx.F16)])
def test_paged_decode_steps(cuda, m, t):
    """Twelve eager steps, then as many replays of the captured step, pages filling up one after another."""
    torch = cuda
    torch.manual_seed(m)
    model = _model(torch)
    step = decode.PagedDecodeStep(model, m, heads=8, kv_heads=2, n_pages=8 * m + 1, max_pages=9, page_size=3, cache_type=t)
    host = HostStep(torch, step, torch.float16 if t == qvx.F16 else torch.float32)
    for i in range(24):
        x = torch.randn((m, 512), device="cuda")
        want_x, want = host.run(x)
        step.x.copy_(x)
        if i == 12:
            step.capture()
        if i < 12:
            step.run(torch.cuda.current_stream().cuda_stream)
        else:
            step.replay()
        torch.cuda.synchronize()
        assert step.lens.tolist() == [i + 1] * m and step.taken.tolist() == [m * (i // 3 + 1), 0]
        _near(step.x, want_x, 8e-3)
        _near(step.logits, want, 8e-3)


def test_paged_decode_step_without_pages_left(cuda):
    """The pool runs out: the status says so and the lengths stand still."""
    torch = cuda
    step = decode.PagedDecodeStep(_model(torch, layers=1), 2, heads=8, kv_heads=2, n_pages=3, max_pages=4, page_size=2)
    s = torch.cuda.current_stream().cuda_stream
    for i in range(4):
        step.x.normal_()
        step.run(s)
        torch.cuda.synchronize()
        assert step.lens.tolist() == [min(i + 1, 2)] * 2
        assert step.taken.tolist() == ([2, 0] if i < 2 else [2, qvx.MAP_PAGES])
        assert bool(step.x.isfinite().all())


def test_paged_decode_step_refuses_models(cuda):
    torch = cuda
    model = _model(torch, layers=1)
    with pytest.raises(ValueError):
        decode.PagedDecodeStep(model, 1, heads=7, kv_heads=1, n_pages=4, max_pages=2)
    with pytest.raises(ValueError):
        decode.PagedDecodeStep(model, 1, heads=8, kv_heads=4, n_pages=4, max_pages=2)
    with pytest.raises(ValueError):
        decode.PagedDecodeStep(model, 1, heads=8, kv_heads=2, n_pages=4, max_pages=2, cache_type=qvx.Q4_0)
    model.norms[0]["ffn_norm"] = None
    with pytest.raises(ValueError):
        decode.PagedDecodeStep(model, 1, heads=8, kv_heads=2, n_pages=4, max_pages=2)


def test_speech_decoder_layer(cuda):
    """Three candidates of a speech decoder: products with bias, attention to their own tokens over the cache and to
    their windows' states (one product for keys and values, read where it stands), token after token."""
    torch = cuda
    torch.manual_seed(5)
    d, heads, hd, n, frames = 256, 4, 64, 3, 150
    w = {k: _weight(torch, qvx.Q8_0, rows, d, i) for i, (k, rows) in enumerate(
        (("qkv", 3 * d), ("o", d), ("cq", d), ("ckv", 2 * d), ("co", d)))}
    bias = {k: 0.1 * torch.randn(x.rows, device="cuda") for k, x in w.items()}

    def product(k, x):
        out = torch.empty((x.shape[0], w[k].rows), device="cuda")
        assert qvx.qmatmul_n_bias(out.data_ptr(), w[k].data.data_ptr(), w[k].type, x.data_ptr(), bias[k].data_ptr(),
                                  x.shape[0], w[k].rows, d, torch.cuda.current_stream().cuda_stream) == qvx.OK
        return out

    audio = torch.randn((n * frames, d), device="cuda")
    kv = product("ckv", audio).to(torch.float16).view(n, frames, 2, heads, hd)
    states = qvx.KvStates.of(kv[:, :, 0], kv[:, :, 1])
    lens = torch.tensor([150, 7, 64], dtype=torch.int32, device="cuda")
    page, pages = 4, 9
    size = qvx.kv_page_bytes(qvx.F32, heads, page, hd)
    cache = qvx.KvCache.of(*(torch.zeros((pages, size), dtype=torch.uint8, device="cuda") for _ in range(2)), qvx.F32, page,
                           heads, hd)
    still = qvx.Rope.of(torch.zeros(0, dtype=torch.float64, device="cuda"))  # learned positions: nothing turns
    held = torch.zeros(n, dtype=torch.int32, device="cuda")
    new, taken = torch.ones_like(held), torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.full((n, 3), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, device="cuda").to(torch.int32)
    past_k, past_v = [], []
    for step in range(9):
        x = torch.randn((n, d), device="cuda")
        held, _, slots, pos, _, taken = qvx.kv_map_t(held, new, table, page, free, taken, n)
        qkv = product("qkv", x).view(n, 3, heads, hd)
        q = qvx.rope_kv_t(qkv[:, 0], qkv[:, 1], qkv[:, 2], pos, still, cache, slots)
        assert torch.equal(q, qkv[:, 0])
        a = qvx.attn_paged_t(q, cache, table, held)
        past_k.append(qkv[:, 1].cpu().double())
        past_v.append(qkv[:, 2].cpu().double())
        k, v = torch.stack(past_k, 2), torch.stack(past_v, 2)  # [n, heads, tokens, hd]
        p = torch.softmax((k @ q.cpu().double().unsqueeze(-1)).squeeze(-1) * hd ** -0.5, -1)
        _near(a, (p.unsqueeze(2) @ v).squeeze(2), 2e-5)
        y = x + product("o", a.view(n, d))
        cq = product("cq", y).view(n, heads, hd)
        ca = qvx.attn_cross_t(cq, states, lens=lens)
        for b in range(n):
            kk, vv = (kv[b, : int(lens[b]), i].cpu().double().transpose(0, 1) for i in range(2))
            p = torch.softmax((kk @ cq[b].cpu().double().unsqueeze(-1)).squeeze(-1) * hd ** -0.5, -1)
            _near(ca[b], (p.unsqueeze(1) @ vv).squeeze(1), 2e-5)
        assert bool((y + product("co", ca.view(n, d))).isfinite().all())
    assert taken.tolist() == [9, 0]


def test_paged_decode_step_of_a_file(cuda, tmp_path):
    """A file's own rotation: neighbours form the pairs, half of a head turns, base and divisors as the file gives them.
    What the step leaves in q and stores in the fp32 cache is the projections' outputs turned in 64 bits; the bar is the
    rotation's own (32 u of the largest value) and what a projection of the same activations repeats bit by bit."""
    from gguf_build import GgufBuilder
    torch = cuda
    rng = np.random.default_rng(8)
    d, heads, kv_heads, hd, rot, ffn, base = 512, 8, 2, 64, 32, 512, 700.0
    b = (GgufBuilder(3).str("general.architecture", "llama").u32("general.alignment", 32).u32("llama.block_count", 1)
         .u32("llama.embedding_length", d).u32("llama.feed_forward_length", ffn).u32("llama.attention.head_count", heads)
         .u32("llama.attention.head_count_kv", kv_heads).f32("llama.rope.freq_base", base)
         .u32("llama.rope.dimension_count", rot).str("llama.rope.scaling.type", "linear").f32("llama.rope.scaling.factor", 2.0))
    factors = (1.0 + rng.random(rot // 2)).astype(np.float32)
    tensors = [("rope_freqs.weight", [rot // 2], factors)]
    tensors += [(n, [d], (1.0 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for n in
                ("blk.0.attn_norm.weight", "blk.0.ffn_norm.weight", "output_norm.weight")]
    tensors += [(f"blk.0.{n}.weight", [cols, rows], (rng.standard_normal((rows, cols)) * cols ** -0.5).astype(np.float32))
                for n, rows, cols in (("attn_q", d, d), ("attn_k", kv_heads * hd, d), ("attn_v", kv_heads * hd, d),
                                      ("attn_output", d, d), ("ffn_gate", ffn, d), ("ffn_up", ffn, d), ("ffn_down", d, ffn))]
    tensors.append(("token_embd.weight", [d, 64], rng.standard_normal((64, d)).astype(np.float32)))
    data = bytearray()
    for name, dims, x in tensors:
        b.tensor(name, dims, qvx.F32, len(data))
        data += x.tobytes()
    path = tmp_path / "model.gguf"
    path.write_bytes(b.build(32, data=bytes(data)))
    step = decode.PagedDecodeStep(decode.Model.from_gguf(path).fused_ops(), 2, heads, kv_heads, n_pages=8, max_pages=3,
                                  page_size=4, cache_type=qvx.F32)
    layer, norms = step.model.layers[0], step.model.norms[0]
    for t in range(6):
        x = torch.randn((2, d), device="cuda")
        step.x.copy_(x)
        step.run(torch.cuda.current_stream().cuda_stream)
        w = layer["wqk"]
        qk = qvx.qmatmul_rmsnorm_t(w.data, w.type, x, norms["attn_norm"], step.model.eps, w.rows, w.cols)
        qk = qk.cpu().double().numpy().reshape(2, heads + kv_heads, hd)
        angle = t * base ** (-np.arange(rot // 2) * 2 / rot) / 2.0 / factors.astype(np.float64)
        a, c = qk[..., 0:rot:2].copy(), qk[..., 1:rot:2].copy()
        qk[..., 0:rot:2], qk[..., 1:rot:2] = a * np.cos(angle) - c * np.sin(angle), a * np.sin(angle) + c * np.cos(angle)
        bar = 32 * 2.0 ** -24 * np.abs(qk).max()
        got = step.qk.cpu().double().numpy().reshape(2, heads + kv_heads, hd)[:, :heads]
        assert np.abs(got - qk[:, :heads]).max() <= bar
        page = step.table.cpu().numpy()[:, t // 4]
        stored = step.caches[0].tensors[0].cpu().contiguous().view(torch.float32).view(8, kv_heads, 4, hd)
        assert np.abs(stored[page, :, t % 4].double().numpy() - qk[:, heads:]).max() <= bar
    assert step.taken.tolist() == [4, 0] and bool(step.logits.isfinite().all())


def test_paged_decode_step_without_pages_left_changes_nothing(cuda):
    """Lengths, table and every byte of the cache stand still, eager and replayed, and the step goes on once the caller has
    handed pages back."""
    torch = cuda
    step = decode.PagedDecodeStep(_model(torch, layers=1), 2, heads=8, kv_heads=2, n_pages=3, max_pages=4, page_size=2)
    for _ in range(2):
        step.x.normal_()
        step.run(torch.cuda.current_stream().cuda_stream)
    step.capture()
    before = [x.clone() for x in (step.table, step.lens, *step.pages)]
    for replay in (False, True, True):
        step.x.normal_()
        step.replay() if replay else step.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert step.taken.tolist() == [2, qvx.MAP_PAGES]
        assert all(torch.equal(a, b) for a, b in zip(before, (step.table, step.lens, *step.pages)))
    step.lens.zero_()  # both requests end: their pages go back
    step.table.fill_(-1)
    step.taken.zero_()
    step.x.normal_()
    step.replay()
    torch.cuda.synchronize()
    assert step.taken.tolist() == [2, 0] and step.lens.tolist() == [1, 1] and bool(step.logits.isfinite().all())


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32, qvx.Q8_0))
@pytest.mark.parametrize("scale_mul", (2.4e-4, 1e-4))
def test_paged_decode_step_weighs_its_tokens(cuda, t, scale_mul):
    """The step's attention by itself, on logits that leave weight to several tokens: what it leaves in `attn` against the
    softmax in 64 bits of its rotated queries on the keys and values that its cache holds.  Bar: that of the attention's
    own tests; a scale a tenth off, put into the reference, passes it in some row of every step from two tokens on."""
    torch = cuda
    torch.manual_seed(3)
    heads, hk, hd, m, page, u = 8, 2, 64, 3, 3, 2.0 ** -24
    model = _model(torch, layers=1)
    w = model.layers[0]["wqk"]
    qvx.fill_synthetic_t(w.data, w.type, w.rows, w.cols, seed=77, scale_mul=scale_mul)
    step = decode.PagedDecodeStep(model, m, heads=heads, kv_heads=hk, n_pages=8 * m + 1, max_pages=9, page_size=page, cache_type=t)
    for i in range(20):
        visible = []
        step.x.normal_()
        step.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        q = step.qk[:, : heads * hd].cpu().double().view(m, heads, hd).numpy()
        got, table = step.attn.cpu().double().view(m, heads, hd).numpy(), step.table.cpu().long()
        for b in range(m):
            kv = []
            for x in step.caches[0].tensors:
                raw = x[table[b, : i // page + 1].cuda()].cpu().contiguous()
                if t == qvx.Q8_0:
                    cut = hk * page * hd
                    x = raw[:, :cut].contiguous().view(torch.int8).double().view(-1, hk, page, hd // 32, 32)
                    x = x * raw[:, cut: cut + cut // 16].contiguous().view(torch.float16).double().view(-1, hk, page, hd // 32, 1)
                else:
                    used = hk * page * hd * (2 if t == qvx.F16 else 4)
                    x = raw[:, :used].contiguous().view(torch.float16 if t == qvx.F16 else torch.float32).double()
                kv.append(x.reshape(-1, hk, page, hd).transpose(1, 2).reshape(-1, hk, hd)[: i + 1].numpy())
            for h in range(heads):
                k, v = kv[0][:, h // 4], kv[1][:, h // 4]
                s = k @ q[b, h] * hd ** -0.5
                p = np.exp(s - s.max())
                p /= p.sum()
                size = (np.abs(k) @ np.abs(q[b, h])).max() * hd ** -0.5
                bar = 2 * u * ((hd + 3) * size + i + 9) * np.abs(v).max()
                assert np.abs(got[b, h] - p @ v).max() <= bar
                wrong = np.exp(1.1 * (s - s.max()))
                visible.append(bool(np.abs(wrong @ v / wrong.sum() - p @ v).max() > 2 * bar))
        assert i < 1 or any(visible)


def test_paged_decode_step_stays_on_its_device(cuda, monkeypatch):
    """The step's launches go to the current device: with another one current it is refused, eager and in a capture."""
    torch = cuda
    step = decode.PagedDecodeStep(_model(torch, layers=1), 1, heads=8, kv_heads=2, n_pages=4, max_pages=2)
    step.run(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "current_device", lambda: step.x.device.index + 1)
        with pytest.raises(ValueError, match="device"):
            step.run(stream)
        with pytest.raises(ValueError, match="device"):
            step.capture()
    step.capture()
    step.replay()
    torch.cuda.synchronize()
    assert step.lens.tolist() == [2]
