"""The shared cache's calls in the steps that use them: decode.PagedDecodeStep with norms of q and k, behind a window, behind
shared prefixes, with forks, releases and compaction between its steps; and a prompt in pieces followed by samples of it,
call by call.  Reference and tolerance of the steps are test_gpu_serving.py's: 4e-3 a layer; of the calls, those of
test_gpu_window.py."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from qorvix_amd import decode
from test_gpu_serving import HostStep, _model, _near
from test_gpu_window import HALF, U, attend, seen

pytestmark = pytest.mark.gpu


class HostShared(HostStep):
    """HostStep with norms of the q and k heads, a window, and sequences that become copies of others."""

    def __init__(self, torch, step, dtype, window=None, sinks=0):
        super().__init__(torch, step, dtype)
        self.window, self.sinks = window, sinks

    def turn(self, x, pos):
        return super().turn(x, pos)

    def fork(self, source, to):
        for a, b in zip(source, to):
            for l in range(len(self.k)):
                self.k[l][b], self.v[l][b] = list(self.k[l][a]), list(self.v[l][a])
            self.t[b] = self.t[a]

    def empty(self, rows):
        for b in rows:
            for l in range(len(self.k)):
                self.k[l][b], self.v[l][b] = [], []
            self.t[b] = 0

    def norm(self, x, w):
        if w is None:
            return x
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.s.model.eps) * w.cpu().double().numpy()

    def run(self, x):
        torch, s, model = self.torch, self.s, self.s.model
        hd, g = s.head_dim, s.heads // s.kv_heads
        x = x.clone()
        for l, w in enumerate(model.layers):
            an, fn = model.norms[l]["attn_norm"], model.norms[l]["ffn_norm"]
            qn, kn = model.norms[l].get("q_norm"), model.norms[l].get("k_norm")
            qk = qvx.qmatmul_rmsnorm_t(w["wqk"].data, w["wqk"].type, x, an, model.eps, w["wqk"].rows, w["wqk"].cols)
            v = qvx.qmatmul_rmsnorm_t(w["wv"].data, w["wv"].type, x, an, model.eps, w["wv"].rows, w["wv"].cols)
            qk, v = qk.cpu().double().numpy(), v.cpu().double().numpy()
            attn = np.zeros((s.m, s.heads * hd))
            for b in range(s.m):
                q = self.turn(self.norm(qk[b, : s.heads * hd].reshape(-1, hd), qn), self.t[b])
                self.k[l][b].append(self.rounded(self.turn(self.norm(qk[b, s.heads * hd:].reshape(-1, hd), kn), self.t[b])))
                self.v[l][b].append(self.rounded(v[b].reshape(-1, hd)))
                keys, vals = np.stack(self.k[l][b]), np.stack(self.v[l][b])
                see = np.ones((1, len(keys)), bool) if self.window is None else seen(len(keys), 1, self.window, self.sinks)
                for h in range(s.heads):
                    attn[b, h * hd:(h + 1) * hd] = attend(q[h: h + 1], keys[:, h // g], vals[:, h // g], see, hd ** -0.5)[0]
            a = torch.from_numpy(attn.astype(np.float32)).cuda()
            x += qvx.qmatmul_t(w["wo"].data, w["wo"].type, a, w["wo"].rows, w["wo"].cols)
            gu, down = w["ffn_gateup"], w["ffn_down"]
            h = qvx.qmatmul_swiglu_t(gu.data, gu.type, x, gu.rows // 2, gu.cols, fn, model.eps)
            x += qvx.qmatmul_t(down.data, down.type, h, down.rows, down.cols)
        self.t = [t + 1 for t in self.t]
        lm = model.lm_head
        return x, qvx.qmatmul_rmsnorm_t(lm.data, lm.type, x, model.output_norm, model.eps, lm.rows, lm.cols)


def _both(torch, step, host, n, tol=8e-3, replay=False):
    for _ in range(n):
        x = torch.randn((step.m, 512), device="cuda")
        want_x, want = host.run(x)
        step.x.copy_(x)
        if replay:
            step.replay()
        else:
            step.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert step.taken.tolist()[1] == 0 and step.lens.tolist() == host.t
        _near(step.x, want_x, tol)
        _near(step.logits, want, tol)


@pytest.mark.parametrize("which", [("q_norm", "k_norm"), ("q_norm",), ("k_norm",)])
def test_norms_of_q_and_k(cuda, which):
    torch = cuda
    torch.manual_seed(1)
    model = _model(torch)
    for norms in model.norms:
        for k in which:
            norms[k] = 1.0 + 0.3 * torch.randn(64, device="cuda")
    step = decode.PagedDecodeStep(model, 3, heads=8, kv_heads=2, n_pages=30, max_pages=9, page_size=4)
    host = HostShared(torch, step, torch.float16)
    _both(torch, step, host, 6)
    step.capture()
    _both(torch, step, host, 6, replay=True)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (5, 2), (100, 1)])
def test_a_window(cuda, window, sinks):
    torch = cuda
    torch.manual_seed(2)
    step = decode.PagedDecodeStep(_model(torch), 2, heads=8, kv_heads=2, n_pages=20, max_pages=9, page_size=3, window=window,
                                  sinks=sinks)
    host = HostShared(torch, step, torch.float16, window, sinks)
    _both(torch, step, host, 10)
    step.capture()
    _both(torch, step, host, 6, replay=True)


@pytest.mark.parametrize("window,sinks,page", [(1, 0, 1), (5, 0, 3), (6, 4, 3), (4, 3, 2), (64, 0, 4)])
def test_pages_behind_a_window_go_back(cuda, window, sinks, page):
    torch = cuda
    torch.manual_seed(5)
    step = decode.PagedDecodeStep(_model(torch, layers=1), 2, heads=8, kv_heads=2, n_pages=2 * (-(-sinks // page) + -(-window // page) + 3),
                                  max_pages=30, page_size=page, window=window, sinks=sinks)
    host = HostShared(torch, step, torch.float16, window, sinks)
    for _ in range(6):
        _both(torch, step, host, page + 1)
        step.trim()
        n = host.t[0]
        kept = [j for j in range(-(-n // page)) if (j + 1) * page > n - window + 1 or j * page < sinks]
        assert [j for j in range(30) if int(step.table[0, j]) >= 0] == kept and step.taken.tolist() == [2 * len(kept), 0]


@pytest.mark.parametrize("groups", [0, 1, 2])
def test_forks_between_steps(cuda, groups):
    """Sequences that become copies of others, and go on on their own, in every layer; pages that move in between."""
    torch = cuda
    torch.manual_seed(3)
    m, page = 4, 3
    step = decode.PagedDecodeStep(_model(torch), m, heads=8, kv_heads=2, n_pages=40, max_pages=12, page_size=page,
                                  shared_groups=groups)
    host = HostShared(torch, step, torch.float16)
    _both(torch, step, host, 7)
    step.fork([0, 0], [1, 3])
    host.fork([0, 0], [1, 3])
    if groups:  # sequences 0 and 1 begin alike, and 2 and 3 do not: their group shares nothing
        step.groups.copy_(torch.tensor([0, 2, 4][: groups] + [m], dtype=torch.int32))
        step.shared[0] = 7 // page * page if groups == 2 else 0
    _both(torch, step, host, 4)
    step.compact()
    used = int((step.table >= 0).sum()) - int(step.extra.sum())
    assert step.taken.tolist() == [used, 0] and int(step.table.max()) == used - 1
    step.capture()
    _both(torch, step, host, 4, replay=True)
    if groups:
        step.shared.zero_()
    step.fork([3], [0])
    host.fork([3], [0])
    step.release([2])
    host.empty([2])
    _both(torch, step, host, 3, replay=True)
    step.release(range(m))
    assert step.taken.tolist() == [0, 0] and int(step.extra.sum()) == 0 and int(step.table.max()) == -1
    assert sorted(step.free.tolist()) == list(range(40))


def test_refusals(cuda):
    torch = cuda
    model = _model(torch, layers=1)
    for kw in (dict(window=0), dict(sinks=2), dict(window=4, sinks=-1), dict(shared_groups=3), dict(window=4, shared_groups=1)):
        with pytest.raises(ValueError, match="PagedDecodeStep"):
            decode.PagedDecodeStep(model, 2, heads=8, kv_heads=2, n_pages=4, max_pages=2, **kw)
    step = decode.PagedDecodeStep(model, 2, heads=8, kv_heads=2, n_pages=4, max_pages=2)
    for a, b in (([0], [0]), ([0, 1], [1, 0]), ([0], [2]), ([-1], [0]), ([0, 0], [1, 1]), ([0], [])):
        with pytest.raises(ValueError, match="PagedDecodeStep"):
            step.fork(a, b)
    model.norms[0]["q_norm"] = torch.ones(32, device="cuda")
    with pytest.raises(ValueError, match="q and k heads"):
        decode.PagedDecodeStep(model, 2, heads=8, kv_heads=2, n_pages=4, max_pages=2)


@pytest.mark.parametrize("t,q_type", [(qvx.F16, qvx.F32), (qvx.F16, qvx.F16), (qvx.BF16, qvx.BF16), (qvx.F32, qvx.F32), (qvx.Q8_0, qvx.F32)])
@pytest.mark.parametrize("window,sinks", [(1 << 20, 0), (50, 3)])
def test_a_prompt_in_pieces_and_samples_of_it(cuda, t, q_type, window, sinks):
    """kv_map, norm_rope_kv and attn_window over a prompt in two pieces; forks of it; tokens of their own by attn_shared (or behind
    the window); then the pages compacted and one more token: each against the formula on what the cache holds."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(4)
    n, hq, hk, d, page, width, n_pages = 6, 8, 2, 64, 16, 20, 70
    kind = {qvx.F32: torch.float32, qvx.F16: torch.float16, qvx.BF16: torch.bfloat16}
    size = qvx.kv_page_bytes(t, hk, page, d)
    raw = torch.zeros((n_pages, 2 * size), dtype=torch.uint8, device="cuda")
    cache = qvx.KvCache.of(raw[:, :size], raw[:, size:], t, page, hk, d)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    free, taken, lens = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32), ints([0, 0]), ints([0] * n)
    extra = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    w = 1 + 0.2 * torch.randn((2, d), generator=g, device="cuda")
    norm = qvx.QkNorm.of(w[0], w[1], 1e-6)
    rope = qvx.Rope.of(10000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device="cuda") * 2 / d))

    def held(b, i):
        """What the cache holds of sequence b: [heads, tokens, d] in 64 bits."""
        m = int(lens[b])
        x = raw[table[b, : -(-m // page)].long(), i * size: (i + 1) * size].cpu()
        if t == qvx.Q8_0:
            at = hk * page * d
            quant = x[:, :at].contiguous().view(torch.int8).double().view(-1, hk, page, d // 32, 32)
            vals = quant * x[:, at: at * 17 // 16].contiguous().view(torch.float16).double().view(-1, hk, page, d // 32, 1)
            vals = vals.reshape(-1, hk, page, d)
        else:
            vals = x[:, : hk * page * d * (4 if t == qvx.F32 else 2)].contiguous().view(kind[t]).double().view(-1, hk, page, d)
        return vals.transpose(1, 2).reshape(-1, hk, d)[:m].transpose(0, 1).numpy()

    def tokens(new):
        """New tokens appended, and their queries as the cache's calls leave them."""
        nonlocal lens, taken
        rows = sum(new)
        lens_, offsets, slots, pos, _, taken_ = qvx.kv_map_t(lens, ints(new), table, page, free, taken, rows + 2)
        lens, taken = lens_, taken_
        assert taken.tolist()[1] == 0
        q, k, v = (torch.randn((rows + 2, h, d), generator=g, device="cuda") for h in (hq, hk, hk))
        q = qvx.norm_rope_kv_t(q, k, v, pos, norm, rope, cache, slots, dtype=kind[q_type])
        return q, offsets, rows

    def check(q, out, new, win, first, groups=(), shared=()):
        got, qh = out.double().cpu().numpy(), q.double().cpu().numpy()
        at = 0
        for b, k in enumerate(new):
            keys, vals = held(b, 0), held(b, 1)
            for i, most in enumerate(shared):  # the shared tokens are the first sequence's, also for one emptied in between
                if groups[i] <= b < groups[i + 1]:
                    most = min(most, int(lens[b]))
                    keys, vals = (np.concatenate([held(groups[i], j)[:, :most], x[:, most:]], 1) for j, x in enumerate((keys, vals)))
            see = seen(int(lens[b]), k, win, first)
            for h in range(hq):
                want, most = attend(qh[at: at + k, h], keys[h // 4], vals[h // 4], see, d ** -0.5)
                vmax = np.abs(vals).max() if vals.size else 0.0
                bar = 2 * U * ((d + 3) * most + int(lens[b]) + 10) * vmax + HALF[q_type] * np.abs(want)
                bar = bar + (HALF[q_type] * vmax if q_type != qvx.F32 else 0)
                assert (np.abs(got[at: at + k, h] - want) <= bar).all(), (b, h)
            at += k

    for new in ([90, 0, 0, 0, 0, 0], [75, 0, 40, 0, 0, 0]):
        q, offsets, rows = tokens(new)
        out = qvx.attn_window_t(q, cache, table, lens, window, sinks, offsets)
        check(q, out, new, window, sinks)
        assert (out[rows:] == 0).all()
    pairs, count = qvx.kv_fork_t(ints([0, 0, 0, 2]), ints([1, 3, 4, 5]), table, page, lens, extra, free, taken)
    qvx.kv_copy_t([cache], pairs, count)
    assert taken.tolist()[1] == 0 and lens.tolist() == [165, 165, 40, 165, 165, 40]
    order = ints([0, 1, 3, 4, 2, 5])  # the samples of a prompt side by side
    table, lens = table[order.long()].contiguous(), lens[order.long()].contiguous()
    for step in range(3):
        q, offsets, rows = tokens([1] * n)
        q = q[:n].contiguous()
        if window > 1000:
            groups, shared = [0, 4, 6], [165 // page * page, 40 // page * page]
            out = qvx.attn_shared_t(q, cache, table, lens, ints(shared), ints(groups))
            check(q, out, [1] * n, window, sinks, groups, shared)
        else:
            out = qvx.attn_window_t(q, cache, table, lens, window, sinks)
            check(q, out, [1] * n, window, sinks)
        if step == 1:
            qvx.kv_free_t(ints([1]), table, lens, extra, free, taken)
            assert lens.tolist()[1] == 0
            pairs, moved = qvx.kv_compact_t(table, extra, free, taken)
            qvx.kv_copy_t([cache], pairs, moved[:1])
            assert moved.tolist()[1] == taken.tolist()[0]


@pytest.mark.parametrize("width,key_length", [(64, None), (64, 64), (512, None), (32, None)])
def test_a_files_norms_of_q_and_k(cuda, tmp_path, width, key_length):
    """Norms of a head's width are the step's own; others stay among what it does not compute, and are refused."""
    from gguf_build import GgufBuilder
    torch = cuda
    rng = np.random.default_rng(9)
    d, heads, kv_heads, hd, ffn = 512, 8, 2, 64, 512
    b = (GgufBuilder(3).str("general.architecture", "llama").u32("general.alignment", 32).u32("llama.block_count", 1)
         .u32("llama.embedding_length", d).u32("llama.feed_forward_length", ffn).u32("llama.attention.head_count", heads)
         .u32("llama.attention.head_count_kv", kv_heads).f32("llama.rope.freq_base", 10000.0))
    if key_length:
        b.u32("llama.attention.key_length", key_length)
    weights = [(1.0 + 0.3 * rng.standard_normal(width)).astype(np.float32) for _ in range(2)]
    tensors = [(n, [d], (1.0 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for n in
               ("blk.0.attn_norm.weight", "blk.0.ffn_norm.weight", "output_norm.weight")]
    tensors += [(f"blk.0.attn_{n}_norm.weight", [width], w) for n, w in zip("qk", weights)]
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
    model = decode.Model.from_gguf(path).fused_ops()
    make = lambda: decode.PagedDecodeStep(model, 2, heads, kv_heads, n_pages=8, max_pages=3, page_size=4,  # noqa: E731
                                          rotation=decode.Rotation())
    if width != hd:
        assert model.left_out == ["blk.0.attn_q_norm.weight", "blk.0.attn_k_norm.weight"]
        with pytest.raises(ValueError, match="attn_q_norm"):
            make()
        return
    assert model.left_out == []
    for k, w in zip(("q_norm", "k_norm"), weights):
        assert np.array_equal(model.norms[0][k].cpu().numpy(), w)
    step = make()
    _both(torch, step, HostShared(torch, step, torch.float16), 5)
