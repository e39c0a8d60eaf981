"""The shared cache's calls at the ends of their ranges: byte offsets past 32 bits, lengths next to 2^31, the most forks of a call,
batches past a wave, streams beside the current one and graphs that run at once."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from test_gpu_attention import U, Cache
from test_gpu_window import HALF, attend, check

pytestmark = pytest.mark.gpu


def _ints(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("t", (qvx.BF16, qvx.Q8_0))
def test_pages_past_four_gib(cuda, t):
    """Append, copies and attention on pages whose byte offsets pass 32 bits, against the same on pages at the start: equal bits."""
    torch = cuda
    page, hk, d, n, m = 128, 8, 128, 1000, 3
    size = qvx.kv_page_bytes(t, hk, page, d)
    n_pages = (5 << 30) // size
    ids = _ints(torch, [0, n_pages - 1, n_pages - 5, 3, n_pages - 9, n_pages // 2, n_pages - 2, n_pages - 3, n_pages - 20, n_pages - 21])
    here = _ints(torch, [8, 1, 2, 3, 4, 5, 6, 7, 9, 10])
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    q, kk, vv = (torch.randn((n, h, d), device="cuda") for h in (16, hk, hk))
    rope = qvx.Rope.of(10000.0 ** -(torch.arange(64, dtype=torch.float64, device="cuda") / 64))
    norm = qvx.QkNorm.of(torch.rand(d, device="cuda"), torch.rand(d, device="cuda"))
    outs = []
    for pages, p in ((n_pages, ids), (11, here)):
        k, v = (torch.zeros((pages, size), dtype=torch.uint8, device="cuda") for _ in range(2))
        c = qvx.KvCache.of(k, v, t, page, hk, d)
        turned = qvx.norm_rope_kv_t(q, kk, vv, at, norm, rope, c, p[(at // page).long()] * page + at % page)
        qvx.kv_copy_t([c], torch.stack([p[[7, 7]], p[[8, 9]]], 1).contiguous())
        table = p[None, :8].repeat(m, 1)
        table[1, 7], table[2, 7] = p[8], p[9]
        lens = _ints(torch, [n, n - 3, n - 40])
        wide = torch.cat([table, torch.full((m, 400), -1, dtype=torch.int32, device="cuda")], 1)
        last = turned[-m:].contiguous()
        outs.append([turned, qvx.attn_window_t(turned, c, table[:1], lens[:1], 1 << 30),
                     qvx.attn_window_t(turned, c, table[:1], lens[:1], 300, 5), qvx.attn_window_t(last, c, table, lens, 500, 9),
                     qvx.attn_shared_t(last, c, table, lens, _ints(torch, [7 * page])),
                     qvx.attn_shared_t(last, c, wide, lens, _ints(torch, [7 * page])), k[p.long()], v[p.long()]])
        if t == qvx.BF16:
            outs[-1].append(qvx.attn_window_t(turned.bfloat16(), c, table[:1], lens[:1], 300, 5))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("t", (qvx.F16, qvx.F32))
@pytest.mark.parametrize("width", [127, 128])
@pytest.mark.parametrize("new", [1, 60])
def test_lengths_next_to_2_31(cuda, t, width, new):
    """All columns are one page, so the keys repeat; a window and first tokens of them."""
    torch = cuda
    page, d, window, sinks = (1 << 24) - 1, 8, 100, 20
    size = qvx.kv_page_bytes(t, 1, page, d)
    k, v = (torch.empty((1, size), dtype=torch.uint8, device="cuda") for _ in range(2))
    kind = torch.float16 if t == qvx.F16 else torch.float32
    planes = [x.view(kind).view(-1)[: page * d].view(page, d) for x in (k, v)]
    for x in planes:
        x.normal_()
    c = qvx.KvCache.of(k, v, t, page, 1, d)
    n = width * page - 3
    q = torch.randn((new, 1, d), device="cuda")
    got = qvx.attn_window_t(q, c, torch.zeros((1, width), dtype=torch.int32, device="cuda"), _ints(torch, [n]), window, sinks)
    keys = np.concatenate([np.arange(sinks), np.arange(n - new - window + 1, n)])
    kh, vh = (x[torch.from_numpy(keys % page).cuda()].double().cpu().numpy() for x in planes)
    p = n - new + np.arange(new)[:, None]
    see = (keys[None] <= p) & ((keys[None] > p - window) | (keys[None] < sinks))
    want, most = attend(q[:, 0].double().cpu().numpy(), kh, vh, see, d ** -0.5)
    err = np.abs(got[:, 0].double().cpu().numpy() - want).max()
    # weights of many fp32 rows on 16-bit keys go in two fp16 parts, 2^-22 of each: with the rest as in test_gpu_window.py
    assert err <= (2 * U * ((d + 3) * most + len(keys) + 10) + 2.0 ** -22) * np.abs(vh).max()


def test_the_most_forks(cuda):
    """16384 forks of two rows in one call: every fork shares a page and takes one."""
    torch = cuda
    n, page = 16384, 4
    table = torch.full((n + 2, 2), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(n + 100, device="cuda").to(torch.int32)
    table[:2] = free[:4].view(2, 2)
    lens = torch.zeros(n + 2, dtype=torch.int32, device="cuda")
    lens[0], lens[1] = 6, 8  # the second's last page is full
    extra, taken = torch.zeros(n + 100, dtype=torch.int32, device="cuda"), _ints(torch, [4, 0])
    source = (torch.arange(n, device="cuda") % 3 == 2).to(torch.int32)
    to = 2 + torch.randperm(n, device="cuda").to(torch.int32)
    fresh = free[4:]
    pairs, count = qvx.kv_fork_t(source, to, table, page, lens, extra, free, taken)
    part = (source == 0).nonzero()[:, 0]
    k = part.shape[0]
    assert taken.tolist() == [4 + k, 0] and count.tolist() == [k]
    assert torch.equal(pairs[:k, 0], table[0, 1].expand(k)) and torch.equal(pairs[:k, 1], fresh[:k])
    assert torch.equal(table[to.long()[part], 1], fresh[:k]) and bool((table[to.long()[part], 0] == table[0, 0]).all())
    assert bool((table[to.long()[source == 1]] == table[1]).all()) and torch.equal(lens[to.long()], lens[source.long()])
    held = torch.zeros_like(extra)
    held[table[0, 0].long()], held[table[1].long()] = k, n - k
    assert torch.equal(extra, held)
    qvx.kv_free_t(to, table, lens, extra, free, taken)
    assert taken.tolist() == [4, 0] and not bool(extra.any()) and bool((table[2:] == -1).all())
    assert torch.equal(free[4: 4 + k], fresh[:k].sort().values)


@pytest.mark.parametrize("t,q_type", [(qvx.F16, qvx.F32), (qvx.BF16, qvx.BF16)])
@pytest.mark.parametrize("n", [70, 300])
def test_pieces_of_many_sequences(cuda, t, q_type, n):
    """More sequences than a wave's lanes, and than a workgroup's threads, with more than 48 rows each in the mean."""
    r = np.random.default_rng(n)
    new = [int(x) for x in r.integers(0, 60, n)]
    new[3], new[n - 1] = 0, 200
    lens = [k + int(r.integers(0, 90)) for k in new]
    check(cuda, Cache(cuda, t, lens, 16, 1, 32, seed=n), 4, new, 40, 5, q_type)


@pytest.mark.parametrize("t", (qvx.F16, qvx.BF16))
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
def test_few_new_tokens_over_a_long_past(cuda, t, d):
    """17 to 64 rows a sequence whose keys are split over workgroups and joined, a sequence without new tokens between."""
    for new, window, sinks in (([5, 0, 5], 1 << 20, 0), ([12, 1, 16], 1 << 20, 0), ([16, 0, 9], 700, 33)):
        for q_type in (t, qvx.F32):
            check(cuda, Cache(cuda, t, (5000, 40, 2999), 24, 1, d, seed=d), 5, new, window, sinks, q_type)


@pytest.mark.parametrize("wide", [False, True])
def test_two_graphs_at_once_on_streams_of_their_own(cuda, wide):
    """Each with its own workspace: replays beside each other leave what the calls one by one do."""
    torch = cuda
    lens = [900, 870, 1001, 960]
    c = Cache(torch, qvx.F16, lens, 16, 2, 64, seed=3)
    table = c.dev_table.clone()
    table[:, :50] = table[0, :50]
    if wide:
        table = torch.cat([table, torch.full((4, 1 << 16), -1, dtype=torch.int32, device="cuda")], 1)
    shared, width = _ints(torch, [800]), table.shape[1]
    calls = []
    for i in range(2):
        q = torch.randn((4, 8, 64), device="cuda")
        prompt = torch.randn((80, 8, 64), device="cuda").half()
        outs = [torch.zeros_like(q), torch.zeros_like(prompt)]
        ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in
              (qvx.attn_shared_ws(c.desc, q.dtype, 8, 4, width, 1), qvx.attn_window_ws(c.desc, prompt.dtype, 8, 80, 4, width, 300, 4))]

        def run(q=q, prompt=prompt, outs=outs, ws=ws):
            qvx.attn_shared_t(q, c.desc, table, c.dev_lens, shared, out=outs[0], ws=ws[0])
            qvx.attn_window_t(prompt, c.desc, table, c.dev_lens, 300, 4, out=outs[1], ws=ws[1])
        run()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            run()
        calls.append((q, prompt, outs, run, graph, stream))
    for turn in range(4):
        for q, prompt, outs, _, _, _ in calls:
            q.normal_()
            prompt.normal_()
            for x in outs:
                x.fill_(3.0)
        torch.cuda.synchronize()
        for _, _, _, _, graph, stream in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, outs, run, _, _ in calls:
            got = [x.clone() for x in outs]
            run()
            assert all(torch.equal(a, b) for a, b in zip(got, outs))


@pytest.mark.parametrize("t,q_type", [(qvx.F16, qvx.F16), (qvx.BF16, qvx.F32), (qvx.Q8_0, qvx.F32)])
@pytest.mark.parametrize("hq,hk", [(150, 1), (260, 2)])
def test_groups_of_more_heads_than_a_row_tile(cuda, t, q_type, hq, hk):
    """A query's rows in several row tiles, alone and behind a shared prefix, which the second width reads apart."""
    torch = cuda
    check(cuda, Cache(cuda, t, (70, 333, 20, 1), 16, hk, 32, seed=hq), hq, [1, 7, 3, 1], 50, 3, q_type)
    lens = (300, 291, 400, 290)
    c = Cache(cuda, t, lens, 16, hk, 32, seed=hq + 1)
    c.table[:, :18] = c.table[0, :18]
    q = torch.randn((4, hq, 32), device="cuda").to({qvx.F32: torch.float32, qvx.F16: torch.float16}[q_type])
    for more in (0, 1 << 17):
        table = torch.cat([torch.from_numpy(c.table).cuda(), torch.full((4, more), -1, dtype=torch.int32, device="cuda")], 1)
        got = qvx.attn_shared_t(q, c.desc, table, c.dev_lens, _ints(torch, [288])).double().cpu().numpy()
        for b, n in enumerate(lens):
            k, v = (np.concatenate([c.rows(0, i)[:, :288], c.rows(b, i)[:, 288:]], 1) for i in range(2))
            for h in range(hq):
                g = h // (hq // hk)
                want, most = attend(q[b, h: h + 1].double().cpu().numpy(), k[g], v[g], np.ones((1, n), bool), 32 ** -0.5)
                bar = 2 * U * ((32 + 3) * most + n + 10) * np.abs(v).max() + HALF[q_type] * np.abs(want)
                # rounded weights, of more than 48 rows a group: half a step of each, or what two bf16 parts leave
                bar = bar + (HALF[q_type] if q_type == t else 2.0 ** -18 if t == qvx.BF16 else 0.0) * np.abs(v).max()
                assert (np.abs(got[b, h] - want[0]) <= bar).all()
