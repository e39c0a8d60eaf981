"""Performance cases of the attention operators around the quantized products: page tables from request
lengths (kv_map), rotary positions with the append to the paged cache (rope_kv), attention of one new token
over the paged cache (attn_paged) and cross attention to an encoder's states (attn_cross).

`run` computes them in elementary torch operations, or with the framework's kernels where `own` is set.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": 0, "f16": 1, "q8_0": 8, "bf16": 30}  # ggml type ids
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the bookkeeping of one decode step of 256 running requests, one new token each
        dict(name="map_decode_256", op="map", n=256, held=8192, new=1, page=16),
        # admission of a large batch of prompts beside running requests (ragged, 148 tokens in the mean)
        dict(name="map_prompts_1024", op="map", n=1024, held=2048, new=1024, page=64),
        # the one token of a single user's decode step at the 8B decoder's heads
        dict(name="rope_token", op="rope", n=1, q_heads=32, kv_heads=8, d=128, type="f16", axes=1, page=16),
        # a long prompt with images: positions in time, height and width
        dict(name="rope_prompt_8192", op="rope", n=8192, q_heads=32, kv_heads=8, d=128, type="bf16", axes=3, page=32),
        # the first tokens of a chat: nothing to split, latency alone
        dict(name="paged_short", op="paged", n=1, longest=33, mixed=False, q_heads=32, kv_heads=8, d=128, type="f16",
             page=16),
        # a server's running batch: lengths from a few tokens to 8192
        dict(name="paged_mixed_48", op="paged", n=48, longest=8192, mixed=True, q_heads=32, kv_heads=8, d=128,
             type="f16", page=16),
        # one user with a very long document: a single sequence has to fill the card
        dict(name="paged_long_131071", op="paged", n=1, longest=131071, mixed=False, q_heads=32, kv_heads=8, d=128,
             type="bf16", page=64),
        # a full batch over the quantised cache
        dict(name="paged_q8_64", op="paged", n=64, longest=4096, mixed=False, q_heads=32, kv_heads=8, d=128,
             type="q8_0", page=32),
        # a head for every query head and an unrounded cache, odd lengths
        dict(name="paged_f32_mha", op="paged", n=20, longest=1777, mixed=True, q_heads=16, kv_heads=16, d=64,
             type="f32", page=24),
        # a speech decoder's step: 5 candidates, one token each, on 1500 frames
        dict(name="cross_step_1500", op="cross", n=5, queries=1, states=1500, mixed=False, q_heads=20, kv_heads=20,
             d=64, type="f16", q_type="f32"),
        # an image model's queries on 77 text states, guided and unguided, 40 values a head
        dict(name="cross_image_77", op="cross", n=2, queries=4096, states=77, mixed=False, q_heads=8, kv_heads=8, d=40,
             type="f16", q_type="f16"),
        # transcripts of several windows at once: ragged prompts on ragged audio
        dict(name="cross_prompts_1500", op="cross", n=16, queries=448, states=1500, mixed=True, q_heads=20, kv_heads=20,
             d=64, type="bf16", q_type="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["map", "rope", "paged", "paged", "cross", "cross"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "map":
        n = _log(rng, 1, 1024)
        return dict(op=op, n=n, held=_log(rng, 1, 8192), new=rng.choice([1, _log(rng, 1, 1024)]), page=page)
    if op == "rope":
        kv, d = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 80, 96, 128])
        return dict(op=op, n=_log(rng, 1, 6000), q_heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, d=d,
                    type=rng.choice(["f32", "f16", "bf16"]), axes=rng.choice([1, 3]), page=page)
    if op == "paged":
        kv, kind = rng.choice([1, 2, 4, 8]), rng.choice(["f32", "f16", "bf16", "q8_0"])
        d = rng.choice([64, 96, 128, 256] if kind == "q8_0" else [40, 64, 80, 96, 128, 256])
        most = int(2.5e8) // (kv * _item(kind, d))  # tokens in all
        longest = min(_log(rng, 1, 65536), most)
        n = max(1, min(_log(rng, 1, 128), most // longest))
        return dict(op=op, n=n, longest=longest, mixed=rng.random() < 0.5, q_heads=kv * rng.choice([1, 2, 4, 7, 8]),
                    kv_heads=kv, d=d, type=kind, page=page)
    kv, d = rng.choice([4, 8, 12, 20]), rng.choice([40, 64, 80, 128, 160])
    kind = rng.choice(["f16", "bf16"])
    states, queries = _log(rng, 16, 4096), rng.choice([1, _log(rng, 2, 4096)])
    n = max(1, min(_log(rng, 1, 16), int(2e9) // (queries * states * kv * d)))
    return dict(op=op, n=n, queries=queries, states=states, mixed=rng.random() < 0.5, q_heads=kv * rng.choice([1, 2]),
                kv_heads=kv, d=d, type=kind, q_type=rng.choice([kind, "f32"]) if queries == 1 else kind)


# ---- sizes that a case stands for -----------------------------------------------------------------------

def _spread(n, longest, mixed):
    """n lengths up to `longest`: all of them that, or from short to long with the logarithm evenly spread."""
    if not mixed:
        return [longest] * n
    return [max(1, round(longest ** ((i + 1) / n))) for i in range(n)]


def _cross_lengths(c):
    """Queries and states of each sequence: all as many, or from a quarter of the most to the most, against each other."""
    part = [(i + 1 + c["n"] / 3) / (4 * c["n"] / 3) if c["mixed"] else 1.0 for i in range(c["n"])]
    nq, ns = ([max(1, round(most * p)) for p in part] for most in (c["queries"], c["states"]))
    return nq, ns[::-1]


def _map_lengths(c):
    return _spread(c["n"], c["held"], True), _spread(c["n"], c["new"], True)


def _ceil(a, b):
    return -(-a // b)


def _item(kind, d):
    """Bytes of the d values of one token and head."""
    return {"f32": 4 * d, "f16": 2 * d, "bf16": 2 * d, "q8_0": d + d // 16}[kind]


def work(case):
    c = case
    if c["op"] == "map":
        held, new = _map_lengths(c)
        touched = sum(_ceil(h + k, c["page"]) - h // c["page"] for h, k in zip(held, new))
        fresh = sum(_ceil(h + k, c["page"]) - _ceil(h, c["page"]) for h, k in zip(held, new))
        return {"bytes": 16 * c["n"] + 4 * touched + 4 * fresh + 12 * sum(new), "flops": 0}
    if c["op"] == "rope":
        heads = c["q_heads"] + c["kv_heads"]
        per = 4 * c["d"] * (2 * c["q_heads"] + 2 * c["kv_heads"]) + 2 * c["kv_heads"] * _item(c["type"], c["d"])
        return {"bytes": c["n"] * (per + 4 * c["axes"] + 4), "flops": c["n"] * heads * c["d"] * 3}
    if c["op"] == "paged":
        lens = _spread(c["n"], c["longest"], c["mixed"])
        pages = sum(_ceil(n, c["page"]) for n in lens)
        return {"bytes": 2 * sum(lens) * c["kv_heads"] * _item(c["type"], c["d"]) + 4 * pages
                + 8 * c["n"] * c["q_heads"] * c["d"], "flops": 4 * sum(lens) * c["q_heads"] * c["d"]}
    nq, ns = _cross_lengths(c)
    size = 2 * sum(nq) * c["q_heads"] * _item(c["q_type"], c["d"]) + 2 * sum(ns) * c["kv_heads"] * _item(c["type"], c["d"])
    return {"bytes": size, "flops": 4 * c["q_heads"] * c["d"] * sum(a * b for a, b in zip(nq, ns))}


# ---- what a program has in hand before the call -----------------------------------------------------------

class _State:
    pass


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEVICE)


def _randn(shape, g, kind="f32", mul=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * mul).to(TORCH[kind])


def _tables(lens, page, width, g):
    """A table whose rows hold each sequence's pages in random order (-1 behind them), and how many pages there are."""
    used = [_ceil(n, page) for n in lens]
    total = sum(used)
    pages = torch.randperm(total + 3, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEVICE)
    col = torch.arange(width, device=DEVICE)
    start = _ints([0] + list(np.cumsum(used))[:-1], torch.int64)
    mine = col[None, :] < _ints(used)[:, None]
    table[mine] = pages[(start[:, None] + col[None, :])[mine]]
    return table, total + 3, pages[total:]


def _cache(c, n_pages, g):
    """The pages of a cache [n_pages, page bytes], K and V: each heads x tokens x values; Q8_0 with the quants of a
    page first and the fp16 scales of their blocks of 32 behind them."""
    values = c["kv_heads"] * c["page"] * c["d"]
    if c["type"] != "q8_0":
        return [_randn((n_pages, values), g, c["type"]) for _ in range(2)]
    out = []
    for _ in range(2):
        quants = torch.randint(-127, 128, (n_pages, values), generator=g, device=DEVICE, dtype=torch.int8)
        scales = (torch.rand((n_pages, values // 32), generator=g, device=DEVICE) * 0.01 + 0.01).to(torch.float16)
        out.append(torch.cat([quants.view(torch.uint8), scales.view(torch.uint8)], 1))
    return out


def _prepare_map(s, c, g):
    held, new = _map_lengths(c)
    order = torch.randperm(c["n"], generator=g, device=DEVICE).tolist()
    held, new = [held[i] for i in order], [new[i] for i in reversed(order)]
    s.width = _ceil(c["held"] + c["new"], c["page"]) + 2  # the longest request that the program admits
    s.table, used, _ = _tables(held, c["page"], s.width, g)
    fresh = sum(_ceil(h + k, c["page"]) - _ceil(h, c["page"]) for h, k in zip(held, new))
    s.free = used + torch.randperm(fresh + 12, generator=g, device=DEVICE).to(torch.int32)
    s.taken = _ints([7, 0])  # pages of the list that earlier steps took
    s.held, s.new, s.rows = _ints(held), _ints(new), sum(new) + 5  # a padded batch


def _prepare_rope(s, c, g):
    n, hq, hk, d = c["n"], c["q_heads"], c["kv_heads"], c["d"]
    s.qk = _randn((n, (hq + hk) * d), g)  # q and k as one stacked product leaves them
    s.v = _randn((n, hk * d), g)
    pages = _ceil(n, c["page"]) + 3
    s.k_cache, s.v_cache = _cache(c, pages, g)
    s.slots = torch.randperm(pages * c["page"], generator=g, device=DEVICE)[:n].to(torch.int32)
    s.pos = torch.randint(0, 131072, (c["axes"], n), generator=g, device=DEVICE, dtype=torch.int32)
    half = d // 2
    s.freq = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
    share = half // 4  # a quarter of the pairs in time, three eighths each in height and width
    axis = [0] * half if c["axes"] == 1 else [0] * share + [1 + 2 * (i - share) // (half - share) for i in range(share, half)]
    s.axis = _ints(axis, torch.uint8)


def _prepare_paged(s, c, g):
    lens = _spread(c["n"], c["longest"], c["mixed"])
    order = torch.randperm(c["n"], generator=g, device=DEVICE).tolist()
    lens = [lens[i] for i in order]
    s.width = max(_ceil(n, c["page"]) for n in lens) + 1
    s.table, pages, _ = _tables(lens, c["page"], s.width, g)
    s.k_cache, s.v_cache = _cache(c, pages, g)
    s.lens = _ints(lens)
    s.q = _randn((c["n"], c["q_heads"], c["d"]), g, mul=1.5)


def _prepare_cross(s, c, g):
    nq, ns = _cross_lengths(c)
    s.most = max(nq)
    s.offsets = _ints([0] + list(np.cumsum(nq)))
    s.lens = _ints(ns)
    s.q = _randn((sum(nq), c["q_heads"], c["d"]), g, c["q_type"], 1.5)
    s.kv = _randn((c["n"], max(ns), 2, c["kv_heads"], c["d"]), g, c["type"])  # as one stacked projection leaves them


def _own_handles(s, c):
    """What a program keeps beside its tensors: outputs, cache and state descriptions, workspaces."""
    import qorvix_amd as qvx
    s.qvx = qvx
    if c["op"] == "map":
        s.lens, s.offsets, s.slots, s.pos, s.seq, s.taken_out = (
            torch.empty(n, dtype=torch.int32, device=DEVICE) for n in (c["n"], c["n"] + 1, s.rows, s.rows, s.rows, 2))
    if c["op"] in ("rope", "paged"):
        s.cache = qvx.KvCache.of(s.k_cache, s.v_cache, TYPES[c["type"]], c["page"], c["kv_heads"], c["d"])
    if c["op"] == "rope":
        s.q_out = torch.empty((c["n"], c["q_heads"] * c["d"]), device=DEVICE)
        s.rope = qvx.Rope.of(s.freq, s.axis, c["axes"], qvx.ROPE_HALVES)
    if c["op"] == "paged":
        s.out = torch.empty((c["n"], c["q_heads"], c["d"]), device=DEVICE)
        s.ws = torch.empty(qvx.attn_paged_ws(s.cache, c["q_heads"], c["n"], s.width), dtype=torch.uint8, device=DEVICE)
    if c["op"] == "cross":
        s.out = torch.empty_like(s.q)
        s.states = qvx.KvStates.of(s.kv[:, :, 0], s.kv[:, :, 1])
        s.ws = torch.empty(qvx.attn_cross_ws(s.states, s.q.dtype, c["q_heads"], s.q.shape[0], c["n"]),
                           dtype=torch.uint8, device=DEVICE)


def prepare(case, seed):
    s = _State()
    s.case = case
    g = _generator(seed)
    {"map": _prepare_map, "rope": _prepare_rope, "paged": _prepare_paged, "cross": _prepare_cross}[case["op"]](s, case, g)
    if own:
        _own_handles(s, case)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------

def _plain_map(s):
    page, rows = s.case["page"], s.rows
    held, new = s.held.long(), s.new.long()
    ends = torch.cumsum(new, 0)
    first, last = (held + page - 1) // page, (held + new + page - 1) // page
    before = torch.cumsum(last - first, 0) - (last - first)
    col = torch.arange(s.width, device=DEVICE)
    fresh = (col >= first[:, None]) & (col < last[:, None])
    at = torch.where(fresh, s.taken[0].long() + before[:, None] + col - first[:, None], 0)
    table = torch.where(fresh, s.free[at], s.table)
    t = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(ends, t, right=True)
    live = t < ends[-1]
    b = torch.where(live, seq, 0)
    pos = torch.where(live, held[b] + t - (ends[b] - new[b]), 0)
    slots = torch.where(live, table[b, pos // page].long() * page + pos % page, -1)
    taken = torch.stack([s.taken[0].long() + (last - first).sum(), torch.zeros_like(ends[-1])])
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    i32 = torch.int32
    return [table, (held + new).to(i32), offsets.to(i32), slots.to(i32), pos.to(i32),
            torch.where(live, seq, -1).to(i32), taken.to(i32)]


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_rope(s):
    c = s.case
    n, hq, hk, d, page = c["n"], c["q_heads"], c["kv_heads"], c["d"], c["page"]
    angle = s.pos[s.axis.long()].double().t() * s.freq  # [tokens, pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q, k = s.qk[:, :hq * d].view(n, hq, d), s.qk[:, hq * d:].view(n, hk, d)
    slots = s.slots.long()
    for cache, x in ((s.k_cache, _rotate(k, cos, sin)), (s.v_cache, s.v.view(n, hk, d))):
        cache.view(-1, hk, page, d)[slots // page, :, slots % page] = x.to(cache.dtype)
    return [_rotate(q, cos, sin).reshape(n, hq * d), s.k_cache, s.v_cache]


def _values(pages, c):
    """A cache's values [pages, heads, page, d] in 32 bits."""
    shape = (pages.shape[0], c["kv_heads"], c["page"], c["d"])
    if c["type"] != "q8_0":
        return pages.view(shape).float()
    split = c["kv_heads"] * c["page"] * c["d"]
    quants = pages[:, :split].view(torch.int8).float().view(*shape[:3], c["d"] // 32, 32)
    return (quants * pages[:, split:].view(torch.float16).float().view(*shape[:3], -1, 1)).view(shape)


def _softmax_product(q, k, v, lens, scale):
    """q [n, heads, rows, d] on k, v [n, heads, keys, d] of which the first lens[n] count."""
    logits = torch.matmul(q, k.transpose(-1, -2)) * scale
    live = torch.arange(k.shape[2], device=DEVICE) < lens[:, None]
    logits = logits.masked_fill(~live[:, None, None], -math.inf)
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return torch.matmul(e, v) / e.sum(-1, keepdim=True)


def _plain_paged(s):
    c = s.case
    n, hq, hk, d = c["n"], c["q_heads"], c["kv_heads"], c["d"]
    pages = s.table.clamp(min=0).long()
    if c["type"] == "q8_0":  # the pages in use, decoded once
        k, v = (_values(cache, c)[pages] for cache in (s.k_cache, s.v_cache))
    else:
        k, v = (cache.view(-1, hk, c["page"], d)[pages].float() for cache in (s.k_cache, s.v_cache))
    k, v = (x.transpose(1, 2).reshape(n, hk, -1, d) for x in (k, v))
    o = _softmax_product(s.q.view(n, hk, hq // hk, d), k, v, s.lens, 1.0 / math.sqrt(d))
    return o.reshape(n, hq, d)


def _plain_cross(s):
    c = s.case
    n, hq, hk, d = c["n"], c["q_heads"], c["kv_heads"], c["d"]
    group = hq // hk
    k, v = (s.kv[:, :, i].transpose(1, 2).float() for i in range(2))
    row = s.offsets[:-1, None].long() + torch.arange(s.most, device=DEVICE)  # a padded batch of the queries
    q = s.q[row.clamp(max=s.q.shape[0] - 1)].float()  # [n, most, hq, d]
    q = q.view(n, s.most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * s.most, d)
    o = _softmax_product(q, k, v, s.lens, 1.0 / math.sqrt(d))
    o = o.view(n, hk, group, s.most, d).permute(0, 3, 1, 2, 4).reshape(n, s.most, hq, d)
    t = torch.arange(s.q.shape[0], device=DEVICE)
    seq = (t[:, None] >= s.offsets[None, 1:]).sum(1)
    return o[seq, t - s.offsets[seq].long()].to(s.q.dtype)


# ---- the framework's kernels ---------------------------------------------------------------------------------

def _own(s):
    qvx, c = s.qvx, s.case
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "map":
        rc = qvx.kv_map(s.held.data_ptr(), s.new.data_ptr(), c["n"], s.table.data_ptr(), s.width, c["page"],
                        s.free.data_ptr(), s.free.shape[0], s.taken.data_ptr(), s.taken_out.data_ptr(),
                        s.lens.data_ptr(), s.offsets.data_ptr(), s.slots.data_ptr(), s.pos.data_ptr(),
                        s.seq.data_ptr(), s.rows, stream)
        out = [s.table, s.lens, s.offsets, s.slots, s.pos, s.seq, s.taken_out]
    elif c["op"] == "rope":
        hq, hk, d = c["q_heads"], c["kv_heads"], c["d"]
        qk = s.qk.data_ptr()
        rc = qvx.rope_kv(s.q_out.data_ptr(), hq * d, qk, (hq + hk) * d, hq, qk + 4 * hq * d, (hq + hk) * d,
                         s.v.data_ptr(), hk * d, c["n"], d, s.rope, s.pos.data_ptr(), c["n"], s.cache,
                         s.slots.data_ptr(), stream)
        out = [s.q_out, s.k_cache, s.v_cache]
    elif c["op"] == "paged":
        rc = qvx.attn_paged(s.out.data_ptr(), c["q_heads"] * c["d"], s.q.data_ptr(), c["q_heads"] * c["d"], c["q_heads"],
                            s.cache, s.table.data_ptr(), s.width, s.lens.data_ptr(), c["n"], 1.0 / math.sqrt(c["d"]),
                            s.ws.data_ptr(), s.ws.numel(), stream)
        out = s.out
    else:
        rc = qvx.attn_cross(s.out.data_ptr(), c["q_heads"] * c["d"], s.q.data_ptr(), c["q_heads"] * c["d"],
                            TYPES[c["q_type"]], c["q_heads"], s.offsets.data_ptr(), s.q.shape[0], s.states,
                            s.lens.data_ptr(), c["n"], 1.0 / math.sqrt(c["d"]), s.ws.data_ptr(), s.ws.numel(), stream)
        out = s.out
    if rc != qvx.OK:
        raise qvx.QvxError(rc, c["op"])
    return out


def run(state):
    if own:
        return _own(state)
    return {"map": _plain_map, "rope": _plain_rope, "paged": _plain_paged, "cross": _plain_cross}[state.case["op"]](state)


# ---- the same results in 64 bits -------------------------------------------------------------------------------

def _attend(q, k, v, scale):
    """One sequence and group of heads: q [rows, d], k and v [keys, d], in 64 bits."""
    w = torch.softmax((q @ k.t()) * scale, dim=-1)
    return w @ v


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence; the page tables are whole numbers and have none."""
    c = case
    if c["op"] == "map":
        return None
    s = _State()
    s.case = c
    g = _generator(seed)
    {"rope": _prepare_rope, "paged": _prepare_paged, "cross": _prepare_cross}[c["op"]](s, c, g)
    hq, hk, d = c["q_heads"], c["kv_heads"], c["d"]
    group = hq // hk
    if c["op"] == "rope":
        where = s.pos.double()[s.axis.long(), :]  # [pairs, tokens]
        turn = torch.polar(torch.ones_like(where), where * s.freq[:, None]).t()[:, None, :]

        def turned(x):
            z = torch.complex(x[..., : d // 2].double(), x[..., d // 2:].double()) * turn
            return torch.cat([z.real, z.imag], -1)

        x = s.qk.view(c["n"], hq + hk, d)
        out = [turned(x[:, :hq]).reshape(c["n"], hq * d)]
        page, off = torch.div(s.slots.long(), c["page"], rounding_mode="floor"), s.slots.long() % c["page"]
        for cache, new in ((s.k_cache, turned(x[:, hq:])), (s.v_cache, s.v.view(c["n"], hk, d).double())):
            full = cache.double().view(-1, hk, c["page"], d).transpose(1, 2).contiguous()
            full[page, off] = new
            out.append(full.transpose(1, 2).reshape(cache.shape))
        return out
    scale = 1.0 / math.sqrt(d)
    if c["op"] == "paged":
        out = torch.zeros((c["n"], hq, d), dtype=torch.float64, device=DEVICE)
        for i, length in enumerate(s.lens.tolist()):
            pages = s.table[i, : _ceil(length, c["page"])].long()
            rows = []
            for cache in (s.k_cache, s.v_cache):
                got = cache[pages]
                if c["type"] == "q8_0":
                    at = hk * c["page"] * d
                    steps = got[:, at:].contiguous().view(torch.float16).double()
                    got = got[:, :at].contiguous().view(torch.int8).double() * steps.repeat_interleave(32, dim=1)
                rows.append(got.double().view(-1, hk, c["page"], d).transpose(1, 2).reshape(-1, hk, d)[:length])
            for h in range(hk):
                mine = slice(h * group, (h + 1) * group)
                out[i, mine] = _attend(s.q[i, mine].double(), rows[0][:, h], rows[1][:, h], scale)
        return out
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    edges = s.offsets.tolist()
    for i, length in enumerate(s.lens.tolist()):
        k, v = (s.kv[i, :length, j].double() for j in range(2))
        for h in range(hq):
            rows = slice(edges[i], edges[i + 1])
            out[rows, h] = _attend(s.q[rows, h].double(), k[:, h // group], v[:, h // group], scale)
    return out
