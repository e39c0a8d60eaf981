"""Performance cases of the operators of a cache that requests share: norms of q and k with the rotary positions and
the append (norm_rope_kv), attention with a window and a few first tokens (attn_window), attention of a batch that
shares long prefixes (attn_shared), and the pages' own upkeep: forks, copies, releases and compaction (kv_fork,
kv_copy, kv_free, kv_compact).

`run` computes them in elementary torch operations, or with the framework's kernels where `own` is set.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": 0, "f16": 1, "q8_0": 8, "bf16": 30}  # ggml type ids
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # the one token of a single user's decode step at the 8B decoder's heads
        dict(name="turn_token", op="turn", n=1, q_heads=32, kv_heads=8, d=128, rot=128, pairs=False, each=False, type="f16",
             q_type="f32", page=16),
        # a server's decode step, odd in number: half of each head turned, neighbours paired, weights of their own for each head
        dict(name="turn_batch_301", op="turn", n=301, q_heads=16, kv_heads=4, d=96, rot=48, pairs=True, each=True, type="f32",
             q_type="f32", page=24),
        # a long prompt, its queries rounded for the 16-bit matrix cores
        dict(name="turn_prompt_8192", op="turn", n=8192, q_heads=32, kv_heads=8, d=128, rot=128, pairs=False, each=False,
             type="bf16", q_type="bf16", page=32),
        # a server's running batch: lengths from a few tokens to 32768, pages behind the window given back
        dict(name="window_step_48", op="window", n=48, longest=32768, mixed=True, new=1, window=4096, sinks=4, freed=True,
             q_heads=32, kv_heads=8, d=128, type="f16", q_type="f32", page=16),
        # a window over the quantised cache, with a system prompt that stays visible
        dict(name="window_q8_16", op="window", n=16, longest=20000, mixed=False, new=1, window=8192, sinks=100, freed=False,
             q_heads=32, kv_heads=8, d=128, type="q8_0", q_type="f32", page=32),
        # ragged pieces of long prompts behind what the cache holds of them
        dict(name="window_prompts_3", op="window", n=3, longest=6000, mixed=True, new=2500, window=1024, sinks=4, freed=False,
             q_heads=32, kv_heads=8, d=128, type="bf16", q_type="bf16", page=64),
        # five candidates of one prompt: latency
        dict(name="shared_few_5", op="shared", n=5, groups=1, prefix=700, rest=40, mixed=True, q_heads=32, kv_heads=8, d=128,
             type="f16", q_type="f32", page=16),
        # a server whose requests all begin with the same long instructions
        dict(name="shared_batch_64", op="shared", n=64, groups=1, prefix=8192, rest=512, mixed=True, q_heads=32, kv_heads=8,
             d=128, type="f16", q_type="f32", page=16),
        # samples of several prompts at once, queries rounded as the cache is
        dict(name="shared_groups_96", op="shared", n=96, groups=6, prefix=5000, rest=1000, mixed=True, q_heads=16, kv_heads=4,
             d=64, type="bf16", q_type="bf16", page=24),
        # a small beam search's step: every candidate goes on from one of the last step's, which are then given back
        dict(name="beam_8", op="beam", n=8, prompt=208, rest=50, layers=2, kv_heads=8, d=128, type="f16", page=16),
        # many samples of a long prompt, all layers of a small model
        dict(name="beam_128", op="beam", n=128, prompt=4096, rest=120, layers=16, kv_heads=8, d=128, type="f16", page=16),
        # a pool that requests of all lengths left in pieces
        dict(name="compact_4500", op="compact", n=200, pages=4500, used=0.6, layers=8, kv_heads=8, d=128, type="bf16", page=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["turn", "turn", "window", "window", "window", "shared", "shared", "shared", "beam", "compact"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == "turn":
        d = rng.choice([64, 80, 96, 128, 256])
        kind = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, n=_log(rng, 1, 4000), q_heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, d=d,
                    rot=rng.choice([d, d, d // 2, 32]), pairs=rng.random() < 0.4, each=rng.random() < 0.3, type=kind,
                    q_type=rng.choice(["f32", kind]), page=page)
    if op == "window":
        new = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1500)])
        kind = rng.choice(["f32", "f16", "bf16", "q8_0"] if new < 9 else ["f16", "bf16"])
        d = rng.choice([64, 96, 128] if kind == "q8_0" else [40, 64, 80, 128, 256])
        group, window = rng.choice([1, 2, 4, 7, 8]), _log(rng, 16, 8192)
        longest = min(max(new, _log(rng, 16, 65536)), int(2e8) // (kv * _item(kind, d)))
        n = min(_log(rng, 1, 64), int(2e8) // (longest * kv * _item(kind, d)))
        n = max(1, min(n, int(6e8) // (kv * group * new * (window + new))))
        return dict(op=op, n=n, longest=longest, mixed=rng.random() < 0.6, new=new, window=window,
                    sinks=rng.choice([0, 1, 4, 4, rng.randint(5, 200)]), freed=rng.random() < 0.5, q_heads=kv * group,
                    kv_heads=kv, d=d, type=kind, q_type=kind if new >= 9 else rng.choice(["f32", "f32", "bf16"]), page=page)
    if op == "shared":
        kind = rng.choice(["f32", "f16", "f16", "bf16", "bf16", "q8_0"])
        d = rng.choice([64, 96, 128] if kind == "q8_0" else [40, 64, 80, 128, 256])
        group, prefix, rest = rng.choice([1, 2, 4, 8]), _log(rng, 64, 8192), _log(rng, 1, 700)
        n = max(2, min(_log(rng, 2, 96), int(7e8) // ((prefix + rest) * kv * d * 4)))
        return dict(op=op, n=n, groups=rng.choice([1, 1, min(n, rng.randint(2, 6))]), prefix=prefix, rest=rest,
                    mixed=rng.random() < 0.6, q_heads=kv * group, kv_heads=kv, d=d, type=kind,
                    q_type=rng.choice(["f32", "f32", kind if kind in ("f16", "bf16") else "f32"]), page=page)
    d, layers, kind = rng.choice([64, 128]), rng.randint(1, 12), rng.choice(["f32", "f16", "bf16"])
    if op == "beam":
        return dict(op=op, n=_log(rng, 2, 96), prompt=page * _log(rng, 1, 2000 // page), rest=_log(rng, 1, 100), layers=layers,
                    kv_heads=kv, d=d, type=kind, page=min(page, 32))
    return dict(op=op, n=_log(rng, 4, 200), pages=_log(rng, 100, 4000), used=rng.uniform(0.2, 0.9), layers=rng.randint(1, 6),
                kv_heads=kv, d=d, type=kind, page=min(page, 16))


# ---- sizes that a case stands for -----------------------------------------------------------------------

def _spread(n, longest, mixed):
    """n lengths up to `longest`: all of them that, or from short to long with the logarithm evenly spread."""
    if not mixed:
        return [longest] * n
    return [max(1, round(longest ** ((i + 1) / n))) for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


def _item(kind, d):
    """Bytes of the d values of one token and head."""
    return {"f32": 4 * d, "f16": 2 * d, "bf16": 2 * d, "q8_0": d + d // 16}[kind]


def _window_lengths(c):
    """Tokens of each sequence, and how many of them are new."""
    lens = _spread(c["n"], c["longest"], c["mixed"])
    most = [c["new"]] * c["n"] if c["new"] == 1 else _spread(c["n"], c["new"], c["mixed"])
    return lens, [min(a, b) for a, b in zip(lens, most)]


def _shared_lengths(c):
    """Sequences of each group, shared tokens (whole pages) of each group, tokens of each sequence."""
    size = [c["n"] // c["groups"] + (g < c["n"] % c["groups"]) for g in range(c["groups"])]
    prefix = [max(p, c["prefix"] // 4) for p in _spread(c["groups"], c["prefix"], c["mixed"])]
    rest = _spread(c["n"], c["rest"], c["mixed"])
    group = [g for g in range(c["groups"]) for _ in range(size[g])]
    return size, [p // c["page"] * c["page"] for p in prefix], [prefix[g] + r for g, r in zip(group, rest)]


def _page_bytes(c):
    return c["kv_heads"] * c["page"] * _item(c["type"], c["d"])


def work(case):
    c = case
    if c["op"] == "turn":
        heads = c["q_heads"] + c["kv_heads"]
        per = 4 * c["d"] * (c["q_heads"] + 2 * c["kv_heads"]) + c["q_heads"] * _item(c["q_type"], c["d"]) \
            + 2 * c["kv_heads"] * _item(c["type"], c["d"])
        return {"bytes": c["n"] * (per + 8) + 4 * c["d"] * (heads if c["each"] else 2), "flops": c["n"] * heads * c["d"] * 7}
    if c["op"] == "window":
        lens, new = _window_lengths(c)
        keys = flops = 0
        for n, k in zip(lens, new):
            first = max(n - k - c["window"] + 1, 0)  # the earliest key in any new token's window
            keys += n - first + min(c["sinks"], first)
            w, s = c["window"], c["sinks"]
            flops += sum(min(p + 1, w) + min(s, max(p + 1 - w, 0)) for p in range(n - k, n))
        q = 2 * sum(new) * c["q_heads"] * _item(c["q_type"], c["d"])
        return {"bytes": 2 * keys * c["kv_heads"] * _item(c["type"], c["d"]) + q, "flops": 4 * flops * c["q_heads"] * c["d"]}
    if c["op"] == "shared":
        size, shared, lens = _shared_lengths(c)
        keys = sum(shared) + sum(lens) - sum(a * b for a, b in zip(size, shared))
        return {"bytes": 2 * keys * c["kv_heads"] * _item(c["type"], c["d"]) + 2 * c["n"] * c["q_heads"] * _item(c["q_type"], c["d"]),
                "flops": 4 * sum(lens) * c["q_heads"] * c["d"]}
    if c["op"] == "beam":
        rows = c["n"] * (_ceil(c["prompt"] + c["rest"], c["page"]) + 4)
        return {"bytes": 4 * c["n"] * c["layers"] * _page_bytes(c) + 16 * rows, "flops": 0}
    used = c["used"] * c["pages"]
    moves = used * (1 - c["used"])
    return {"bytes": 4 * moves * c["layers"] * _page_bytes(c) + 8 * used + 16 * c["pages"], "flops": 0}


# ---- what a program has in hand before the call -----------------------------------------------------------

class _State:
    pass


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEVICE)


def _randn(shape, g, kind="f32", mul=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * mul).to(TORCH[kind])


def _perm(n, g):
    return torch.randperm(n, generator=g, device=DEVICE)


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


def _layers(c, pages, g):
    """K and V of all layers [layers, pages, values]."""
    values = c["kv_heads"] * c["page"] * c["d"]
    out = [torch.empty((c["layers"], pages, values), dtype=TORCH[c["type"]], device=DEVICE) for _ in range(2)]
    for x in out:
        x.normal_(generator=g)
    return out


def _table(used, first, g):
    """A table whose row b holds used[b] pages of a random order of sum(used) from id `first` on, -1 behind them."""
    total, width = sum(used), max(used) + 1
    ids = (_perm(total, g) + first).to(torch.int32)
    table = torch.full((len(used), width), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(width, device=DEVICE)[None, :] < _ints(used)[:, None]] = ids
    return table


def _prepare_turn(s, c, g):
    n, hq, hk, d = c["n"], c["q_heads"], c["kv_heads"], c["d"]
    s.qk = _randn((n, (hq + hk) * d), g, mul=3.0)  # q and k as one stacked product leaves them
    s.v = _randn((n, hk * d), g)
    s.q_w, s.k_w = (1 + 0.2 * _randn((h, d) if c["each"] else (1, d), g) for h in (hq, hk))
    pages = _ceil(n, c["page"]) + 3
    s.k_cache, s.v_cache = _cache(c, pages, g)
    s.slots = _perm(pages * c["page"], g)[:n].to(torch.int32)
    s.pos = torch.randint(0, 131072, (n,), generator=g, device=DEVICE, dtype=torch.int32)
    half = c["rot"] // 2
    s.freq = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)


def _prepare_window(s, c, g):
    lens, new = _window_lengths(c)
    order = _perm(c["n"], g).tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    s.table = _table([_ceil(n, c["page"]) for n in lens], 0, g)
    s.width, s.most = s.table.shape[1], max(new)
    pages = int(s.table.max()) + 3
    s.k_cache, s.v_cache = _cache(c, pages, g)
    s.lens, s.offsets = _ints(lens), _ints([sum(new[:i]) for i in range(c["n"] + 1)])
    s.q = _randn((sum(new), c["q_heads"], c["d"]), g, c["q_type"], 1.5)
    if c["freed"]:  # columns that no new token sees went back to the pool
        col = torch.arange(s.width, device=DEVICE) * c["page"]
        first = _ints([n - k - c["window"] + 1 for n, k in zip(lens, new)])[:, None]
        s.table[(col >= c["sinks"]) & (col + c["page"] <= first)] = -1


def _prepare_shared(s, c, g):
    size, shared, lens = _shared_lengths(c)
    page = c["page"]
    group = [i for i in range(c["groups"]) for _ in range(size[i])]
    s.table = _table([_ceil(n, page) for n in lens], 0, g)
    s.width = s.table.shape[1]
    s.groups = _ints([sum(size[:i]) for i in range(c["groups"] + 1)])
    s.shared, s.lens = _ints(shared), _ints(lens)
    lead = s.groups[_ints(group, torch.int64)].long()  # the group's first sequence: its pages are everybody's
    col = torch.arange(s.width, device=DEVICE)
    s.table = torch.where(col * page < s.shared[_ints(group, torch.int64)][:, None], s.table[lead], s.table)
    s.k_cache, s.v_cache = _cache(c, int(s.table.max()) + 2, g)
    s.q = _randn((c["n"], c["q_heads"], c["d"]), g, c["q_type"], 1.5)


def _prepare_beam(s, c, g):
    n, page = c["n"], c["page"]
    prompt = c["prompt"] // page
    rest = _spread(n, c["rest"], True)
    order = _perm(n, g).tolist()
    rest = [rest[i] for i in order]
    tails = [_ceil(r, page) for r in rest]
    spare = 2 * n + 5
    s.pages = prompt + sum(tails) + spare
    ids = _perm(s.pages, g).to(torch.int32)
    own_pages = _table(tails, prompt, g)
    s.width = prompt + own_pages.shape[1]
    s.table = torch.full((2 * n, s.width), -1, dtype=torch.int32, device=DEVICE)
    s.table[:n, :prompt] = torch.arange(prompt, dtype=torch.int32, device=DEVICE)
    s.table[:n, prompt:] = own_pages
    s.table = torch.where(s.table >= 0, ids[s.table.clamp(min=0).long()], s.table)
    s.lens = _ints([prompt * page + r for r in rest] + [0] * n)
    s.extra = torch.zeros(s.pages, dtype=torch.int32, device=DEVICE)
    s.extra[ids[:prompt].long()] = n - 1
    s.free = ids.clone()  # what was handed out, then what is free
    s.taken, s.taken2 = _ints([s.pages - spare, 0]), _ints([0, 0])
    s.k, s.v = _layers(c, s.pages, g)
    pick = torch.randint(0, n, (2, n), generator=g, device=DEVICE, dtype=torch.int32)
    row = torch.arange(n, dtype=torch.int32, device=DEVICE)
    # a step goes on from the rows of one half in the other, whose own rows are then given back; the next one back again
    s.steps = [(pick[0], row + n, row.clone()), (pick[1] + n, row.clone(), row + n)]
    s.at = 0
    s.pairs, s.n_pairs = _ints([[-1, -1]] * n), _ints([0])


def _prepare_compact(s, c, g):
    n, pages = c["n"], c["pages"]
    used = max(1, round(c["used"] * pages))
    n = min(n, used)
    weight = _spread(n, 8, True)
    own_pages = [max(1, used * w // sum(weight)) for w in weight]
    while sum(own_pages) > used:
        own_pages[own_pages.index(max(own_pages))] -= 1
    used = sum(own_pages)
    table = _table(own_pages, 0, g)
    ids = _perm(pages, g).to(torch.int32)
    s.table = torch.where(table >= 0, ids[table.clamp(min=0).long()], table)
    s.free, s.taken = ids, _ints([used, 0])
    s.extra = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    s.extra[ids[:used].long()] = torch.randint(0, 5, (used,), generator=g, device=DEVICE, dtype=torch.int32)
    s.k, s.v = _layers(c, pages, g)
    s.pairs, s.moved = torch.full((max(1, pages // 2), 2), -1, dtype=torch.int32, device=DEVICE), _ints([0, 0])


def _own_handles(s, c):
    """What a program keeps beside its tensors: outputs, cache descriptions, workspaces."""
    import qorvix_amd as qvx
    s.qvx = qvx
    op = c["op"]
    if op in ("turn", "window", "shared"):
        s.cache = qvx.KvCache.of(s.k_cache, s.v_cache, TYPES[c["type"]], c["page"], c["kv_heads"], c["d"])
    if op == "turn":
        s.q_out = torch.empty((c["n"], c["q_heads"] * c["d"]), dtype=TORCH[c["q_type"]], device=DEVICE)
        s.rope = qvx.Rope.of(s.freq, pairing=qvx.ROPE_PAIRS if c["pairs"] else qvx.ROPE_HALVES)
        s.norm = qvx.QkNorm.of(s.q_w if c["each"] else s.q_w[0], s.k_w if c["each"] else s.k_w[0], EPS)
    if op in ("window", "shared"):
        s.out = torch.empty_like(s.q)
        t = TYPES[c["q_type"]]
        need = qvx.attn_window_ws(s.cache, t, c["q_heads"], s.q.shape[0], c["n"], s.width, c["window"], c["sinks"]) \
            if op == "window" else qvx.attn_shared_ws(s.cache, t, c["q_heads"], c["n"], s.width, c["groups"])
        s.ws = torch.empty(need, dtype=torch.uint8, device=DEVICE)
    if op in ("beam", "compact"):
        pages = s.extra.shape[0]
        s.caches = qvx.kv_caches([qvx.KvCache.of(k, v, TYPES[c["type"]], c["page"], c["kv_heads"], c["d"])
                                  for k, v in zip(s.k, s.v)])
        s.ws = torch.empty(qvx.kv_free_ws(pages), dtype=torch.uint8, device=DEVICE)
    if op == "compact":
        s.table_out, s.extra_out, s.free_out = (torch.empty_like(x) for x in (s.table, s.extra, s.free))


def prepare(case, seed):
    s = _State()
    s.case = case
    g = _generator(seed)
    {"turn": _prepare_turn, "window": _prepare_window, "shared": _prepare_shared, "beam": _prepare_beam,
     "compact": _prepare_compact}[case["op"]](s, case, g)
    if own:
        _own_handles(s, case)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------

def _rotate(x, cos, sin, c):
    rot = c["rot"]
    if c["pairs"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_turn(s):
    c = s.case
    n, hq, hk, d, page = c["n"], c["q_heads"], c["kv_heads"], c["d"], c["page"]
    angle = s.pos.double()[:, None] * s.freq  # [tokens, pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q, k = s.qk[:, :hq * d].view(n, hq, d), s.qk[:, hq * d:].view(n, hk, d)
    slots = s.slots.long()
    for cache, x in ((s.k_cache, _rotate(_normed(k, s.k_w), cos, sin, c)), (s.v_cache, s.v.view(n, hk, d))):
        cache.view(-1, hk, page, d)[slots // page, :, slots % page] = x.to(cache.dtype)
    return [_rotate(_normed(q, s.q_w), cos, sin, c).reshape(n, hq * d).to(TORCH[c["q_type"]]), s.k_cache, s.v_cache]


def _tokens(pages, c, page, off):
    """The values [.., heads, d] of the tokens at `off` of the pages `page`, in 32 bits."""
    hk, d = c["kv_heads"], c["d"]
    if c["type"] != "q8_0":
        return pages.view(-1, hk, c["page"], d)[page, :, off].float()
    split = hk * c["page"] * d
    quants = pages[:, :split].view(torch.int8).view(-1, hk, c["page"], d)[page, :, off].float()
    steps = pages[:, split:].view(torch.float16).view(-1, hk, c["page"], d // 32)[page, :, off].float()
    return (quants.unflatten(-1, (d // 32, 32)) * steps[..., None]).flatten(-2)


def _softmax_product(q, k, v, live, scale):
    """q [n, heads, rows, d] on k, v [n, heads, keys, d], where live [n, 1, rows, keys] holds."""
    logits = (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill(~live, -math.inf)
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total == 0, 1.0, total)


def _plain_window(s):
    c = s.case
    n, hq, hk, d, window, sinks = c["n"], c["q_heads"], c["kv_heads"], c["d"], c["window"], c["sinks"]
    group, most = hq // hk, s.most
    new = s.offsets[1:] - s.offsets[:-1]
    held = s.lens - new
    # the keys that any new token of a sequence sees: the sinks, and from the first new token's window on
    near = held[:, None] - window + 1 + torch.arange(min(window + most, s.width * c["page"]), device=DEVICE)
    if window + most > s.width * c["page"]:
        near = torch.arange(s.width * c["page"], device=DEVICE).expand(n, -1)
    far = torch.arange(sinks, device=DEVICE).expand(n, sinks)
    key = torch.cat([far, near], 1)
    good = torch.cat([torch.ones_like(far, dtype=torch.bool), near >= sinks], 1) & (key < s.lens[:, None])
    at = key.clamp(0, s.width * c["page"] - 1).long()
    page = torch.gather(s.table, 1, at // c["page"]).long()
    good &= page >= 0
    k, v = (_tokens(x, c, page.clamp(min=0), at % c["page"]).transpose(1, 2) for x in (s.k_cache, s.v_cache))
    row = torch.arange(most, device=DEVICE)
    pos = held[:, None] + row
    live = (key[:, None] <= pos[..., None]) & ((key[:, None] > pos[..., None] - window) | (key[:, None] < sinks)) & good[:, None]
    at = (s.offsets[:-1, None].long() + row).clamp(max=s.q.shape[0] - 1)  # a padded batch of the queries
    q = s.q[at].float().view(n, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * most, d)
    o = _softmax_product(q, k, v, live[:, None].expand(-1, group, -1, -1).reshape(n, 1, group * most, -1), 1.0 / math.sqrt(d))
    o = o.view(n, hk, group, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, hq, d)
    t = torch.arange(s.q.shape[0], device=DEVICE)
    seq = (t[:, None] >= s.offsets[None, 1:]).sum(1)
    return o[seq, t - s.offsets[seq].long()].to(s.q.dtype)


def _plain_shared(s):
    c = s.case
    n, hq, hk, d, page = c["n"], c["q_heads"], c["kv_heads"], c["d"], c["page"]
    key = torch.arange((s.width - 1) * page, device=DEVICE)
    at = s.table[:, :-1].clamp(min=0).long().repeat_interleave(page, 1)
    k, v = (_tokens(x, c, at, (key % page).expand(n, -1)).transpose(1, 2) for x in (s.k_cache, s.v_cache))
    live = (key < s.lens[:, None])[:, None, None]
    o = _softmax_product(s.q.float().view(n, hk, hq // hk, d), k, v, live, 1.0 / math.sqrt(d))
    return o.reshape(n, hq, d).to(s.q.dtype)


def _plain_beam(s):
    """Forks of the table's rows, copies of their last pages, release of the rows before."""
    c = s.case
    page, pages = c["page"], s.pages
    source, to, gone = (x.long() for x in s.steps[s.at])
    s.at ^= 1
    lens = s.lens[source]
    full, part = (lens // page).long(), lens % page > 0
    col = torch.arange(s.width, device=DEVICE)
    old = s.table[source]
    fresh = s.free[s.taken[0].long() + torch.cumsum(part, 0) - part.long()]
    keep = col < full[:, None]
    s.table[to] = torch.where(keep, old, torch.where((col == full[:, None]) & part[:, None], fresh[:, None], -1))
    s.lens[to] = lens
    count = torch.zeros(pages + 1, dtype=torch.int32, device=DEVICE)
    count.index_add_(0, torch.where(keep, old, pages).flatten().long(), torch.ones(old.numel(), dtype=torch.int32, device=DEVICE))
    s.extra += count[:pages]
    src, dst = old[part, full[part]].long(), fresh[part].long()
    s.k[:, dst], s.v[:, dst] = s.k[:, src], s.v[:, src]
    taken = s.taken[0] + part.sum()

    ids = s.table[gone]
    count = torch.zeros(pages + 1, dtype=torch.int32, device=DEVICE)
    count.index_add_(0, torch.where(ids >= 0, ids, pages).flatten().long(), torch.ones(ids.numel(), dtype=torch.int32, device=DEVICE))
    left = s.extra - count[:pages]
    back = left < 0
    s.extra = left.clamp(min=0)
    taken = taken - back.sum()
    place = torch.where(back, taken + torch.cumsum(back, 0) - 1, pages)  # ascending, in front of what is free
    s.free = torch.cat([s.free, s.free[:1]]).scatter(0, place, torch.arange(pages, dtype=torch.int32, device=DEVICE))[:pages]
    s.table[gone] = -1
    s.lens[gone] = 0
    s.taken = torch.stack([taken, torch.zeros_like(taken)]).to(torch.int32)
    return [s.table, s.lens, s.extra, s.free, s.taken, s.k, s.v]


def _plain_compact(s):
    pages = s.extra.shape[0]
    ids = torch.arange(pages, device=DEVICE)
    listed_free = torch.arange(s.free.shape[0], device=DEVICE) >= s.taken[0]
    used = torch.ones(pages + 1, dtype=torch.bool, device=DEVICE)
    used[torch.where(listed_free, s.free, pages).long()] = False
    used = used[:pages]
    n = used.sum()
    src, dst = torch.nonzero(used & (ids >= n))[:, 0], torch.nonzero(~used & (ids < n))[:, 0]
    to = ids.clone()
    to[src] = dst
    table = torch.where(s.table >= 0, to[s.table.clamp(min=0).long()].to(torch.int32), s.table)
    extra = s.extra.clone()
    extra[dst], extra[src] = s.extra[src], 0
    free = torch.where(listed_free, n + torch.arange(s.free.shape[0], device=DEVICE) - s.taken[0], s.free).to(torch.int32)
    s.k[:, dst], s.v[:, dst] = s.k[:, src], s.v[:, src]
    moved = torch.stack([torch.full_like(n, src.shape[0]), n]).to(torch.int32)  # pages moved, pages in use
    return [table, extra, free, moved, s.k, s.v]


# ---- the framework's kernels ---------------------------------------------------------------------------------

def _own(s):
    qvx, c = s.qvx, s.case
    op, stream = c["op"], torch.cuda.current_stream().cuda_stream
    if op == "turn":
        hq, hk, d = c["q_heads"], c["kv_heads"], c["d"]
        qk = s.qk.data_ptr()
        rc = qvx.norm_rope_kv(s.q_out.data_ptr(), hq * d, TYPES[c["q_type"]], qk, (hq + hk) * d, hq, qk + 4 * hq * d,
                              (hq + hk) * d, s.v.data_ptr(), hk * d, c["n"], d, s.norm, s.rope, s.pos.data_ptr(), c["n"],
                              s.cache, s.slots.data_ptr(), stream)
        out = [s.q_out, s.k_cache, s.v_cache]
    elif op == "window":
        row = c["q_heads"] * c["d"]
        rc = qvx.attn_window(s.out.data_ptr(), row, s.q.data_ptr(), row, TYPES[c["q_type"]], c["q_heads"],
                             s.offsets.data_ptr(), s.q.shape[0], s.cache, s.table.data_ptr(), s.width, s.lens.data_ptr(),
                             c["n"], c["window"], c["sinks"], 1.0 / math.sqrt(c["d"]), s.ws.data_ptr(), s.ws.numel(), stream)
        out = s.out
    elif op == "shared":
        row = c["q_heads"] * c["d"]
        rc = qvx.attn_shared(s.out.data_ptr(), row, s.q.data_ptr(), row, TYPES[c["q_type"]], c["q_heads"], s.cache,
                             s.table.data_ptr(), s.width, s.lens.data_ptr(), c["n"], s.groups.data_ptr(),
                             s.shared.data_ptr(), c["groups"], 1.0 / math.sqrt(c["d"]), s.ws.data_ptr(), s.ws.numel(), stream)
        out = s.out
    elif op == "beam":
        source, to, gone = s.steps[s.at]
        s.at ^= 1
        rows, width, n = s.table.shape[0], s.width, c["n"]
        rc = qvx.kv_fork(source.data_ptr(), to.data_ptr(), n, s.table.data_ptr(), rows, width, c["page"],
                         s.lens.data_ptr(), s.extra.data_ptr(), s.pages, s.free.data_ptr(), s.free.shape[0],
                         s.taken.data_ptr(), s.taken2.data_ptr(), s.pairs.data_ptr(), s.n_pairs.data_ptr(), stream)
        rc = rc or qvx.kv_copy(s.caches, s.pairs.data_ptr(), s.n_pairs.data_ptr(), n, stream)
        rc = rc or qvx.kv_free(gone.data_ptr(), 0, 0, n, s.table.data_ptr(), rows, width, s.lens.data_ptr(),
                               s.extra.data_ptr(), s.pages, s.free.data_ptr(), s.free.shape[0], s.taken2.data_ptr(),
                               s.taken.data_ptr(), s.ws.data_ptr(), s.ws.numel(), stream)
        out = [s.table, s.lens, s.extra, s.free, s.taken, s.k, s.v]
    else:
        pages = s.extra.shape[0]
        rc = qvx.kv_compact(s.table.data_ptr(), s.table_out.data_ptr(), s.table.shape[0], s.table.shape[1],
                            s.extra.data_ptr(), s.extra_out.data_ptr(), pages, s.free.data_ptr(), s.free_out.data_ptr(),
                            s.free.shape[0], s.taken.data_ptr(), s.pairs.data_ptr(), s.moved.data_ptr(), stream)
        rc = rc or qvx.kv_copy(s.caches, s.pairs.data_ptr(), s.moved.data_ptr(), s.pairs.shape[0], stream)
        out = [s.table_out, s.extra_out, s.free_out, s.moved, s.k, s.v]
    if rc != qvx.OK:
        raise qvx.QvxError(rc, op)
    return out


def run(state):
    if own:
        return _own(state)
    return {"turn": _plain_turn, "window": _plain_window, "shared": _plain_shared, "beam": _plain_beam,
            "compact": _plain_compact}[state.case["op"]](state)


# ---- the same results in 64 bits -------------------------------------------------------------------------------

def _decoded(cache, c, pages):
    """The tokens [tokens, heads, d] of a sequence's pages in 64 bits."""
    got = cache[pages]
    if c["type"] == "q8_0":
        at = c["kv_heads"] * c["page"] * c["d"]
        steps = got[:, at:].contiguous().view(torch.float16).double()
        got = got[:, :at].contiguous().view(torch.int8).double() * steps.repeat_interleave(32, dim=1)
    return got.double().view(-1, c["kv_heads"], c["page"], c["d"]).transpose(1, 2).flatten(0, 1)


def _exact_turn(s, c):
    n, hq, hk, d, half = c["n"], c["q_heads"], c["kv_heads"], c["d"], c["rot"] // 2
    where = s.pos.double()[:, None, None] * s.freq
    turn = torch.polar(torch.ones_like(where), where)

    def done(x, w):
        x = x.double()
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS) * w.double()
        a, b = (x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]) if c["pairs"] else (x[..., :half], x[..., half: 2 * half])
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        y = x.clone()
        if c["pairs"]:
            y[..., 0: 2 * half: 2], y[..., 1: 2 * half: 2] = z.real, z.imag
        else:
            y[..., :half], y[..., half: 2 * half] = z.real, z.imag
        return y

    x = s.qk.view(n, hq + hk, d)
    out = [done(x[:, :hq], s.q_w).reshape(n, hq * d)]
    page, off = torch.div(s.slots.long(), c["page"], rounding_mode="floor"), s.slots.long() % c["page"]
    for cache, new in ((s.k_cache, done(x[:, hq:], s.k_w)), (s.v_cache, s.v.view(n, hk, d).double())):
        full = cache.double().view(-1, hk, c["page"], d).transpose(1, 2).contiguous()
        full[page, off] = new
        out.append(full.transpose(1, 2).reshape(cache.shape))
    return out


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence and head by head; pages that move keep their values and have none."""
    c = case
    if c["op"] in ("beam", "compact"):
        return None
    s = _State()
    s.case = c
    g = _generator(seed)
    {"turn": _prepare_turn, "window": _prepare_window, "shared": _prepare_shared}[c["op"]](s, c, g)
    if c["op"] == "turn":
        return _exact_turn(s, c)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    group = c["q_heads"] // c["kv_heads"]
    rows = s.offsets.tolist() if c["op"] == "window" else list(range(c["n"] + 1))
    for i, length in enumerate(s.lens.tolist()):
        col = s.table[i, : _ceil(length, c["page"])].long()
        k, v = (_decoded(x, c, col.clamp(min=0))[:length] for x in (s.k_cache, s.v_cache))
        j = torch.arange(length, device=DEVICE)
        p = length - rows[i + 1] + rows[i] + torch.arange(rows[i + 1] - rows[i], device=DEVICE)[:, None]
        seen = j <= p
        if c["op"] == "window":
            seen = seen & ((p - j < c["window"]) | (j < c["sinks"]))
        for h in range(c["q_heads"]):
            a = s.q[rows[i]: rows[i + 1], h].double() @ k[:, h // group].t() / math.sqrt(c["d"])
            out[rows[i]: rows[i + 1], h] = torch.softmax(a.masked_fill(~seen, -math.inf), -1) @ v[:, h // group]
    return out
