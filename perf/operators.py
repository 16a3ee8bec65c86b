"""The operators of the paged KV cache: what they compute, in plain torch, and the sizes they are used at.

Serving keeps each sequence's keys and values in pages of a pool. A speculative decoder checks a
tree of drafted tokens against the cached ones (tree), a long context is read through the pages
that a cheap score picks (select), accepted or prompt tokens are written to pages (append), slots
are forked, reordered and freed (fork), and the pool is packed so its tail can be given back
(compact).

Pools are bf16 [layers, pages, kv heads, page size, head dim] (without the layer dimension for
attention, which reads one layer); page tables int32 [slots, table width] with -1 for no page;
refs int32 [pages] counts the table rows that hold a page.

`own` False: plain torch, fp32 arithmetic, one rounding at the end. `own` True: iron_b200.
"""

import math
import random

import torch

own = False

NEG = float("-inf")
FLT_MAX = 3.4028234663852886e38


# ---- cases ----------------------------------------------------------------------------------


def listed():
    # head layouts: 32 query / 8 kv heads of 64 (Llama-3.2-1B) and of 128 (Llama-3-8B)
    small = dict(heads=32, kv_heads=8, dim=64, page=64)
    wide = dict(heads=32, kv_heads=8, dim=128, page=64)
    return [
        # one chat sequence, a short context and a small draft: the latency of a call
        dict(name="tree 1x8 short", op="tree", batch=1, nodes=8, lo=301, hi=301, **small),
        # a serving batch at ordinary, ragged lengths
        dict(name="tree 16x26 ragged 4k", op="tree", batch=16, nodes=26, lo=257, hi=4096, **small),
        # wide trees over long contexts: the largest verification step
        dict(name="tree 8x64 32k d128", op="tree", batch=8, nodes=64, lo=16385, hi=32768, **wide),
        # one sequence with a middling context: latency of score, choice and attention
        dict(name="select 1 8k", op="select", batch=1, lo=8190, hi=8190, top=16, **small),
        # a batch of long ragged contexts at head dim 128
        dict(name="select 16 32k d128", op="select", batch=16, lo=2001, hi=32768, top=32, **wide),
        # the largest batch of the decode benchmark at its longest context
        dict(name="select 64 32k", op="select", batch=64, lo=30001, hi=32768, top=64, **small),
        # after a verification step: a few accepted tokens of each tree, every layer
        dict(name="append 16 accepted", op="append", layers=16, slots=16, new=8, take=5, lo=130, hi=2000, summaries=False, **small),
        # prompts entering the cache after prefill, every layer, with the pages' summaries
        dict(name="append 4 prompts 2k", op="append", layers=16, slots=4, new=2048, take=2048, lo=0, hi=70, summaries=True, **small),
        # one prompt sampled four ways
        dict(name="fork 1 into 4", op="fork", layers=16, slots=8, parents=1, filled=4, lo=901, hi=901, **small),
        # beam reordering of a large batch: half of the slots survive, some are freed
        dict(name="fork 128 beams", op="fork", layers=16, slots=128, parents=60, filled=120, lo=70, hi=460, **small),
        # packing a small pool of one layer
        dict(name="compact 300 pages", op="compact", layers=1, pages=300, used=140, moved=50, slots=16, summaries=False, **small),
        # packing a fragmented pool of every layer, summaries with it
        dict(name="compact 1000 pages", op="compact", layers=16, pages=1000, used=600, moved=250, slots=64, summaries=True, **small),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "select", "select", "select", "append", "fork", "compact"])
    heads, kv = rng.choice([(32, 8), (32, 8), (32, 8), (16, 16), (8, 1), (24, 8), (32, 2)])
    c = dict(op=op, heads=heads, kv_heads=kv, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 64, 128]))
    if op in ("tree", "select"):
        c["batch"] = _log(rng, 1, 64)
        # the cache holds at most 2^27 values of each of K and V
        most = min(32768, (1 << 27) // (c["batch"] * kv * c["dim"]))
        c["hi"] = _log(rng, 1, most)
        c["lo"] = rng.randint(max(1, c["hi"] // 8), c["hi"])
        if op == "tree":
            # scores of all rows: at most 2^28
            c["nodes"] = _log(rng, 1, max(1, min(64, (1 << 28) // (c["batch"] * heads * c["hi"]))))
        else:
            c["top"] = _log(rng, 1, 80)
    elif op == "append":
        c.update(layers=rng.randint(1, 16), slots=_log(rng, 1, 64), summaries=rng.random() < 0.5)
        most = min(2048, 50_000_000 // (c["layers"] * c["slots"] * kv * c["dim"]))
        c["new"] = _log(rng, 1, max(1, most))
        c["take"] = rng.randint(1, c["new"])
        c["lo"] = _log(rng, 1, 200) - 1
        c["hi"] = c["lo"] + rng.randint(0, 300)
    elif op == "fork":
        c.update(layers=rng.randint(1, 16), slots=_log(rng, 2, 160))
        c["filled"] = rng.randint(1, c["slots"])
        c["parents"] = rng.randint(1, c["filled"])
        c["lo"] = _log(rng, 1, 300)
        c["hi"] = c["lo"] + rng.randint(0, 200)
        c["layers"] = max(1, min(c["layers"], (1 << 29) // (c["slots"] * (c["hi"] + 2 * c["page"]) * 2 * kv * c["dim"])))
    else:
        c.update(pages=_log(rng, 8, 1000), slots=_log(rng, 1, 64), summaries=rng.random() < 0.5)
        c["layers"] = max(1, min(rng.randint(1, 16), 250_000_000 // (c["pages"] * c["page"] * kv * c["dim"])))
        c["used"] = rng.randint(1, c["pages"] - 1)
        c["moved"] = rng.randint(0, min(c["used"], c["pages"] - c["used"]))
    return c


def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly spread (the seed orders them)."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _pages(n, page):
    return -(-n // page)


def _fork_lens(c):
    """Lengths of the old slots; parents are the first ones. None ends with its page, so every second child costs a copy."""
    lens = _spread(c["lo"], c["hi"], c["slots"])
    return [n + 1 if n % c["page"] == 0 else n for n in lens]


def work(c):
    row = c["kv_heads"] * c["dim"] * 2  # one token's K (or V) in one layer
    if c["op"] == "tree":
        B, N, H = c["batch"], c["nodes"], c["heads"]
        cached = sum(_spread(c["lo"], c["hi"], B))
        table = 4 * sum(_pages(n, c["page"]) for n in _spread(c["lo"], c["hi"], B))
        byts = 2 * row * (cached + B * N) + 2 * B * N * H * c["dim"] * 2 + table + 4 * B * (N + 1)
        return {"bytes": byts, "flops": 4 * N * H * c["dim"] * cached}
    if c["op"] == "select":
        lens = _spread(c["lo"], c["hi"], c["batch"])
        pages = [_pages(n, c["page"]) for n in lens]
        # every page but the last is full
        kept = sum(n if p <= c["top"] else c["top"] * c["page"] - (p * c["page"] - n) for n, p in zip(lens, pages))
        byts = sum(pages) * (c["kv_heads"] * (2 * c["dim"] + 4) + 4) + 2 * row * kept
        byts += 2 * c["batch"] * c["heads"] * c["dim"] * 2 + 4 * c["batch"] * c["kv_heads"] * c["top"]
        return {"bytes": byts, "flops": 4 * c["heads"] * c["dim"] * kept + 4 * sum(pages) * c["kv_heads"] * c["dim"]}
    if c["op"] == "append":
        n = sum(_takes(c))
        return {"bytes": c["layers"] * n * 2 * row * 2 + 8 * c["slots"] + 4 * n, "flops": 0}
    if c["op"] == "fork":
        lens = _fork_lens(c)
        kids = [sum(1 for i in range(c["filled"]) if i % c["parents"] == p) for p in range(c["parents"])]
        rows = sum((k - 1) * (n % c["page"]) for k, n in zip(kids, lens))
        table = sum(_pages(n, c["page"]) for n in lens)
        return {"bytes": c["layers"] * rows * 2 * row * 2 + 8 * table + 8 * _fork_pages(c) + 12 * c["slots"], "flops": 0}
    one = c["layers"] * (2 * row * c["page"] + c["summaries"] * c["kv_heads"] * (2 * c["dim"] + 4))
    return {"bytes": 2 * c["moved"] * one + 8 * c["used"] + 8 * c["pages"], "flops": 0}


def _takes(c):
    """How many rows each slot appends: from one to `take`."""
    return _spread(1 if c["take"] < c["new"] else max(1, c["take"] // 2), c["take"], c["slots"])


def _fork_pages(c):
    return sum(_pages(n, c["page"]) for n in _fork_lens(c)) + c["filled"] + 3


# ---- inputs ---------------------------------------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(rng, lens, page, width, pages):
    """Each slot's pages, drawn without order from the pool: the table and the reference counts."""
    n = _ints([_pages(n, page) for n in lens])
    total = int(n.sum())
    ids = _ints(rng.sample(range(pages), total) + [-1])
    at = torch.arange(width, device="cuda")
    which = (n.cumsum(0) - n)[:, None] + at
    table = ids[torch.where(at < n[:, None], which, torch.full_like(which, total))]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[ids[:total].long()] = 1
    return table.contiguous(), refs


def _summaries(k):
    """Bounds of each page's keys: codes int8 [..., 2, D] and their scale [...]."""
    k = k.float()
    lo, hi = k.amin(-2), k.amax(-2)
    top = torch.maximum(lo.abs().amax(-1), hi.abs().amax(-1))
    scale = top / 127.0
    by = torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    lo, hi = torch.floor(lo / by).clamp(-127, 127), torch.ceil(hi / by).clamp(-127, 127)
    fine = torch.isfinite(top)
    scale = torch.where(fine, scale, torch.full_like(scale, FLT_MAX))
    lo = torch.where(fine[..., None], lo, torch.full_like(lo, -127.0))
    hi = torch.where(fine[..., None], hi, torch.full_like(hi, 127.0))
    return torch.stack([lo, hi], -2).to(torch.int8), scale


def _parents(rng, batch, nodes):
    """Drafted trees: nodes mostly extend a recent one, some start beside the root; the smaller trees of a batch leave their last places unused (-2)."""
    sizes = [nodes] + [rng.randint(max(1, nodes // 2), nodes) for _ in range(batch - 1)]
    pick = lambda i: -1 if i == 0 or rng.random() < 0.1 else rng.randint(max(0, i - 6), i - 1)  # noqa: E731
    return _ints([[pick(i) if i < n else -2 for i in range(nodes)] for n in sizes])


def prepare(case, seed):
    c = case
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    kv, dim, page = c["kv_heads"], c["dim"], c["page"]
    if c["op"] in ("tree", "select"):
        lens = _spread(c["lo"], c["hi"], c["batch"])
        rng.shuffle(lens)
        width = _pages(c["hi"], page) + 1
        pages = sum(_pages(n, page) for n in lens) + 5
        s["table"], _ = _table(rng, lens, page, width, pages)
        s["lens"] = _ints(lens)
        s["k"], s["v"] = _normal(gen, pages, kv, page, dim), _normal(gen, pages, kv, page, dim)
        if c["op"] == "tree":
            # q, k and v of the drafted tokens as the QKV projection leaves them: one row per token
            s["qkv"] = _normal(gen, c["batch"], c["nodes"], c["heads"] + 2 * kv, dim)
            s["parents"] = _parents(rng, c["batch"], c["nodes"])
            s["out"] = torch.zeros(c["batch"], c["nodes"], c["heads"], dim, device="cuda", dtype=torch.bfloat16)
        else:
            # keys of a page resemble one another, so that pages differ in what they offer a query
            s["k"] += _normal(gen, pages, kv, 1, dim)
            s["codes"], s["scales"] = _summaries(s["k"])
            s["q"] = _normal(gen, c["batch"], c["heads"], dim)
            s["out"] = torch.zeros(c["batch"], c["heads"], dim, device="cuda", dtype=torch.bfloat16)
            s["selected"] = torch.zeros(c["batch"], kv, c["top"], device="cuda", dtype=torch.int32)
        return s
    s["status"] = _ints([0])
    if c["op"] == "append":
        lens = _spread(c["lo"], c["hi"], c["slots"])
        rng.shuffle(lens)
        takes = _takes(c)
        rng.shuffle(takes)
        width = _pages(c["hi"] + c["take"], page) + 1
        pages = sum(_pages(n, page) + 1 for n in lens) + sum(_pages(t, page) for t in takes) + 3
        # accepted rows are an ascending choice of the new ones, as the path of a tree is
        index = [sorted(rng.sample(range(c["new"]), t)) + [-1] * (c["new"] - t) for t in takes]
        s["table"], s["refs"] = _table(rng, lens, page, width, pages)
        s["lens"], s["index"], s["lens_out"] = _ints(lens), _ints(index), _ints([0] * c["slots"])
        s["k_new"], s["v_new"] = (_normal(gen, c["layers"], c["slots"], c["new"], kv, dim) for _ in range(2))
    elif c["op"] == "fork":
        lens = _fork_lens(c)
        old = list(range(c["slots"]))
        rng.shuffle(old)  # parent i is slot old[i]
        source = [old[i % c["parents"]] for i in range(c["filled"])] + [-1] * (c["slots"] - c["filled"])
        rng.shuffle(source)
        by_slot = [0] * c["slots"]
        for r, n in zip(old, lens):
            by_slot[r] = n
        pages, width = _fork_pages(c), _pages(c["hi"] + 1, page) + 1
        s["table"], s["refs"] = _table(rng, by_slot, page, width, pages)
        s["lens"], s["source"] = _ints(by_slot), _ints(source)
        s["table_out"], s["lens_out"], s["refs_out"] = (torch.zeros_like(s[n]) for n in ("table", "lens", "refs"))
    else:
        pages, used, moved = c["pages"], c["used"], c["moved"]
        low = rng.sample(range(used), used - moved)
        ids = low + rng.sample(range(used, pages), moved)
        rng.shuffle(ids)
        width = _pages(used, c["slots"]) + 2
        rows, refs = [[] for _ in range(c["slots"])], [0] * pages
        for i, p in enumerate(ids):
            rows[i % c["slots"]].append(p)
            refs[p] = 1
        for r in rows[1::2]:  # every second slot shares its neighbour's first page, as forks do
            r.append(rows[0][0])
            refs[rows[0][0]] += 1
        s["table"], s["refs"] = _ints([r + [-1] * (width - len(r)) for r in rows]), _ints(refs)
        s["table_out"], s["refs_out"], s["used"] = torch.zeros_like(s["table"]), torch.zeros_like(s["refs"]), _ints([0])
    s["k"], s["v"] = (_normal(gen, c["layers"], pages, kv, page, dim) for _ in range(2))
    if c.get("summaries"):
        s["codes"] = torch.randint(-127, 128, (c["layers"], pages, kv, 2, dim), generator=gen, device="cuda", dtype=torch.int8)
        s["scales"] = torch.rand(c["layers"], pages, kv, generator=gen, device="cuda")
    return s


# ---- the plain form -------------------------------------------------------------------------


def _visible(parents):
    """[B, N, N]: whether node j is on the path from the root to node i (i included), False for unused nodes."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    eye = torch.eye(n, device=parents.device)
    bad = (parents < -1) | (parents >= at)
    step = ((parents[..., None] == at) & ~bad[..., None]).float()
    # (I - A)^-1 = I + A + A^2 + ...: every ancestor, exactly
    path = torch.linalg.solve_triangular(eye - step, eye.expand_as(step), upper=False, unitriangular=True) > 0.5
    used = ~(path & bad[:, None, :]).any(-1)
    return path & used[..., None]


def _tree(s):
    c, table = s["case"], s["table"].clamp(min=0).long()
    B, N, H, G, D = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    T = table.shape[1] * c["page"]
    q, kn, vn = s["qkv"].float().split([H, G, G], 2)
    q = q.reshape(B, N, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, -1, D)
    k = torch.cat([s["k"][table].transpose(1, 2).reshape(B, G, T, D).float(), kn.transpose(1, 2)], 2)
    v = torch.cat([s["v"][table].transpose(1, 2).reshape(B, G, T, D).float(), vn.transpose(1, 2)], 2)
    path = _visible(s["parents"])
    cached = (torch.arange(T, device=q.device) < s["lens"][:, None])[:, None].expand(B, N, T)
    seen = torch.cat([cached & path.any(-1, keepdim=True), path], 2)[:, None, :, None]
    scores = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(D)).view(B, G, N, H // G, -1)
    scores = scores.masked_fill_(~seen, NEG)
    top = scores.amax(-1, keepdim=True).clamp(min=-FLT_MAX)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, G, -1, T + N) @ v).view(B, G, N, H // G, D) / total.clamp(min=1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(B, N, H, D).to(torch.bfloat16)


def _select(s):
    c, lens, k_most = s["case"], s["lens"], s["case"]["top"]
    B, H, G, D, page = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    table = s["table"].clamp(min=0).long()
    M = table.shape[1]
    q = s["q"].float().view(B, G, H // G, D)
    top = q.abs().amax((2, 3), keepdim=True)
    q8 = torch.round(q / torch.where(top > 0, top, torch.ones_like(top)) * 127.0)
    up, down = q8.clamp(min=0).sum(2), q8.clamp(max=0).sum(2)  # whole numbers: exact in any order
    codes = s["codes"][table].float()  # [B, M, G, 2, D]
    whole = (codes[:, :, :, 1] * up[:, None]).sum(-1) + (codes[:, :, :, 0] * down[:, None]).sum(-1)
    score = (whole * s["scales"][table]).transpose(1, 2).clamp(-FLT_MAX, FLT_MAX)  # [B, G, M]
    n = ((lens + page - 1) // page)[:, None, None]
    at = torch.arange(M, device=q.device)
    score = torch.where((at == 0) & (k_most > 1) | (at == n - 1), torch.full_like(score, math.inf), score)
    score = score.masked_fill(at >= n, NEG)
    first = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k_most]
    first = torch.where(first < n, first, torch.full_like(first, M)).sort(-1).values
    kept = first < M
    selected = torch.full((B, G, k_most), -1, device=q.device, dtype=torch.int32)
    selected[..., : first.shape[-1]] = torch.where(kept, first, torch.full_like(first, -1)).int()
    ids = torch.gather(table[:, None].expand(B, G, M), 2, first.clamp(max=M - 1))  # [B, G, K]
    head = torch.arange(G, device=q.device)[None, :, None]
    k, v = (s[x][ids, head].float().flatten(2, 3) for x in ("k", "v"))  # [B, G, K * page, D]
    t = (first[..., None] * page + torch.arange(page, device=q.device)).flatten(2)
    scores = (q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill((t >= lens[:, None, None])[:, :, None], NEG)
    p = (scores - scores.amax(-1, keepdim=True).clamp(min=-FLT_MAX)).exp()
    out = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return {"out": out.reshape(B, H, D).to(torch.bfloat16), "selected": selected}


def _append(s):
    c, page = s["case"], s["case"]["page"]
    S, N, M, P = c["slots"], c["new"], s["table"].shape[1], s["refs"].shape[0]
    index, lens, table, refs = s["index"].long(), s["lens"].long(), s["table"], s["refs"]
    take = ((index >= 0) & (index < N)).long().cumprod(1).sum(1)
    at = torch.arange(M, device=index.device)
    touched = (at >= (lens // page)[:, None]) & (at <= ((lens + take - 1).div(page, rounding_mode="floor"))[:, None]) & (take > 0)[:, None]
    shared = (touched & (table >= 0) & (refs[table.clamp(min=0).long()] > 1)).any(1)
    off = (lens + take > M * page) | shared
    need = (touched & (table < 0) & ~off[:, None]).long()
    ends = need.sum(1).cumsum(0)
    spare = (refs <= 0).sum()
    off |= (need.sum(1) > 0) & (ends > spare)
    need = need * ~off[:, None]
    rank = need.flatten().cumsum(0).view(S, M) - 1
    free = torch.argsort((refs > 0).int(), stable=True)  # the lowest free pages first
    table.copy_(torch.where(need > 0, free[rank.clamp(0, P - 1)].int(), table))
    refs[table[need > 0].long()] = 1
    take = take * ~off
    s["lens_out"].copy_(lens + take)
    s["status"].copy_(off.sum())
    slot, j = (torch.arange(N, device=index.device) < take[:, None]).nonzero(as_tuple=True)
    pos = lens[slot] + j
    ids, row = table[slot, pos // page].long(), pos % page
    s["k"][:, ids, :, row] = s["k_new"][:, slot, index[slot, j]].transpose(0, 1)
    s["v"][:, ids, :, row] = s["v_new"][:, slot, index[slot, j]].transpose(0, 1)
    out = {n: s[n] for n in ("k", "v", "table", "refs", "lens_out", "status")}
    if c["summaries"]:
        full = ids[row == page - 1]
        s["codes"][:, full], s["scales"][:, full] = _summaries(s["k"][:, full])
    return out


def _fork(s):
    c, page = s["case"], s["case"]["page"]
    S, M, P = c["slots"], s["table"].shape[1], s["refs"].shape[0]
    source, lens, table, refs = s["source"].long(), s["lens"].long(), s["table"], s["refs"]
    dev = source.device
    slot = torch.arange(S, device=dev)
    old = source.clamp(min=0)
    live = (source >= 0) & (source < S)
    length = torch.where(live, lens[old], torch.zeros_like(old))
    # who keeps a parent's partial page: the parent itself, else its lowest child
    keeper = torch.full((S,), S, device=dev, dtype=torch.long).scatter_reduce(0, old, torch.where(live, slot, S), "amin")
    keeper = torch.where(source == slot, slot, keeper)
    last = length // page
    copy = live & (length % page > 0) & (keeper[old] != slot)
    rank = copy.long().cumsum(0) - 1
    off = copy & (rank >= (refs <= 0).sum())
    copy &= ~off
    length = torch.where(off, torch.zeros_like(length), length)
    fresh = torch.argsort((refs > 0).int(), stable=True)[rank.clamp(0, P - 1)].int()
    at = torch.arange(M, device=dev)
    rows = torch.where(at < (-(-length // page))[:, None], table[old], torch.full_like(table, -1))
    rows = torch.where(copy[:, None] & (at == last[:, None]), fresh[:, None], rows)
    s["refs_out"].copy_(refs)
    s["refs_out"].scatter_add_(0, table.clamp(min=0).long().flatten(), -(table >= 0).int().flatten())
    s["refs_out"].scatter_add_(0, rows.clamp(min=0).long().flatten(), (rows >= 0).int().flatten())
    s["table_out"].copy_(rows)
    s["lens_out"].copy_(length)
    s["status"].copy_(off.sum())
    to, r = (copy[:, None] & (torch.arange(page, device=dev) < (length % page)[:, None])).nonzero(as_tuple=True)
    src, dst = table[old[to], last[to]].long(), fresh[to].long()
    s["k"][:, dst, :, r] = s["k"][:, src, :, r]
    s["v"][:, dst, :, r] = s["v"][:, src, :, r]
    return {n: s[n] for n in ("k", "v", "table_out", "lens_out", "refs_out", "status")}


def _compact(s):
    refs, table = s["refs"], s["table"]
    used = (refs > 0).sum()
    at = torch.arange(refs.shape[0], device=refs.device)
    dst = ((refs <= 0) & (at < used)).nonzero().flatten()
    src = ((refs > 0) & (at >= used)).nonzero().flatten()
    where = at.clone()
    where[src] = dst
    s["table_out"].copy_(torch.where(table >= 0, where[table.clamp(min=0).long()].int(), table))
    s["refs_out"].copy_(refs)
    s["refs_out"][dst] = refs[src]
    s["refs_out"][src] = 0
    s["used"].copy_(used)
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    if s["case"]["summaries"]:
        s["codes"][:, dst], s["scales"][:, dst] = s["codes"][:, src], s["scales"][:, src]
    return {n: s[n] for n in ("k", "v", "table_out", "refs_out", "used")}


def _with_bounds(s, out):
    """The summaries with an operator's outputs, as the bounds that the codes stand for."""
    if "codes" in s:
        out["bounds"] = s["codes"].float() * s["scales"][..., None, None]
    return out


# ---- the framework's calls ------------------------------------------------------------------

_calls = {}


def _call(name, **sizes):
    """The operator of these sizes, made once as a program does at its start."""
    key = (name, tuple(sizes.items()))
    if key not in _calls:
        from iron_b200 import operators

        _calls[key] = getattr(operators, name)(**sizes).get_callable()
    return _calls[key]


def _own(s):
    c = s["case"]
    heads = dict(num_kv_heads=c["kv_heads"], head_dim=c["dim"], page_size=c["page"])
    if c["op"] == "tree":
        H, G = c["heads"], c["kv_heads"]
        call = _call("TreeAttention", batch=c["batch"], num_nodes=c["nodes"], num_heads=H, num_pages=s["k"].shape[0], max_pages=s["table"].shape[1], **heads)
        q, kn, vn = s["qkv"].split([H, G, G], 2)
        call(q, kn, vn, s["k"], s["v"], s["table"], s["lens"], s["parents"], s["out"])
        return s["out"]
    if c["op"] == "select":
        call = _call("PageSelectAttention", batch=c["batch"], num_heads=c["heads"], num_pages=s["k"].shape[0], max_pages=s["table"].shape[1], top_pages=c["top"], **heads)
        call(s["q"], s["k"], s["v"], s["codes"], s["scales"], s["table"], s["lens"], s["out"], s["selected"])
        return {"out": s["out"], "selected": s["selected"]}
    sizes = dict(num_layers=c["layers"], slots=s["table"].shape[0], num_pages=s["refs"].shape[0], max_pages=s["table"].shape[1], summaries="codes" in s, **heads)
    more = (s["codes"], s["scales"]) if "codes" in s else ()
    if c["op"] == "append":
        call = _call("PageAppend", num_new=c["new"], **sizes)
        call(s["k_new"], s["v_new"], s["index"], s["k"], s["v"], s["table"], s["lens"], s["refs"], s["lens_out"], s["status"], *more)
        return {n: s[n] for n in ("k", "v", "table", "refs", "lens_out", "status")}
    if c["op"] == "fork":
        sizes.pop("summaries")
        call = _call("PageFork", **sizes)
        call(s["source"], s["table"], s["lens"], s["refs"], s["k"], s["v"], s["table_out"], s["lens_out"], s["refs_out"], s["status"])
        return {n: s[n] for n in ("k", "v", "table_out", "lens_out", "refs_out", "status")}
    call = _call("PageCompact", **sizes)
    call(s["table"], s["refs"], s["k"], s["v"], s["table_out"], s["refs_out"], s["used"], *more)
    return {n: s[n] for n in ("k", "v", "table_out", "refs_out", "used")}


_plain = dict(tree=_tree, select=_select, append=_append, fork=_fork, compact=_compact)


def run(state):
    out = _own(state) if own else _plain[state["case"]["op"]](state)
    return _with_bounds(state, out) if state["case"]["op"] in ("append", "compact") else out


# ---- 64 bits --------------------------------------------------------------------------------


def _attend64(q, keys, values, scale):
    """softmax(scale q k) v of one row in float64; zeros where there is nothing to see."""
    if keys.shape[-2] == 0:
        return torch.zeros_like(q)
    return torch.softmax(scale * (q @ keys.transpose(-1, -2)), -1) @ values


def _bounds64(c, s):
    """The pages' bounds after an append (one that fits), from each page's rows in float64."""
    page, table = c["page"], s["table"].tolist()
    free = [p for p, r in enumerate(s["refs"].tolist()) if r == 0]
    bounds = s["codes"].double() * s["scales"].double()[..., None, None]
    for slot, (n, index) in enumerate(zip(s["lens"].tolist(), s["index"].tolist())):
        index = [i for i in index if i >= 0]
        rows = s["k_new"][:, slot, index].transpose(1, 2)  # [layers, kv heads, taken, D]
        for at in range(n // page, _pages(n + len(index), page)):
            p = table[slot][at] if table[slot][at] >= 0 else free.pop(0)
            first, last = at * page - n, (at + 1) * page - n
            if last > len(index):
                continue  # not full: no bounds yet
            old = s["k"][:, p, :, : max(0, -first)]
            keys = torch.cat([old, rows[:, :, max(0, first) : last]], 2).double()
            lo, hi = keys.amin(2), keys.amax(2)
            step = keys.abs().amax((2, 3))[..., None] / 127
            bounds[:, p, :, 0], bounds[:, p, :, 1] = torch.floor(lo / step).clamp(min=-127) * step, torch.ceil(hi / step).clamp(max=127) * step
    return bounds


def exact(case, seed):
    c = case
    if c["op"] in ("fork", "compact") or c["op"] == "append" and not c["summaries"]:
        return None  # rows that are moved and whole numbers: nothing is computed
    s = prepare(case, seed)
    if c["op"] == "append":
        return dict.fromkeys(("k", "v", "table", "refs", "lens_out", "status")) | {"bounds": _bounds64(c, s)}
    B, H, G, D, page = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    g, scale = H // G, 1 / math.sqrt(D)
    lens, table = s["lens"].tolist(), s["table"].tolist()

    def rows(pool, ids, heads=slice(None)):
        return pool[torch.tensor(ids, device="cuda")][:, heads].double().transpose(0, 1).reshape(-1, len(ids) * page, D)

    if c["op"] == "tree":
        N = c["nodes"]
        out = torch.zeros(B, N, H, D, dtype=torch.float64, device="cuda")
        parents = s["parents"].tolist()
        for b in range(B):
            n = _pages(lens[b], page)
            K, V = (rows(s[x], table[b][:n])[:, : lens[b]] for x in ("k", "v"))
            x = s["qkv"][b].double()
            sees, used = torch.zeros(N, N, dtype=torch.bool), []
            for i, p in enumerate(parents[b]):
                ok = -1 <= p < i and (p == -1 or used[p])
                used.append(ok)
                if ok:
                    if p >= 0:
                        sees[i] = sees[p]
                    sees[i, i] = True
            sees = sees.cuda()
            on = torch.tensor(used, device="cuda")
            kn, vn = x[:, H : H + G].transpose(0, 1), x[:, H + G :].transpose(0, 1)
            for h in range(G):
                qh = x[:, h * g : h * g + g]  # [N, g, D]
                a = scale * (qh @ K[h].T)
                t = (scale * (qh @ kn[h].T)).masked_fill(~sees[:, None], NEG)
                p = torch.softmax(torch.cat([a, t], -1), -1)
                o = p[..., : a.shape[-1]] @ V[h] + p[..., a.shape[-1] :] @ vn[h]
                out[b, :, h * g : h * g + g] = torch.where(on[:, None, None], o, torch.zeros_like(o))
        return out
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = _pages(lens[b], page)
        ids = torch.tensor(table[b][:n], device="cuda")
        for h in range(G):
            q = s["q"][b, h * g : h * g + g]
            if n > c["top"]:
                top = q.float().abs().max()
                q8 = torch.round(q.float() / top * 127.0).long()  # the definition's own fp32 steps
                lo, hi = s["codes"][ids, h, 0].long(), s["codes"][ids, h, 1].long()
                whole = torch.maximum(q8[:, None] * lo, q8[:, None] * hi).sum((0, 2))
                score = (whole.float() * s["scales"][ids, h]).tolist()
                middle = sorted(range(1, n - 1), key=lambda i: (-score[i], i))
                keep = ([n - 1] + [0] + middle)[: c["top"]]
            else:
                keep = list(range(n))
            keep.sort()
            K, V = (rows(s[x], ids[keep].tolist(), slice(h, h + 1))[0] for x in ("k", "v"))
            valid = len(keep) * page - (n * page - lens[b])  # the last page is always kept
            out[b, h * g : h * g + g] = _attend64(q.double(), K[:valid], V[:valid], scale)
    return {"out": out, "selected": None}
