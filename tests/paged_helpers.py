"""Plain implementations of the paged-cache operators, in 64 bits and host integers."""

import math

import torch


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


class Cache:
    """One layer of a paged cache with random rows; what no sequence owns is NaN."""

    def __init__(self, lens, Hkv, D, page, seed, spare=3, width=None, pages=None, base=0):
        g = gen(seed)
        self.lens_list, self.page, self.D, self.Hkv = list(lens), page, D, Hkv
        need = [-(-n // page) for n in lens]
        self.P = pages or sum(need) + spare
        self.M = width or max(max(need), 1) + 1
        ids = torch.randperm(self.P - base, generator=torch.Generator().manual_seed(seed))[: sum(need)] + base
        if pages is None:
            self.k = torch.full((self.P, Hkv, page, D), math.nan, dtype=torch.bfloat16, device="cuda")
            self.v = self.k.clone()
        else:  # too large to fill
            self.k = torch.empty(self.P, Hkv, page, D, dtype=torch.bfloat16, device="cuda")
            self.v = torch.empty_like(self.k)
        table = torch.full((len(lens), self.M), -1, dtype=torch.int32)
        self.K, self.V, at = [], [], 0
        for s, n in enumerate(lens):
            mine = ids[at : at + need[s]]
            at += need[s]
            table[s, : need[s]] = mine.int()
            K, V = randn(g, Hkv, need[s] * page, D), randn(g, Hkv, need[s] * page, D)
            K[:, n:] = V[:, n:] = math.nan
            if need[s]:
                self.k[mine.cuda()] = K.view(Hkv, need[s], page, D).transpose(0, 1)
                self.v[mine.cuda()] = V.view(Hkv, need[s], page, D).transpose(0, 1)
            self.K.append(K[:, :n])
            self.V.append(V[:, :n])
        self.table = table.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")


def paths(parents):
    out = []
    for i, p in enumerate(parents):
        out.append([i] if p == -1 else out[p] + [i] if 0 <= p < i and out[p] else [])
    return out


def attend(q, k, v, scale):
    """softmax(scale q k^T) v in float64 and the bound on a bf16 kernel's error.

    A kernel rounds its output to bf16: 2^-8 of |out| <= A = sum p |v|. It sums the scores
    in fp32: a logit is off by at most D 2^-24 sum |q| |k| scale (twice that if the sums are
    truncated), which moves the numerator and the denominator by that much of A each."""
    q, k, v = q.double(), k.double(), v.double()
    p = torch.softmax(scale * q @ k.transpose(-1, -2), -1)
    logit = 2 * q.shape[-1] * 2.0**-24 * float((q.abs() @ k.abs().transpose(-1, -2)).max()) * scale
    return p @ v, (p @ v.abs()) * (2.0**-8 + 2 * logit + 2.0**-20)


def tree_reference(cache, q, kn, vn, parents, scale):
    """(out, tolerance) [B, N, Hq, D] in float64, row by row."""
    B, N, Hq, D = q.shape
    g = Hq // cache.Hkv
    out = torch.zeros(B, N, Hq, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for b in range(B):
        for i, path in enumerate(paths(parents[b])):
            if path:
                k = torch.cat([cache.K[b], kn[b, path].transpose(0, 1)], 1)
                v = torch.cat([cache.V[b], vn[b, path].transpose(0, 1)], 1)
                o, t = attend(q[b, i].view(cache.Hkv, g, D), k, v, scale)
                out[b, i], tol[b, i] = o.reshape(Hq, D), t.reshape(Hq, D)
    return out, tol


def summary(keys):
    """codes [..., 2, D] (floats) and scales of pages [..., page, D]."""
    k = keys.float().cpu()
    lo, hi, top = k.amin(-2), k.amax(-2), k.abs().amax((-1, -2))
    scale = top / 127.0
    by = torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    codes = torch.stack([torch.floor(lo / by).clamp(-127, 127), torch.ceil(hi / by).clamp(-127, 127)], -2)
    odd = ~torch.isfinite(top)
    codes[odd] = torch.tensor([[-127.0], [127.0]])
    scale[odd] = torch.finfo(torch.float32).max
    return codes, scale


def select_reference(q, codes, scales, top):
    """Kept pages (ascending) of one kv head: q [g, D], codes [n, 2, D] and scales [n] of its pages in order."""
    n = len(scales)
    x = q.float().cpu()
    a = float(x.abs().max())
    q8 = torch.round(x / a * 127.0).long() if 0 < a < math.inf else torch.zeros_like(x).long()
    lo, hi = codes[:, 0].long().cpu(), codes[:, 1].long().cpu()
    big = torch.finfo(torch.float32).max
    score = ((q8[:, None].clamp(min=0) * hi + q8[:, None].clamp(max=0) * lo).sum((0, 2)).float() * scales.cpu()).clamp(-big, big).tolist()
    order = sorted(range(1, n - 1), key=lambda i: (-score[i], i))
    return sorted(([n - 1] + ([0] if n > 1 else []) + order)[:top]) if n else []


class HostCache:
    """The metadata of a cache as host lists, changed by the rules of the operators."""

    def __init__(self, slots, pages, width, page):
        self.table = [[-1] * width for _ in range(slots)]
        self.lens, self.refs, self.page, self.M = [0] * slots, [0] * pages, page, width

    def free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def append(self, takes):
        """takes[s] rows for slot s. Returns (refused, positions written: (slot, j, page, row))."""
        refused, wrote, total, free = 0, [], 0, self.free()
        plan, short = [], []
        for s, n in enumerate(takes):
            touched = range(self.lens[s] // self.page, (self.lens[s] + n - 1) // self.page + 1) if n else []
            if self.lens[s] + n > self.M * self.page or any(self.table[s][i] >= 0 and self.refs[self.table[s][i]] > 1 for i in touched):
                refused += 1
                plan.append((0, []))
                continue
            need = [i for i in touched if self.table[s][i] < 0]
            total += len(need)
            if need and total > len(free):
                refused += 1
                plan.append((0, []))
                continue
            plan.append((n, [(i, free[total - len(need) + x]) for x, i in enumerate(need)]))
        for s, (n, got) in enumerate(plan):
            for i, p in got:
                self.table[s][i], self.refs[p] = p, 1
            for j in range(n):
                pos = self.lens[s] + j
                wrote.append((s, j, self.table[s][pos // self.page], pos % self.page))
            self.lens[s] += n
        return refused, wrote

    def fork(self, source):
        """Returns (refused, copies: (old page, new page, rows))."""
        S, old, lens = len(self.table), [list(r) for r in self.table], list(self.lens)
        free, copies, refused, rank = self.free(), [], 0, 0
        source = [r if 0 <= r < S else -1 for r in source]
        kids = {r: [s for s in range(S) if source[s] == r] for r in range(S)}
        for s, r in enumerate(source):
            n = lens[r] if r >= 0 else 0
            row = old[r][: -(-n // self.page)] if r >= 0 else []
            keeper = (r if source[r] == r else kids[r][0]) if r >= 0 else None
            if n % self.page and keeper != s:
                if rank < len(free):
                    copies.append((row[-1], free[rank], n % self.page))
                    row = row[:-1] + [free[rank]]
                else:
                    refused, row, n = refused + 1, [], 0
                rank += 1
            self.table[s], self.lens[s] = row + [-1] * (self.M - len(row)), n
        for row, sign in [(r, -1) for r in old] + [(r, 1) for r in self.table]:
            for p in row:
                if p >= 0:
                    self.refs[p] += sign
        return refused, copies

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        src = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(used) if self.refs[p] <= 0]
        where = dict(zip(src, dst))
        for a, b in where.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[where.get(p, p) for p in r] for r in self.table]
        return used, list(where.items())
