"""The order of the barriers in the tcgen05 form of TreeAttention (csrc/tree_attention_tc.cu),
checked on the host for the pieces that a batch is cut into on 148 CTAs.

A wait names a phase of an mbarrier by its parity alone, so it is right only if the phase
before is complete when it starts and the phase after cannot complete before it has ended;
an arrival counts for its own phase only if the one before is complete. `Run` writes down
what each role of a CTA does, in program order, and checks this, and that every buffer is
read between its own write and the next one, from the order that the events have whatever
the timing: program order, and the end of a phase before the end of a wait for it.
"""

import random
import re
from collections import defaultdict
from pathlib import Path

import pytest

TILE, UNIT_COST, MASKS, CTAS = 128, 3, 8, 148


def segments(lens, rows, kv_heads, cta, ctas=CTAS):
    """(rows of the unit, cached tokens, first tile, count) of each segment of one CTA's piece
    (nodes are at most 128: a unit ends with one tile of them)."""
    groups = -(-rows // 256)
    cost = [-(-n // TILE) + 1 + UNIT_COST for n in lens]
    units = [(b, u % groups) for b in range(len(lens)) for u in range(kv_heads * groups)]
    total = sum(c * kv_heads * groups for c in cost)
    pieces = min(ctas, total)
    if cta >= pieces:
        return []
    lo, hi, at, out = total * cta // pieces, total * (cta + 1) // pieces, 0, []
    for b, group in units:
        a, z = max(lo, at), min(hi, at + cost[b])
        if a < z:
            first = max(0, a - at - UNIT_COST)
            count = z - at - UNIT_COST - first
            if count > 0:
                out.append((rows - 256 * group, lens[b], first, count))
        at += cost[b]
    return out


class Run:
    def __init__(self, segs, nodes, D, skip=False):
        """skip: streams wait for their own tiles only and release each twice."""
        self.D, self.S, self.nodes, self.skip = D, 4 if D == 64 else 2, nodes, skip
        self.before = []  # events that each event directly follows
        self.done = {}  # (barrier, phase): the event of its completion
        self.arrivals, self.waits = defaultdict(list), []
        self.writes, self.reads = defaultdict(list), defaultdict(list)
        self.segs, at = [], 0
        for rows, length, first, count in segs:
            both, ctiles = rows > 128, -(-length // TILE)
            own = [[i for i in range(count) if both or i % 2 == s] for s in (0, 1)]
            left = [nodes if first + i >= ctiles else length - (first + i) * TILE for i in range(count)]
            halves = [2 if n > TILE // 2 else 1 for n in left]
            self.segs.append((at, count, both, own, halves, first + count > ctiles))
            at += count
        self.loader()
        self.prepare()
        for s in (0, 1):
            self.mma(s)
            for warp in (0, 1):  # two of the four warps: each counts, and each may lag
                self.softmax(s, warp)

    # -- events ------------------------------------------------------------------------------
    def event(self, *after):
        self.before.append([e for e in after if e is not None])
        return len(self.before) - 1

    def step(self, role):
        role.append(self.event(role[-1] if role else None))
        return role[-1]

    def phase(self, bar, n):
        if n < 0:
            return None
        if (bar, n) not in self.done:
            self.done[bar, n] = self.event(self.phase(bar, n - 1))
        return self.done[bar, n]

    def wait(self, role, bar, n):
        start, end = self.step(role), self.step(role)
        self.before[end].append(self.phase(bar, n))
        self.waits.append((bar, n, start, end))

    def arrive(self, role, bar, n, times=1, after=None):
        """after: what a commit waits for."""
        for _ in range(times):
            e = self.event(self.step(role), after)  # copies arrive some time after they are issued
            self.before[self.phase(bar, n)].append(e)
            self.arrivals[bar, n].append(e)

    # -- the roles ---------------------------------------------------------------------------
    def loader(self):
        role, S = [], self.S
        for at, count, *_ in self.segs:
            for it in range(at, at + count):
                slot, n = it % S, it // S
                if n:
                    self.wait(role, ("kempty", slot), n - 1)
                self.writes["mask", it % MASKS].append(self.step(role))
                self.arrive(role, ("mask", it % MASKS), it // MASKS)
                self.writes["K", slot].append(self.step(role))
                self.arrive(role, ("kfull", slot), n)
                if n:
                    self.wait(role, ("vempty", slot), n - 1)
                self.writes["V", slot].append(self.step(role))
                self.arrive(role, ("vfull", slot), n)

    def prepare(self):
        role, S, trees = [], self.S, 0
        for at, count, both, own, halves, tree in self.segs:
            if tree:
                self.writes["tree", trees % (S + 3)].append(self.step(role))
                self.arrive(role, ("paths", trees % (S + 3)), trees // (S + 3))
                trees += 1
            for it in range(at, at + count):
                self.wait(role, ("vfull", it % S), it // S)
                self.reads["mask", it % MASKS].append((it // MASKS, self.step(role)))
                self.arrive(role, ("vready", it % S), it // S)

    def mma(self, s):
        role, S, c = [], self.S, dict(k=0, v=0, sn=0, pc=0, q=0)
        whole = self.D == 64  # one S of a whole tile, else one per half

        def pass_k(upto):
            while c["k"] < upto and not self.skip:
                self.wait(role, ("kfull", c["k"] % S), c["k"] // S)
                self.arrive(role, ("kempty", c["k"] % S), c["k"] // S)
                c["k"] += 1

        def pass_v(upto):
            while c["v"] < upto and not self.skip:
                self.wait(role, ("vready", c["v"] % S), c["v"] // S)
                self.arrive(role, ("vempty", c["v"] % S), c["v"] // S)
                c["v"] += 1

        issued = [None]

        def issue():  # a batch of MMAs, complete some time after; a commit waits for all so far
            issued[0] = self.event(self.step(role), issued[0])
            return issued[0]

        def scores(it, last, twice):
            pass_k(it)
            self.wait(role, ("kfull", it % S), it // S)
            if c["sn"]:
                self.wait(role, ("sfree", s), c["sn"] - 1)
            e = issue()
            self.writes["S", s].append(e)
            self.arrive(role, ("sfull", s), c["sn"], after=e)
            c["sn"] += 1
            self.reads["K", it % S].append((it // S, e))
            self.reads["Q", s].append((c["q"] - 1, e))
            if last:
                self.arrive(role, ("kempty", it % S), it // S, 2 if twice else 1, after=e)
                c["k"] = it + 1

        def values(it, last, twice):
            pass_v(it)
            self.wait(role, ("vready", it % S), it // S)
            self.wait(role, ("pfull", s), c["pc"])
            e = issue()
            self.arrive(role, ("pvdone", s), c["pc"], after=e)
            self.reads["V", it % S].append((it // S, e))
            self.reads["P", s].append((c["pc"], e))
            c["pc"] += 1
            if last:
                self.arrive(role, ("vempty", it % S), it // S, 2 if twice else 1, after=e)
                c["v"] = it + 1

        for at, count, both, own, halves, tree in self.segs:
            mine = own[s]
            twice = self.skip and not both
            if mine:
                self.wait(role, ("qfull", s), c["q"])
                c["q"] += 1
                k = halves[mine[0]]
                scores(at + mine[0], whole or k == 1, twice)
                pass_v(at)
            for j, i in enumerate(mine):
                nxt = mine[j + 1] if j + 1 < len(mine) else None
                for h in range(k):
                    if not whole and h + 1 < k:
                        scores(at + i, h + 2 == k, twice)
                    elif h + 1 == k and nxt is not None:
                        scores(at + nxt, whole or halves[nxt] == 1, twice)
                    values(at + i, h + 1 == k, twice)
                k = halves[nxt] if nxt is not None else 0
            pass_k(at + count)
            pass_v(at + count - 1)

    def softmax(self, s, warp):
        role, S, c = [], self.S, dict(sc=0, vc=0, j=0, q=0, trees=0)
        whole = self.D == 64

        def load_q(seg):
            if seg[3][s]:
                if warp == 0:
                    self.writes["Q", s].append(self.step(role))
                self.arrive(role, ("qfull", s), c["q"])
                c["q"] += 1

        if self.segs:
            load_q(self.segs[0])
        for k, (at, count, both, own, halves, tree) in enumerate(self.segs):
            mine = own[s]
            for j, i in enumerate(mine):
                it = at + i
                for h in range(halves[i]):
                    if h == 0 or not whole:
                        self.wait(role, ("sfull", s), c["sc"])
                        c["sc"] += 1
                    if h == 0:
                        self.wait(role, ("mask", it % MASKS), it // MASKS)
                        if tree and j == len(mine) - 1:
                            t = c["trees"] % (S + 3)
                            self.wait(role, ("paths", t), c["trees"] // (S + 3))
                            self.reads["tree", t].append((c["trees"] // (S + 3), self.step(role)))
                        self.reads["mask", it % MASKS].append((it // MASKS, self.step(role)))
                    self.reads["S", s].append((c["sc"] - 1, self.step(role)))
                    if not whole or h == halves[i] - 1:
                        self.arrive(role, ("sfree", s), c["sc"] - 1)
                    if c["vc"]:
                        self.wait(role, ("pvdone", s), c["vc"] - 1)
                    if warp == 0:
                        self.writes["P", s].append(self.step(role))
                    self.arrive(role, ("pfull", s), c["vc"])
                    c["vc"] += 1
            c["trees"] += tree
            if k + 1 < len(self.segs):
                load_q(self.segs[k + 1])
            if mine:
                self.wait(role, ("pvdone", s), c["vc"] - 1)
            if not both and own[1]:
                if s == 1:
                    self.arrive(role, ("other",), c["j"])
                    self.wait(role, ("joined",), c["j"])
                else:
                    self.wait(role, ("other",), c["j"])
                    self.step(role)
                    self.arrive(role, ("joined",), c["j"])
                c["j"] += 1

    # -- the checks --------------------------------------------------------------------------
    def faults(self):
        n = len(self.before)
        after, missing = [[] for _ in range(n)], [0] * n
        for e, b in enumerate(self.before):
            missing[e] = len(b)
            for x in b:
                after[x].append(e)
        ready, past, order = [e for e in range(n) if not missing[e]], [0] * n, 0
        while ready:
            e = ready.pop()
            order += 1
            past[e] |= 1 << e
            for x in after[e]:
                past[x] |= past[e]
                missing[x] -= 1
                if not missing[x]:
                    ready.append(x)
        if order < n:
            return ["a deadlock"]
        precedes = lambda a, b: bool(past[b] >> a & 1)  # noqa: E731
        out = []
        for bar, phase, start, end in self.waits:
            if phase and not precedes(self.done[bar, phase - 1], start):
                out.append(f"{bar}: a wait for phase {phase} may start before phase {phase - 1} is complete")
            if (bar, phase + 1) in self.done and not precedes(end, self.done[bar, phase + 1]):
                out.append(f"{bar}: phase {phase + 1} may complete under a wait for phase {phase}")
        counts = {"kempty": 2, "vempty": 2, "sfree": 2, "pfull": 2, "qfull": 2, "other": 2, "joined": 2}
        for (bar, phase), events in self.arrivals.items():
            want = counts.get(bar[0], 1)
            if len(events) > want or len(events) < want and (bar, phase + 1) in self.done:
                out.append(f"{bar}: {len(events)} arrivals in phase {phase}")
            out += [f"{bar}: an arrival of phase {phase} may come before phase {phase - 1} is complete"
                    for e in events if phase and not precedes(self.done[bar, phase - 1], e)]
        for what, reads in self.reads.items():
            w = self.writes[what]
            for version, e in reads:
                if not precedes(w[version], e):
                    out.append(f"{what}: version {version} may be read before it is written")
                if version + 1 < len(w) and not precedes(e, w[version + 1]):
                    out.append(f"{what}: version {version} may be overwritten while it is read")
        return out


def check(lens, nodes, Hq, Hkv, D, ctas=CTAS, skip=False):
    """The faults of every different piece of a batch."""
    rows, seen, out = nodes * (Hq // Hkv), set(), []
    for cta in range(ctas):
        segs = tuple(segments(lens, rows, Hkv, cta, ctas))
        # only the last tile's fill counts of a length
        key = tuple((r > 128, -(-n // TILE) - f if f + c > n // TILE else -1, (n - 1) % TILE // 64 if n else 0, c) for r, n, f, c in segs)
        if key not in seen:
            seen.add(key)
            out += Run(segs, nodes, D, skip).faults()
    return out


BATCHES = {
    "many tiles per piece": [4096, 2999, 2049, 100, 3100, 0, 4000, 640],
    "uniform": [2048] * 16,
    "edges": [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 255, 257, 511],
    "empty slots": [0] * 8 + [700, 0, 0, 0, 1500, 128] + [0] * 20 + [64, 65, 3000],
    "all empty": [0] * 64,
    "one long": [9000, 0, 0],
}


def test_sizes_are_the_kernels():
    src = (Path(__file__).parents[1] / "iron_b200/csrc/tree_attention_tc.cu").read_text()
    for line in (f"kTile = {TILE};", "kStages = D == 64 ? 4 : 2;", "kTrees = kStages + 3;", f"kMasks = {MASKS};",
                 f"kUnitCost = {UNIT_COST};", "kScores = D == 64 ? 128 : 64;"):
        assert re.search(re.escape(line), src), line


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nodes,Hq,Hkv", [(9, 32, 8), (20, 32, 8), (32, 32, 8), (40, 32, 8), (100, 8, 2)])
@pytest.mark.parametrize("batch", BATCHES)
def test_waits_tell_their_phase_from_every_other(batch, nodes, Hq, Hkv, D):
    assert check(BATCHES[batch], nodes, Hq, Hkv, D) == []


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed, D):
    rng = random.Random(seed)
    lens = [rng.choice([0, 0, 64, 128, rng.randint(1, 4096)]) for _ in range(rng.choice([3, 16, 40]))]
    assert check(lens, rng.choice([9, 12, 26, 32, 33, 64]), 32, 8, D, ctas=rng.choice([132, 148])) == []


def test_streams_that_pass_their_own_tiles_alone_are_found():
    """The order in which a stream neither waits for nor releases the other one's tiles."""
    found = check(BATCHES["many tiles per piece"], 20, 32, 8, 128, skip=True)
    assert {f.split("'")[1] for f in found} == {"kfull", "vready"}
    assert check(BATCHES["empty slots"], 16, 32, 8, 64, skip=True)
    # with more than 128 rows both streams have every tile
    assert check(BATCHES["many tiles per piece"], 64, 32, 8, 128, skip=True) == []
