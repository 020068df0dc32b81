"""The barriers of chunk attention over the 8-bit cache (csrc/kv_fp8_chunk.cu), walked through in random orders.

A wait knows a phase by its parity alone: it must never be met by a barrier that is two phases off, nothing may be overwritten that
somebody still has to read, and everybody has to come to an end.  The model has the kernel's roles: copies, warps that turn codes into
tiles (two of them, which may be a block apart), the warp that issues products, the tensor core (in the order of issue) and the softmax
groups; in pairs of CTAs each CTA has its own, and the first one's issuer works for both."""
import random

import pytest

STAGES, META, RING = 2, 4, {"two": 3, "dual": 4, "pair": 6}


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.done = count, count, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.done = self.count, self.done + 1

    def passes(self, phase):
        """What the hardware says to the phase's parity; it has to be the truth."""
        says = (self.done & 1) != (phase & 1)
        assert says == (self.done > phase), (self.done, phase)
        return says


class Kernel:
    """``items``: (tiles, blocks) each."""

    def __init__(self, form, items, rng):
        self.form, self.items, self.rng = form, items, rng
        self.ctas, self.ring, self.halves = 2 if form == "pair" else 1, RING[form], 1 if form == "pair" else 2
        C = range(self.ctas)
        one = lambda n: [[Barrier(1) for _ in range(n)] for _ in C]
        self.st_full, self.kv_empty, self.q_empty, self.s_full, self.o_full = one(STAGES), one(self.ring), one(1), one(2), one(4)
        self.st_empty = [[Barrier(2) for _ in range(STAGES)] for _ in C]
        self.kv_full, self.q_full = [Barrier(2 * self.ctas) for _ in range(self.ring)], Barrier(self.ctas)
        self.p_full, self.meet = [Barrier(self.ctas) for _ in range(4)], Barrier(2)
        self.stage = [[None] * STAGES for _ in C]
        self.tile = [[[None, None] for _ in range(self.ring)] for _ in C]          # of the two warps that turn codes
        self.meta = [[None] * META for _ in C]
        self.s, self.p, self.o, self.q = ([[None] * n for _ in C] for n in (2, 4, 2, 1))
        self.queue, self.issued = [], False

    def copies(self, c):
        n = slot = 0
        uses = [0] * STAGES
        for i, (tiles, blocks) in enumerate(self.items):
            if blocks == 0:
                continue
            yield self.q_empty[c][0], n - 1
            n += 1
            self.q[c][0] = i
            self.q_full.arrive()
            for j in range(blocks):
                yield self.st_empty[c][slot], uses[slot] - 1
                self.stage[c][slot] = (i, j)
                self.st_full[c][slot].arrive()
                uses[slot] += 1
                slot = (slot + 1) % STAGES

    def turn(self, c, w):
        st = slot = n = 0
        seen, uses = [0] * STAGES, [0] * self.ring
        for i, (tiles, blocks) in enumerate(self.items):
            for j in range(blocks):
                yield self.st_full[c][st], seen[st]
                seen[st] += 1
                if w == 0:
                    self.meta[c][n % META] = (i, j)
                n += 1
                for what in "KV":
                    yield self.kv_empty[c][slot], uses[slot] - 1
                    uses[slot] += 1
                    assert self.stage[c][st] == (i, j)
                    self.tile[c][slot][w] = (i, j, what)
                    yield None
                    self.kv_full[slot].arrive()
                    slot = (slot + 1) % self.ring
                self.st_empty[c][st].arrive()
                st = (st + 1) % STAGES

    # products and commits, in the order of issue
    def scores(self, g, slot, i, j):
        self.queue.append(("S", g, slot, i, j))
        self.commit(self.s_full, g)

    def values(self, g, h, slot, i, j, first):
        self.queue.append(("O", g, h, slot, i, j, first))

    def commit(self, bars, k):
        self.queue.append(("commit", [b[k] for b in bars]))

    def issue(self):
        slot = n_q = 0
        done, uses = [0, 0], [0] * self.ring
        dual, pair = self.form == "dual", self.form == "pair"
        for i, (tiles, blocks) in enumerate(self.items):
            if blocks == 0:
                continue
            yield self.q_full, n_q
            n_q += 1
            if dual:
                first = slot
                at = lambda t: (first + t) % self.ring
                phase = lambda t: uses[at(t)] + t // self.ring

                def scores(j):
                    yield self.kv_full[at(2 * j)], phase(2 * j)
                    self.scores(j & 1, at(2 * j), i, j)
                    self.commit(self.kv_empty, at(2 * j))
                    if j + 1 == blocks:
                        self.commit(self.q_empty, 0)

                for j in range(min(blocks, 2)):
                    yield from scores(j)
                for j in range(blocks):
                    g, t = j & 1, 2 * j + 1
                    yield self.kv_full[at(t)], phase(t)
                    for h in range(2):
                        yield self.p_full[g * 2 + h], done[g] >> 1
                        done[g] += 1
                        self.values(g, h, at(t), i, j, j < 2 and h == 0)
                        self.commit(self.o_full, g * 2 + h)
                        if h == 1:
                            self.commit(self.kv_empty, at(t))
                    if j + 2 < blocks:
                        yield from scores(j + 2)
                for t in range(2 * blocks):
                    uses[at(t)] += 1
                slot = at(2 * blocks)
                continue

            def next_tile():
                nonlocal slot
                yield self.kv_full[slot], uses[slot]
                uses[slot] += 1
                slot = (slot + 1) % self.ring

            sk = slot
            yield from next_tile()
            for g in range(tiles):
                self.scores(g, sk, i, 0)
            self.commit(self.kv_empty, sk)
            if blocks == 1:
                self.commit(self.q_empty, 0)
            for j in range(blocks):
                more, sv = j + 1 < blocks, slot
                yield from next_tile()
                sk = slot
                if pair and more:
                    yield from next_tile()
                for g in range(tiles):
                    for h in range(self.halves):
                        last = h + 1 == self.halves
                        yield self.p_full[g * 2 + h], done[g] // self.halves
                        done[g] += 1
                        self.values(g, h, sv, i, j, j == 0 and h == 0)
                        if pair:
                            if more:
                                self.scores(g, sk, i, j + 1)
                            else:
                                self.commit(self.o_full, g * 2)
                            if g == tiles - 1:
                                self.commit(self.kv_empty, sv)
                                if more:
                                    self.commit(self.kv_empty, sk)
                                if j + 2 == blocks:
                                    self.commit(self.q_empty, 0)
                            continue
                        self.commit(self.o_full, g * 2 + h)
                        if last and g == tiles - 1:
                            self.commit(self.kv_empty, sv)
                        if not more or not last:
                            continue
                        if g == 0:
                            yield from next_tile()
                        self.scores(g, sk, i, j + 1)
                        if g == tiles - 1:
                            self.commit(self.kv_empty, sk)
                            if j + 2 == blocks:
                                self.commit(self.q_empty, 0)
        self.issued = True

    def tensor(self):
        while not self.issued or self.queue:
            if not self.queue:
                yield None
                continue
            yield None
            op = self.queue.pop(0)
            if op[0] == "commit":
                for b in op[1]:
                    b.arrive()
                continue
            for c in range(self.ctas):
                if op[0] == "S":
                    _, g, slot, i, j = op
                    assert self.tile[c][slot] == [(i, j, "K")] * 2 and self.q[c][0] == i
                    assert self.s[c][g] is None and self.p[c][2 * g] is None and self.p[c][2 * g + 1] is None
                    self.s[c][g] = (i, j)
                else:
                    _, g, h, slot, i, j, first = op
                    assert self.tile[c][slot] == [(i, j, "V")] * 2 and self.p[c][2 * g + h] == (i, j)
                    assert self.o[c][g] is None if first else self.o[c][g][0] == i
                    self.o[c][g] = (i, j, h)
                    self.p[c][2 * g + h] = None

    def softmax(self, c, g):
        parts = blocks_all = ended = met = 0
        dual, H = self.form == "dual", self.halves
        for i, (tiles, blocks) in enumerate(self.items):
            if not dual and g > 0 and tiles == 1:
                blocks_all += blocks
                continue
            n = H * ((blocks + 1 - g) // 2 if dual else blocks)
            for k in range(n):
                j, h = (k // H * 2 + g if dual else k // H), k % H
                if h == 0:
                    yield self.s_full[c][g], parts // H
                parts += 1
                assert self.s[c][g] == (i, j) and self.meta[c][(blocks_all + j) % META] == (i, j)
                yield None
                if k and self.rng.random() < 0.5:          # a reference that moves: O as far as it is known
                    if h == 1:
                        yield self.o_full[c][g * 2], (parts - 1) // H
                    assert self.o[c][g] == ((i, j, 0) if h else (i, j - (2 if dual else 1), H - 1))
                assert self.s[c][g] == (i, j) and self.meta[c][(blocks_all + j) % META] == (i, j)
                self.p[c][2 * g + h] = (i, j)
                if h + 1 == H:
                    self.s[c][g] = None
                self.p_full[2 * g + h].arrive()
            last = blocks_all + blocks
            blocks_all = last
            if n:
                yield self.o_full[c][g * 2 + H - 1], ended if H == 1 else (parts - 1) >> 1
                ended += 1
            if dual:
                self.meet.arrive()
                yield self.meet, met
                met += 1
            for of in range(2) if dual else (g,):          # what the results are made of
                own = H * ((blocks + 1 - of) // 2) if dual else n
                if own:
                    assert self.o[c][of] == (i, (blocks - 1 - (blocks - 1 - of) % 2) if dual else blocks - 1, H - 1)
            yield None
            if dual:
                self.meet.arrive()
                yield self.meet, met
                met += 1
            self.o[c][g] = None

    def run(self):
        C = range(self.ctas)
        agents = [self.issue(), self.tensor(), *(self.copies(c) for c in C), *(self.turn(c, w) for c in C for w in range(2)),
                  *(self.softmax(c, g) for c in C for g in range(2))]
        at = {a: next(a, "end") for a in agents}
        while True:
            live = [a for a in agents if at[a] != "end"]
            if not live:
                return
            ready = [a for a in live if at[a] is None or at[a][0].passes(at[a][1])]
            assert any(a is not agents[1] or self.queue for a in ready), "nobody can go on"
            # now and then one agent goes as far as it can, so that the others are far behind
            a = self.rng.choice(ready)
            for _ in range(self.rng.choice([1, 1, 3, 40])):
                at[a] = next(a, "end")
                if at[a] == "end" or (at[a] is not None and not at[a][0].passes(at[a][1])):
                    break


@pytest.mark.parametrize("form", ["two", "dual", "pair"])
def test_no_wait_is_met_by_another_phase_and_all_come_to_an_end(form):
    rng = random.Random(11)
    cases = [[(2, 5)], [(1, 1)], [(2, 1)] * 6, [(1, 2), (2, 3), (1, 0), (2, 1), (1, 1), (1, 4)], [(2, 0)], [(2, 2), (1, 1), (1, 1), (2, 9)]]
    cases += [[(rng.randint(1, 2), rng.randint(0, 4)) for _ in range(rng.randint(1, 7))] for _ in range(20)]
    for items in cases:
        for _ in range(12):
            Kernel(form, [(1, b) for _, b in items] if form == "dual" else items, rng).run()
